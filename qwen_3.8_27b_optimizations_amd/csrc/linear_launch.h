// linear_launch.h -- the kernels of linear attention as linear.hip launches them.
#pragma once

#include <hip/hip_runtime.h>

#include "iq4xs_mi355x.h"

namespace iq4xs {

struct LinearArgs;
int64_t linear_step_grid(const iq4xs_linear_attention_args& args);
void launch_linear_step(const LinearArgs& a, int dk, int dv, int type, int64_t grid, hipStream_t stream);

}  // namespace iq4xs
