// linear_internal.h -- launchers of linear attention; arguments are checked by the C ABI (attention_api.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "iq4xs_mi355x.h"

namespace iq4xs {

// hipErrorInvalidConfiguration: a call whose launches would be too large.
hipError_t linear_attention_workspace(const iq4xs_linear_attention_args& args, size_t* bytes);
// The same, and hipErrorInvalidValue for a workspace that is too small or not aligned to 256 bytes.
hipError_t launch_linear_attention(const iq4xs_linear_attention_args& args, void* ws, size_t ws_bytes, hipStream_t stream);

}  // namespace iq4xs
