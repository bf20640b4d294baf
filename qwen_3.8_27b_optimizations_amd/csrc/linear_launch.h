// linear_launch.h -- the kernels of linear attention as linear.hip launches them.
#pragma once

#include <hip/hip_runtime.h>

#include "linear_plan.h"

namespace iq4xs {

struct LinearArgs;

// 2^decays of a segment, times log2(e): part * 2^exponent.
struct SegmentDecay {
    float part;
    int exponent;
};

// Segments of `length` tokens that sequences are cut into; with one there are no states.
struct LinearSegments {
    float* states;  // [places of `kept`][heads][dk][dv]: a sequence's own, and what each segment leaves (the first) or adds
    SegmentDecay* decays;  // [places of `kept`][heads] what each keeps of the state that it begins with
    int count, length;
    SegmentPlaces runs, kept;
    bool join_rows;
    int64_t grid;
};

// units: of 32 columns of a head's state.
void launch_linear_steps(const LinearArgs& a, int dk, int dv, int type, int64_t units, hipStream_t stream);
void launch_linear_chunks(const LinearArgs& a, const LinearSegments& segments, int dk, int dv, int type,
                          hipStream_t stream);

}  // namespace iq4xs
