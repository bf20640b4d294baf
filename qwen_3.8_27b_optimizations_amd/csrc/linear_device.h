// linear_device.h -- what the kernels of linear attention share: their arguments, sequences and states.
#pragma once

#include <math.h>

#include "attention_device.h"

namespace iq4xs {

struct LinearArgs {
    const void *q, *k, *v;
    const float* decay;
    const int32_t* starts;
    float* states;
    const int64_t *from_slots, *to_slots;
    void* out;
    int64_t q_stride, k_stride, v_stride, decay_stride, slots;
    int total, most_q, seqs, heads, group, out_type;  // group: heads that share one of q and k
    float scale;
};

// Rows [first, first + count) of a sequence, cut to what the arguments allow.
struct Rows {
    int first, count;
};
__device__ inline Rows rows_of(const LinearArgs& a, int seq) {
    Rows r;
    r.first = a.starts[seq];
    const int64_t n = (int64_t)a.starts[seq + 1] - r.first;
    int64_t count = n < a.most_q ? n : a.most_q;
    if (r.first < 0) count = 0;
    if (count > a.total - (int64_t)r.first) count = a.total - (int64_t)r.first;
    r.count = count > 0 ? (int)count : 0;
    return r;
}

// The state of a sequence and head, [dk][dv], NULL for none.
__device__ inline float* state_at(const LinearArgs& a, const int64_t* slots, int seq, int head, int size) {
    if (!slots) return nullptr;
    const int64_t slot = slots[seq];
    return slot >= 0 && slot < a.slots ? a.states + (slot * a.heads + head) * size : nullptr;
}

// Decays below -200 are zeros beside any fp32 number, and sums of them keep their bits; a NaN stays.
__device__ inline float decay_at(const LinearArgs& a, int64_t row, int head) {
    const float g = a.decay[row * a.decay_stride + head];
    return g < -200.0f ? -200.0f : g;
}

}  // namespace iq4xs
