// linear_plan.h -- which kernel takes a call of linear attention, and the segments of its sequences.  Plain arithmetic in a
// header of its own, so that the host tests compile the same rules.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "iq4xs_mi355x.h"

namespace iq4xs {

// Columns of a state that a workgroup of the kernel of chunks takes: 128 while their accumulators fit the registers.
inline int linear_chunk_columns(int dk, int dv) { return dk == 256 || dv == 64 ? 64 : 128; }

struct LinearPlan {
    bool steps;           // token by token
    int segments;         // of the longest sequence
    int length;           // tokens of a segment, a multiple of 64
    int64_t units;        // of 32 columns of a head's state, token by token
    size_t state_bytes;   // states that segments begin with
    size_t decay_bytes;   // and what segments keep of them
};

// False: its launches would be too large.
inline bool linear_plan(const iq4xs_linear_attention_args& g, int64_t cus, LinearPlan& p) {
    constexpr int64_t MOST = 0x7FFFFFFF;
    const int64_t most = g.most_q < g.total ? g.most_q : g.total;
    p = {true, 1, (int)((most + 63) / 64 * 64), 0, 0, 0};
    if (g.seqs > MOST / g.heads / 8) return false;  // 32 columns of 256 at a time
    p.units = g.seqs * g.heads * (g.dv / 32);
    if (most <= 16) return true;
    p.steps = false;
    // Segments: as long as makes work for the workgroups that the CUs hold at once, two each of bf16 inputs and one of others,
    // whose parts fill LDS, and none less than 256 tokens.  Their states cost half of the work again, so only where the
    // longest sequence would take half as long again as that.
    const int64_t units = g.heads * (g.dv / linear_chunk_columns(g.dk, g.dv));
    const int64_t slots = (g.in_type == IQ4XS_TYPE_BF16 ? 2 : 1) * cus;
    int64_t length = (g.total * units + slots - 1) / slots;
    if (length < 256) length = 256;
    if (2 * most > 3 * length) {
        const int64_t segments = (most + length - 1) / length;
        p.length = (int)(((most + segments - 1) / segments + 63) / 64 * 64);
        p.segments = (int)((most + p.length - 1) / p.length);
    }
    if (p.segments > 1) {
        const int64_t places = g.seqs * p.segments * g.heads;
        p.state_bytes = (size_t)places * g.dk * g.dv * sizeof(float);
        p.decay_bytes = ((size_t)places * sizeof(float) + 255) / 256 * 256;
    }
    return g.seqs * units <= MOST / p.segments;
}

}  // namespace iq4xs
