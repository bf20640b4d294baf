// linear_plan.h -- which kernel takes a call of linear attention, the segments of its sequences, and where workgroups and states
// of segments are counted.  Plain arithmetic in a header of its own, so that the host tests compile the same rules; the kernels
// use the part on places.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "iq4xs_mi355x.h"

#ifndef IQ4XS_BOTH
#ifdef __HIPCC__
#define IQ4XS_BOTH __host__ __device__
#else
#define IQ4XS_BOTH
#endif
#endif

namespace iq4xs {

// Numbers for the segments of each sequence that no other has, from what a kernel knows of one sequence: its first row and its
// index.  First place rows * row / length + each * seq, and as many as it has segments.
//   rows 0, each the segments of the longest: seqs * each of them
//   rows 1, each 1: total / length + seqs, as ceil(n / length) is no more than the whole lengths that end within n rows and one
//   rows 2, each 0: 2 * total / length, for sequences of two segments and more, as ceil(m) <= floor(2 m) where m > 1
// One long prompt among many single tokens has few segments, which the first of these does not see, and few that are kept,
// which the second does not.
struct SegmentPlaces {
    int rows, each, length;
    IQ4XS_BOTH int64_t of(int row, int seq) const {  // 2 * row is below 2^32
        return (uint32_t)rows * (uint32_t)row / (uint32_t)length + (int64_t)each * seq;
    }
};
inline int64_t places_in(const SegmentPlaces& p, int64_t total, int64_t seqs) { return p.of((int)total, (int)seqs); }

// Sequences of three segments and more are joined: with more sequences than these rows, by the only one of every 2 * length
// rows that lies in the first 2 * length of a sequence.
inline int64_t joining_rows(int64_t total, int length) { return (total + 2 * (int64_t)length - 1) / (2 * (int64_t)length); }

// Columns of a state that a workgroup of the kernel of chunks takes: 128 while their accumulators fit the registers.
inline int linear_chunk_columns(int dk, int dv) { return dk == 256 || dv == 64 ? 64 : 128; }

constexpr size_t SEGMENT_DECAY_BYTES = 8;

struct LinearPlan {
    bool steps;           // token by token
    int segments;         // of the longest sequence
    int length;           // tokens of a segment, a multiple of 64
    int64_t units;        // of 32 columns of a head's state, token by token
    SegmentPlaces runs;   // workgroups, for each head and its columns
    SegmentPlaces kept;   // states of segments
    bool join_rows;       // whether sequences are joined by joining_rows, or one by one
    int64_t grid;
    size_t state_bytes;   // states that segments begin with
    size_t decay_bytes;   // and what segments keep of them
};

// False: its launches would be too large.
inline bool linear_plan(const iq4xs_linear_attention_args& g, int64_t cus, LinearPlan& p) {
    constexpr int64_t MOST = 0x7FFFFFFF;
    const int64_t most = g.most_q < g.total ? g.most_q : g.total;
    p = {};
    p.steps = true;
    p.segments = 1;
    p.length = (int)(most < MOST - 63 ? (most + 63) / 64 * 64 : MOST);  // one segment: as long as any sequence
    if (g.seqs > MOST / g.heads / 8) return false;  // 32 columns of 256 at a time
    p.units = g.seqs * g.heads * (g.dv / 32);
    // Token by token while that is no slower: a chunk's work hardly grows with its tokens, a step's does (64 heads of 128 x
    // 128, steps and chunks in turn.  64 sequences of 4, 5, 8 and 16 tokens: bf16 114, 125, 154, 238 us and 113, 113, 114, 118;
    // fp16 111, 122, 154, 236 and 155, 155, 156, 159; fp32 124, 135, 169, 268 and 175, 176, 180, 190.  8 sequences of 4, 5 and
    // 8: bf16 17, 18, 22 and 17, 18, 18; of 5, 8 and 12: fp16 18, 22, 27 and 23, 23, 23.  One of 5 and 8: bf16 11, 11 and 11,
    // 11; of 8 and 12: fp16 11, 14 and 11, 11.  Between, 4 of 8 fp16 tokens lose 3 us: 14 and 11).
    if (most <= (g.in_type == IQ4XS_TYPE_BF16 ? 4 : 8)) return true;
    p.steps = false;
    // Segments: as long as makes work for the workgroups that the CUs hold at once, two each of bf16 inputs and one of others,
    // whose parts fill LDS, and none less than 256 tokens (4096 tokens of 64 heads, bf16: 8 segments 117 us, 4 147, 11 135).
    // Their states cost half of the work again, so only where the longest sequence would take half as long again as that
    // (5 prompts of 987 to 4001 tokens, fp16: 471 us whole, 664 in up to 2 segments).
    const int64_t units = g.heads * (g.dv / linear_chunk_columns(g.dk, g.dv));
    const int64_t slots = (g.in_type == IQ4XS_TYPE_BF16 ? 2 : 1) * cus;
    int64_t length = (g.total * units + slots - 1) / slots;
    if (length < 256) length = 256;
    if (2 * most > 3 * length) {
        const int64_t segments = (most + length - 1) / length;
        p.length = (int)(((most + segments - 1) / segments + 63) / 64 * 64);
        p.segments = (int)((most + p.length - 1) / p.length);
    }
    const SegmentPlaces places[] = {{0, p.segments, p.length}, {1, 1, p.length}, {2, 0, p.length}};
    p.runs = p.kept = places[0];
    if (p.segments > 1) {
        for (int i = 1; i < 3; ++i) {
            const int64_t n = places_in(places[i], g.total, g.seqs);
            if (i == 1 && n < places_in(p.runs, g.total, g.seqs)) p.runs = places[i];
            if (n < places_in(p.kept, g.total, g.seqs)) p.kept = places[i];
        }
        p.join_rows = joining_rows(g.total, p.length) < g.seqs;
        if (g.seqs * g.heads > MOST / 64) return false;  // the launch that joins them: 1024 elements of 256 x 256 each
        const size_t states = (size_t)places_in(p.kept, g.total, g.seqs) * g.heads;
        p.state_bytes = states * g.dk * g.dv * sizeof(float);
        p.decay_bytes = (states * SEGMENT_DECAY_BYTES + 255) / 256 * 256;
    }
    const int64_t runs = places_in(p.runs, g.total, g.seqs);
    if (runs > MOST / units) return false;
    p.grid = runs * units;
    return true;
}

}  // namespace iq4xs
