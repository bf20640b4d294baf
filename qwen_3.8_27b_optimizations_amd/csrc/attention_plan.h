// attention_plan.h -- which kernel takes an attention call, how the keys are split over workgroups, and which keys a row
// sees.  Plain arithmetic in a header of its own, so that the host tests compile the same rules; the kernels use the part
// on keys.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "iq4xs_mi355x.h"

#ifdef __HIPCC__
#define IQ4XS_BOTH __host__ __device__
#else
#define IQ4XS_BOTH
#endif

namespace iq4xs {

// One sequence of the call, cut to what the arguments allow.
struct Sequence {
    int first, fresh;  // its rows in q: first row, count
    int keys;          // cached tokens
    int seen_from;     // first key that the first row sees, a multiple of 32: where split 0 begins
    const int32_t* pages;
};

template <typename Args>
IQ4XS_BOTH inline int least_key(const Args& a, const Sequence& s, int total_fresh, int token) {
    const int64_t lo = (int64_t)s.keys - total_fresh + token + 1 - a.window;
    return a.window > 0 && lo > 0 ? (lo < s.keys ? (int)lo : s.keys) : 0;
}
template <typename Args>
IQ4XS_BOTH inline int end_key(const Args& a, const Sequence& s, int total_fresh, int token) {
    const int64_t hi = (int64_t)s.keys - total_fresh + token + 1;
    return !a.causal || hi > s.keys ? s.keys : hi > 0 ? (int)hi : 0;
}

// total_fresh: the new tokens as the positions count them; s.fresh of them are rows to compute.
template <typename Args>
IQ4XS_BOTH inline Sequence sequence(const Args& a, int seq, int& total_fresh) {
    Sequence s;
    s.first = a.starts[seq];
    total_fresh = a.starts[seq + 1] - s.first;
    s.fresh = total_fresh < a.most_q ? total_fresh : a.most_q;
    if (s.first < 0) s.fresh = 0;
    if (s.fresh > a.total - s.first) s.fresh = a.total - s.first;
    int64_t keys = a.kv_len[seq];
    keys = keys < a.most_kv ? keys : a.most_kv;
    keys = keys < (a.width << a.c.shift) ? keys : a.width << a.c.shift;
    s.keys = keys > 0 ? (int)keys : 0;
    s.seen_from = least_key(a, s, total_fresh, 0) & ~31;
    s.pages = a.table + (int64_t)seq * a.width;
    return s;
}

// The split that a key belongs to.  The last one goes on to the end: lengths are read on the device, and a sequence of more
// new tokens than most_q may see more keys than the splits were planned for (with a window, its first row's lies further
// back).
template <typename Args>
IQ4XS_BOTH inline int split_of(const Args& a, const Sequence& s, int key) {
    const int split = (key - s.seen_from) / a.chunk;
    return split < a.splits ? split : a.splits - 1;
}

// The keys [k0, k1) that a workgroup of rows that see some of [lo, hi) takes as its split; false: none, and no rows to
// write either.
template <typename Args>
IQ4XS_BOTH inline bool split_keys(const Args& a, const Sequence& s, int lo, int hi, int split, int& k0, int& k1) {
    const int64_t from = s.seen_from + (int64_t)split * a.chunk, to = from + a.chunk;
    const bool last = split + 1 == a.splits;
    if (a.splits > 1 && (hi <= from || (!last && to <= lo))) return false;
    k0 = from < (lo & ~31) ? lo & ~31 : (int)from;
    k1 = last || hi < to ? hi : (int)to;
    return true;
}

// The splits that hold keys of a row that sees [lo, hi): first and last, which is before the first if there are none.
template <typename Args>
IQ4XS_BOTH inline void splits_of(const Args& a, const Sequence& s, int lo, int hi, int& first, int& last) {
    first = split_of(a, s, lo);
    last = hi > lo ? split_of(a, s, hi - 1) : first - 1;
}

// Where the sums of a row that sees the keys [lo, hi) go: with one split, to the outputs, from the workgroup of that
// split; with several, to its place in the workspace, from every workgroup that has them, and the joining kernel writes
// the outputs, as it does for a row that sees nothing.
enum RowEnd { ROW_OUT, ROW_PART, ROW_NONE };

template <typename Args>
IQ4XS_BOTH inline bool one_split(const Args& a, const Sequence& s, int lo, int hi) {
    return a.splits == 1 || (hi > lo && split_of(a, s, lo) == split_of(a, s, hi - 1));
}
template <typename Args>
IQ4XS_BOTH inline RowEnd row_end(const Args& a, const Sequence& s, int lo, int hi, int split) {
    if (!one_split(a, s, lo, hi)) return ROW_PART;
    return a.splits == 1 || split_of(a, s, lo) == split ? ROW_OUT : ROW_NONE;
}

// What a call launches.
struct AttentionPlan {
    int tiles;      // 16-row tiles of a workgroup that streams the cache, or 0: the kernel of many rows
    int row_tiles;  // workgroups for the rows of a sequence and cache head
    int splits, chunk;
    int64_t grid;
};

// Whether the outputs show a rounding of an 8-bit cache's keys to fp16: all but bf16 ones do.
inline bool exact_keys(const iq4xs_paged_attention_args& g) { return g.out_type != IQ4XS_TYPE_BF16 || g.lse; }

inline int64_t at_most(int64_t x, int64_t most) { return x < most ? x : most; }

// Positions are below 2^31: a window of that many and more hides nothing, and sums with it could pass 64 bits.
inline int64_t window_of(const iq4xs_paged_attention_args& g) { return g.window < 0x7FFFFFFF ? g.window : 0; }

// Keys of a sequence that count: their places, and those of a few steps past the end, are ints in the kernels.
inline int most_kv_of(const iq4xs_paged_attention_args& g) {
    return (int)at_most(g.most_kv, ((int64_t)1 << 31) - 4096);
}

inline AttentionPlan plan_of(const iq4xs_paged_attention_args& g, int64_t cus) {
    const int64_t group = g.q_heads / g.cache->heads, most_q = g.most_q < g.total ? g.most_q : g.total;
    AttentionPlan p;
    // Where the kernel of few rows ends: at two 16-row tiles, beyond which reading the keys again for the third costs more
    // than the other kernel's idle rows (8 sequences of 9001 keys, 40 rows a cache head, of 64, 128, 256 channels: 16-bit
    // caches 90, 82, 80 us here and 70, 58, 66 there, 8-bit ones for bf16 outputs 88, 77, 96 and 72, 59, 71; 32 rows: 64,
    // 61, 58 and 73, 57, 66, and 55, 51, 68 and 74, 57, 70).  With exact 8-bit keys, which cost the other kernel more, at 64
    // rows, with heads of 256 at 48 (48 rows: 87, 77, 95 and 102, 82, 112; 64 rows: 91, 82, 125 and 106, 84, 115; 128 rows:
    // 163, 150, 246 and 107, 95, 123).  One tile at a time where two do not fit the registers or leave most of the second
    // empty.
    const int64_t rows = most_q * group;
    const bool codes = g.cache->type == IQ4XS_TYPE_Q8, wide = g.cache->head_dim == 256;
    if (rows > (codes && exact_keys(g) ? wide ? 48 : 64 : 32))
        p.tiles = 0;
    else
        p.tiles = rows <= 16 || (codes && (wide || (rows > 32 && rows <= 48))) ? 1 : 2;
    const int64_t tile = p.tiles ? 16 * p.tiles : 128, row_tiles = (most_q * group + tile - 1) / tile;
    // the keys of a sequence that some row sees; a window's first key lies anywhere in a step of 32
    int64_t span = g.most_kv;
    const int64_t window = window_of(g);
    if (window > 0 && window + most_q + 32 < span) span = window + most_q + 32;
    const int64_t pairs = g.seqs * g.cache->heads * row_tiles;
    int64_t splits;
    if (p.tiles) {
        // One sequence, whose splits are alike: the workgroups that the CUs hold at once (by registers; one for each CU
        // keeps enough 16-bit keys on their way), none with less than 128 keys, 32 for a wave.  Several, which may
        // differ: up to eight times as many, in whole rounds (a few more than a round cost another: 8 x 2 tokens over
        // 9001 keys of 8-bit heads of 256 40 us, 61 in one split more), while they have 512 keys (1024 of 256 channels).
        const int64_t held = g.cache->head_dim == 64 ? 4 : g.cache->head_dim == 256 ? 1 : p.tiles == 2 ? 2 : codes ? 3 : 2;
        const int64_t one = g.seqs == 1 && !codes && g.cache->head_dim == 128 ? 1 : held;
        const int64_t round = one * cus / pairs;  // splits of one
        if (round == 0) {
            splits = at_most((8 * held * cus + pairs - 1) / pairs, (span + 511) / 512);
        } else {
            const int64_t least = g.cache->head_dim == 256 ? 1024 : 512;
            const int64_t rounds = g.seqs == 1 ? 1 : at_most(8, span / (least * round));
            splits = at_most(round * (rounds > 1 ? rounds : 1), (span + 127) / 128);
        }
    } else {
        // the workgroups that the CUs hold at once, none with less than 512 keys: one with heads of 256 (a 1024-token
        // prompt 48 us, 60 with two), two with 128 (33, 58 with four), and of 64, where they hold three, two for one
        // sequence (16 tokens over 32768 keys 40, 47 with four) and four for several, whose lengths differ (8 x 8 tokens
        // over 2250 to 9001 keys 54, 65 with two; 80 and 75 over 9001 each, 106 and 87 for 32 x 16 over 1024 to 4096)
        const int64_t held = wide ? 1 : g.cache->head_dim == 64 && g.seqs > 1 ? 4 : 2;
        splits = at_most((held * cus + pairs - 1) / pairs, (span + 511) / 512);
    }
    const int64_t chunk = ((span + splits - 1) / splits + 127) / 128 * 128;
    p.splits = (int)((span + chunk - 1) / chunk);
    p.chunk = (int)chunk;
    p.row_tiles = (int)(row_tiles < 0x7FFFFFFF ? row_tiles : 0x7FFFFFFF);
    p.grid = pairs * p.splits;
    return p;
}

// The plan of a call, unless its launches would be too large: a workgroup for each row and head, without whose limit the
// plan's products could pass 64 bits, and the plan's own.
inline bool plan_fits(const iq4xs_paged_attention_args& g, int64_t cus, AttentionPlan& p) {
    constexpr int64_t MOST = 0x7FFFFFFF;
    if (g.total > MOST / g.q_heads) return false;
    p = plan_of(g, cus);
    return p.grid <= MOST;
}

inline size_t part_bytes(const iq4xs_paged_attention_args& g, int splits) {
    return splits > 1 ? (size_t)splits * g.total * g.q_heads * g.cache->head_dim * sizeof(float) : 0;
}

}  // namespace iq4xs
