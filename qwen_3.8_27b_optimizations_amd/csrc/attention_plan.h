// attention_plan.h -- which kernel takes an attention call, how the keys are split over workgroups, and which keys a row
// sees.  Plain arithmetic in a header of its own, so that the host tests compile the same rules; the kernels use the part
// on keys.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <type_traits>

#include "iq4xs_mi355x.h"

#ifdef __HIPCC__
#define IQ4XS_BOTH __host__ __device__
#else
#define IQ4XS_BOTH
#endif

namespace iq4xs {

// Where keys end that count.
constexpr int KEYS_END = (int)(((int64_t)1 << 31) - 4096);

// One sequence of the call, cut to what the arguments allow.
struct Sequence {
    int first, fresh;  // its rows in q: first row, count
    int keys;          // cached tokens
    int seen_from;     // first key that the first row sees, a multiple of 32: where split 0 begins
    const int32_t* pages;
    int skip;  // calls with first tokens or a shared prefix: keys that are not among the row's range [least, end)
};

// What a launch of a call with first tokens or a shared prefix is of: all of the former; of the latter the prefixes, a
// group of sequences in a sequence's place, or what comes after them.
enum Pass { PASS_SINKS, PASS_PREFIX, PASS_OWN };

// Whether the arguments are those of such a launch (they say MORE).
template <typename Args, typename = void>
struct HasMore : std::false_type {};
template <typename Args>
struct HasMore<Args, std::void_t<decltype(Args::MORE)>> : std::true_type {};

template <typename Args>
IQ4XS_BOTH inline int least_key(const Args& a, const Sequence& s, int total_fresh, int token) {
    const int64_t lo = (int64_t)s.keys - total_fresh + token + 1 - a.window;
    const int least = a.window > 0 && lo > 0 ? (lo < s.keys ? (int)lo : s.keys) : 0;
    if constexpr (HasMore<Args>::value) return least > s.skip ? least : s.skip;
    return least;
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
    s.skip = 0;
    s.seen_from = least_key(a, s, total_fresh, 0) & ~31;
    s.pages = a.table + (int64_t)seq * a.width;
    return s;
}

// The group that holds a sequence, -1 if none does or it has sequences that the call has not; NULL is one group of all.
template <typename Args>
IQ4XS_BOTH inline int group_of(const Args& a, int seq) {
    if (!a.group_first) return 0;
    int from = 0, to = a.groups;  // the groups before `from` begin at seq or before it, those from `to` on after it
    while (from < to) {
        const int mid = (from + to) / 2;
        if (a.group_first[mid] <= seq)
            from = mid + 1;
        else
            to = mid;
    }
    if (from == 0 || seq >= a.group_first[from]) return -1;
    return a.group_first[from - 1] >= 0 && a.group_first[from] <= a.all_seqs ? from - 1 : -1;
}

// Shared tokens of a group, cut to what the arguments allow.
template <typename Args>
IQ4XS_BOTH inline int shared_keys(const Args& a, int group) {
    if (group < 0) return 0;
    int64_t n = a.shared_len[group];
    n = n < a.most_shared ? n : a.most_shared;
    n = n < (a.width << a.c.shift) ? n : a.width << a.c.shift;
    return n > 0 ? (int)n : 0;
}

// The sequence of a launch with first tokens or of a shared prefix's; with PASS_PREFIX `seq` is a group, whose sequences'
// rows are one sequence's.
template <typename Args>
IQ4XS_BOTH inline Sequence sequence_more(const Args& a, int seq, int& total_fresh) {
    Sequence s;
    if (a.pass == PASS_SINKS) {
        s = sequence(a, seq, total_fresh);
        s.skip = a.sinks < s.keys ? a.sinks : s.keys;
    } else if (a.pass == PASS_PREFIX) {
        const int from = a.group_first ? a.group_first[seq] : 0, to = a.group_first ? a.group_first[seq + 1] : a.all_seqs;
        const bool some = from >= 0 && to <= a.all_seqs && from < to;
        s.first = some ? a.starts[from] : 0;
        total_fresh = some ? a.starts[to] - s.first : 0;
        s.fresh = total_fresh < a.most_q ? total_fresh : a.most_q;
        if (s.first < 0) s.fresh = 0;
        if (s.fresh > a.total - s.first) s.fresh = a.total - s.first;
        s.keys = shared_keys(a, seq);
        s.pages = a.table + (int64_t)(some ? from : 0) * a.width;
        s.skip = 0;
    } else {
        s = sequence(a, seq, total_fresh);
        const int skip = shared_keys(a, group_of(a, seq));
        int64_t keys = a.kv_len[seq];
        keys = keys < (int64_t)skip + a.most_kv ? keys : (int64_t)skip + a.most_kv;
        keys = keys < (a.width << a.c.shift) ? keys : a.width << a.c.shift;
        keys = keys < KEYS_END ? keys : KEYS_END;
        s.keys = keys > 0 ? (int)keys : 0;
        s.skip = skip < s.keys ? skip : s.keys;
    }
    s.seen_from = least_key(a, s, total_fresh, 0) & ~31;
    if (a.pass == PASS_SINKS) {
        // split 0's first tokens count as keys of its range, as far as that goes: a step less for its waves (8 x 5 tokens, a
        // window of 2048, 64 first tokens, 8-bit heads of 256: 39.1 us, 41.3 with a whole range behind them)
        const int first = (s.skip + 31) & ~31;
        s.seen_from -= first < a.chunk ? first : a.chunk;
    }
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

// The same of a launch with first tokens: split 0 has them too, the keys [0, extra) of the rows, before those of its range,
// which may be empty then.
template <typename Args>
IQ4XS_BOTH inline bool split_keys_more(const Args& a, const Sequence& s, int lo, int hi, int split, int& k0, int& k1,
                                       int& extra) {
    extra = a.pass == PASS_SINKS && split == 0 ? (s.skip < hi ? s.skip : hi) : 0;
    if (!split_keys(a, s, lo, hi, split, k0, k1)) {
        if (extra <= 0) return false;
        k0 = k1 = 0;
    }
    if (extra < 0) extra = 0;
    if (k1 < k0) k1 = k0;
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

// The same of a launch with first tokens.  A row that sees some sees key 0, in split 0, whatever its range; the parts of a
// shared prefix's launches are always joined.
template <typename Args>
IQ4XS_BOTH inline bool one_split_more(const Args& a, const Sequence& s, int lo, int hi) {
    if (a.pass != PASS_SINKS) return false;
    if (a.splits == 1) return true;
    if (hi <= lo) return hi > 0 && s.skip > 0;
    return split_of(a, s, lo) == split_of(a, s, hi - 1) && (s.skip == 0 || split_of(a, s, lo) == 0);
}
template <typename Args>
IQ4XS_BOTH inline RowEnd row_end_more(const Args& a, const Sequence& s, int lo, int hi, int split) {
    if (!one_split_more(a, s, lo, hi)) return ROW_PART;
    return a.splits == 1 || (hi > lo ? split_of(a, s, lo) : 0) == split ? ROW_OUT : ROW_NONE;
}

// Where the parts of a row lie that are joined: `before` of them from 0 on, `after` from `from` on.
struct RowParts {
    int before, from, after;
    IQ4XS_BOTH int count() const { return before + after; }
    IQ4XS_BOTH int at(int i) const { return i < before ? i : from + i - before; }
};
template <typename Args>
IQ4XS_BOTH inline RowParts row_parts(const Args& a, const Sequence& s, int lo, int hi) {
    int first, last;
    splits_of(a, s, lo, hi, first, last);
    if (hi <= lo) first = last + 1;
    if (a.pass == PASS_SINKS) {
        const int before = hi > 0 && s.skip > 0 && (first > 0 || hi <= lo);
        return {before, first, last - first + 1};
    }
    // s.skip: the shared tokens, as far as the sequence reaches; the prefix's parts lie before the others
    return {0, a.prefix_splits + first, last - first + 1};
}
// The parts of the prefix, of a group that shares `keys` tokens.
template <typename Args>
IQ4XS_BOTH inline int prefix_parts(const Args& a, int keys) {
    if (keys <= 0) return 0;
    const int last = (keys - 1) / a.prefix_chunk;
    return (last < a.prefix_splits ? last : a.prefix_splits - 1) + 1;
}

// The keys that a workgroup goes through, KEYS at a time: [k0, k1), and before them as many steps as the first tokens
// [0, extra) take.  Steps are at `base` from start on; those before k0 are of first tokens.
template <int KEYS, bool MORE>
struct KeySteps {
    int k0, k1, extra, start;
    IQ4XS_BOTH KeySteps(int k0, int k1, int extra)
        : k0(k0), k1(k1), extra(extra), start(MORE ? k0 - (extra + KEYS - 1) / KEYS * KEYS : k0) {}
    IQ4XS_BOTH bool is_first(int base) const { return MORE && base < k0; }
    IQ4XS_BOTH int place(int base) const { return is_first(base) ? base - start : base; }  // first key of the step
    IQ4XS_BOTH int stop(int base) const { return is_first(base) ? extra : k1; }             // where its keys end
    // whether rows that all see [lo, hi) see the whole step
    IQ4XS_BOTH bool all_see(int base, int lo, int hi) const {
        if (is_first(base)) return place(base) + KEYS <= (extra < hi ? extra : hi);
        return base >= lo && base + KEYS <= hi;
    }
    // of a row that sees [lo, hi): what it sees of the step's kind
    IQ4XS_BOTH int lo_in(int base, int lo) const { return is_first(base) ? 0 : lo; }
    IQ4XS_BOTH int hi_in(int base, int hi) const { return is_first(base) && extra < hi ? extra : hi; }
};

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
inline int most_kv_of(const iq4xs_paged_attention_args& g) { return (int)at_most(g.most_kv, KEYS_END); }

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
    // the keys of a sequence that some row sees; a window's first key lies anywhere in a step of 32.  No more than count: a
    // call may name lengths whose splits, rounded up to 128 keys, are no ints.
    int64_t span = most_kv_of(g);
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

// Sums of `splits` splits for every row and head.
inline size_t parts_bytes(const iq4xs_paged_attention_args& g, int splits) {
    return (size_t)splits * g.total * g.q_heads * g.cache->head_dim * sizeof(float);
}

// Whether first tokens are more than the window shows: a window as long as the longest sequence hides none.
inline bool sinks_matter(const iq4xs_paged_attention_args& g, int64_t sinks) {
    return sinks > 0 && window_of(g) > 0 && window_of(g) < g.most_kv;
}

// The launch over the prefixes of a call as one over groups: their rows all see all of it.
inline iq4xs_paged_attention_args prefix_call(const iq4xs_paged_attention_args& g, const iq4xs_shared_prefix& x) {
    iq4xs_paged_attention_args p = g;
    p.seqs = x.groups;
    p.most_q = x.most_rows;
    p.most_kv = at_most(x.most_len, KEYS_END);
    p.causal = 0;
    return p;
}

// Each sequence by itself: a call without shared prefixes.
inline iq4xs_paged_attention_args each_call(const iq4xs_paged_attention_args& g, const iq4xs_shared_prefix& x) {
    iq4xs_paged_attention_args p = g;
    p.most_kv = at_most(x.most_len, KEYS_END) + at_most(g.most_kv, KEYS_END);
    return p;
}

struct SharedPlan {
    bool once;
    AttentionPlan prefix, own;  // with `once`; the latter else each sequence's whole
    int parts() const { return once ? prefix.splits + own.splits : own.splits > 1 ? own.splits : 0; }
};

// Once costs two more launches, each sequence by itself reads shared keys again, though from caches that hold them: 8 heads of
// 128, one token each, fp16, 4096 shared tokens, 8, 16 and 32 sequences 29, 32, 37 us once and 21, 34, 56 each; 16384, 2, 4
// and 64 sequences 26, 28, 74 and 22, 34, 317; 8 bits 4 heads of 256, 4 tokens each, 4096, 16 and 32 sequences 77, 81 and 66,
// 117: from 2^26 elements of keys read again on.  Between 2^25 and 2^26 the sides differ by type (4 fp16 sequences behind 16384
// 28 once and 34 each, but 16 of 8 bits behind 4096 42 and 32), and there is no third launch each by itself.
// 128 rows of a sequence and head on each: the products bound such calls, of which there are no fewer, but those of a last tile
// that is hardly used (64 tokens of 64 heads on 8, fp16, 16384 shared: 4, 8 and 16 sequences 179, 331, 630 once and 166, 311,
// 585 each; 24 tokens, 192 rows, 95, 162, 285 and 95, 171, 297; 17 tokens, 136 rows, 80, 127, 204 and 89, 162, 287; behind
// 4096 tokens 17 take 51, 66, 79 and 41, 63, 89).  A caller that knows such rows says so by `path`.
inline bool shared_once(const iq4xs_paged_attention_args& g, const iq4xs_shared_prefix& x) {
    if (x.path != IQ4XS_SHARED_AUTO) return x.path == IQ4XS_SHARED_ONCE;
    const int64_t most_q = g.most_q < g.total ? g.most_q : g.total;
    if (most_q * (g.q_heads / g.cache->heads) >= 128) return false;
    const int64_t again = g.seqs > x.groups ? g.seqs - x.groups : 0, each = (int64_t)g.cache->heads * g.cache->head_dim;
    return again > 0 && x.most_len > ((int64_t)1 << 26) / each / again;
}

inline bool shared_plan_fits(const iq4xs_paged_attention_args& g, const iq4xs_shared_prefix& x, int64_t cus,
                             SharedPlan& p) {
    p.once = shared_once(g, x);
    if (!p.once) return plan_fits(each_call(g, x), cus, p.own);
    if (!plan_fits(prefix_call(g, x), cus, p.prefix) || !plan_fits(g, cus, p.own)) return false;
    if (p.prefix.tiles == 0 && p.prefix.splits > 1) {
        // groups' prefixes are mostly alike: no workgroup more than the CUs hold at once, or it takes as long again (two
        // groups of 350 rows over 8187 tokens of heads of 256, 8 bits: 264 workgroups 135 us, 240 97)
        const int64_t rows = p.prefix.grid / p.prefix.splits, held = g.cache->head_dim == 256 ? 1 : 2;
        int64_t splits = held * cus / rows;
        if (splits < 1) splits = 1;
        if (splits < p.prefix.splits) {
            const int64_t keys = at_most(x.most_len, KEYS_END);
            p.prefix.chunk = (int)(((keys + splits - 1) / splits + 127) / 128 * 128);
            p.prefix.splits = (int)((keys + p.prefix.chunk - 1) / p.prefix.chunk);
            p.prefix.grid = rows * p.prefix.splits;
        }
    }
    return true;
}

}  // namespace iq4xs
