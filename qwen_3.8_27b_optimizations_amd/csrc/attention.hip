// attention.hip -- attention of new tokens over the paged cache: which kernel takes a call, how the keys are split, and
// the joining of the splits.
#include "attention_core.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

// One workgroup for each row and head: the splits' sums, each group of head_dim / 4 lanes taking every so-manieth split
// with a running maximum, then the groups in order.  Rows of one split were written by their kernel.
constexpr int JOIN_THREADS = 256;

template <int D>
__global__ __launch_bounds__(JOIN_THREADS) void join_splits_kernel(AttentionArgs a) {
    constexpr int LANES = D / 4, GROUPS = JOIN_THREADS / LANES;
    __shared__ f4 so[GROUPS][LANES];
    __shared__ float sm[GROUPS], sl[GROUPS], sr[GROUPS];
    const int head = blockIdx.x % a.q_heads, row = blockIdx.x / a.q_heads;
    const int seq = sequence_of(a.starts, a.seqs, row, threadIdx.x % 64);
    if (seq < 0 || seq >= a.seqs) return;
    int total_fresh;
    const Sequence s = sequence(a, seq, total_fresh);
    const int token = row - s.first;
    if (token >= s.fresh) return;
    const int lo = least_key(a, s, total_fresh, token), hi = end_key(a, s, total_fresh, token);
    if (one_split(a, s, lo, hi)) return;
    const int from = (lo - s.seen_from) / a.chunk, to = hi > lo ? (hi - 1 - s.seen_from) / a.chunk : from - 1;
    const int g = threadIdx.x / LANES, c = threadIdx.x % LANES;
    const int64_t out = (int64_t)row * a.q_heads + head, step = (int64_t)a.total * a.q_heads;
    float m = -FLT_MAX, l = 0.0f, rounded = 0.0f;
    f4 o{0, 0, 0, 0};
#pragma unroll 4
    for (int i = from + g; i <= to; i += GROUPS) {
        const int64_t at = i * step + out;
        const float4 ml = *reinterpret_cast<const float4*>(a.part_ml + 4 * at);
        const f4 v = *reinterpret_cast<const f4*>(a.part + at * D + 4 * c);
        const float up = fmaxf(m, ml.x), old = __builtin_amdgcn_exp2f(m - up), now = __builtin_amdgcn_exp2f(ml.x - up);
        m = up;
        l = l * old + ml.y * now;
        rounded = rounded * old + ml.z * now;
        o = o * old + v * now;
    }
    so[g][c] = o;
    if (c == 0) {
        sm[g] = m;
        sl[g] = l;
        sr[g] = rounded;
    }
    __syncthreads();
    if (g > 0) return;
    float best = sm[0];
#pragma unroll
    for (int i = 1; i < GROUPS; ++i) best = fmaxf(best, sm[i]);
    float sum = 0.0f, weights = 0.0f;
    f4 v{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const float f = __builtin_amdgcn_exp2f(sm[i] - best);
        sum += sl[i] * f;
        weights += sr[i] * f;
        v += so[i][c] * f;
    }
    store4(a.out, out * D + 4 * c, a.out_type, sum == 0.0f ? f4{0, 0, 0, 0} : v / weights);
    if (a.lse && c == 0) a.lse[out] = sum == 0.0f ? -INFINITY : (best + __log2f(sum)) * 0.69314718056f;
}

// The same with a wave for JOIN_EACH consecutive pairs of row and head: head_dim / 64 channels in a lane, the splits one
// after another.
constexpr int JOIN_EACH = 4;

template <int D>
__global__ __launch_bounds__(JOIN_THREADS) void join_splits_of_many_kernel(AttentionArgs a) {
    typedef float Part __attribute__((ext_vector_type(D / 64)));
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t pairs = (int64_t)a.total * a.q_heads, step = pairs;
    int64_t out = ((int64_t)blockIdx.x * (JOIN_THREADS / 64) + wave) * JOIN_EACH;
    int before = -1, from = 0, to = -1;
    bool skip = true;
    for (int e = 0; e < JOIN_EACH && out < pairs; ++e, ++out) {
        const int row = (int)(out / a.q_heads);
        if (row != before) {
            before = row;
            const int seq = sequence_of(a.starts, a.seqs, row, lane);
            skip = seq < 0 || seq >= a.seqs;
            if (!skip) {
                int total_fresh;
                const Sequence s = sequence(a, seq, total_fresh);
                const int token = row - s.first;
                skip = token >= s.fresh;
                if (!skip) {
                    const int lo = least_key(a, s, total_fresh, token), hi = end_key(a, s, total_fresh, token);
                    skip = one_split(a, s, lo, hi);
                    from = (lo - s.seen_from) / a.chunk;
                    to = hi > lo ? (hi - 1 - s.seen_from) / a.chunk : from - 1;
                }
            }
        }
        if (skip) continue;
        float m = -FLT_MAX, l = 0.0f, rounded = 0.0f;
        Part o = (Part)(0.0f);
#pragma unroll 4
        for (int i = from; i <= to; ++i) {
            const int64_t at = i * step + out;
            const float4 ml = *reinterpret_cast<const float4*>(a.part_ml + 4 * at);
            const Part v = *reinterpret_cast<const Part*>(a.part + at * D + D / 64 * lane);
            const float up = fmaxf(m, ml.x), old = __builtin_amdgcn_exp2f(m - up), now = __builtin_amdgcn_exp2f(ml.x - up);
            m = up;
            l = l * old + ml.y * now;
            rounded = rounded * old + ml.z * now;
            o = o * old + v * now;
        }
        const Part y = l == 0.0f ? (Part)(0.0f) : o / rounded;
        const int64_t at = out * D + D / 64 * lane;
#pragma unroll
        for (int c = 0; c < D / 64; ++c) {
            float z;
            if constexpr (D == 64)
                z = y[0];
            else
                z = y[c];
            if (a.out_type == IQ4XS_TYPE_F32)
                static_cast<float*>(a.out)[at + c] = z;
            else if (a.out_type == IQ4XS_TYPE_F16)
                static_cast<_Float16*>(a.out)[at + c] = (_Float16)z;
            else
                static_cast<__bf16*>(a.out)[at + c] = (__bf16)z;
        }
        if (a.lse && lane == 0) a.lse[out] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718056f;
    }
}

// What a call launches.
struct AttentionPlan {
    int tiles;      // 16-row tiles of a workgroup that streams the cache, or 0: the kernel of many rows
    int row_tiles;  // workgroups for the rows of a sequence and cache head
    int splits, chunk;
    int64_t grid;
};

// Whether the outputs show a rounding of an 8-bit cache's keys to fp16: all but bf16 ones do.
static bool exact_keys(const iq4xs_paged_attention_args& g) { return g.out_type != IQ4XS_TYPE_BF16 || g.lse; }

static int64_t at_most(int64_t x, int64_t most) { return x < most ? x : most; }

// Positions are below 2^31: a window of that many and more hides nothing, and sums with it could pass 64 bits.
static int64_t window_of(const iq4xs_paged_attention_args& g) { return g.window < 0x7FFFFFFF ? g.window : 0; }

static AttentionPlan plan_of(const iq4xs_paged_attention_args& g) {
    const int64_t group = g.q_heads / g.cache->heads, most_q = g.most_q < g.total ? g.most_q : g.total;
    AttentionPlan p;
    // Where the kernel of few rows ends: at two 16-row tiles, beyond which reading the keys again for the third costs more
    // than the other kernel's idle rows (40 rows: 75 against 54 us with 16-bit caches, 48 rows of an 8-bit one for bf16
    // outputs 94 against 72 of 256 channels, 64 against 57 of 128).  With exact 8-bit keys, which cost the other kernel
    // more, at 64 rows, with heads of 256 at 48 (64 rows of 64, 128, 256 channels: 66, 70, 121 against 99, 79, 115 us; 128
    // rows: 110, 118, 218 against 93, 87, 116).  One tile at a time where two do not fit the registers or leave most of the
    // second empty.
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
    const int64_t pairs = g.seqs * g.cache->heads * row_tiles, cus = device_cu_count();
    int64_t splits;
    if (p.tiles) {
        // One sequence, whose splits are alike: the workgroups that the CUs hold at once (by registers; one for each CU
        // keeps enough 16-bit keys on their way), none with less than 128 keys, 32 for a wave.  Several, which may
        // differ: up to eight times as many, in whole rounds (a few more than a round cost another: 8 sequences of 9001
        // keys of 256 channels 53 us in 9 splits, 35 in 8), while they have 512 keys (1024 of 256 channels).
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
        // the workgroups that the CUs hold at once, none with less than 512 keys: one with heads of 256 (1024-token
        // prompt 94 us with two, 50 with one), two with 128, and of 64, where they hold three, two for one sequence and
        // four for several, whose lengths differ (16 tokens over 32768 keys 43 us with two, 50 with four; 8 x 8 tokens 65
        // and 54)
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

static size_t part_bytes(const iq4xs_paged_attention_args& g, int splits) {
    return splits > 1 ? (size_t)splits * g.total * g.q_heads * g.cache->head_dim * sizeof(float) : 0;
}

size_t paged_attention_workspace(const iq4xs_paged_attention_args& g) {
    const int splits = plan_of(g).splits;
    return part_bytes(g, splits) + part_bytes(g, splits) / g.cache->head_dim * 4;
}

hipError_t launch_paged_attention(const iq4xs_paged_attention_args& g, void* ws, hipStream_t stream) {
    clear_launch_error();
    const AttentionPlan p = plan_of(g);
    const int D = g.cache->head_dim;
    float* part = static_cast<float*>(ws);
    const AttentionArgs a{cache_pages(*g.cache), g.q, g.out, g.lse, g.table, g.starts, g.kv_len, part,
                          p.splits > 1 ? part + part_bytes(g, p.splits) / sizeof(float) : nullptr, g.q_stride,
                          g.table_width, (int)g.total, (int)g.most_q, (int)g.most_kv, (int)window_of(g), (int)g.seqs,
                          g.q_heads, g.q_heads / g.cache->heads, g.out_type, g.causal, p.splits, p.chunk, p.row_tiles,
                          g.scale * 1.44269504089f};
    const int64_t join = g.total * g.q_heads;
    if (p.grid > 0x7FFFFFFF || join > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    if (p.tiles)
        launch_stream_attention(a, D, p.tiles, g.type, g.cache->type, p.grid, stream);
    else
        launch_tile_attention(a, D, g.type, g.cache->type, exact_keys(g), p.grid, stream);
    if (p.splits > 1) {
        const dim3 threads(JOIN_THREADS);
        // a workgroup for each costs 1.3 ns; a wave for four is slower while there are few, whose splits then wait for
        // each other (4 x 64 tokens, 16384 pairs: 84 us of a call in all, 78 so; 8 x 8 tokens, 4096 pairs: 47 and 50)
        const bool many = join >= 16384;
        const int64_t each = JOIN_THREADS / 64 * JOIN_EACH;
        const dim3 blocks((unsigned)(many ? (join + each - 1) / each : join));
        if (many && D == 64)
            hipLaunchKernelGGL((join_splits_of_many_kernel<64>), blocks, threads, 0, stream, a);
        else if (many && D == 128)
            hipLaunchKernelGGL((join_splits_of_many_kernel<128>), blocks, threads, 0, stream, a);
        else if (many)
            hipLaunchKernelGGL((join_splits_of_many_kernel<256>), blocks, threads, 0, stream, a);
        else if (D == 64)
            hipLaunchKernelGGL((join_splits_kernel<64>), blocks, threads, 0, stream, a);
        else if (D == 128)
            hipLaunchKernelGGL((join_splits_kernel<128>), blocks, threads, 0, stream, a);
        else
            hipLaunchKernelGGL((join_splits_kernel<256>), blocks, threads, 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace iq4xs
