// attention.hip -- attention of new tokens over the paged cache: its launches (by attention_plan.h), and the joining of the
// splits.
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
    if (token < 0 || token >= s.fresh) return;  // below zero: starts that fall
    const int lo = least_key(a, s, total_fresh, token), hi = end_key(a, s, total_fresh, token);
    if (one_split(a, s, lo, hi)) return;
    int from, to;
    splits_of(a, s, lo, hi, from, to);
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
                skip = token < 0 || token >= s.fresh;
                if (!skip) {
                    const int lo = least_key(a, s, total_fresh, token), hi = end_key(a, s, total_fresh, token);
                    skip = one_split(a, s, lo, hi);
                    splits_of(a, s, lo, hi, from, to);
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

static size_t workspace_of(const iq4xs_paged_attention_args& g, const AttentionPlan& p) {
    return part_bytes(g, p.splits) + part_bytes(g, p.splits) / g.cache->head_dim * 4;
}

hipError_t paged_attention_workspace(const iq4xs_paged_attention_args& g, size_t* bytes) {
    AttentionPlan p;
    if (!plan_fits(g, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    *bytes = workspace_of(g, p);
    return hipSuccess;
}

hipError_t launch_paged_attention(const iq4xs_paged_attention_args& g, void* ws, size_t ws_bytes, hipStream_t stream) {
    AttentionPlan p;
    if (!plan_fits(g, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    const size_t need = workspace_of(g, p);
    if (ws_bytes < need || (need && (!ws || reinterpret_cast<uintptr_t>(ws) % 256 != 0))) return hipErrorInvalidValue;
    clear_launch_error();
    const int D = g.cache->head_dim;
    float* part = static_cast<float*>(ws);
    const AttentionArgs a{cache_pages(*g.cache), g.q, g.out, g.lse, g.table, g.starts, g.kv_len, part,
                          p.splits > 1 ? part + part_bytes(g, p.splits) / sizeof(float) : nullptr, g.q_stride,
                          g.table_width, (int)g.total, (int)g.most_q, most_kv_of(g), (int)window_of(g), (int)g.seqs,
                          g.q_heads, g.q_heads / g.cache->heads, g.out_type, g.causal, p.splits, p.chunk, p.row_tiles,
                          g.scale * 1.44269504089f};
    const int64_t join = g.total * g.q_heads;
    if (p.tiles)
        launch_stream_attention(a, D, p.tiles, g.type, g.cache->type, p.grid, stream);
    else
        launch_tile_attention(a, D, g.type, g.cache->type, exact_keys(g), p.grid, stream);
    if (p.splits > 1) {
        const dim3 threads(JOIN_THREADS);
        // a workgroup for each costs 1.3 ns; a wave for four is slower while there are few, whose splits then wait for
        // each other (of a call in all, 64 heads: one token over 4096 keys 12 us, 25 so; 8 x 8 tokens, 4096 pairs, 67 and
        // 68; 4 x 64 over 8192 keys, 16384 pairs, 107 and 93)
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
