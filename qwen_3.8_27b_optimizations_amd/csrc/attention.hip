// attention.hip -- attention of new tokens over the paged cache: its launches (by attention_plan.h), also with first tokens
// beside a window or a prefix that sequences share, and the joining of the splits.
#include "attention_core.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

// The parts of a row that are to be joined; false: none, as no call computes the row or its kernel wrote it.
template <typename Args>
__device__ inline bool parts_of_row(const Args& a, int row, int lane, RowParts& parts) {
    const int all = [&] {
        if constexpr (HasMore<Args>::value) return a.all_seqs;
        return a.seqs;
    }();
    const int seq = sequence_of(a.starts, all, row, lane);
    if (seq < 0 || seq >= all) return false;
    int total_fresh;
    Sequence s;
    if constexpr (HasMore<Args>::value)
        s = sequence_more(a, seq, total_fresh);
    else
        s = sequence(a, seq, total_fresh);
    const int token = row - s.first;
    if (token < 0 || token >= s.fresh) return false;  // below zero: starts that fall
    const int lo = least_key(a, s, total_fresh, token), hi = end_key(a, s, total_fresh, token);
    if constexpr (HasMore<Args>::value) {
        if (one_split_more(a, s, lo, hi)) return false;
        parts = row_parts(a, s, lo, hi);
        if (a.pass == PASS_SINKS) return true;
        const int group = group_of(a, seq);
        parts.before = prefix_parts(a, shared_keys(a, group));
        if (parts.before == 0) return true;
        const int from = a.group_first ? a.group_first[group] : 0;
        return row - a.starts[from] < a.prefix_rows;
    } else {
        if (one_split(a, s, lo, hi)) return false;
        int from, to;
        splits_of(a, s, lo, hi, from, to);
        parts = {0, from, to - from + 1};
        return true;
    }
}

// One workgroup for each row and head: the splits' sums, each group of head_dim / 4 lanes taking every so-manieth split
// with a running maximum, then the groups in order.  Rows of one split were written by their kernel.
constexpr int JOIN_THREADS = 256;

template <int D, typename Args>
__global__ __launch_bounds__(JOIN_THREADS) void join_splits_kernel(Args a) {
    constexpr int LANES = D / 4, GROUPS = JOIN_THREADS / LANES;
    __shared__ f4 so[GROUPS][LANES];
    __shared__ float sm[GROUPS], sl[GROUPS], sr[GROUPS];
    const int head = blockIdx.x % a.q_heads, row = blockIdx.x / a.q_heads;
    RowParts parts;
    if (!parts_of_row(a, row, threadIdx.x % 64, parts)) return;
    const int g = threadIdx.x / LANES, c = threadIdx.x % LANES;
    const int64_t out = (int64_t)row * a.q_heads + head, step = (int64_t)a.total * a.q_heads;
    float m = -FLT_MAX, l = 0.0f, rounded = 0.0f;
    f4 o{0, 0, 0, 0};
#pragma unroll 4
    for (int i = g; i < parts.count(); i += GROUPS) {
        const int64_t at = parts.at(i) * step + out;
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

template <int D, typename Args>
__global__ __launch_bounds__(JOIN_THREADS) void join_splits_of_many_kernel(Args a) {
    typedef float Part __attribute__((ext_vector_type(D / 64)));
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int64_t pairs = (int64_t)a.total * a.q_heads, step = pairs;
    int64_t out = ((int64_t)blockIdx.x * (JOIN_THREADS / 64) + wave) * JOIN_EACH;
    int before = -1;
    RowParts parts{0, 0, 0};
    bool skip = true;
    for (int e = 0; e < JOIN_EACH && out < pairs; ++e, ++out) {
        const int row = (int)(out / a.q_heads);
        if (row != before) {
            before = row;
            skip = !parts_of_row(a, row, lane, parts);
        }
        if (skip) continue;
        float m = -FLT_MAX, l = 0.0f, rounded = 0.0f;
        Part o = (Part)(0.0f);
#pragma unroll 4
        for (int i = 0; i < parts.count(); ++i) {
            const int64_t at = parts.at(i) * step + out;
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

template <typename Args>
static void launch_join(const Args& a, int D, hipStream_t stream) {
    const int64_t join = (int64_t)a.total * a.q_heads;
    const dim3 threads(JOIN_THREADS);
    // a workgroup for each costs 1.3 ns; a wave for four is slower while there are few, whose splits then wait for
    // each other (of a call in all, 64 heads: one token over 4096 keys 12 us, 25 so; 8 x 8 tokens, 4096 pairs, 67 and
    // 68; 4 x 64 over 8192 keys, 16384 pairs, 107 and 93)
    const bool many = join >= 16384;
    const int64_t each = JOIN_THREADS / 64 * JOIN_EACH;
    const dim3 blocks((unsigned)(many ? (join + each - 1) / each : join));
    if (many && D == 64)
        hipLaunchKernelGGL((join_splits_of_many_kernel<64, Args>), blocks, threads, 0, stream, a);
    else if (many && D == 128)
        hipLaunchKernelGGL((join_splits_of_many_kernel<128, Args>), blocks, threads, 0, stream, a);
    else if (many)
        hipLaunchKernelGGL((join_splits_of_many_kernel<256, Args>), blocks, threads, 0, stream, a);
    else if (D == 64)
        hipLaunchKernelGGL((join_splits_kernel<64, Args>), blocks, threads, 0, stream, a);
    else if (D == 128)
        hipLaunchKernelGGL((join_splits_kernel<128, Args>), blocks, threads, 0, stream, a);
    else
        hipLaunchKernelGGL((join_splits_kernel<256, Args>), blocks, threads, 0, stream, a);
}

template <typename Args>
static void launch_rows(const Args& a, const iq4xs_paged_attention_args& g, const AttentionPlan& p, hipStream_t stream) {
    if (p.tiles)
        launch_stream_attention(a, g.cache->head_dim, p.tiles, g.type, g.cache->type, p.grid, stream);
    else
        launch_tile_attention(a, g.cache->head_dim, g.type, g.cache->type, exact_keys(g), p.grid, stream);
}

static bool enough(const void* ws, size_t ws_bytes, size_t need) {
    return ws_bytes >= need && (!need || (ws && reinterpret_cast<uintptr_t>(ws) % 256 == 0));
}

// The kernels' arguments, parts[splits][total][q_heads] from the workspace's beginning, `splits` of them in all.
static AttentionArgs args_of(const iq4xs_paged_attention_args& g, const AttentionPlan& p, void* ws, int splits) {
    float* part = static_cast<float*>(ws);
    return {cache_pages(*g.cache), g.q, g.out, g.lse, g.table, g.starts, g.kv_len, part,
            splits > 0 ? part + parts_bytes(g, splits) / sizeof(float) : nullptr, g.q_stride, g.table_width, (int)g.total,
            (int)g.most_q, most_kv_of(g), (int)window_of(g), (int)g.seqs, g.q_heads, g.q_heads / g.cache->heads,
            g.out_type, g.causal, p.splits, p.chunk, p.row_tiles, g.scale * 1.44269504089f};
}

static size_t workspace_of(const iq4xs_paged_attention_args& g, int splits) {
    return parts_bytes(g, splits) + parts_bytes(g, splits) / g.cache->head_dim * 4;
}
static size_t workspace_of(const iq4xs_paged_attention_args& g, const AttentionPlan& p) {
    return p.splits > 1 ? workspace_of(g, p.splits) : 0;
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
    if (!enough(ws, ws_bytes, workspace_of(g, p))) return hipErrorInvalidValue;
    clear_launch_error();
    const AttentionArgs a = args_of(g, p, ws, p.splits > 1 ? p.splits : 0);
    launch_rows(a, g, p, stream);
    if (p.splits > 1) launch_join(a, g.cache->head_dim, stream);
    return hipGetLastError();
}

hipError_t launch_sinks_attention(const iq4xs_paged_attention_args& g, int64_t sinks, void* ws, size_t ws_bytes,
                                  hipStream_t stream) {
    if (!sinks_matter(g, sinks)) return launch_paged_attention(g, ws, ws_bytes, stream);
    AttentionPlan p;
    if (!plan_fits(g, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    if (!enough(ws, ws_bytes, workspace_of(g, p))) return hipErrorInvalidValue;
    clear_launch_error();
    const MoreArgs a{args_of(g, p, ws, p.splits > 1 ? p.splits : 0), PASS_SINKS, (int)at_most(sinks, KEYS_END), nullptr,
                     nullptr, 0, 0, (int)g.seqs, 0, 0, 0};
    launch_rows(a, g, p, stream);
    if (p.splits > 1) launch_join(a, g.cache->head_dim, stream);
    return hipGetLastError();
}

hipError_t shared_attention_workspace(const iq4xs_paged_attention_args& g, const iq4xs_shared_prefix& x, size_t* bytes) {
    SharedPlan p;
    if (!shared_plan_fits(g, x, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    *bytes = workspace_of(g, p.parts());
    return hipSuccess;
}

hipError_t launch_shared_attention(const iq4xs_paged_attention_args& g, const iq4xs_shared_prefix& x, void* ws,
                                   size_t ws_bytes, hipStream_t stream) {
    SharedPlan p;
    if (!shared_plan_fits(g, x, device_cu_count(), p)) return hipErrorInvalidConfiguration;
    if (!p.once) return launch_paged_attention(each_call(g, x), ws, ws_bytes, stream);
    if (!enough(ws, ws_bytes, workspace_of(g, p.parts()))) return hipErrorInvalidValue;
    clear_launch_error();
    const iq4xs_paged_attention_args prefix = prefix_call(g, x);
    const MoreArgs first{args_of(prefix, p.prefix, ws, p.parts()), PASS_PREFIX, 0, x.first, x.len, (int)x.groups,
                         (int)at_most(x.most_len, KEYS_END), (int)g.seqs, p.prefix.splits, p.prefix.chunk,
                         (int)x.most_rows};
    launch_rows(first, prefix, p.prefix, stream);
    MoreArgs own{args_of(g, p.own, ws, p.parts()), PASS_OWN, 0, x.first, x.len, (int)x.groups, first.most_shared,
                 (int)g.seqs, p.prefix.splits, p.prefix.chunk, (int)x.most_rows};
    own.part += p.prefix.splits * g.total * g.q_heads * g.cache->head_dim;
    own.part_ml += p.prefix.splits * g.total * g.q_heads * 4;
    launch_rows(own, g, p.own, stream);
    own.part = first.part;
    own.part_ml = first.part_ml;
    launch_join(own, g.cache->head_dim, stream);
    return hipGetLastError();
}

}  // namespace iq4xs
