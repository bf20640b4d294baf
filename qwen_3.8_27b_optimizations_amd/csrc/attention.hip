// attention.hip -- attention of new tokens over the paged cache.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q k_j - max),  lse = max + log(sum_j w_j)
//
// in one pass over the keys with the running maximum m and sum l of the softmax: a tile of keys raises m to m', what
// is held is scaled by exp(m - m').  One wave for each row and head, 64 keys at a time, a key for each lane.
#include <math.h>

#include "attention_device.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

constexpr int ROW_WAVES = 4;

struct AttentionArgs {
    CachePages c;
    const void* q;
    void* out;
    float* lse;
    const int32_t *table, *starts, *kv_len;
    int64_t q_stride, width, total, most_q, most_kv, window;
    int seqs, q_heads, out_type, causal;
    float scale;
};

template <typename T>
__device__ inline float element(const void* p, const _Float16*, int64_t row, int D, int c) {
    return (float)static_cast<const T*>(p)[row * D + c];
}
template <>
__device__ inline float element<int8_t>(const void* p, const _Float16* scales, int64_t row, int D, int c) {
    return (float)static_cast<const int8_t*>(p)[row * D + c] * (float)scales[row * (D / 32) + c / 32];
}

template <int D, typename Q, typename KV>
__global__ __launch_bounds__(64 * ROW_WAVES) void row_attention_kernel(AttentionArgs a) {
    __shared__ float qs[ROW_WAVES][D];
    __shared__ float ws[ROW_WAVES][64];
    __shared__ int64_t at[ROW_WAVES][64];
    constexpr int OWN = D / 64;
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
    const int64_t unit = (int64_t)blockIdx.x * ROW_WAVES + wave;
    const int64_t row = unit / a.q_heads;
    if (row >= a.total) return;
    const int head = (int)(unit % a.q_heads), kv_head = head / (a.q_heads / a.c.heads);
    const int seq = sequence_of(a.starts, a.seqs, row, lane);
    if (seq < 0 || seq >= a.seqs) return;
    const int first = a.starts[seq], fresh = a.starts[seq + 1] - first;
    const int64_t step = row - first;
    if (step >= a.most_q) return;
    int64_t keys = a.kv_len[seq];
    keys = keys < a.most_kv ? keys : a.most_kv;
    keys = keys < (a.width << a.c.shift) ? keys : a.width << a.c.shift;
    const int64_t p = keys - fresh + step;
    int64_t hi = a.causal && p + 1 < keys ? p + 1 : keys;
    int64_t lo = a.window > 0 && p + 1 - a.window > 0 ? p + 1 - a.window : 0;

    for (int c = lane; c < D; c += 64)
        qs[wave][c] = (float)static_cast<const Q*>(a.q)[row * a.q_stride + head * D + c];
    float m = -INFINITY, l = 0.0f, o[OWN] = {};
    for (int64_t base = lo; base < hi; base += 64) {
        const int64_t key = base + lane;
        int page = -1;
        if (key < hi) page = a.table[seq * a.width + (key >> a.c.shift)];
        const bool seen = page >= 0 && page < a.c.pages;
        const int64_t kr = seen ? page_row(a.c, page, kv_head, (int)key & ((1 << a.c.shift) - 1)) : -1;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float s = -INFINITY;
        if (seen) {
            s = 0.0f;
            for (int c = 0; c < D; ++c) s += qs[wave][c] * element<KV>(a.c.k, a.c.ks, kr, D, c);
            s *= a.scale;
        }
        float top = s;
        for (int x = 32; x > 0; x /= 2) top = fmaxf(top, __shfl_xor(top, x, 64));
        top = fmaxf(top, m);
        const float ref = top == -INFINITY ? 0.0f : top;
        const float keep = __expf(m - ref), w = seen ? __expf(s - ref) : 0.0f;
        m = top;
        float sum = w;
        for (int x = 32; x > 0; x /= 2) sum += __shfl_xor(sum, x, 64);
        l = l * keep + sum;
        ws[wave][lane] = w;
        at[wave][lane] = kr;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int i = 0; i < OWN; ++i) o[i] *= keep;
        for (int j = 0; j < 64; ++j) {
            const int64_t vr = at[wave][j];
            if (vr < 0) continue;
            for (int i = 0; i < OWN; ++i) o[i] += ws[wave][j] * element<KV>(a.c.v, a.c.vs, vr, D, lane + 64 * i);
        }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    for (int i = 0; i < OWN; ++i) {
        const int64_t e = (row * a.q_heads + head) * D + lane + 64 * i;
        const float x = l == 0.0f ? 0.0f : o[i] * inv;
        if (a.out_type == IQ4XS_TYPE_F32)
            static_cast<float*>(a.out)[e] = x;
        else if (a.out_type == IQ4XS_TYPE_F16)
            static_cast<_Float16*>(a.out)[e] = (_Float16)x;
        else
            static_cast<__bf16*>(a.out)[e] = (__bf16)x;
    }
    if (a.lse && lane == 0) a.lse[row * a.q_heads + head] = l == 0.0f ? -INFINITY : m + logf(l);
}

size_t paged_attention_workspace(const iq4xs_paged_attention_args&) { return 0; }

template <int D>
void launch_rows(const AttentionArgs& a, int type, int cache_type, dim3 grid, dim3 block, hipStream_t stream) {
    if (cache_type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((row_attention_kernel<D, _Float16, _Float16>), grid, block, 0, stream, a);
    else if (cache_type == IQ4XS_TYPE_BF16)
        hipLaunchKernelGGL((row_attention_kernel<D, __bf16, __bf16>), grid, block, 0, stream, a);
    else if (type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((row_attention_kernel<D, _Float16, int8_t>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((row_attention_kernel<D, __bf16, int8_t>), grid, block, 0, stream, a);
}

hipError_t launch_paged_attention(const iq4xs_paged_attention_args& g, void*, hipStream_t stream) {
    clear_launch_error();
    const AttentionArgs a{cache_pages(*g.cache), g.q, g.out, g.lse, g.table, g.starts, g.kv_len, g.q_stride,
                          g.table_width, g.total, g.most_q, g.most_kv, g.window, (int)g.seqs, g.q_heads, g.out_type,
                          g.causal, g.scale};
    const int64_t grid = (g.total * g.q_heads + ROW_WAVES - 1) / ROW_WAVES;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    const dim3 blocks((unsigned)grid), threads(64 * ROW_WAVES);
    if (g.cache->head_dim == 64)
        launch_rows<64>(a, g.type, g.cache->type, blocks, threads, stream);
    else if (g.cache->head_dim == 128)
        launch_rows<128>(a, g.type, g.cache->type, blocks, threads, stream);
    else
        launch_rows<256>(a, g.type, g.cache->type, blocks, threads, stream);
    return hipGetLastError();
}

}  // namespace iq4xs
