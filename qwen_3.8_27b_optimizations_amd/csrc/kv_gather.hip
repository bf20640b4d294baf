// kv_gather.hip -- cached tokens of sequences read back as dense rows.
//
// A copy, bound by HBM: 32768 tokens of an 8-bit cache of 8 heads of 128 to fp16 in 46 us (4.5 TB/s), 37 sequences in bf16
// 52 us (5.0 TB/s).  A wave takes a token's heads, keys and values, 8 channels for each lane and load; the
// sequence of a row is the number of starts at or below it, counted 64 at a time.
#include "attention_device.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

constexpr int GATHER_WAVES = 4;

struct GatherArgs {
    CachePages c;
    const int32_t* table;
    const int32_t* starts;
    void *k_out, *v_out;
    int64_t width, total;
    int seqs;
};

template <typename Out>
struct Row8;
template <>
struct Row8<float> {
    static __device__ void store(float* p, f4 a, f4 b) {
        *reinterpret_cast<f4*>(p) = a;
        *reinterpret_cast<f4*>(p + 4) = b;
    }
};
template <>
struct Row8<_Float16> {
    static __device__ void store(_Float16* p, f4 a, f4 b) {
        *reinterpret_cast<h8*>(p) = __builtin_convertvector(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), h8);
    }
};
template <>
struct Row8<__bf16> {
    static __device__ void store(__bf16* p, f4 a, f4 b) {
        *reinterpret_cast<b8*>(p) = __builtin_convertvector(__builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7), b8);
    }
};

template <typename T>
__device__ inline void load8(const void* p, const _Float16*, int64_t row, int D, int c, f4& a, f4& b) {
    a = load4(static_cast<const T*>(p) + row * D + c);
    b = load4(static_cast<const T*>(p) + row * D + c + 4);
}
// codes times their group's scale, exact in fp32
template <>
__device__ inline void load8<int8_t>(const void* p, const _Float16* scales, int64_t row, int D, int c, f4& a, f4& b) {
    const u2 w = *reinterpret_cast<const u2*>(static_cast<const int8_t*>(p) + row * D + c);
    const float s = (float)scales[row * (D / 32) + c / 32];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = (float)((int)(w.x << (24 - 8 * i)) >> 24) * s;
        b[i] = (float)((int)(w.y << (24 - 8 * i)) >> 24) * s;
    }
}

template <int D, typename In, typename Out>
__global__ __launch_bounds__(64 * GATHER_WAVES) void kv_gather_kernel(GatherArgs a) {
    constexpr int L = D / 8, HEADS = 64 / L;
    const int lane = threadIdx.x % 64, l = lane % L, sub = lane / L;
    const int64_t row = (int64_t)blockIdx.x * GATHER_WAVES + threadIdx.x / 64;
    if (row >= a.total) return;
    const int seq = sequence_of(a.starts, a.seqs, row, lane);
    int page = -1, off = 0;
    if (seq >= 0 && seq < a.seqs) {
        const int64_t j = row - a.starts[seq];
        off = (int)j & ((1 << a.c.shift) - 1);
        // j below zero: starts that fall
        if (j >= 0 && (j >> a.c.shift) < a.width) page = a.table[seq * a.width + (j >> a.c.shift)];
    }
    const bool there = page >= 0 && page < a.c.pages;
    for (int head = sub; head < 2 * a.c.heads; head += HEADS) {
        const bool key = head < a.c.heads;
        const int h = key ? head : head - a.c.heads;
        f4 x{0, 0, 0, 0}, y{0, 0, 0, 0};
        if (there)
            load8<In>(key ? a.c.k : a.c.v, key ? a.c.ks : a.c.vs, page_row(a.c, page, h, off), D, 8 * l, x, y);
        Row8<Out>::store(static_cast<Out*>(key ? a.k_out : a.v_out) + (row * a.c.heads + h) * D + 8 * l, x, y);
    }
}

template <int D, typename In>
void launch_to(const GatherArgs& a, int out_type, dim3 grid, dim3 block, hipStream_t stream) {
    if (out_type == IQ4XS_TYPE_F32)
        hipLaunchKernelGGL((kv_gather_kernel<D, In, float>), grid, block, 0, stream, a);
    else if (out_type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((kv_gather_kernel<D, In, _Float16>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((kv_gather_kernel<D, In, __bf16>), grid, block, 0, stream, a);
}

template <int D>
void launch_from(const GatherArgs& a, int type, int out_type, dim3 grid, dim3 block, hipStream_t stream) {
    if (type == IQ4XS_TYPE_F16)
        launch_to<D, _Float16>(a, out_type, grid, block, stream);
    else if (type == IQ4XS_TYPE_BF16)
        launch_to<D, __bf16>(a, out_type, grid, block, stream);
    else
        launch_to<D, int8_t>(a, out_type, grid, block, stream);
}

hipError_t launch_kv_gather(const iq4xs_kv_cache& cache, const int32_t* table, int64_t width, const int32_t* starts,
                            int64_t seqs, void* k_out, void* v_out, int64_t total, int out_type, hipStream_t stream) {
    clear_launch_error();
    const GatherArgs a{cache_pages(cache), table, starts, k_out, v_out, width, total, (int)seqs};
    const int64_t grid = (total + GATHER_WAVES - 1) / GATHER_WAVES;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    const dim3 blocks((unsigned)grid), threads(64 * GATHER_WAVES);
    if (cache.head_dim == 64)
        launch_from<64>(a, cache.type, out_type, blocks, threads, stream);
    else if (cache.head_dim == 128)
        launch_from<128>(a, cache.type, out_type, blocks, threads, stream);
    else
        launch_from<256>(a, cache.type, out_type, blocks, threads, stream);
    return hipGetLastError();
}

}  // namespace iq4xs
