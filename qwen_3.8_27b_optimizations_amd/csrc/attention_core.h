// attention_core.h -- what the two attention kernels share: their arguments, matrix products, and the outputs.
#pragma once

#include <float.h>
#include <math.h>

#include "attention_device.h"
#include "attention_plan.h"

namespace iq4xs {

typedef float fx16 __attribute__((ext_vector_type(16)));

struct AttentionArgs {
    CachePages c;
    const void* q;
    void* out;
    float* lse;
    const int32_t *table, *starts, *kv_len;
    float* part;      // [splits][total][q_heads][D] unnormalised sums, with splits > 1
    float* part_ml;   // [splits][total][q_heads][4] their maxima (in powers of two), sums of weights, and of rounded ones
    int64_t q_stride, width;
    int total, most_q, most_kv, window;  // window 0: none
    int seqs, q_heads, group, out_type, causal;
    int splits, chunk;  // keys of a split, a multiple of 128
    int row_tiles;
    float scale;  // times log2(e)
};

// A launch of a call with first tokens or with a shared prefix.
struct MoreArgs : AttentionArgs {
    static constexpr bool MORE = true;
    int pass, sinks;
    const int32_t* group_first;  // [groups + 1] first sequence of each, or NULL
    const int32_t* shared_len;   // [groups]
    int groups, most_shared, all_seqs;
    int prefix_splits, prefix_chunk, prefix_rows;  // of the prefixes' launch: rows of a group that it took
};

// Pairs of 16-bit numbers as masks: 0xFFFF where a number is an infinity or NaN and `which` says so of its sign (0 or 1)
// and of being NaN.
template <uint32_t EXPONENT, typename Which>
__device__ inline u4 odd_pairs(u4 x, Which which) {
    u4 out;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        out[p] = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t y = x[p] >> (16 * h) & 0xFFFFu;
            if ((y & EXPONENT) == EXPONENT && which(y >> 15 != 0, (y & ~EXPONENT & 0x7FFFu) != 0))
                out[p] |= 0xFFFFu << (16 * h);
        }
    }
    return out;
}

// What the kernels do with pairs of 16-bit numbers: `finite` keeps those (0 for the others), `above` has ones where
// there is +Inf or NaN, `below` where there is -Inf or NaN.
template <uint32_t E, uint32_t ONE>
struct Pairs {
    static constexpr uint32_t EXPONENT = E, ONES = ONE;
    static __device__ u4 finite(u4 x) {
        return x & ~odd_pairs<E>(x, [](bool, bool) { return true; });
    }
    static __device__ u4 above(u4 x) {
        return odd_pairs<E>(x, [](bool minus, bool nan) { return nan || !minus; }) & ONE;
    }
    static __device__ u4 below(u4 x) {
        return odd_pairs<E>(x, [](bool minus, bool nan) { return nan || minus; }) & ONE;
    }
};

template <typename T>
struct Matrix;
template <>
struct Matrix<_Float16> : Pairs<0x7C00u, 0x3C003C00u> {
    // Weights are 2^(z - m), in 16 bits for their product with the values.  m is set so that the row's largest weight is
    // 2^LARGEST then, and moves when one passes 2^(LARGEST + 8).  fp16 holds 2^15, and has its full bits down to 2^-14: as
    // far up as it goes, since a key that takes nearly all of the weight may have a value of nothing, and then the
    // small weights make the output.  At 2^0 weights 17 nats below the largest were two fifths off or zero, at 2^7 half a
    // hundredth.
    static constexpr float LARGEST = 7.0f;
    static __device__ f4 mma16(u4 a, u4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    static __device__ fx16 mma32(u4 a, u4 b, fx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    static __device__ uint32_t pack(float x, float y) {
        return __builtin_bit_cast(uint32_t, h2{(_Float16)x, (_Float16)y});
    }
    // A pair of weights onto a sum, exact products and one fp32 sum (fp16 below its normal range too).  What the values'
    // sum is divided by has to be the sum of the weights as they are rounded, or a row of one key is off by its
    // weight's rounding, and rows of few keys by most of theirs.
    static __device__ float add(uint32_t pair, float sum) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, pair), h2{(_Float16)1, (_Float16)1}, sum, false);
    }
    static __device__ uint32_t scaled(uint32_t x, float by) {
        const h2 v = __builtin_bit_cast(h2, x);
        return pack((float)v.x * by, (float)v.y * by);
    }
};
template <>
struct Matrix<__bf16> : Pairs<0x7F80u, 0x3F803F80u> {
    static constexpr float LARGEST = 0.0f;  // fp32's range
    static __device__ f4 mma16(u4 a, u4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ fx16 mma32(u4 a, u4 b, fx16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ uint32_t pack(float x, float y) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, b2{(__bf16)x, (__bf16)y});
    }
    static __device__ float add(uint32_t pair, float sum) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, pair), b2{(__bf16)1.0f, (__bf16)1.0f}, sum, false);
    }
    static __device__ uint32_t scaled(uint32_t x, float by) {
        return pack(__uint_as_float(x << 16) * by, __uint_as_float(x & 0xFFFF0000u) * by);
    }
};

// x of this lane and of the lanes 16, 32 and 48 away, which hold other keys of the same row.
__device__ inline float max_of_quarters(float x) {
    u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ inline float sum_of_quarters(float x) {
    u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r.x) + __uint_as_float(r.y);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// The same for the lane 32 away.
__device__ inline float max_of_halves(float x) {
    const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ inline float sum_of_halves(float x) {
    const u2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

// bf16 queries of a row for an 8-bit cache, as fp16 with a power of two taken out: 2^-e q, exact down to 2^-14 of the
// row's largest element.  `top` is the largest magnitude of the row as bf16 bits, in every lane that holds a part of it.
__device__ inline int query_exponent(uint32_t top) {
    const float size = __uint_as_float(top << 16);
    return size > 0.0f && size <= FLT_MAX ? ilogbf(size) : 0;
}
template <int N>
__device__ inline uint32_t query_top(const u4 (&q)[N]) {
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t u = q[c][w] & 0x7FFF7FFFu;
            top = top > (u & 0xFFFFu) ? top : u & 0xFFFFu;
            top = top > u >> 16 ? top : u >> 16;
        }
    return top;
}
template <int N>
__device__ inline void queries_to_f16(u4 (&q)[N], int e) {
#pragma unroll
    for (int c = 0; c < N; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w)
            q[c][w] = Matrix<_Float16>::pack(ldexpf(__uint_as_float(q[c][w] << 16), -e),
                                             ldexpf(__uint_as_float(q[c][w] & 0xFFFF0000u), -e));
}

}  // namespace iq4xs
