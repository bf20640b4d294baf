// attention_device.h -- types, vector accesses and the paged cache's addressing, shared by the kernels of the
// attention half of a layer (qk_rope.hip, kv_gather.hip, attention.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "iq4xs_mi355x.h"

namespace iq4xs {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// The cache as kernels take it: page is 1 << shift.
struct CachePages {
    void* k;
    void* v;
    _Float16* ks;
    _Float16* vs;
    int pages, heads, shift;
};

inline CachePages cache_pages(const iq4xs_kv_cache& c) {
    return {c.k, c.v, static_cast<_Float16*>(c.k_scales), static_cast<_Float16*>(c.v_scales), (int)c.pages, c.heads,
            __builtin_ctz((unsigned)c.page)};
}

// Index of token `off` of a page's head, in tokens of one head; times head_dim (or head_dim / 32) it passes 32 bits in a
// long cache.
__device__ inline int64_t page_row(const CachePages& c, int page, int head, int off) {
    return (((int64_t)page * c.heads + head) << c.shift) + off;
}

// Four consecutive elements as fp32.
__device__ inline f4 load4(const float* p) { return *reinterpret_cast<const f4*>(p); }
__device__ inline f4 load4(const _Float16* p) {
    return __builtin_convertvector(*reinterpret_cast<const h4*>(p), f4);
}
__device__ inline f4 load4(const __bf16* p) {
    const u2 w = *reinterpret_cast<const u2*>(p);
    return f4{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
              __uint_as_float(w.y & 0xFFFF0000u)};
}

// Four fp32 values rounded to `type` (nearest even) at element i of p.
__device__ inline void store4(void* p, int64_t i, int type, f4 x) {
    if (type == IQ4XS_TYPE_F32)
        *reinterpret_cast<f4*>(static_cast<float*>(p) + i) = x;
    else if (type == IQ4XS_TYPE_F16)
        *reinterpret_cast<h4*>(static_cast<_Float16*>(p) + i) = __builtin_convertvector(x, h4);
    else
        *reinterpret_cast<b4*>(static_cast<__bf16*>(p) + i) = __builtin_convertvector(x, b4);
}

// The sequence that holds `row`, whose starts never fall: -1 before the first, seqs past the last.  All lanes of a wave
// with the same row.
__device__ inline int sequence_of(const int32_t* starts, int seqs, int64_t row, int lane) {
    int seq = -1;
    for (int s = 0; s <= seqs; s += 64) {
        const int i = s + lane;
        const int n = __popcll(__ballot(i <= seqs && starts[i <= seqs ? i : 0] <= row));
        seq += n;
        if (n < 64) break;
    }
    return seq;
}

}  // namespace iq4xs
