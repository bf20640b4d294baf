// qk_rope.hip -- norm of queries and keys for each head and the position rotation, into dense rows or a paged cache.
//
//   y = x * rsqrt(mean(x^2) + eps) * gain;  pair i of the first rot channels, (a, b):
//   (a cos t - b sin t, b cos t + a sin t),  t = pos * freq[i]
//
// One pass over the data, bound by HBM at many tokens (4096 tokens of 64 + 8 heads of 128 in fp32: 64 us, 4.7 TB/s; 2048
// into an 8-bit cache 34 us, 4.3 TB/s) and by latency at few.  A head is held by head_dim / 8 lanes of 8
// channels, as two chunks of 4 picked so that both channels of every pair lie in one lane (half layout: chunk l and
// chunk l + rot/8; interleaved: neighbours), so the rotation needs no exchange, and cosine and sine are computed once
// for a lane's four pairs and used for every head it takes.  The angle is reduced to turns in 64 bits (positions reach
// 2^31, where 32 bits hold nothing of it); cosine and sine of the remainder are fp32's.
#include "attention_device.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

constexpr int QK_WAVES = 4;

struct QkArgs {
    const void *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;
    const int32_t* pos;
    const double* freqs;
    const float *q_gamma, *k_gamma;
    const int64_t* slots;  // null: dense
    void *q_out, *k_out;
    int64_t units;  // tokens * splits
    int q_heads, k_heads, rot, half, out_type, splits, steps;
    float eps;
    CachePages c;
    int cache_type;
};

// Maximum of bit patterns of magnitudes over the lanes of a 32-channel group: NaN is above every number.
template <int kLanes>
__device__ inline uint32_t group_umax(uint32_t v) {
#pragma unroll
    for (int o = 1; o < kLanes; o *= 2) {
        const uint32_t w = __shfl_xor(v, o, 64);
        v = w > v ? w : v;
    }
    return v;
}

// Eight consecutive channels of a head (channel 8 * l) as codes, the group's scale by its first lane of four.
__device__ inline void store_q8(int8_t* codes, _Float16* scales, int64_t row, int D, int l, f4 a, f4 b) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = __float_as_uint(a[i]) & 0x7FFFFFFFu, y = __float_as_uint(b[i]) & 0x7FFFFFFFu;
        top = x > top ? x : top;
        top = y > top ? y : top;
    }
    const float amax = __uint_as_float(group_umax<4>(top));
    float d = amax / 127.0f;
    d = d > 65504.0f / 127.0f ? 65504.0f / 127.0f : d;  // NaN passes
    // That is 516 in fp16, and 127 times it past fp16: what fp16 holds takes the scale below, whose codes it holds too, and
    // only what it does not comes back as an infinity there.
    if (amax < 65520.0f && d > 515.5f) d = 515.5f;
    const _Float16 dh = (_Float16)d;
    const float df = (float)dh;
    uint32_t w[2] = {0, 0};
    if (df > 0.0f) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float x = fminf(fmaxf(__builtin_rintf(a[i] / df), -127.0f), 127.0f);
            const float y = fminf(fmaxf(__builtin_rintf(b[i] / df), -127.0f), 127.0f);
            w[0] |= ((uint32_t)(int)x & 0xFFu) << (8 * i);
            w[1] |= ((uint32_t)(int)y & 0xFFu) << (8 * i);
        }
    }
    *reinterpret_cast<u2*>(codes + row * D + 8 * l) = u2{w[0], w[1]};
    if ((l & 3) == 0) scales[row * (D / 32) + l / 4] = dh;
}

template <int D, typename In>
__global__ __launch_bounds__(64 * QK_WAVES) void qk_norm_rope_kernel(QkArgs a) {
    constexpr int L = D / 8, HEADS = 64 / L;  // lanes of a head, heads of a wave at a time
    __shared__ float rows[QK_WAVES][HEADS][D];  // rotated keys on their way to codes, private to the wave's lanes
    const int wave = threadIdx.x / 64, lane = threadIdx.x % 64, l = lane % L, sub = lane / L;
    const int64_t unit = (int64_t)blockIdx.x * QK_WAVES + wave;
    if (unit >= a.units) return;
    const int64_t token = unit / a.splits;
    const int first = (int)(unit % a.splits) * a.steps * HEADS;
    const bool append = a.slots != nullptr;
    const int heads = a.q_heads + a.k_heads * (append ? 2 : 1);

    // this lane's chunks of 4 channels
    const int turned = a.rot / 8;
    const bool turns = l < turned;
    const int ca = !a.half ? 2 * l : (turns ? l : 2 * l), cb = !a.half || !turns ? ca + 1 : l + turned;
    float cs[4], sn[4];
    if (turns) {
        const double pos = (double)a.pos[token];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double turn = pos * a.freqs[4 * l + i] * 0.15915494309189533577;
            sincospif(2.0f * (float)(turn - __builtin_rint(turn)), &sn[i], &cs[i]);
        }
    }
    int64_t slot = -1;
    if (append) {
        slot = a.slots[token];
        if (slot >= ((int64_t)a.c.pages << a.c.shift)) slot = -1;
    }

    // a step's heads are loaded a step ahead
    auto fetch = [&](int head, f4& u, f4& w) {
        if (head >= heads) return;
        const bool query = head < a.q_heads, key = head < a.q_heads + a.k_heads;
        const int h = head - (query ? 0 : key ? a.q_heads : a.q_heads + a.k_heads);
        const In* x = (query ? static_cast<const In*>(a.q) + token * a.q_stride
                       : key ? static_cast<const In*>(a.k) + token * a.k_stride
                             : static_cast<const In*>(a.v) + token * a.v_stride) + h * D;
        u = load4(x + 4 * (key ? ca : 2 * l));
        w = load4(x + 4 * (key ? cb : 2 * l + 1));
    };
    f4 u_next, w_next;
    fetch(first + sub, u_next, w_next);
    for (int step = 0; step < a.steps; ++step) {
        const int head = first + step * HEADS + sub;
        if (head >= heads) return;  // a head's lanes leave together
        f4 u = u_next, w = w_next;
        if (step + 1 < a.steps) fetch(head + HEADS, u_next, w_next);
        const int kind = head < a.q_heads ? 0 : head < a.q_heads + a.k_heads ? 1 : 2;
        const int h = head - (kind == 0 ? 0 : kind == 1 ? a.q_heads : a.q_heads + a.k_heads);
        if (kind == 2) {
            if (slot < 0) continue;
            const int64_t row = page_row(a.c, (int)(slot >> a.c.shift), h, (int)slot & ((1 << a.c.shift) - 1));
            if (a.cache_type == IQ4XS_TYPE_Q8) {
                store_q8(static_cast<int8_t*>(a.c.v), a.c.vs, row, D, l, u, w);
            } else {
                store4(a.c.v, row * D + 8 * l, a.cache_type, u);
                store4(a.c.v, row * D + 8 * l + 4, a.cache_type, w);
            }
            continue;
        }
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += u[i] * u[i] + w[i] * w[i];
#pragma unroll
        for (int o = 1; o < L; o *= 2) ss += __shfl_xor(ss, o, 64);
        const float scale = rsqrtf(ss * (1.0f / D) + a.eps);
        const float* gain = kind == 0 ? a.q_gamma : a.k_gamma;
        u *= scale;
        w *= scale;
        if (gain) {
            u *= load4(gain + 4 * ca);
            w *= load4(gain + 4 * cb);
        }
        if (turns) {
            if (a.half) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = u[i], r = w[i];
                    u[i] = p * cs[i] - r * sn[i];
                    w[i] = r * cs[i] + p * sn[i];
                }
            } else {
                const f4 p = u, r = w;
                u = f4{p.x * cs[0] - p.y * sn[0], p.y * cs[0] + p.x * sn[0], p.z * cs[1] - p.w * sn[1],
                       p.w * cs[1] + p.z * sn[1]};
                w = f4{r.x * cs[2] - r.y * sn[2], r.y * cs[2] + r.x * sn[2], r.z * cs[3] - r.w * sn[3],
                       r.w * cs[3] + r.z * sn[3]};
            }
        }
        if (kind == 0 || !append) {
            void* out = kind == 0 ? a.q_out : a.k_out;
            const int64_t row = (token * (kind == 0 ? a.q_heads : a.k_heads) + h) * D;
            store4(out, row + 4 * ca, a.out_type, u);
            store4(out, row + 4 * cb, a.out_type, w);
            continue;
        }
        if (slot < 0) continue;
        const int64_t row = page_row(a.c, (int)(slot >> a.c.shift), h, (int)slot & ((1 << a.c.shift) - 1));
        if (a.cache_type != IQ4XS_TYPE_Q8) {
            store4(a.c.k, row * D + 4 * ca, a.cache_type, u);
            store4(a.c.k, row * D + 4 * cb, a.cache_type, w);
            continue;
        }
        // codes go by groups of 32 channels in a row: the lanes trade their chunks through LDS, which a wave's
        // accesses reach in program order
        float* r = rows[wave][sub];
        *reinterpret_cast<f4*>(r + 4 * ca) = u;
        *reinterpret_cast<f4*>(r + 4 * cb) = w;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        u = *reinterpret_cast<const f4*>(r + 8 * l);
        w = *reinterpret_cast<const f4*>(r + 8 * l + 4);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        store_q8(static_cast<int8_t*>(a.c.k), a.c.ks, row, D, l, u, w);
    }
}

hipError_t launch_qk_norm_rope(const iq4xs_qk_norm_rope_args& g, const iq4xs_kv_cache* cache, hipStream_t stream) {
    clear_launch_error();
    QkArgs a{g.q, g.k, g.v, g.q_stride, g.k_stride, g.v_stride, g.pos, g.freqs, g.q_gamma, g.k_gamma,
             cache ? g.slots : nullptr, g.q_out, g.k_out, 0, g.q_heads, g.k_heads, g.rot, g.rope == IQ4XS_ROPE_HALF,
             g.out_type, 1, 1, g.eps, cache ? cache_pages(*cache) : CachePages{}, cache ? cache->type : 0};
    const int at_once = 512 / g.head_dim;
    const int steps = (g.q_heads + g.k_heads * (cache ? 2 : 1) + at_once - 1) / at_once;
    // a token's heads go to as many waves as give every CU 16: fewer leave it idle (256 tokens of 64 + 8 heads of 128 22.6
    // us in one wave each, 11.2 so), more compute more cosines (1024 tokens: 21.7 us with 64 waves, 15.2 so)
    const int64_t splits = (16 * (int64_t)device_cu_count() + g.tokens - 1) / g.tokens;
    a.splits = (int)(splits < steps ? splits : steps);
    a.steps = (steps + a.splits - 1) / a.splits;
    a.units = g.tokens * a.splits;
    const int64_t grid = (a.units + QK_WAVES - 1) / QK_WAVES;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    const dim3 blocks((unsigned)grid), threads(64 * QK_WAVES);
#define IQ4XS_LAUNCH(D, T) hipLaunchKernelGGL((qk_norm_rope_kernel<D, T>), blocks, threads, 0, stream, a)
#define IQ4XS_TYPES(D)                                         \
    if (g.in_type == IQ4XS_TYPE_F32) IQ4XS_LAUNCH(D, float);   \
    else if (g.in_type == IQ4XS_TYPE_F16) IQ4XS_LAUNCH(D, _Float16); \
    else IQ4XS_LAUNCH(D, __bf16)
    if (g.head_dim == 64) {
        IQ4XS_TYPES(64);
    } else if (g.head_dim == 128) {
        IQ4XS_TYPES(128);
    } else {
        IQ4XS_TYPES(256);
    }
#undef IQ4XS_TYPES
#undef IQ4XS_LAUNCH
    return hipGetLastError();
}

}  // namespace iq4xs
