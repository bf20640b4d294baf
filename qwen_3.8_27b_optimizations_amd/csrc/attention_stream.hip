// attention_stream.hip -- attention of few rows over the paged cache: single tokens and short drafts.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q k_j - m),  lse = m + log(sum_j w_j)
//
// The rows of a cache head (its new tokens times the query heads that read it, token by token) are the columns of
// 16 x 16 matrix products: S^T = K Q^T and O^T = V^T W^T.  Bound by reading the cache, so everything is arranged around
// that read:
// - a wave goes through its keys alone, 32 at a time, straight from memory into registers: no LDS and no barrier in the
//   loop.  Keys arrive as the product's left operand; of the values a lane takes 8 keys by head_dim / 16 channels and
//   turns them there with byte permutations, 1 for every 2 elements;
// - the result of S^T holds, in each lane, weights of exactly the 8 keys whose values the lane took, for one row: they
//   are the right operand of O^T as they stand;
// - the four waves of a workgroup and the splits of a long cache go through different keys; the waves join in LDS, the
//   splits in a second launch.
// The running maximum of a row moves only when a key passes it by 2^8 (in powers of two): weights up to 2^8 times the
// largest are as exact in 16 bits, and the sums need no rescaling in most steps.
// A step's loads are issued a step ahead, its pages looked up two ahead, and none has a condition, so that each wait is
// for what it needs.  Registers decide how many workgroups a CU holds: 4 with heads of 64, 2 with 128 (3 of an 8-bit
// cache), 1 with 256; staging through LDS, two steps of a wave at once and three waves a SIMD by spilling were slower.
// Measured: 131072 keys of 8 heads of 128, one token: 96 us, 5.6 TB/s (fp16), 54 us, 5.3 TB/s (8 bits); 64 sequences of up
// to 16384 tokens: 211 us, 5.0 TB/s.  4096 keys: 6 us, of them latency (a dependent chain of table, keys, scores and
// values), and 4 of the joining launch.  With more rows vector work grows beside the read: 8 sequences of 40 rows over
// 8-bit heads of 256 94 us, of which reading is 19.
// An 8-bit cache's codes become fp16 (exact); a key's scales (one for 32 channels) multiply the parts of its score in
// fp32, the values' scales multiply their codes in fp16 (half a step of 2^-11), and the weights go as two fp16 numbers, so
// that this rounding is left, and that of weights below 2^-21 of the largest, whose second part is below fp16's normal
// range (2^-32 of the largest each).  bf16 queries for it become fp16 with a power of
// two taken out of each row, exact down to 2^-14 of the row's largest element.
//
// First tokens beside a window are further steps before those of the window, of the first split, with masks of their own: 64
// sequences of up to 32768 tokens, window 4096, 4 first tokens, 64 heads on 8 of 128, bf16: 157 us of a call's 168 (4.8 TB/s
// of the call); 8 x 5 tokens over a window of 2048 and 64 first tokens, 8-bit heads of 256: 35 of 39 us.
#include "attention_core.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

constexpr int STREAM_WAVES = 4;
constexpr int STEP_KEYS = 32;  // of a wave at a time

// The rows' queries, right operand of S^T: in registers, of 256 channels in LDS (every wave has the same), where the
// registers do not hold them beside a step and the sums.
template <int D, int NT>
struct Queries {
    u4 own[NT][D / 32];
    __device__ u4 at(int i, int c) const { return own[i][c]; }
};
template <int NT>
struct Queries<256, NT> {
    const u4* own;  // of this lane; [tile][8][64 lanes]
    __device__ u4 at(int i, int c) const { return own[(8 * i + c) * 64]; }
};

// Two tiles of 16 keys as they lie in the cache, in the lanes that use them.
template <int D, typename KV>
struct Step {
    static constexpr int OWN = D / 16;  // channels of a value in a lane
    u4 k[2][D / 32];
    u4 v[8][OWN / 8 ? OWN / 8 : 1];

    __device__ void load_keys(const AttentionArgs& a, const int64_t (&row)[2], int n, int j) {
        const uint16_t* p = static_cast<const uint16_t*>(a.c.k);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
                k[t][c] = *reinterpret_cast<const u4*>(p + row[t] * D + n * D + 32 * c + 8 * j);
    }
    __device__ void load_values(const AttentionArgs& a, const int64_t (&row)[2], int n, int j) {
        const uint16_t* p = static_cast<const uint16_t*>(a.c.v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t* r = p + row[e / 4] * D + (4 * j + e % 4) * D;
            if constexpr (OWN == 4) {
                const u2 w = *reinterpret_cast<const u2*>(r + 4 * n);
                v[e][0] = u4{w.x, w.y, 0, 0};
            } else {
#pragma unroll
                for (int h = 0; h < OWN / 8; ++h) v[e][h] = *reinterpret_cast<const u4*>(r + 128 * h + 8 * n);
            }
        }
    }
    template <int NT>
    __device__ void scores(const Queries<D, NT>& q, f4 (&s)[NT][2], int) const {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                s[i][t] = f4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < D / 32; ++c) s[i][t] = Matrix<KV>::mma16(k[t][c], q.at(i, c), s[i][t]);
            }
    }
    // Left operand of O^T for the lane's channel t: its 8 keys, two for each word.
    __device__ u4 values(int t) const {
        u4 x;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const int h = t / 8, w = (t % 8) / 2;
            x[p] = __builtin_amdgcn_perm(v[2 * p + 1][h][w], v[2 * p][h][w], t % 2 ? 0x07060302u : 0x05040100u);
        }
        return x;
    }
    __device__ void share_scales(int) {}
    __device__ void prepare_values(int) {}
    __device__ bool some_odd() const { return false; }
    // Clears the values outside the slots of the mask and those that are not finite; whether there were such inside.
    __device__ bool keep_finite(u4 slots) {
        uint32_t odd = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t keep = slots[e / 2] >> (16 * (e % 2)) & 1 ? ~0u : 0u;
#pragma unroll
            for (int h = 0; h < (OWN / 8 ? OWN / 8 : 1); ++h) {
                const u4 x = v[e][h] & keep, f = Matrix<KV>::finite(x), y = x ^ f;
                odd |= y.x | y.y | y.z | y.w;
                v[e][h] = f;
            }
        }
        return odd != 0;
    }
    using Weight = KV;
};

// codes: bytes of `hi` and `lo` at place b as a pair of fp16 numbers (1024 + code + 128, then less 1152: both exact)
__device__ inline h2 code_pair(uint32_t hi, uint32_t lo, int b) {
    const uint32_t sel = 0x0C040C00u + 0x00010001u * b;
    const uint32_t w = __builtin_amdgcn_perm(hi, lo, sel) | 0x64006400u;
    return __builtin_bit_cast(h2, w) - h2{(_Float16)1152, (_Float16)1152};
}

// Codes: a lane loads 16 of a key at once, so that a load's segments are whole 64-byte pieces, and lanes of the two halves
// of the wave trade 8 of them, so that each product is over one group of 32.  The scales of the 32 keys and values of a
// step are one load for the wave, lane l those of key l or value l - 32, and are handed round through LDS.
template <int D>
struct Step<D, int8_t> {
    static constexpr int OWN = D / 16, WORDS = D / 64, HALVES = D == 256 ? 2 : 1, GROUPS = D / 32;
    u4 k[2][D / 64];
    uint32_t v[8][WORDS];
    h2 pair[HALVES][4];
    typedef _Float16 Scales __attribute__((ext_vector_type(GROUPS)));
    Scales scale;
    _Float16* shared;  // [64][GROUPS], of this wave

    __device__ void load_keys(const AttentionArgs& a, const int64_t (&row)[2], int n, int j) {
        const int8_t* p = static_cast<const int8_t*>(a.c.k);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
                k[t][c] = *reinterpret_cast<const u4*>(p + row[t] * D + n * D + 64 * c + 16 * j);
        // row[j % 2], as a sum: the compiler would index the pair in memory
        const int64_t mine = row[0] + ((row[1] - row[0]) & -(int64_t)(j & 1));
        const _Float16* s = (j < 2 ? a.c.ks : a.c.vs) + (mine + n) * GROUPS;
        scale = *reinterpret_cast<const Scales*>(s);
    }
    __device__ void load_values(const AttentionArgs& a, const int64_t (&row)[2], int n, int j) {
        const int8_t* p = static_cast<const int8_t*>(a.c.v);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int8_t* r = p + row[e / 4] * D + (4 * j + e % 4) * D;
            if constexpr (OWN == 4) {
                v[e][0] = *reinterpret_cast<const uint32_t*>(r + 4 * n);
            } else {
#pragma unroll
                for (int h = 0; h < HALVES; ++h) {
                    const u2 w = *reinterpret_cast<const u2*>(r + 128 * h + 8 * n);
                    v[e][2 * h] = w.x;
                    v[e][2 * h + 1] = w.y;
                }
            }
        }
    }
    __device__ void share_scales(int lane) const {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        *reinterpret_cast<Scales*>(shared + lane * GROUPS) = scale;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    template <int NT>
    __device__ void scores(const Queries<D, NT>& q, f4 (&s)[NT][2], int lane) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            // of the lane's four keys of the tile
            const Scales* from = reinterpret_cast<const Scales*>(shared + (16 * t + 4 * (lane / 16)) * GROUPS);
            const Scales ks[4] = {from[0], from[1], from[2], from[3]};
#pragma unroll
            for (int i = 0; i < NT; ++i) s[i][t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < GROUPS; ++c) {
                // lanes 0 to 31 hold channels 64 (c / 2) + 0..31 of the key, the others 32..63
                const u4 both = k[t][c / 2] ^ 0x80808080u;
                const u2 x0 = __builtin_amdgcn_permlane32_swap(both.x, both.z, false, false);
                const u2 x1 = __builtin_amdgcn_permlane32_swap(both.y, both.w, false, false);
                u4 x;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const uint32_t b = w < 2 ? (c % 2 ? x0.y : x0.x) : (c % 2 ? x1.y : x1.x);
                    const uint32_t z = __builtin_amdgcn_perm(b, b, w % 2 ? 0x0C030C02u : 0x0C010C00u) | 0x64006400u;
                    x[w] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, z) - h2{(_Float16)1152, (_Float16)1152});
                }
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const f4 part = Matrix<_Float16>::mma16(x, q.at(i, c), f4{0, 0, 0, 0});
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        s[i][t][r] = __builtin_fmaf((float)ks[r][c], part[r], s[i][t][r]);
                    }
                }
            }
        }
    }
    __device__ void prepare_values(int lane) {
        flip_codes();
        take_scales(lane);
    }
    __device__ void flip_codes() {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int w = 0; w < WORDS; ++w) v[e][w] ^= 0x80808080u;
    }
    __device__ void take_scales(int lane) {
        const int n = lane % 16, j = lane / 16;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const _Float16* from = shared + (32 + 16 * (p / 2) + 4 * j + 2 * (p % 2)) * GROUPS +
                                       (OWN == 4 ? n / 8 : 4 * h + n / 4);
                pair[h][p] = h2{from[0], from[GROUPS]};
            }
    }
    __device__ u4 values(int t) const {
        u4 x;
#pragma unroll
        for (int p = 0; p < 4; ++p)
            x[p] = __builtin_bit_cast(uint32_t, code_pair(v[2 * p + 1][t / 4], v[2 * p][t / 4], t % 4) * pair[t / 8][p]);
        return x;
    }
    // Whether a scale of the step, of a key or a value, is not finite, or so large that codes may pass fp16: above 515.5,
    // 127 times which is the last that rounds to one.
    __device__ bool some_odd() const {
        bool odd = false;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const _Float16 x = scale[g];
            odd = odd || (__builtin_bit_cast(uint16_t, x) & 0x7FFFu) > 0x6007u;
        }
        return __any(odd);
    }
    // Clears the scales outside the slots of the mask, and those that are not finite or large; whether there were such
    // inside.
    __device__ bool keep_finite(u4 slots) {
        bool odd = false;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint32_t x = __builtin_bit_cast(uint32_t, pair[h][p]) & slots[p], over = large_halves(x);
                odd = odd || over != 0;
                pair[h][p] = __builtin_bit_cast(h2, x & ~over);
            }
        return odd;
    }
    // Puts in the scales' place the large ones among them that are finite, times 2^-12, so that no code makes an infinity
    // of them; whether there are any.
    __device__ bool large_scales(u4 slots, int lane) {
        take_scales(lane);
        uint32_t some = 0;
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint32_t x = __builtin_bit_cast(uint32_t, pair[h][p]) & slots[p];
                const uint32_t f = Matrix<_Float16>::finite(u4{x & large_halves(x), 0, 0, 0}).x;
                some |= f;
                pair[h][p] = __builtin_bit_cast(h2, f) * h2{(_Float16)0x1p-12f, (_Float16)0x1p-12f};
            }
        return __any(some != 0);
    }
    static __device__ uint32_t large_halves(uint32_t x) {
        return ((x & 0x7FFFu) > 0x6007u ? 0xFFFFu : 0u) | ((x >> 16 & 0x7FFFu) > 0x6007u ? 0xFFFF0000u : 0u);
    }
    using Weight = _Float16;
};

// The lane's 8 keys of a step as word masks: pairs of 16-bit slots whose key lies in [lo, hi).
__device__ inline u4 slots_in(int base, int j, int lo, int hi) {
    const int from = lo - base - 4 * j, to = hi - base - 4 * j;
    u4 m;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int in = (p < 2 ? 0 : 16) + 2 * (p % 2);
        m[p] = (in >= from && in < to ? 0xFFFFu : 0u) | (in + 1 >= from && in + 1 < to ? 0xFFFF0000u : 0u);
    }
    return m;
}

template <int D, typename Q, typename KV, int NT, typename Args>
__global__ __launch_bounds__(64 * STREAM_WAVES, D == 256 ? 1 : 2) void stream_attention_kernel(Args a) {
    constexpr bool MORE = HasMore<Args>::value;
    constexpr int OWN = D / 16, PART = D == 64 ? 64 : 128;
    using W = typename Step<D, KV>::Weight;
    constexpr uint32_t ONES = Matrix<W>::ONES;
    // values of an 8-bit cache are rounded, so weights are not: they go as two fp16 numbers, high and rest
    constexpr bool EXACT = sizeof(KV) == 1;
    __shared__ float so[STREAM_WAVES][16][PART + 4];
    __shared__ float sm[STREAM_WAVES][16], sl[STREAM_WAVES][16], sr[STREAM_WAVES][16];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int n = lane % 16, j = lane / 16;
    unsigned x = blockIdx.x;
    const int head = x % a.c.heads;
    x /= a.c.heads;
    const int seq = x % a.seqs;
    x /= a.seqs;
    const int tile = x % a.row_tiles, split = x / a.row_tiles;
    int total_fresh;
    Sequence s;
    if constexpr (MORE)
        s = sequence_more(a, seq, total_fresh);
    else
        s = sequence(a, seq, total_fresh);
    const int rows = s.fresh * a.group, row0 = tile * 16 * NT;
    if (row0 >= rows) return;
    const int last = (rows < row0 + 16 * NT ? rows : row0 + 16 * NT) - 1;
    const int token0 = row0 / a.group, token1 = last / a.group;
    // keys that some row of the tile sees, and those that all see
    const int any_lo = least_key(a, s, total_fresh, token0), any_hi = end_key(a, s, total_fresh, token1);
    const int all_lo = least_key(a, s, total_fresh, token1), all_hi = end_key(a, s, total_fresh, token0);
    int k0, k1, extra = 0;
    if constexpr (MORE) {
        if (!split_keys_more(a, s, any_lo, any_hi, split, k0, k1, extra)) return;
    } else {
        if (!split_keys(a, s, any_lo, any_hi, split, k0, k1)) return;
    }
    const KeySteps<STEP_KEYS, MORE> span(k0, k1, extra);
    const int start = span.start;

    // this lane's rows and their keys (lanes without a row repeat the last)
    int token[NT], lo[NT], hi[NT];
    float factor[NT];
    u4 q[NT][D / 32];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const int r = row0 + 16 * i + n <= last ? row0 + 16 * i + n : last;
        token[i] = r / a.group;
        lo[i] = least_key(a, s, total_fresh, token[i]);
        hi[i] = end_key(a, s, total_fresh, token[i]);
        // the channels that the keys' lanes hold
        const int channel = sizeof(KV) == 1 ? 16 * (j % 2) + 8 * (j / 2) : 8 * j;
        const int64_t at = (int64_t)(s.first + token[i]) * a.q_stride + (head * a.group + r % a.group) * D + channel;
        const u4* p = reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.q) + at);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) q[i][c] = p[4 * c];
        factor[i] = a.scale;
        if constexpr (sizeof(KV) == 1 && sizeof(Q) == 2 && __is_same(Q, __bf16)) {
            // the largest magnitudes of a row's four lanes, as numbers (a NaN lets the others through)
            const int e = query_exponent(__float_as_uint(max_of_quarters(__uint_as_float(query_top(q[i]) << 16))) >> 16);
            factor[i] = ldexpf(a.scale, e);
            queries_to_f16(q[i], e);
        }
    }

    Queries<D, NT> queries;
    if constexpr (D == 256) {
        __shared__ u4 sq[NT][D / 32][64];
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
                if (wave == 0) sq[i][c][lane] = q[i][c];
        __syncthreads();
        queries.own = &sq[0][0][lane];
    } else {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) queries.own[i][c] = q[i][c];
    }

    f4 o[NT][OWN];
    float m[NT], l[NT], rounded[NT];  // of the weights as they are and, where they are rounded, so
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        m[i] = -FLT_MAX;
        l[i] = rounded[i] = 0.0f;
#pragma unroll
        for (int t = 0; t < OWN; ++t) o[i][t] = f4{0, 0, 0, 0};
    }

    // Where tile t of the step at `base` lies; a tile past the end or on no page of the cache reads page 0 and is masked.
    // Its pages are looked up a step before they are wanted, tile t's in lane t: a load without a condition, issued ahead of
    // the step's keys, so that waiting for it is not waiting for them.
    auto look_up = [&](int base) {
        const int key = span.place(base) + 16 * (lane % 2);
        const int32_t* p = key < span.stop(base) ? s.pages + (key >> a.c.shift) : a.starts;
        return *p;
    };
    auto find = [&](int base, int pages, int64_t(&row)[2], bool(&there)[2]) {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int key = span.place(base) + 16 * t, page = __builtin_amdgcn_readlane(pages, t);
            there[t] = key < span.stop(base) && page >= 0 && page < a.c.pages;
            row[t] = page_row(a.c, there[t] ? page : 0, head, there[t] ? key & ((1 << a.c.shift) - 1) : 0);
        }
    };

    // the lane's slots of a step whose keys some row sees
    auto seen = [&](int base, const bool(&there)[2]) {
        u4 some = slots_in(span.place(base), j, span.lo_in(base, any_lo), span.hi_in(base, any_hi));
        if (!there[0]) some.x = some.y = 0;
        if (!there[1]) some.z = some.w = 0;
        return some;
    };

    bool odd = false;
    Step<D, KV> step;
    if constexpr (sizeof(KV) == 1) {
        __shared__ __attribute__((aligned(16))) _Float16 scales[STREAM_WAVES][64 * (D / 32)];
        step.shared = scales[wave];
    }
    int64_t row[2];
    bool there[2];
    int base = start + STEP_KEYS * wave, pages = 0;
    if (base < k1) {
        const int first = look_up(base);
        pages = look_up(base + STEP_KEYS * STREAM_WAVES);
        find(base, first, row, there);
        step.load_keys(a, row, n, j);
        __builtin_amdgcn_sched_barrier(0);  // keys first, as in the loop, or its waits count too few
        step.load_values(a, row, n, j);
    }
    // the queries are there before the loop begins: a wait for them inside it would be one for every load after them
    if constexpr (D != 256) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int c = 0; c < D / 32; ++c) asm volatile("" : "+v"(queries.own[i][c]));
    }
    while (base < k1) {
        const int next = base + STEP_KEYS * STREAM_WAVES;
        int64_t next_row[2];
        bool next_there[2];
        find(next, pages, next_row, next_there);
        pages = look_up(next + STEP_KEYS * STREAM_WAVES);
        __builtin_amdgcn_sched_barrier(0);
        // an infinity times a weight's second part may be NaN: with codes, what may not be finite is always cleared
        const bool finite = !step.some_odd();
        f4 z[NT][2];
        step.share_scales(lane);
        step.scores(queries, z, lane);
        // past the last step every lane reads one place: loads without a condition let the waits count exactly
        const int next_n = next < k1 ? n : 0, next_j = next < k1 ? j : 0;
        step.load_keys(a, next_row, next_n, next_j);
        // Scores of heads of 256 come out in accumulation registers; they leave them here.  Left to itself the compiler
        // read them in the blocks below, the last 6 wait states after its product, which takes 8, and got it unfinished.
        if constexpr (D == 256 && !EXACT) {
#pragma unroll
            for (int i = 0; i < NT; ++i) asm volatile("" : "+v"(z[i][0]), "+v"(z[i][1]));
        }
        const bool full = finite && there[0] && there[1] && span.all_see(base, all_lo, all_hi);
        u4 w[NT], w_rest[EXACT ? NT : 1];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            float top = -INFINITY;
            const int at0 = span.place(base) + 4 * j;
            const int from = span.lo_in(base, lo[i]) - at0, to = span.hi_in(base, hi[i]) - at0;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    z[i][t][r] *= factor[i];
                    if (__builtin_expect(!full, 0)) {
                        if (!there[t] || 16 * t + r < from || 16 * t + r >= to) z[i][t][r] = -INFINITY;
                    }
                    top = fmaxf(top, z[i][t][r]);
                }
            if (__builtin_expect(__any(top > m[i] + (Matrix<W>::LARGEST + 8.0f)), 0)) {
                const float up = fmaxf(max_of_quarters(top) - Matrix<W>::LARGEST, m[i]), keep = __builtin_amdgcn_exp2f(m[i] - up);
                m[i] = up;
                l[i] *= keep;
                rounded[i] *= keep;
#pragma unroll
                for (int t = 0; t < OWN; ++t) o[i][t] *= keep;
            }
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(z[i][e / 4][e % 4] - m[i]);
                l[i] += p[e];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t both = Matrix<W>::pack(p[2 * e], p[2 * e + 1]);
                w[i][e] = both;
                if constexpr (!EXACT) rounded[i] = Matrix<W>::add(both, rounded[i]);
                if constexpr (EXACT) {
                    const h2 high = __builtin_bit_cast(h2, both);
                    w_rest[i][e] = Matrix<W>::pack(p[2 * e] - (float)high.x, p[2 * e + 1] - (float)high.y);
                }
            }
        }
        step.prepare_values(lane);
        // a weight of zero times an infinity is NaN: where rows differ in what they see, what no row sees and what is not
        // finite is cleared; the latter comes again after the last step
        if (__builtin_expect(!full, 0)) odd = step.keep_finite(seen(base, there)) || odd;
#pragma unroll
        for (int t = 0; t < OWN; ++t) {
            const u4 x = step.values(t);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                o[i][t] = Matrix<W>::mma16(x, w[i], o[i][t]);
                if constexpr (EXACT) o[i][t] = Matrix<W>::mma16(x, w_rest[i], o[i][t]);
            }
            if (t % 4 == 3) __builtin_amdgcn_sched_barrier(0);
        }
        step.load_values(a, next_row, next_n, next_j);
        base = next;
        there[0] = next_there[0];
        there[1] = next_there[1];
    }

    if (__builtin_expect(__any(odd), 0)) {
        if constexpr (EXACT) {
            // values of large scales come with the weights as they are now, and may be infinities too: those after them
            for (base = start + STEP_KEYS * wave; base < k1; base += STEP_KEYS * STREAM_WAVES) {
                find(base, look_up(base), row, there);
                step.load_keys(a, row, n, j);
                step.share_scales(lane);
                if (!step.large_scales(seen(base, there), lane)) continue;
                f4 z[NT][2];
                u4 w[NT], w_rest[NT];
                step.scores(queries, z, lane);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    u4 sees = slots_in(span.place(base), j, span.lo_in(base, lo[i]), span.hi_in(base, hi[i]));
                    if (!there[0]) sees.x = sees.y = 0;
                    if (!there[1]) sees.z = sees.w = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float p[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float x = z[i][e / 2][2 * (e % 2) + h] * factor[i] - m[i];
                            p[h] = sees[e] >> (16 * h) & 1 ? __builtin_amdgcn_exp2f(x) : 0.0f;
                        }
                        const uint32_t both = Matrix<W>::pack(p[0], p[1]);
                        const h2 high = __builtin_bit_cast(h2, both);
                        w[i][e] = both;
                        w_rest[i][e] = Matrix<W>::pack(p[0] - (float)high.x, p[1] - (float)high.y);
                    }
                }
                step.load_values(a, row, n, j);
                step.flip_codes();
#pragma unroll
                for (int t = 0; t < OWN; ++t) {
                    const u4 x = step.values(t);
#pragma unroll
                    for (int i = 0; i < NT; ++i) {
                        f4 part = Matrix<W>::mma16(x, w[i], f4{0, 0, 0, 0});
                        part = Matrix<W>::mma16(x, w_rest[i], part);
                        o[i][t] += part * 0x1p12f;
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
        // values that are not finite reach the rows that see them as infinities (a NaN as both)
        for (base = start + STEP_KEYS * wave; base < k1; base += STEP_KEYS * STREAM_WAVES) {
            find(base, look_up(base), row, there);
            if (!EXACT && there[0] && there[1] && span.all_see(base, all_lo, all_hi)) continue;
            step.load_keys(a, row, n, j);
            step.load_values(a, row, n, j);
            step.share_scales(lane);
            step.prepare_values(lane);
#pragma unroll
            for (int t = 0; t < OWN; ++t) {
                const u4 x = step.values(t) & seen(base, there);
#pragma unroll
                for (int i = 0; i < NT; ++i) {
                    const u4 sees = slots_in(span.place(base), j, span.lo_in(base, lo[i]), span.hi_in(base, hi[i])) & ONES;
                    const f4 plus = Matrix<W>::mma16(Matrix<W>::above(x), sees, f4{0, 0, 0, 0});
                    const f4 minus = Matrix<W>::mma16(Matrix<W>::below(x), sees, f4{0, 0, 0, 0});
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        if (plus[r] > 0.0f) o[i][t][r] += INFINITY;
                        if (minus[r] > 0.0f) o[i][t][r] -= INFINITY;
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }

    // the waves' sums join in LDS, 16 rows and up to 128 channels at a time, in the waves' order
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        const float lw = sum_of_quarters(l[i]), rw = EXACT ? lw : sum_of_quarters(rounded[i]);
        __syncthreads();
        if (j == 0) {
            sm[wave][n] = m[i];
            sl[wave][n] = lw;
            sr[wave][n] = rw;
        }
        __syncthreads();
        float top = sm[0][n];
#pragma unroll
        for (int w = 1; w < STREAM_WAVES; ++w) top = fmaxf(top, sm[w][n]);
        const float f = __builtin_amdgcn_exp2f(m[i] - top);
#pragma unroll
        for (int part = 0; part < D / PART; ++part) {
            if (part) __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < PART / 16; t += 4) {
                    const int u = 8 * part + t;
                    *reinterpret_cast<f4*>(&so[wave][n][(4 * j + r) * (PART / 16) + t]) =
                        f4{o[i][u][r] * f, o[i][u + 1][r] * f, o[i][u + 2][r] * f, o[i][u + 3][r] * f};
                }
            __syncthreads();
            constexpr int LANES = PART / 4, AT_ONCE = 64 * STREAM_WAVES / LANES;
            for (int y = threadIdx.x / LANES; y < 16; y += AT_ONCE) {
                const int r = row0 + 16 * i + y, c = threadIdx.x % LANES * 4;
                if (r > last) continue;
                float best = sm[0][y];
#pragma unroll
                for (int w = 1; w < STREAM_WAVES; ++w) best = fmaxf(best, sm[w][y]);
                float sum = 0.0f, weights = 0.0f;
                f4 v{0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < STREAM_WAVES; ++w) {
                    const float f = __builtin_amdgcn_exp2f(sm[w][y] - best);
                    sum += sl[w][y] * f;
                    weights += sr[w][y] * f;
                    v += *reinterpret_cast<const f4*>(&so[w][y][c]);
                }
                const int tok = r / a.group, h = head * a.group + r % a.group;
                const int64_t out = (int64_t)(s.first + tok) * a.q_heads + h;
                const int row_lo = least_key(a, s, total_fresh, tok), row_hi = end_key(a, s, total_fresh, tok);
                RowEnd end;
                if constexpr (MORE)
                    end = row_end_more(a, s, row_lo, row_hi, split);
                else
                    end = row_end(a, s, row_lo, row_hi, split);
                if (end == ROW_OUT) {
                    store4(a.out, out * D + PART * part + c, a.out_type, sum == 0.0f ? f4{0, 0, 0, 0} : v / weights);
                    if (a.lse && part == 0 && c == 0)
                        a.lse[out] = sum == 0.0f ? -INFINITY : (best + __log2f(sum)) * 0.69314718056f;
                } else if (end == ROW_PART) {
                    const int64_t at = (int64_t)split * a.total * a.q_heads + out;
                    *reinterpret_cast<f4*>(a.part + at * D + PART * part + c) = v;
                    if (part == 0 && c == 0) *reinterpret_cast<float4*>(a.part_ml + 4 * at) = make_float4(best, sum, weights, 0.0f);
                }
            }
        }
    }
}

template <int D, int NT, typename Args>
void launch_types(const Args& a, int type, int cache_type, dim3 grid, hipStream_t stream) {
    const dim3 block(64 * STREAM_WAVES);
    if (cache_type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((stream_attention_kernel<D, _Float16, _Float16, NT, Args>), grid, block, 0, stream, a);
    else if (cache_type == IQ4XS_TYPE_BF16)
        hipLaunchKernelGGL((stream_attention_kernel<D, __bf16, __bf16, NT, Args>), grid, block, 0, stream, a);
    else if constexpr (D == 256 && NT == 2)
        return;  // not asked for: two tiles of codes do not fit the registers
    else if (type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((stream_attention_kernel<D, _Float16, int8_t, NT, Args>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((stream_attention_kernel<D, __bf16, int8_t, NT, Args>), grid, block, 0, stream, a);
}

template <int D, typename Args>
void launch_tiles(const Args& a, int tiles, int type, int cache_type, dim3 grid, hipStream_t stream) {
    if (tiles == 1)
        launch_types<D, 1>(a, type, cache_type, grid, stream);
    else
        launch_types<D, 2>(a, type, cache_type, grid, stream);
}

template <typename Args>
void launch_stream_attention(const Args& a, int head_dim, int tiles, int type, int cache_type, int64_t grid,
                             hipStream_t stream) {
    const dim3 blocks((unsigned)grid);
    if (head_dim == 64)
        launch_tiles<64>(a, tiles, type, cache_type, blocks, stream);
    else if (head_dim == 128)
        launch_tiles<128>(a, tiles, type, cache_type, blocks, stream);
    else
        launch_tiles<256>(a, tiles, type, cache_type, blocks, stream);
}
#ifdef IQ4XS_ATTENTION_MORE
template void launch_stream_attention(const MoreArgs&, int, int, int, int, int64_t, hipStream_t);
#else
template void launch_stream_attention(const AttentionArgs&, int, int, int, int, int64_t, hipStream_t);
#endif

}  // namespace iq4xs
