// linear_chunk.hip -- linear attention with a decay for each head, in chunks of tokens: prompts and long drafts.
//
// With G the sum of decays from a chunk's beginning and S the state there,
//   o_i = scale (exp(G_i) q_i^T S + sum_{j <= i} exp(G_i - G_j) (q_i k_j) v_j)
//   S  <- exp(G_C) S + sum_j exp(G_C - G_j) k_j v_j^T
#include "attention_core.h"
#include "iq4xs_internal.h"
#include "lds_device.h"
#include "linear_device.h"
#include "linear_launch.h"

namespace iq4xs {

constexpr int CHUNK_WAVES = 4, CHUNK_THREADS = 64 * CHUNK_WAVES;

// Numbers as sums of bf16 parts: as many as hold the input types exactly.
template <typename T>
constexpr int parts_of = __is_same(T, float) ? 3 : __is_same(T, _Float16) ? 2 : 1;

__device__ inline uint32_t high_halves(float x0, float x1) {
    return __builtin_amdgcn_perm(__float_as_uint(x1), __float_as_uint(x0), 0x07060302u);
}
__device__ inline float high_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xFFFF0000u); }

// A pair of fp32 numbers: leading 8 bits, the next 8, and (N = 3) the last 8; the last of two parts is rounded.
template <int N>
__device__ inline void split(float x0, float x1, uint32_t (&p)[N]) {
    p[0] = high_halves(x0, x1);
    x0 -= high_part(x0);
    x1 -= high_part(x1);
    if constexpr (N == 3) {
        p[1] = high_halves(x0, x1);
        x0 -= high_part(x0);
        x1 -= high_part(x1);
    }
    p[N - 1] = Matrix<__bf16>::pack(x0, x1);
}

// Eight consecutive elements as they come from memory.
template <typename T>
struct Piece {
    u4 w[sizeof(T) / 2];
    __device__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const u4*>(p)[i];
    }
    __device__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i / 4][i % 4]);
        const uint32_t x = w[0][i / 2] >> (16 * (i % 2));
        if constexpr (__is_same(T, _Float16)) return (float)__builtin_bit_cast(_Float16, (uint16_t)x);
        return __uint_as_float(x << 16);
    }
    __device__ void clear(bool all) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i)
            if (all) w[i] = u4{0, 0, 0, 0};
    }
    __device__ bool finite(int i) const { return fabsf(at(i)) <= FLT_MAX; }
    __device__ bool finite() const {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < 8; ++i) ok = ok && finite(i);
        return ok;
    }
    __device__ void clear_at(int i) {
        if constexpr (sizeof(T) == 4)
            w[i / 4][i % 4] = 0;
        else
            w[0][i / 2] &= i % 2 ? 0xFFFFu : 0xFFFF0000u;
    }
    __device__ void parts(u4 (&p)[parts_of<T>]) const {
        if constexpr (__is_same(T, __bf16)) {
            p[0] = w[0];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = at(2 * i), x1 = at(2 * i + 1);
                if constexpr (__is_same(T, _Float16)) {
                    const uint32_t high = Matrix<__bf16>::pack(x0, x1);
                    p[0][i] = high;
                    p[1][i] = Matrix<__bf16>::pack(x0 - __uint_as_float(high << 16), x1 - high_part(__uint_as_float(high)));
                } else {
                    uint32_t y[3];
                    split<3>(x0, x1, y);
                    p[0][i] = y[0];
                    p[1][i] = y[1];
                    p[2][i] = y[2];
                }
            }
        }
    }
};

// A tile in LDS: ROWS rows of CHANNELS bf16 numbers, 16-byte pieces exchanged within a row so that 16 rows' pieces of one
// place lie in 16 places.
template <int ROWS, int CHANNELS>
struct ChunkTile {
    static constexpr int ROW = 2 * CHANNELS, BYTES = ROWS * ROW, PIECES = CHANNELS / 8;
    static constexpr int LOADS = ROWS * PIECES / CHUNK_THREADS;  // pieces of a thread
    static __device__ int place(int row, int piece) {
        return piece ^ (PIECES >= 16 ? row & 15 : PIECES == 8 ? (row >> 1) & 7 : 0);
    }
    static __device__ uint32_t at(int row, int piece) { return row * ROW + 16 * place(row, piece); }
};

// 8 tokens of the lane's channel, as the left or right operand of a product over tokens: rows row0 to row0 + 7 of the lane's
// group of 16, which reads channels 4 (lane % 4) of `piece`'s half `half`.
template <typename Tile>
__device__ inline u4 eight_tokens(uint32_t tile, int row0, int piece, int half, int lane) {
    const int row = row0 + lane % 16 / 4;
    const u2 x = read_column(tile + Tile::at(row, piece) + 8 * half), y = read_column(tile + Tile::at(row + 4, piece) + 8 * half);
    return u4{x.x, x.y, y.x, y.y};
}

// DK by DVT of a head's state belong to a workgroup, DVT / 4 columns to a wave, in accumulators.  OUT: parts that outputs
// are made of.
template <int DK, int DVT, int C, typename T, int OUT, bool STATE_ONLY>
__global__ __launch_bounds__(CHUNK_THREADS, 2) void linear_chunk_kernel(LinearArgs a, LinearSegments seg, int dv) {
    constexpr int IN = parts_of<T>, NT = DVT / 64, KS = DK / 32, TS = C / 32, IT = C / 16;
    using KTile = ChunkTile<C, DK>;
    using VTile = ChunkTile<C, DVT>;
    using PTile = ChunkTile<C, C>;
    static_assert(KTile::LOADS * CHUNK_THREADS == C * KTile::PIECES && VTile::LOADS * CHUNK_THREADS == C * VTile::PIECES,
                  "pieces are dealt out evenly");
    __shared__ __attribute__((aligned(1024))) uint8_t qs[STATE_ONLY ? 1 : IN][STATE_ONLY ? 16 : KTile::BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t ks[IN][KTile::BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t vs[IN][VTile::BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t ps[STATE_ONLY ? 1 : OUT][STATE_ONLY ? 16 : PTile::BYTES];
    __shared__ double sum[C];             // of decays up to a token, times log2(e)
    __shared__ float from_start[C], to_end[C];
    __shared__ int odd, odd_from[DVT];    // whether values are not finite, and a channel's first token of such
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int n = lane % 16, j = lane / 16;

    // heads that share q and k, and the columns of one head, are multiples of qk_heads apart
    unsigned x = blockIdx.x;
    const int qk_heads = a.heads / a.group, spread = x % a.heads;
    const int head = spread % qk_heads * a.group + spread / qk_heads;
    x /= a.heads;
    const int tile = x % (dv / DVT);
    x /= dv / DVT;
    const int part = x % seg.count, seq = x / seg.count;
    const Rows all = rows_of(a, seq);
    const int begin = part * seg.length;
    if (begin >= all.count) return;
    const bool last = begin + seg.length >= all.count;
    if (STATE_ONLY && last) return;
    const int end = last ? all.count : begin + seg.length;

    const uint32_t q_at = lds_address(qs), k_at = lds_address(ks), v_at = lds_address(vs), p_at = lds_address(ps);
    const T* q = static_cast<const T*>(a.q) + (head / a.group) * DK;
    const T* k = static_cast<const T*>(a.k) + (head / a.group) * DK;
    const T* v = static_cast<const T*>(a.v) + head * dv + tile * DVT;

    // state: column n of the wave's tile u, rows 32 s + 8 j + 4 t + r
    const int base = DVT / 4 * wave;  // of the wave's columns
    auto column = [&](int u, int m) { return NT == 2 ? base + 8 * (m / 4) + 4 * u + m % 4 : base + m; };
    f4 S[KS][2][NT];
    const float* from = STATE_ONLY ? nullptr
                        : part == 0 && last ? state_at(a, a.from_slots, seq, head, DK * dv)
                                            : seg.states + ((int64_t)(seq * seg.count + part) * a.heads + head) * DK * dv;
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    S[s][t][u][r] = from ? from[(32 * s + 8 * j + 4 * t + r) * dv + tile * DVT + column(u, n)] : 0.0f;
    if constexpr (!STATE_ONLY) {
        for (int i = threadIdx.x; i < OUT * PTile::BYTES / 16; i += CHUNK_THREADS)
            *reinterpret_cast<u4*>(&ps[0][16 * i]) = u4{0, 0, 0, 0};  // above the diagonal
    }

    Piece<T> qn[STATE_ONLY ? 1 : KTile::LOADS], kn[KTile::LOADS], vn[VTile::LOADS];
    float gn;
    // rows past the end read the last one, and are cleared on their way into LDS
    auto fetch = [&](int chunk) {
        auto row = [&](int i) { return (int64_t)(all.first + (chunk + i < end ? chunk + i : end - 1)); };
#pragma unroll
        for (int l = 0; l < KTile::LOADS; ++l) {
            const int i = threadIdx.x + l * CHUNK_THREADS;
            if constexpr (!STATE_ONLY) qn[l].load(q + row(i / KTile::PIECES) * a.q_stride + 8 * (i % KTile::PIECES));
            kn[l].load(k + row(i / KTile::PIECES) * a.k_stride + 8 * (i % KTile::PIECES));
        }
#pragma unroll
        for (int l = 0; l < VTile::LOADS; ++l) {
            const int i = threadIdx.x + l * CHUNK_THREADS;
            vn[l].load(v + row(i / VTile::PIECES) * a.v_stride + 8 * (i % VTile::PIECES));
        }
        gn = decay_at(a, row(lane % C), head);
    };
    // The first `count` rows of the chunk that was fetched, zeros behind them.  A value that is not finite would reach the
    // rows before it (a weight of zero times an infinity): it becomes zero, and its channel NaN from its row on.
    auto put = [&](int count) {
        auto store = [&](uint8_t* to, int bytes, uint32_t at, const u4* p) {
#pragma unroll
            for (int i = 0; i < IN; ++i) *reinterpret_cast<u4*>(to + i * bytes + at) = p[i];
        };
        u4 p[IN];
#pragma unroll
        for (int l = 0; l < KTile::LOADS; ++l) {
            const int i = threadIdx.x + l * CHUNK_THREADS, row = i / KTile::PIECES;
            const uint32_t at = KTile::at(row, i % KTile::PIECES);
            if constexpr (!STATE_ONLY) {
                qn[l].parts(p);
                store(qs[0], KTile::BYTES, at, p);
            }
            Piece<T> y = kn[l];
            y.clear(row >= count);
            y.parts(p);
            store(ks[0], KTile::BYTES, at, p);
        }
#pragma unroll
        for (int l = 0; l < VTile::LOADS; ++l) {
            const int i = threadIdx.x + l * CHUNK_THREADS, row = i / VTile::PIECES;
            Piece<T> y = vn[l];
            y.clear(row >= count);
            if (__builtin_expect(!y.finite(), 0)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (y.finite(e)) continue;
                    y.clear_at(e);
                    atomicMin(&odd_from[8 * (i % VTile::PIECES) + e], row);
                }
                odd = 1;
            }
            y.parts(p);
            store(vs[0], VTile::BYTES, VTile::at(row, i % VTile::PIECES), p);
        }
        if (wave == 0 && lane < C) {
            double g = lane < count ? (double)gn * 1.4426950408889634 : 0.0;
#pragma unroll
            for (int d = 1; d < C; d *= 2) {
                const double before = __shfl_up(g, d);
                if (lane >= d) g += before;
            }
            const double whole = __shfl(g, C - 1);
            sum[lane] = g;
            from_start[lane] = __builtin_amdgcn_exp2f((float)g);
            to_end[lane] = __builtin_amdgcn_exp2f((float)(whole - g));
        }
    };

    double decayed = 0.0;  // of the segment so far, times log2(e)
    auto compute = [&](int chunk, int count, bool some_odd) {
        if constexpr (!STATE_ONLY) {
            // weighted scores of tiles on and below the diagonal: keys 16 kt + 4 j + r of query 16 it + n
#pragma unroll
            for (int i = 0; i < (IT * (IT + 1) / 2 + CHUNK_WAVES - 1) / CHUNK_WAVES; ++i) {
                const int which = i * CHUNK_WAVES + wave;
                if (which >= IT * (IT + 1) / 2) break;
                const int it = which >= 6 ? 3 : which >= 3 ? 2 : which >= 1 ? 1 : 0, kt = which - it * (it + 1) / 2;
                f4 z{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u4 x[IN], y[IN];
#pragma unroll
                    for (int p = 0; p < IN; ++p) {
                        x[p] = read_row(k_at + p * KTile::BYTES + KTile::at(16 * kt + n, 4 * s + j));
                        y[p] = read_row(q_at + p * KTile::BYTES + KTile::at(16 * it + n, 4 * s + j));
                    }
#pragma unroll
                    for (int p = IN - 1; p >= 0; --p)
#pragma unroll
                        for (int o = IN - 1; o >= 0; --o)
                            if (p + o < OUT) z = Matrix<__bf16>::mma16(x[p], y[o], z);
                }
                const int query = 16 * it + n, key = 16 * kt + 4 * j;
                const double g = sum[query];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = __builtin_amdgcn_exp2f((float)(g - sum[key + r])) * a.scale;
                    z[r] = key + r <= query ? z[r] * w : 0.0f;
                }
                uint32_t lo2[OUT], hi2[OUT];
                split<OUT>(z[0], z[1], lo2);
                split<OUT>(z[2], z[3], hi2);
#pragma unroll
                for (int p = 0; p < OUT; ++p)
                    *reinterpret_cast<u2*>(&ps[p][PTile::at(query, key / 8) + 2 * (key % 8)]) = u2{lo2[p], hi2[p]};
            }
        }
        // the wave's values: channels of tile u by tokens 32 t + 8 j + e
        u4 V[TS][NT][IN];
#pragma unroll
        for (int t = 0; t < TS; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int p = 0; p < IN; ++p) {
                    const uint32_t at = v_at + p * VTile::BYTES;
                    V[t][u][p] = NT == 2 ? eight_tokens<VTile>(at, 32 * t + 8 * j, base / 8 + lane % 4, u, lane)
                                         : eight_tokens<VTile>(at, 32 * t + 8 * j, base / 8 + lane % 4 / 2, lane % 2, lane);
                }
        if constexpr (!STATE_ONLY) {
            f4 O[IT][NT];
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int u = 0; u < NT; ++u) O[i][u] = f4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u4 x[NT][OUT];
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t y[OUT];
                        split<OUT>(S[s][e / 2][u][2 * (e % 2)], S[s][e / 2][u][2 * (e % 2) + 1], y);
#pragma unroll
                        for (int p = 0; p < OUT; ++p) x[u][p][e] = y[p];
                    }
#pragma unroll
                for (int i = 0; i < IT; ++i) {
                    u4 y[IN];
#pragma unroll
                    for (int p = 0; p < IN; ++p)
                        y[p] = read_row(q_at + p * KTile::BYTES + KTile::at(16 * i + n, 4 * s + j));
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int p = OUT - 1; p >= 0; --p)
#pragma unroll
                            for (int o = IN - 1; o >= 0; --o)
                                if (p + o < OUT) O[i][u] = Matrix<__bf16>::mma16(x[u][p], y[o], O[i][u]);
                }
            }
            __syncthreads();  // weighted scores are there
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const float w = from_start[16 * i + n] * a.scale;
#pragma unroll
                for (int u = 0; u < NT; ++u) O[i][u] *= w;
#pragma unroll
                for (int t = 0; t <= i / 2; ++t) {
                    u4 y[OUT];
#pragma unroll
                    for (int p = 0; p < OUT; ++p) y[p] = read_row(p_at + p * PTile::BYTES + PTile::at(16 * i + n, 4 * t + j));
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int p = OUT - 1; p >= 0; --p)
#pragma unroll
                            for (int o = IN - 1; o >= 0; --o)
                                if (p + o < OUT) O[i][u] = Matrix<__bf16>::mma16(V[t][u][o], y[p], O[i][u]);
                }
                const int row = 16 * i + n;
                if (__builtin_expect(some_odd, 0)) {
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (row >= odd_from[column(u, 4 * j + r)]) O[i][u][r] = NAN;
                }
                if (row < count) {
                    const int64_t at = ((int64_t)(all.first + chunk + row) * a.heads + head) * dv + tile * DVT;
#pragma unroll
                    for (int u = 0; u < NT; ++u) store4(a.out, at + column(u, 4 * j), a.out_type, O[i][u]);
                }
            }
        }
        // values times what is left of them at the chunk's end, and the state's update
        const float keep = from_start[C - 1];
        u4 W[TS][NT][3];
#pragma unroll
        for (int t = 0; t < TS; ++t) {
            const float* w = &to_end[32 * t + 8 * j];
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x0 = 0.0f, x1 = 0.0f;
#pragma unroll
                    for (int p = IN - 1; p >= 0; --p) {
                        x0 += __uint_as_float(V[t][u][p][e] << 16);
                        x1 += high_part(__uint_as_float(V[t][u][p][e]));
                    }
                    uint32_t y[3];
                    split<3>(x0 * w[2 * e], x1 * w[2 * e + 1], y);
#pragma unroll
                    for (int p = 0; p < 3; ++p) W[t][u][p][e] = y[p];
                }
        }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int u = 0; u < NT; ++u) S[s][h][u] *= keep;
#pragma unroll
                for (int t = 0; t < TS; ++t) {
                    u4 x[IN];
#pragma unroll
                    for (int p = 0; p < IN; ++p)
                        x[p] = eight_tokens<KTile>(k_at + p * KTile::BYTES, 32 * t + 8 * j, 4 * s + lane % 4, h, lane);
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int o = 2; o >= 0; --o)
#pragma unroll
                            for (int p = IN - 1; p >= 0; --p)
                                if (p + o < 3) S[s][h][u] = Matrix<__bf16>::mma16(x[p], W[t][u][o], S[s][h][u]);
                }
            }
        if (__builtin_expect(some_odd, 0)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const float x = odd_from[column(u, n)] < C ? NAN : 0.0f;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) S[s][h][u] += x;
            }
            __syncthreads();
            for (int i = threadIdx.x; i < DVT; i += CHUNK_THREADS) odd_from[i] = C;
            if (threadIdx.x == 0) odd = 0;
        }
        if constexpr (STATE_ONLY) decayed += sum[C - 1];
    };

    for (int i = threadIdx.x; i < DVT; i += CHUNK_THREADS) odd_from[i] = C;
    if (threadIdx.x == 0) odd = 0;
    fetch(begin);
    for (int chunk = begin; chunk < end; chunk += C) {
        const int count = end - chunk < C ? end - chunk : C;
        __syncthreads();  // the chunk before is done with
        put(count);
        __syncthreads();
        const bool some_odd = odd != 0;
        if (chunk + C < end) fetch(chunk + C);
        compute(chunk, count, some_odd);
    }

    float* to = STATE_ONLY ? seg.states + ((int64_t)(seq * seg.count + part + 1) * a.heads + head) * DK * dv
                : last     ? state_at(a, a.to_slots, seq, head, DK * dv)
                           : nullptr;
    if (to) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        to[(32 * s + 8 * j + 4 * t + r) * dv + tile * DVT + column(u, n)] = S[s][t][u][r];
    }
    if constexpr (STATE_ONLY) {
        if (threadIdx.x == 0 && tile == 0)
            seg.decays[(seq * seg.count + part) * (int64_t)a.heads + head] = __builtin_amdgcn_exp2f((float)decayed);
    }
}

// The states that segments begin with, from the sequence's own and what each segment adds: in place, the first included.
__global__ __launch_bounds__(256) void join_segments_kernel(LinearArgs a, LinearSegments seg, int size) {
    const int pieces = size / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int piece = (int)(at % pieces), head = (int)(at / pieces % a.heads), seq = (int)(at / pieces / a.heads);
    if (seq >= a.seqs) return;
    const Rows all = rows_of(a, seq);
    if (all.count <= seg.length) return;
    const float* from = state_at(a, a.from_slots, seq, head, size);
    f4 s = from ? load4(from + 4 * piece) : f4{0, 0, 0, 0};
    const int count = (all.count + seg.length - 1) / seg.length;
    for (int i = 0; i < count; ++i) {
        const int64_t place = (int64_t)(seq * seg.count + i) * a.heads + head;
        f4* p = reinterpret_cast<f4*>(seg.states + place * size + 4 * piece);
        if (i > 0) s = s * seg.decays[place - a.heads] + *p;
        *p = s;
    }
}

template <int DK, int DVT, int C, typename T, int OUT>
static void launch(const LinearArgs& a, const LinearSegments& seg, int dv, hipStream_t stream) {
    const dim3 block(CHUNK_THREADS), grid((unsigned)((int64_t)a.seqs * seg.count * a.heads * (dv / DVT)));
    if (seg.count > 1) {
        hipLaunchKernelGGL((linear_chunk_kernel<DK, DVT, C, T, OUT, true>), grid, block, 0, stream, a, seg, dv);
        const int64_t pieces = (int64_t)a.seqs * a.heads * DK * dv / 4;
        hipLaunchKernelGGL(join_segments_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, a, seg, DK * dv);
    }
    hipLaunchKernelGGL((linear_chunk_kernel<DK, DVT, C, T, OUT, false>), grid, block, 0, stream, a, seg, dv);
}

template <int DK, typename T, int OUT>
static void launch_columns(const LinearArgs& a, const LinearSegments& seg, int dv, hipStream_t stream) {
    constexpr int C = parts_of<T> == 1 && DK < 256 ? 64 : 32;
    if constexpr (DK == 256) {
        launch<DK, 64, C, T, OUT>(a, seg, dv, stream);
    } else {
        if (linear_chunk_columns(DK, dv) == 64)
            launch<DK, 64, C, T, OUT>(a, seg, dv, stream);
        else
            launch<DK, 128, C, T, OUT>(a, seg, dv, stream);
    }
}

template <int DK>
static void launch_types(const LinearArgs& a, const LinearSegments& seg, int dv, int type, hipStream_t stream) {
    const bool exact = a.out_type == IQ4XS_TYPE_F32;
    if (type == IQ4XS_TYPE_F32)
        launch_columns<DK, float, 3>(a, seg, dv, stream);
    else if (type == IQ4XS_TYPE_F16 && exact)
        launch_columns<DK, _Float16, 3>(a, seg, dv, stream);
    else if (type == IQ4XS_TYPE_F16)
        launch_columns<DK, _Float16, 2>(a, seg, dv, stream);
    else if (exact)
        launch_columns<DK, __bf16, 3>(a, seg, dv, stream);
    else
        launch_columns<DK, __bf16, 2>(a, seg, dv, stream);
}

void launch_linear_chunks(const LinearArgs& a, const LinearSegments& seg, int dk, int dv, int type, hipStream_t stream) {
    if (dk == 64)
        launch_types<64>(a, seg, dv, type, stream);
    else if (dk == 128)
        launch_types<128>(a, seg, dv, type, stream);
    else
        launch_types<256>(a, seg, dv, type, stream);
}

}  // namespace iq4xs
