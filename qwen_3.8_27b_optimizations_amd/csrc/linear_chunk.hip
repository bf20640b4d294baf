// linear_chunk.hip -- linear attention with a decay for each head, in chunks of tokens: prompts and long drafts.
//
// With G the sum of decays from a chunk's beginning and S the state there,
//   o_i = scale (exp(G_i) q_i^T S + sum_{j <= i} exp(G_i - G_j) (q_i k_j) v_j)
//   S  <- exp(G_C) S + sum_j exp(G_C - G_j) k_j v_j^T
//
// Four products of 16 x 16 x 32 on matrix units for each chunk of 32 tokens.  States and sums are fp32 and inputs 16 bits, so
// what is fp32 (the state, values times their weights, weighted scores, fp32 inputs) goes as a sum of bf16 parts, which
// have fp32's range: three for the state's update and fp32 outputs, two for what makes 16-bit outputs.  Exponents of
// weights are differences of 64-bit sums, since a large decay would take the bits of the small ones behind it.
// - A workgroup has DK x 64 or DK x 128 of a head's state in accumulators through all chunks of its segment; a wave has whole
//   columns, so that only weighted scores pass between waves.  The state's accumulators hold, in each lane, 8 rows of a
//   column: the left operand of S^T Q^T as they stand, and values read as columns serve V^T P^T and the update alike.
// - LDS holds queries once, keys and values twice: the next chunk goes in beside this one's products (where three parts
//   have no room for that, after them).  Two waits of the workgroup for each chunk.
// - Decays go into the accumulators as whole powers of two, which rounds nothing, with each chunk that comes to one; the rest
//   is in the scales of what is read and added, so that the accumulators never hold more than the state.
//   (Up to 2^40 in the scales saves 3 of 117 us of the 4096 tokens below, and large values overflow.  Fractions in the
//   accumulators, without a rest: 116 us, and 7.0e-7 for 4.8e-7 of error in the states of the prompts below.)  Scales are
//   made for as many chunks as there are waves at a time, a chunk to a wave.
// - A long sequence is cut into segments side by side: a first pass leaves what each adds to the state, a launch joins them,
//   and the second pass begins with the states.
// Bound by vector instructions (parts of the state and of the weighted values: about as many issue cycles as the products
// take) and by the chain read, multiply, exchange, multiply, wait of each chunk, with two waves to a SIMD to hide it.
// Measured: 4096 tokens, 64 heads of 128 x 128 on 16 of q and k, bf16: 117 us (traced 40 for the states, 10 to join them, 80),
// of which memory takes 34; a chunk 2.1 us of a CU.  5 prompts of 987 to 4001 tokens, 32 heads of 128 x 256, fp16 to fp32:
// 471 us, 1.85 TB/s.  One prompt of 4096 tokens beside 63 single ones, bf16: 217 us for 138 of memory.
// Slower or no faster: 64 columns of fp16 on four waves, two workgroups to a CU (473 and 474 us of the prompts, 131 and 116 of
// 4 x 1024 tokens), chunks of 64 tokens (an earlier second pass 82 us for 70: registers), one tile of columns on
// eight waves for bf16 (77 and 79), three workgroups to a CU (87), single buffers (490 and 474 us of the prompts, earlier),
// scales by one wave a chunk ahead (as fast alone, but the pass over states waits for it), fp16 inputs as they are with
// the state in fp16's range (500 us: keeping the range costs what the parts do), sums of earlier segments in each
// workgroup instead of a launch that joins (96 against 64 + 12 us).
#include "attention_core.h"
#include "iq4xs_internal.h"
#include "lds_device.h"
#include "linear_device.h"
#include "linear_launch.h"

namespace iq4xs {

constexpr int CHUNK = 32;  // tokens

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
        if constexpr (sizeof(T) == 4) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, w[i / 4][i % 4] & 0x7FFFFFFFu);
            return top < 0x7F800000u;
        } else {
            typedef uint16_t s2 __attribute__((ext_vector_type(2)));
            s2 top{0, 0};
#pragma unroll
            for (int i = 0; i < 4; ++i)
                top = __builtin_elementwise_max(top, __builtin_bit_cast(s2, w[0][i] & 0x7FFF7FFFu));
            return max(top.x, top.y) < (__is_same(T, _Float16) ? 0x7C00 : 0x7F80);
        }
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
// place lie in 16 places (reads of rows), and those of 4 rows in 4 groups of places (reads of columns).
template <int ROWS, int CHANNELS>
struct ChunkTile {
    static constexpr int ROW = 2 * CHANNELS, BYTES = ROWS * ROW, PIECES = CHANNELS / 8;
    static __device__ int place(int row, int piece) {
        return piece ^ (PIECES >= 16 ? (row & 3) << 2 | (row >> 2 & 3) : PIECES == 8 ? (row & 2) << 1 | (row >> 2 & 3) : 0);
    }
    static __device__ uint32_t at(int row, int piece) { return row * ROW + 16 * place(row, piece); }
};

// Sums over this lane and those before it.
template <int CTRL, int ROWS>
__device__ inline double plus_moved(double x) {
    const u2 w = __builtin_bit_cast(u2, x);
    const u2 y{(uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.x, CTRL, ROWS, 0xF, false),
               (uint32_t)__builtin_amdgcn_update_dpp(0, (int)w.y, CTRL, ROWS, 0xF, false)};
    return x + __builtin_bit_cast(double, y);
}
__device__ inline double running_sum(double x) {
    x = plus_moved<0x111, 0xF>(x);  // 1, 2, 4 and 8 lanes on within 16
    x = plus_moved<0x112, 0xF>(x);
    x = plus_moved<0x114, 0xF>(x);
    x = plus_moved<0x118, 0xF>(x);
    x = plus_moved<0x142, 0xA>(x);     // the last of 16 to the next 16
    return plus_moved<0x143, 0xC>(x);  // and the last of 32 to the next 32
}

// 2^x where x is large: its whole part apart, so that the rest keeps its bits.
__device__ inline float exp2_of(double x) {
    const double whole = rint(x);
    return ldexpf(__builtin_amdgcn_exp2f((float)(x - whole)), (int)whole);
}
// The same apart, `part` in (1/2, 1].
__device__ inline SegmentDecay exp2_parts(double x) {
    const double whole = ceil(x);
    return {__builtin_amdgcn_exp2f((float)(x - whole)), (int)fmin(fmax(whole, -10000.0), 10000.0)};
}

// Four tokens of the lane's channel and the four after them, as the left or right operand of a product over tokens.
template <typename Tile>
__device__ inline u4 eight_tokens(uint32_t at) {
    const u2 x = read_column(at), y = read_column((at ^ 16) + 4 * Tile::ROW);
    return u4{x.x, x.y, y.x, y.y};
}

// Eight fp32 values rounded to `type`.
__device__ inline void store8(void* p, int type, f4 x, f4 y) {
    if (type == IQ4XS_TYPE_F32) {
        static_cast<f4*>(p)[0] = x;
        static_cast<f4*>(p)[1] = y;
        return;
    }
    typedef float f8 __attribute__((ext_vector_type(8)));
    const f8 v = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    if (type == IQ4XS_TYPE_F16)
        *static_cast<h8*>(p) = __builtin_convertvector(v, h8);
    else
        *static_cast<b8*>(p) = __builtin_convertvector(v, b8);
}

// The last sequence that begins at a place or before it, -1 if none does: a 64th of the sequences left at a time.
// before(first row, index): whether it does, which later ones never do again.
template <typename Before>
__device__ inline int last_sequence(const LinearArgs& a, int lane, Before before) {
    int seq = -1, from = 0, left = a.seqs;
    while (left > 0) {
        const int step = (left + 63) / 64, i = lane * step;
        const int n = __popcll(__ballot(i < left && before(a.starts[i < left ? from + i : from], from + i)));
        if (n == 0) break;
        seq = from + (n - 1) * step;
        left = min(step, from + left - seq) - 1;
        from = seq + 1;
    }
    return seq;
}

// What a chunk's decays come to.
template <int C>
struct ChunkScales {
    double sum[C];        // of decays up to a token, times log2(e)
    float from_start[C];  // of the accumulators in an output: 2^sum, the output's scale, and 2^held as the chunk begins
    float to_end[C];      // of a token in the accumulators: 2^(whole - sum), and 2^-held as the chunk ends
    float by;             // power of two that the accumulators go down by before the chunk's tokens come to them
};

// DK by 16 NT WAVES of a head's state belong to a workgroup, 16 NT columns to a wave, in accumulators.  OUT: parts of the
// state and of weights that outputs are made of.  AHEAD: whether the next chunk's keys and values have room in LDS beside
// this one's.
template <int DK, int NT, int WAVES, typename T, int OUT, bool STATE_ONLY, bool AHEAD>
__global__ __launch_bounds__(64 * WAVES, 2) void linear_chunk_kernel(LinearArgs a, LinearSegments seg, int dv) {
    constexpr int C = CHUNK, IN = parts_of<T>, KS = DK / 32, IT = C / 16, DVT = 16 * NT * WAVES, THREADS = 64 * WAVES;
    // products of parts p and o count while p + o is below OUT
    constexpr int BUFFERS = AHEAD ? 2 : 1;
    // whether the accumulators are multiplied beside the products of their update, every time, or before them, where there is
    // something to do: 2048 tokens of 32 heads of 256 x 256, fp16 258 and 263 us, fp32 333 and 341; 5 prompts of 128 x 256,
    // fp16 479 and 471, 4096 tokens of 128 x 128, bf16 118 and 117
    constexpr bool DECAY_BESIDE = KS * IN >= 16;
    using KTile = ChunkTile<C, DK>;
    using VTile = ChunkTile<C, DVT>;
    using PTile = ChunkTile<C, C>;
    constexpr int K_LOADS = C * KTile::PIECES / THREADS, V_LOADS = C * VTile::PIECES / THREADS;  // pieces of a thread
    static_assert(K_LOADS * THREADS == C * KTile::PIECES && V_LOADS * THREADS == C * VTile::PIECES, "dealt out evenly");
    constexpr int K_BYTES = IN * KTile::BYTES, V_BYTES = IN * VTile::BYTES;  // of a buffer
    __shared__ __attribute__((aligned(1024))) uint8_t qs[STATE_ONLY ? 1024 : K_BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t ks[BUFFERS * K_BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t vs[BUFFERS * V_BYTES];
    __shared__ __attribute__((aligned(1024))) uint8_t ps[STATE_ONLY ? 1024 : OUT * PTile::BYTES];
    __shared__ ChunkScales<C> scales[WAVES];  // of as many chunks at a time
    __shared__ double wholes[WAVES];
    __shared__ int odd[2], odd_from[2][DVT];  // whether values are not finite, and a channel's first token of such
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int n = lane % 16, j = lane / 16;

    // heads that share q and k, and the columns of one head, are multiples of qk_heads apart
    unsigned x = blockIdx.x;
    const int qk_heads = a.heads / a.group, spread = x % a.heads;
    const int head = spread % qk_heads * a.group + spread / qk_heads;
    x /= a.heads;
    const int tile = x % (dv / DVT);
    x /= dv / DVT;
    int seq;
    int64_t part64;
    Rows all;
    if (seg.runs.rows == 0) {
        seq = x / seg.runs.each;
        part64 = x % seg.runs.each;
        all = rows_of(a, seq);
    } else {
        seq = last_sequence(a, lane, [&](int row, int i) { return seg.runs.of(max(row, 0), i) <= x; });
        if (seq < 0) return;
        all = rows_of(a, seq);
        if (all.count == 0) return;
        part64 = x - seg.runs.of(all.first, seq);
    }
    if (part64 < 0 || part64 * seg.length >= all.count) return;
    const int part = (int)part64, begin = part * seg.length;
    const bool last = all.count - begin <= seg.length;
    if (STATE_ONLY && last) return;
    const int end = last ? all.count : begin + seg.length;

    // Where this lane reads: rows n, piece j; columns by groups of 16 lanes that read 4 rows of 4 pieces' halves.  Other
    // pieces are exclusive ors away, other rows sums; 4 rows on are a piece's neighbour.
    const int r4 = lane % 16 / 4, base = 16 * NT * wave;  // base: of the wave's columns
    uint32_t q_row = lds_address(qs) + KTile::at(n, j), k_row = lds_address(ks) + KTile::at(n, j);
    uint32_t p_row = lds_address(ps) + PTile::at(n, j), k_column = lds_address(ks) + KTile::at(8 * j + r4, lane % 4);
    uint32_t v_column = lds_address(vs) + (NT == 2 ? VTile::at(8 * j + r4, base / 8 + lane % 4)
                                                   : VTile::at(8 * j + r4, base / 8 + lane % 4 / 2) + 8 * (lane % 2));
    const T* q = static_cast<const T*>(a.q) + (head / a.group) * DK;
    const T* k = static_cast<const T*>(a.k) + (head / a.group) * DK;
    const T* v = static_cast<const T*>(a.v) + head * dv + tile * DVT;

    // state: column n of the wave's tile u, rows 32 s + 8 j + 4 t + r
    auto column = [&](int u, int m) { return NT == 2 ? base + 8 * (m / 4) + 4 * u + m % 4 : base + m; };
    auto state_place = [&](auto* state, int s, int t, int u, int r) {
        const uint32_t lane_off = (8 * j * dv + tile * DVT + column(u, n)) * (uint32_t)sizeof(float);
        using P = decltype(state);
        return reinterpret_cast<P>((char*)(state + (32 * s + 4 * t + r) * dv) + lane_off);
    };
    f4 S[KS][2][NT];
    // place of the sequence's first segment among those that are kept
    const int64_t kept = seg.count > 1 ? seg.kept.of(all.first, seq) * a.heads + head : 0;
    auto segment_state = [&](int i) { return seg.states + (kept + (int64_t)i * a.heads) * DK * dv; };
    // The first segment goes on from the sequence's state, in both passes: the pass over states leaves a copy of it, since
    // the last segment may write it while others begin.
    const float* from = part == 0 && (STATE_ONLY || last) ? state_at(a, a.from_slots, seq, head, DK * dv)
                        : STATE_ONLY                      ? nullptr
                                                          : segment_state(part);
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u) S[s][t][u] = f4{0, 0, 0, 0};
    if (from) {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[s][t][u][r] = *state_place(from, s, t, u, r);
    }
    if constexpr (STATE_ONLY) {
        if (part == 0) {
            float* copy = segment_state(0);
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r) *state_place(copy, s, t, u, r) = S[s][t][u][r];
        }
    }

    Piece<T> qn[STATE_ONLY ? 1 : K_LOADS], kn[K_LOADS], vn[V_LOADS];
    // places of this thread's pieces in a chunk, in bytes; rows past the end read the last one, and are cleared on their way
    // into LDS
    uint32_t q_off[K_LOADS], k_off[K_LOADS], v_off[V_LOADS];
    auto places = [&](int count) {
        auto row = [&](int i) { return (uint32_t)(i < count ? i : count - 1); };
#pragma unroll
        for (int l = 0; l < K_LOADS; ++l) {
            const int i = threadIdx.x + l * THREADS, channel = 8 * (i % KTile::PIECES);
            q_off[l] = (row(i / KTile::PIECES) * (uint32_t)a.q_stride + channel) * sizeof(T);
            k_off[l] = (row(i / KTile::PIECES) * (uint32_t)a.k_stride + channel) * sizeof(T);
        }
#pragma unroll
        for (int l = 0; l < V_LOADS; ++l) {
            const int i = threadIdx.x + l * THREADS;
            v_off[l] = (row(i / VTile::PIECES) * (uint32_t)a.v_stride + 8 * (i % VTile::PIECES)) * sizeof(T);
        }
    };
    auto fetch = [&](int chunk) {
        if (end - chunk < C) places(end - chunk);
        const int64_t row = all.first + chunk;
        auto at = [&](const T* p, int64_t stride, uint32_t off) {
            return reinterpret_cast<const T*>(reinterpret_cast<const char*>(p + row * stride) + off);
        };
#pragma unroll
        for (int l = 0; l < K_LOADS; ++l) {
            if constexpr (!STATE_ONLY) qn[l].load(at(q, a.q_stride, q_off[l]));
            kn[l].load(at(k, a.k_stride, k_off[l]));
        }
#pragma unroll
        for (int l = 0; l < V_LOADS; ++l) vn[l].load(at(v, a.v_stride, v_off[l]));
    };
    // The first `count` rows of the chunk that was fetched, zeros behind them, into a buffer.  A value that is not finite
    // would reach the rows before it (a weight of zero times an infinity): it becomes zero, and its channel NaN from its row
    // on.
    auto put = [&](int count, int parity) {
        const int buffer = AHEAD ? parity : 0;
        auto store = [&](uint8_t* to, int bytes, uint32_t at, const u4* p) {
#pragma unroll
            for (int i = 0; i < IN; ++i) *reinterpret_cast<u4*>(to + i * bytes + at) = p[i];
        };
        u4 p[IN];
#pragma unroll
        for (int l = 0; l < K_LOADS; ++l) {
            const int i = threadIdx.x + l * THREADS, row = i / KTile::PIECES;
            const uint32_t at = KTile::at(row, i % KTile::PIECES);
            if constexpr (!STATE_ONLY) {
                qn[l].parts(p);
                store(qs, KTile::BYTES, at, p);
            }
            if (count < C) kn[l].clear(row >= count);
            kn[l].parts(p);
            store(ks + buffer * K_BYTES, KTile::BYTES, at, p);
        }
#pragma unroll
        for (int l = 0; l < V_LOADS; ++l) {
            const int i = threadIdx.x + l * THREADS, row = i / VTile::PIECES;
            if (count < C) vn[l].clear(row >= count);
            if (__builtin_expect(!vn[l].finite(), 0)) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (vn[l].finite(e)) continue;
                    vn[l].clear_at(e);
                    atomicMin(&odd_from[parity][8 * (i % VTile::PIECES) + e], row);
                }
                odd[parity] = 1;
            }
            vn[l].parts(p);
            store(vs + buffer * V_BYTES, VTile::BYTES, VTile::at(row, i % VTile::PIECES), p);
        }
    };

    // What the accumulators hold is the state times 2^-rest, the rest of the segment's decays over whole powers of two: these go
    // into the accumulators, which rounds nothing, and the rest, in [0, 1), into the scales of what is read and added.  The
    // scales of the next chunks, one to a wave (scanning the decays of one chunk after another would keep the other waves
    // waiting for the one that does).
    double decayed = 0.0;  // the segment's decays up to the next scales, times log2(e)
    float gn;
    auto decays = [&](int chunk) {  // of the wave's chunk of those from `chunk` on, ahead of their use
        const int i = chunk + C * wave + lane % C;
        const int64_t row = all.first + (i < end ? i : end - 1);
        gn = a.decay[row * a.decay_stride + head];
    };
    auto scale = [&](int chunk) {
        const int mine = chunk + C * wave;
        // decays below -200 are zeros beside any fp32 number, those above 200 infinities, and sums of them keep their bits;
        // what is not finite stays
        gn = gn < -200.0f ? -200.0f : gn > 200.0f && gn <= FLT_MAX ? 200.0f : gn;
        const double g = running_sum(mine + lane < end ? (double)gn * 1.4426950408889634 : 0.0);
        if (lane == C - 1) wholes[wave] = g;
        __syncthreads();
        double before = decayed;  // the wave's chunk
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const double x = wholes[i];
            if (i < wave) before += x;
            decayed += x;
        }
        const double whole = wholes[wave], after = before + whole, from = floor(before), down = floor(after);
        ChunkScales<C>& to = scales[wave];
        if (lane < C) {
            to.sum[lane] = g;
            to.from_start[lane] = exp2_of(g + (before - from)) * a.scale;
            to.to_end[lane] = exp2_of(whole - g - (after - down));
        }
        if (lane == 0) to.by = ldexpf(1.0f, (int)(down - from));
        decays(chunk + C * WAVES);
    };

    const uint32_t out_bytes = a.out_type == IQ4XS_TYPE_F32 ? 4 : 2;
    for (int i = threadIdx.x; i < 2 * DVT; i += THREADS) odd_from[i / DVT][i % DVT] = C;
    if (threadIdx.x < 2) odd[threadIdx.x] = 0;
    if constexpr (!STATE_ONLY) {
        for (int i = threadIdx.x; i < OUT * PTile::BYTES / 16; i += THREADS)
            *reinterpret_cast<u4*>(&ps[16 * i]) = u4{0, 0, 0, 0};  // above the diagonal
    }
    __syncthreads();
    decays(begin);
    places(C);
    fetch(begin);
    put(end - begin, 0);
    if (begin + C < end) fetch(begin + C);
    __syncthreads();
    bool was_odd = false;
    for (int chunk = begin, which = 0; chunk < end; chunk += C, ++which) {
        const int parity = which % 2;
        const bool more = chunk + C < end;
        const int count = end - chunk;
        if (which % WAVES == 0) {
            scale(chunk);
            __syncthreads();
        }
        const ChunkScales<C>& sc = scales[which % WAVES];
        // the places along a row are cheaper computed than kept
        asm volatile("" : "+v"(q_row), "+v"(k_row), "+v"(p_row), "+v"(k_column), "+v"(v_column));
        const uint32_t k_buffer = AHEAD ? parity * K_BYTES : 0, v_buffer = AHEAD ? parity * V_BYTES : 0;
        if (__builtin_expect(was_odd, 0)) {
            for (int i = threadIdx.x; i < DVT; i += THREADS) odd_from[parity ^ 1][i] = C;
            if (threadIdx.x == 0) odd[parity ^ 1] = 0;
            if (STATE_ONLY) __syncthreads();  // before the next chunk says which of its values are; else below
        }
        f4 O[IT][NT];
        if constexpr (!STATE_ONLY) {
            // weighted scores of tiles on and below the diagonal: keys 16 kt + 4 j + r of query 16 it + n; weights below 2^-126
            // are zeros
            if (wave < 3) {
                const int it = wave > 0, kt = wave > 1;
                f4 z{0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u4 x[IN], y[IN];
#pragma unroll
                    for (int p = 0; p < IN; ++p) {
                        x[p] = read_row((k_row ^ 64 * s) + k_buffer + p * KTile::BYTES + 16 * kt * KTile::ROW);
                        y[p] = read_row((q_row ^ 64 * s) + p * KTile::BYTES + 16 * it * KTile::ROW);
                    }
#pragma unroll
                    for (int p = IN - 1; p >= 0; --p)
#pragma unroll
                        for (int o = IN - 1; o >= 0; --o)
                            if (p + o < OUT) z = Matrix<__bf16>::mma16(x[p], y[o], z);
                }
                const int query = 16 * it + n, key = 16 * kt + 4 * j;
                const double g = sc.sum[query];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = __builtin_amdgcn_exp2f((float)(g - sc.sum[key + r])) * a.scale;
                    z[r] = key + r <= query ? z[r] * w : 0.0f;
                }
                uint32_t lo[OUT], hi[OUT];
                split<OUT>(z[0], z[1], lo);
                split<OUT>(z[2], z[3], hi);
#pragma unroll
                for (int p = 0; p < OUT; ++p)
                    *reinterpret_cast<u2*>(&ps[p * PTile::BYTES + PTile::at(query, key / 8) + 2 * (key % 8)]) = u2{lo[p], hi[p]};
            }
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int u = 0; u < NT; ++u) O[i][u] = f4{0, 0, 0, 0};
            // a step's queries are read while the step before it is multiplied
            u4 y[2][IT][IN];
            auto queries = [&](int s) {
#pragma unroll
                for (int i = 0; i < IT; ++i)
#pragma unroll
                    for (int p = 0; p < IN; ++p)
                        y[s % 2][i][p] = read_row((q_row ^ 64 * s) + p * KTile::BYTES + 16 * i * KTile::ROW);
            };
            queries(0);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if (s + 1 < KS) queries(s + 1);
                __builtin_amdgcn_sched_barrier(0);
                u4 x[NT][OUT];
#pragma unroll
                for (int u = 0; u < NT; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t z[OUT];
                        split<OUT>(S[s][e / 2][u][2 * (e % 2)], S[s][e / 2][u][2 * (e % 2) + 1], z);
#pragma unroll
                        for (int p = 0; p < OUT; ++p) x[u][p][e] = z[p];
                    }
#pragma unroll
                for (int p = OUT - 1; p >= 0; --p)
#pragma unroll
                    for (int o = IN - 1; o >= 0; --o)
#pragma unroll
                        for (int i = 0; i < IT; ++i)
#pragma unroll
                            for (int u = 0; u < NT; ++u)
                                if (p + o < OUT) O[i][u] = Matrix<__bf16>::mma16(x[u][p], y[s % 2][i][o], O[i][u]);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const float w = sc.from_start[16 * i + n];
#pragma unroll
                for (int u = 0; u < NT; ++u) O[i][u] *= w;
            }
            __syncthreads();  // weighted scores are there, queries done with
        }
        if (AHEAD && more) {
            put(end - chunk - C, parity ^ 1);
            if (chunk + 2 * C < end) fetch(chunk + 2 * C);
        }
        // keys of a step of the state's update, read while the step before it is multiplied
        u4 kx[2][2][IN];
        auto keys = [&](int s) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int p = 0; p < IN; ++p)
                    kx[s % 2][h][p] = eight_tokens<KTile>((k_column ^ 64 * s) + 8 * h + k_buffer + p * KTile::BYTES);
        };
        // the wave's values: channels of tile u by tokens 8 j + e
        u4 V[NT][IN];
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int p = 0; p < IN; ++p) V[u][p] = eight_tokens<VTile>(v_column + v_buffer + 8 * u + p * VTile::BYTES);
        const bool some_odd = odd[parity] != 0;
        float w[8];
        const float by = sc.by;
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = sc.to_end[8 * j + e];
        u4 y[IT][OUT];
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int i = 0; i < IT; ++i)
#pragma unroll
                for (int p = 0; p < OUT; ++p) y[i][p] = read_row(p_row + p * PTile::BYTES + 16 * i * PTile::ROW);
        }
        keys(0);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!STATE_ONLY) {
#pragma unroll
            for (int p = OUT - 1; p >= 0; --p)
#pragma unroll
                for (int o = IN - 1; o >= 0; --o)
#pragma unroll
                    for (int i = 0; i < IT; ++i)
#pragma unroll
                        for (int u = 0; u < NT; ++u)
                            if (p + o < OUT) O[i][u] = Matrix<__bf16>::mma16(V[u][o], y[i][p], O[i][u]);
        }
        auto decay = [&](int s) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int u = 0; u < NT; ++u) S[s][h][u] *= by;
        };
        if (!DECAY_BESIDE && by != 1.0f) {
#pragma unroll
            for (int s = 0; s < KS; ++s) decay(s);
        }
        // values times what is left of them at the chunk's end, and the state's update
        u4 W[NT][3];
#pragma unroll
        for (int u = 0; u < NT; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x0 = __uint_as_float(V[u][IN - 1][e] << 16), x1 = high_part(__uint_as_float(V[u][IN - 1][e]));
#pragma unroll
                for (int p = IN - 2; p >= 0; --p) {
                    x0 += __uint_as_float(V[u][p][e] << 16);
                    x1 += high_part(__uint_as_float(V[u][p][e]));
                }
                uint32_t z[3];
                split<3>(x0 * w[2 * e], x1 * w[2 * e + 1], z);
#pragma unroll
                for (int p = 0; p < 3; ++p) W[u][p][e] = z[p];
            }
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s + 1 < KS) keys(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            if (DECAY_BESIDE && s == 0) decay(0);
            if (DECAY_BESIDE && s + 1 < KS) decay(s + 1);
#pragma unroll
            for (int o = 2; o >= 0; --o)
#pragma unroll
                for (int p = IN - 1; p >= 0; --p)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int u = 0; u < NT; ++u)
                            if (p + o < 3) S[s][h][u] = Matrix<__bf16>::mma16(kx[s % 2][h][p], W[u][o], S[s][h][u]);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!STATE_ONLY) {
            char* out = static_cast<char*>(a.out) + (int64_t)(all.first + chunk) * a.heads * dv * out_bytes;
#pragma unroll
            for (int i = 0; i < IT; ++i) {
                const int row = 16 * i + n;
                if (__builtin_expect(some_odd, 0)) {
#pragma unroll
                    for (int u = 0; u < NT; ++u)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (row >= odd_from[parity][column(u, 4 * j + r)]) O[i][u][r] = NAN;
                }
                if (row < count) {
                    // two tiles' columns of a lane lie one after another
                    const uint32_t at = ((uint32_t)row * a.heads + head) * dv + tile * DVT + column(0, 4 * j);
                    char* to = out + at * out_bytes;
                    if constexpr (NT == 2)
                        store8(to, a.out_type, O[i][0], O[i][NT - 1]);
                    else
                        store4(to, 0, a.out_type, O[i][0]);
                }
            }
        }
        if (__builtin_expect(some_odd, 0)) {
#pragma unroll
            for (int u = 0; u < NT; ++u) {
                const float x = odd_from[parity][column(u, n)] < C ? NAN : 0.0f;
#pragma unroll
                for (int s = 0; s < KS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) S[s][h][u] += x;
            }
        }
        was_odd = some_odd;
        __syncthreads();  // keys and values are done with, and the next there
        if (!AHEAD && more) {
            put(end - chunk - C, parity ^ 1);
            if (chunk + 2 * C < end) fetch(chunk + 2 * C);
            __syncthreads();
        }
    }

    if (STATE_ONLY && tile == 0 && threadIdx.x == 0)
        seg.decays[kept + (int64_t)part * a.heads] = exp2_parts(decayed);
    float* to = STATE_ONLY ? segment_state(part + 1)
                : last     ? state_at(a, a.to_slots, seq, head, DK * dv)
                           : nullptr;
    if (!to) return;
    const float rest = exp2_of(decayed - floor(decayed));
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int u = 0; u < NT; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    *state_place(to, s, t, u, r) = S[s][t][u][r] * rest;
}

// The states that segments begin with, in the place of what each adds, from the third on.  Bound by memory: 16 bytes read and
// 16 written of a piece, all segments' reads on their way at once (7 segments of 4 MiB: 10 us, 5.6 TB/s).
__global__ __launch_bounds__(256) void join_segments_kernel(LinearArgs a, LinearSegments seg, int size) {
    const int pieces = size / 4;
    const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int piece = (int)(at % pieces), head = (int)(at / pieces % a.heads);
    const int64_t which = at / pieces / a.heads, row = which * 2 * seg.length;
    const int seq = seg.join_rows ? last_sequence(a, threadIdx.x % 64, [&](int start, int) { return start <= row; }) : (int)which;
    if (seq < 0 || seq >= a.seqs) return;
    const Rows all = rows_of(a, seq);
    const int count = (int)((all.count + (int64_t)seg.length - 1) / seg.length);
    if (count < 3 || (seg.join_rows && row - all.first >= 2 * (int64_t)seg.length)) return;
    const int64_t first = seg.kept.of(all.first, seq) * a.heads + head;
    f4* p = reinterpret_cast<f4*>(seg.states + first * size + 4 * piece);
    const int64_t step = (int64_t)a.heads * pieces;
    f4 s = p[step];
#pragma unroll 8
    for (int i = 2; i < count; ++i) {
        // of a state that grows, 2^decays alone may pass what fp32 holds
        const SegmentDecay d = seg.decays[first + (i - 1) * (int64_t)a.heads];
        const f4 x = p[i * step];
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] = ldexpf(s[e] * d.part, d.exponent) + x[e];
        p[i * step] = s;
    }
}

template <int DK, int NT, int WAVES, typename T, int OUT>
static void launch(const LinearArgs& a, const LinearSegments& seg, int dv, hipStream_t stream) {
    // 160 KiB of LDS: queries of all parts once, keys and values twice
    constexpr int ROWS = 2 * CHUNK * parts_of<T>, COLUMNS = 16 * NT * WAVES;
    constexpr bool AHEAD = ROWS * (3 * DK + 2 * COLUMNS) + 12 * 1024 <= 160 * 1024;
    const dim3 block(64 * WAVES), grid((unsigned)seg.grid);
    if (seg.count > 1) {
        hipLaunchKernelGGL((linear_chunk_kernel<DK, NT, WAVES, T, 2, true, AHEAD>), grid, block, 0, stream, a, seg, dv);
        const int64_t joins = seg.join_rows ? joining_rows(a.total, seg.length) : a.seqs;
        const int64_t pieces = joins * a.heads * DK * dv / 4;
        hipLaunchKernelGGL(join_segments_kernel, dim3((unsigned)((pieces + 255) / 256)), dim3(256), 0, stream, a, seg, DK * dv);
    }
    hipLaunchKernelGGL((linear_chunk_kernel<DK, NT, WAVES, T, OUT, false, AHEAD>), grid, block, 0, stream, a, seg, dv);
}

template <int DK, typename T, int OUT>
static void launch_columns(const LinearArgs& a, const LinearSegments& seg, int dv, hipStream_t stream) {
    if (linear_chunk_columns(DK, dv) == 64)
        launch<DK, 1, 4, T, OUT>(a, seg, dv, stream);
    else if constexpr (DK == 64)
        launch<DK, 2, 4, T, OUT>(a, seg, dv, stream);
    else if constexpr (DK == 128 && parts_of<T> == 1)
        launch<DK, 2, 4, T, OUT>(a, seg, dv, stream);
    else if constexpr (DK == 128)
        launch<DK, 1, 8, T, OUT>(a, seg, dv, stream);
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
