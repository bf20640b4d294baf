// attention_tile.hip -- attention of many rows over the paged cache: prompts, chunks of prompts and longer drafts.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q k_j - m),  lse = m + log(sum_j w_j)
//
// A workgroup takes 128 rows of a cache head (new tokens times the query heads that read it, token by token, so that
// rows of one token share every key) and goes through the keys in tiles; each of its four waves has 32 rows as the
// columns of 32 x 32 matrix products, S^T = K Q^T and O^T = V^T W^T.  Bound by the matrix products, and next to them by
// the exponentials (a quarter of the rate of other vector operations: 16 for every 16 x 32 x 32 products), so:
// - tiles of keys and values reach LDS by asynchronous copies, the next tile's in flight during this tile's products;
//   pieces of 16 bytes are exchanged within a row so that reads of rows (keys) and of columns (values, turned by the
//   LDS on their way) touch every bank once;
// - S^T leaves in each lane the weights of one row, for exactly the keys whose values the second product wants from
//   that lane: weights stay in registers;
// - two workgroups share a CU, so that one's products run beside the other's exponentials;
// - the running maximum of a row moves only when a key passes it by 2^8 (in powers of two);
// - the scores of the next 32 keys, the weights of these and the value products of those before are one stream of
//   instructions, in the order written.
// Measured: 2048 tokens over 16384 keys of 128 channels, 64 query heads on 8: 1020 to 1150 us from card to card, 900 to
// 1010 TFLOP/s of fp16 (1440 is what a large library product reaches); on a card of 1022 bf16 took 966, 64 channels 1224,
// 256 1127.  Matrix units are busy about half of the time and vector units as long, with little overlap; LDS has no
// conflicts.
// An 8-bit cache whose outputs are bf16 alone: keys and values become fp16 on their way into LDS (half a step of 2^-11
// each, an eighth of what such outputs show).  In fp16 outputs that would be 1.7 to 2.4 times the error of their own
// rounding, and log-sum-exps would be off by 1e-5, so for these (EXACT) keys stay codes, exact in fp16, whose scales
// multiply the parts of a score in fp32, and weights go as two fp16 numbers: half as many products again and as many
// vector operations.  bf16 queries become fp16 with a power of two taken out of each row.  2048 tokens over 16384 keys
// of 128 channels on that card: 1222 us with rounded keys, 1835 with exact ones (of 64 channels 1413 and 2182, of 256
// 1517 and 2603); the kernel of few rows takes 2428 (2911, 4960).
#include <type_traits>

#include "attention_core.h"
#include "attention_internal.h"
#include "iq4xs_internal.h"

namespace iq4xs {

constexpr int TILE_WAVES = 4, TILE_ROWS = 32 * TILE_WAVES;

__device__ inline uint32_t lds_address(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)(const_cast<void*>(p));
}

// 16 bytes for each lane, from global base + offset to LDS at lds + 16 * lane, asynchronously (lds the same in all
// lanes).  As asm: the compiler would let every later LDS read wait for it.  The kernel waits before the barrier that
// ends a tile.
__device__ inline void copy_to_lds(const void* base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "s"(lds)
                 : "memory", "m0");
}
__device__ inline void wait_for_copies() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

__device__ inline u4 read_row(uint32_t lds) {
    return *reinterpret_cast<__attribute__((address_space(3))) const u4*>((uintptr_t)lds);
}
// Four keys of the lane's channel: 16 lanes read 4 rows of 16 channels and each gets a column.
__device__ inline u2 read_column(uint32_t lds) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(
        u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<__attribute__((address_space(3))) s4*>((uintptr_t)lds)));
}

// Geometry of a tile in LDS: KEYS rows of 2 * D bytes, 16-byte pieces exchanged within a row.
template <int D>
struct Tile {
    static constexpr int KEYS = 64;
    static constexpr int ROW = 2 * D, BYTES = KEYS * ROW;
    static constexpr int PIECES = D / 8;               // of a row
    static constexpr int ROWS = 64 / PIECES;           // of 64 pieces
    static constexpr int LOADS = KEYS * PIECES / 256;  // for each lane
    // Places are exclusive ors: place(row, piece) = place(row', piece) ^ place(row - row', 0) where row' are the row's
    // bits within a load.
    // keys are read by rows: 16 rows' pieces of one place lie in 16 places
    static __device__ int key_place(int row, int piece) {
        return piece ^ (D == 64 ? (row >> 1) & 7 : row & 15);
    }
    // values by columns: 4 rows' groups of 4 pieces lie apart
    static __device__ int value_place(int row, int piece) {
        return piece ^ (D == 64 ? ((row >> 1) & 1) << 2 : (row & 3) << 2);
    }
};

// 16-byte piece of 8 codes as fp16, times the scale of their group or (SCALED false) as they are.
template <bool SCALED>
__device__ inline u4 codes_to_f16(u2 w, _Float16 scale) {
    u4 x;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const uint32_t b = (p < 2 ? w.x : w.y) ^ 0x80808080u;
        const uint32_t z = __builtin_amdgcn_perm(b, b, p % 2 ? 0x0C030C02u : 0x0C010C00u) | 0x64006400u;
        const h2 v = __builtin_bit_cast(h2, z) - h2{(_Float16)1152, (_Float16)1152};
        x[p] = __builtin_bit_cast(uint32_t, SCALED ? v * h2{scale, scale} : v);
    }
    return x;
}

template <int D, typename Q, typename KV, bool EXACT>
__global__ __launch_bounds__(64 * TILE_WAVES, D == 256 ? 1 : 2) void tile_attention_kernel(AttentionArgs a) {
    using T = Tile<D>;
    constexpr bool CODES = sizeof(KV) == 1;
    using W = typename std::conditional<CODES, _Float16, KV>::type;
    using M = Matrix<W>;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2][2][T::BYTES];  // [buffer][keys, values]
    // of exact keys, in the order in which a lane's scores want them: the 4 keys of every 8, half by half
    __shared__ __attribute__((aligned(16))) _Float16 key_scales[EXACT ? 2 : 1][D / 32][T::KEYS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    const int n = lane % 32, half = lane / 32;

    unsigned x = blockIdx.x;
    const int head = x % a.c.heads;
    x /= a.c.heads;
    const int seq = x % a.seqs;
    x /= a.seqs;
    // the last rows see the most keys: first
    const int tile = a.row_tiles - 1 - x % a.row_tiles, split = x / a.row_tiles;
    int total_fresh;
    const Sequence s = sequence(a, seq, total_fresh);
    const int rows = s.fresh * a.group, row0 = tile * TILE_ROWS;
    if (row0 >= rows) return;
    const int last = (rows < row0 + TILE_ROWS ? rows : row0 + TILE_ROWS) - 1;
    const int token0 = row0 / a.group, token1 = last / a.group;
    // keys that some row sees, and those that all see
    const int any_lo = least_key(a, s, total_fresh, token0), any_hi = end_key(a, s, total_fresh, token1);
    const int all_lo = least_key(a, s, total_fresh, token1), all_hi = end_key(a, s, total_fresh, token0);
    int k0, k1;
    if (!split_keys(a, s, any_lo, any_hi, split, k0, k1)) return;

    // this lane's row (lanes without one repeat the last)
    const int wave0 = row0 + 32 * wave;
    const int r = wave0 + n <= last ? wave0 + n : last, token = r / a.group;
    const int lo = least_key(a, s, total_fresh, token), hi = end_key(a, s, total_fresh, token);
    const int query_head = head * a.group + r % a.group;

    u4 q[D / 16];
    float factor = fabsf(a.scale);
    {
        const u4* p = reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.q) +
                                                  (int64_t)(s.first + token) * a.q_stride + query_head * D + 8 * half);
#pragma unroll
        for (int c = 0; c < D / 16; ++c) q[c] = p[2 * c];
        if constexpr (CODES && __is_same(Q, __bf16)) {
            const int e =
                query_exponent(__float_as_uint(max_of_halves(__uint_as_float(query_top(q) << 16))) >> 16);
            factor = ldexpf(factor, e);
            queries_to_f16(q, e);
        }
        // a negative scale goes with the queries; one of zero must not meet the -Inf of hidden keys
        if (a.scale < 0.0f) {
#pragma unroll
            for (int c = 0; c < D / 16; ++c) q[c] ^= 0x80008000u;
        }
        factor = fmaxf(factor, FLT_MIN);
    }

    fx16 o[D / 32];
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -FLT_MAX, l = 0.0f, rounded = 0.0f;  // sums of the weights as they are and, where they are rounded, so

    const uint32_t at = lds_address(lds);
    // wave w brings a tile's rows 16 w to 16 w + 15, which lie in one page; a page that is not in the cache, or past the
    // keys, is read as page 0 and masked
    const int bring = 16 * wave, piece = lane % T::PIECES, in_load = lane / T::PIECES;
    constexpr int PARTS = T::KEYS / 16;
    // Pages of a tile, looked up a tile before they are wanted: of its 16 keys i in lane i.  A load without a condition,
    // waited for where `locate` uses it; waiting at once would be waiting for the tiles on their way (2048 tokens over
    // 16384 keys: 1116 us, and 1032 so).
    int looked_up;
    auto look_up = [&](int base) {
        const int key = base + 16 * (lane % PARTS);
        const int32_t* p = key < k1 ? s.pages + (key >> a.c.shift) : a.starts;
        looked_up = *p;
    };
    // of the tile at `base`, which was looked up: which 16 keys are not there, and where this wave's rows begin
    auto locate = [&](int base, uint32_t& lacking) {
        const bool held = base + 16 * (lane % PARTS) < k1 && looked_up >= 0 && looked_up < a.c.pages;
        lacking = ~(uint32_t)__ballot(held) & ((1u << PARTS) - 1);
        const int page = __builtin_amdgcn_readlane(looked_up, wave);
        const bool there = !(lacking >> wave & 1);
        return page_row(a.c, there ? page : 0, head, there ? (base + bring) & ((1 << a.c.shift) - 1) : 0);
    };
    // rows of one side (0 keys, 1 values) on their way to a buffer; of an 8-bit cache into registers, from which `put`
    // takes them
    // heads of 256 have no registers for both sides at once: keys are fetched when the values have been put
    constexpr bool IN_TURN = CODES && D == 256;
    u2 code[IN_TURN ? 1 : 2][CODES ? T::LOADS : 1];
    _Float16 code_scale[IN_TURN ? 1 : 2][CODES ? T::LOADS : 1];
    uint32_t load_at[2] = {(uint32_t)(in_load * T::ROW + 16 * T::key_place(in_load, piece)),
                           (uint32_t)(in_load * T::ROW + 16 * T::value_place(in_load, piece))};
    auto turn = [&](int side, int i) {
        return 16u * (side ? T::value_place(i * T::ROWS, 0) : T::key_place(i * T::ROWS, 0));
    };
    auto fetch = [&](int side, int64_t row, int buffer) {
        asm volatile("" : "+v"(load_at[side]));  // a load's place is cheaper computed than kept
        const void* from = side ? a.c.v : a.c.k;
        if constexpr (CODES) {
            const int8_t* p = static_cast<const int8_t*>(from) + row * D;
            const _Float16* sc = (side ? a.c.vs : a.c.ks) + row * (D / 32);
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) {
                const int rr = i * T::ROWS;
                code[IN_TURN ? 0 : side][i] = *reinterpret_cast<const u2*>(p + rr * D + 8 * (unsigned)lane);
                code_scale[IN_TURN ? 0 : side][i] = sc[rr * (D / 32) + (unsigned)lane / 4];
            }
        } else {
            const uint8_t* p = static_cast<const uint8_t*>(from) + row * T::ROW;
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) {
                copy_to_lds(p + i * T::ROWS * T::ROW, load_at[side] ^ turn(side, i),
                            at + (buffer * 2 + side) * T::BYTES + (bring + i * T::ROWS) * T::ROW);
            }
        }
    };
    // An infinity times a weight's second part is NaN: exact products want none in LDS; `odd` says that there were such.
    int odd = 0;
    auto put = [&](int side, int buffer, int base = 0, uint32_t missing = 0) {
        if constexpr (CODES) {
            asm volatile("" : "+v"(load_at[side]));
            bool large = false;  // scales past 65504 / 127, whose values may not be finite
            if (EXACT && side == 1) {
#pragma unroll
                for (int i = 0; i < T::LOADS; ++i) {
                    const _Float16 by = code_scale[IN_TURN ? 0 : 1][i];
                    large = large || (__builtin_bit_cast(uint16_t, by) & 0x7FFFu) > 0x6007u;
                }
                large = __any(large);
            }
#pragma unroll
            for (int i = 0; i < T::LOADS; ++i) {
                const u2 c = code[IN_TURN ? 0 : side][i];
                const _Float16 by = code_scale[IN_TURN ? 0 : side][i];
                u4* to = reinterpret_cast<u4*>(&lds[buffer][side][(bring + i * T::ROWS) * T::ROW] +
                                               (load_at[side] ^ turn(side, i)));
                if (EXACT && side == 0) {
                    const int rr = bring + i * T::ROWS + in_load;
                    *to = codes_to_f16<false>(c, by);
                    if (piece % 4 == 0)
                        key_scales[buffer][piece / 4][rr / 32 * 32 + rr / 4 % 2 * 16 + rr % 32 / 8 * 4 + rr % 4] = by;
                } else {
                    u4 v = codes_to_f16<true>(c, by);
                    if (__builtin_expect(large, 0)) {
                        const int rr = bring + i * T::ROWS + in_load, key = base + rr;
                        const u4 f = M::finite(v), x = v ^ f;
                        odd |= key >= any_lo && key < any_hi && !(missing >> (rr / 16) & 1) &&
                               (x.x | x.y | x.z | x.w) != 0;
                        v = f;
                    }
                    *to = v;
                }
            }
        }
    };

    // the values of a tile once more, what no row sees cleared
    auto again = [&](int base, int buffer, uint32_t missing) {
        for (int i = threadIdx.x; i < T::KEYS * T::PIECES; i += 64 * TILE_WAVES) {
            const int rr = i / T::PIECES, p = i % T::PIECES, key = base + rr;
            u4 v{0, 0, 0, 0};
            if (key >= any_lo && key < any_hi && !(missing >> (rr / 16) & 1)) {
                const int64_t row = page_row(a.c, s.pages[key >> a.c.shift], head, key & ((1 << a.c.shift) - 1));
                if constexpr (CODES)
                    v = codes_to_f16<true>(*reinterpret_cast<const u2*>(static_cast<const int8_t*>(a.c.v) + row * D + 8 * p),
                                     a.c.vs[row * (D / 32) + p / 4]);
                else
                    v = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.c.v) + row * D + 8 * p);
            }
            *reinterpret_cast<u4*>(&lds[buffer][1][rr * T::ROW + 16 * T::value_place(rr, p)]) = v;
        }
    };

    // where this lane reads: keys by rows n, values by columns
    const int column = lane % 16, value_row = 4 * half + column / 4;
    uint32_t key_at = at + n * T::ROW + 16 * T::key_place(n, half);
    uint32_t value_at = at + T::BYTES + value_row * T::ROW + 8 * (column % 2) +
                        16 * T::value_place(value_row, 2 * ((lane / 16) % 2) + (column % 4) / 2);
    // pieces 2 c further along a row of keys, 4 t of values, and `more` bytes on: the exchange of pieces is an exclusive
    // or within 16 (8 with heads of 64)
    auto key_piece = [&](uint32_t from, int c, int more) {
        return read_row((from ^ (32 * c & (T::ROW < 256 ? 127 : 255))) + (32 * c & ~255) + more);
    };
    auto value_piece = [&](uint32_t from, int t, int more) {
        const uint32_t to = (from ^ (64 * t & (T::ROW < 256 ? 127 : 255))) + (64 * t & ~255) + more;
        const u2 x0 = read_column(to), x1 = read_column(to + 8 * T::ROW);
        return u4{x0.x, x0.y, x1.x, x1.y};
    };

    // `z` are scores of 32 keys at `base`: hidden ones go, the running maximum moves if it must, and with it the sums and
    // the weights `w` still to be used.
    auto raise = [&](fx16& z, int base, uint32_t lacking, bool edge, u4(&w)[2]) {
        if (__builtin_expect(edge, 0)) {
            const int from = lo - base - 4 * half, to = hi - base - 4 * half;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int in = 8 * (i / 4) + i % 4;
                z[i] = in >= from && in < to && !(lacking >> (in / 16) & 1) ? z[i] : -INFINITY;
            }
        }
        float top = z[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, z[i]);
        top *= factor;
        if (__builtin_expect(__any(top > m + (M::LARGEST + 8.0f)), 0)) {
            // whole powers of two, so that scaling the 16-bit weights is exact
            const float up = fmaxf(ceilf(max_of_halves(top)) - M::LARGEST, m), keep = __builtin_amdgcn_exp2f(m - up);
            m = up;
            l *= keep;
            rounded *= keep;
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                o[t] *= keep;
                if constexpr (D == 256) {  // back where the products keep them, one at a time
                    asm volatile("" : "+a"(o[t]));
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int p = 0; p < 4; ++p) w[k][p] = M::scaled(w[k][p], keep);
        }
    };
    // A pair of weights of the scores z.
    auto weigh = [&](const fx16& z, int i, u4(&w)[2]) {
        const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i], factor, -m));
        const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i + 1], factor, -m));
        l += x0 + x1;
        uint32_t pair = M::pack(x0, x1);
        rounded = M::add(pair, rounded);
        asm volatile("" : "+v"(pair), "+v"(l), "+v"(rounded));  // here, not where they are used
        w[i / 8][i % 8 / 2] = pair;
    };
    // A step's products in turn, those of the scores (place c of the queries) between those of the values (16 keys k,
    // channels t); its operands from LDS are read AHEAD products before.
    constexpr int PRODUCTS = D / 8, AHEAD = 4;
    auto piece_of = [&](int i, uint32_t keys, uint32_t values) {
        const int j = i / 2;
        return i % 2 == 0 ? key_piece(keys, j, 0) : value_piece(values, j % (D / 32), 16 * (j / (D / 32)) * T::ROW);
    };
    auto begin = [&](uint32_t keys, uint32_t values, u4(&f)[AHEAD]) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) f[i] = piece_of(i, keys, values);
    };
    // The scores `next` of 32 keys, the weights of the scores `z`, and the product of the weights `w` before them with
    // their values.  The order is kept as written: beside each product its share of the weights.
    auto step = [&](uint32_t keys, uint32_t values, u4(&f)[AHEAD], fx16& next, const fx16& z, const u4(&w)[2],
                    u4(&w_next)[2]) {
#pragma unroll
        for (int i = 0; i < 16; ++i) next[i] = 0.0f;
#pragma unroll
        for (int i = 0; i < PRODUCTS; ++i) {
            const int j = i / 2;
            if (i % 2 == 0)
                next = M::mma32(f[i % AHEAD], q[j], next);
            else
                o[j % (D / 32)] = M::mma32(f[i % AHEAD], w[j / (D / 32)], o[j % (D / 32)]);
            if (i + AHEAD < PRODUCTS) f[i % AHEAD] = piece_of(i + AHEAD, keys, values);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e * PRODUCTS / 8 == i || (PRODUCTS == 8 && e == i)) weigh(z, 2 * e, w_next);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // A weight of zero times an infinity is NaN.  Where rows differ in what they see, values that no row sees and values
    // that are not finite are cleared in LDS; the latter come again after the last tile.
    auto clear = [&](int base, int buffer, uint32_t missing) {
        uint32_t some = 0;
        for (int i = threadIdx.x; i < T::KEYS * T::PIECES; i += 64 * TILE_WAVES) {
            const int key = base + i / T::PIECES;
            u4* p = reinterpret_cast<u4*>(&lds[buffer][1][16 * i]);
            const bool seen = key >= any_lo && key < any_hi && !(missing >> (i / T::PIECES / 16) & 1);
            const u4 v = *p, f = seen ? M::finite(v) : u4{0, 0, 0, 0}, x = v ^ f;
            some |= seen ? x.x | x.y | x.z | x.w : 0u;
            *p = f;
        }
        odd = __syncthreads_or(odd | (some != 0));
    };

    if constexpr (EXACT) {
        // A tile's 32 keys in turn: their scores, weights and product with the values; the next tile's codes are on their
        // way meanwhile.
        uint32_t lacking;
        look_up(k0);
        int64_t row = locate(k0, lacking);
        fetch(0, row, 0);
        if (IN_TURN) put(0, 0);
        fetch(1, row, 0);
        if (!IN_TURN) put(0, 0);
        put(1, 0, k0, lacking);
        look_up(k0 + T::KEYS);
        int buffer = 0;
        for (int base = k0; base < k1; base += T::KEYS, buffer ^= 1) {
            asm volatile("" : "+v"(looked_up));
            __syncthreads();
            const bool edge = lacking != 0 || base < all_lo || base + T::KEYS > all_hi, more = base + T::KEYS < k1;
            if (__builtin_expect(edge, 0)) clear(base, buffer, lacking);
            const uint32_t was_lacking = lacking;
            if (more) {
                row = locate(base + T::KEYS, lacking);
                fetch(0, row, buffer ^ 1);
                if (!IN_TURN) fetch(1, row, buffer ^ 1);
                look_up(base + 2 * T::KEYS);
            }
            asm volatile("" : "+v"(key_at), "+v"(value_at));
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const uint32_t from = buffer * 2 * T::BYTES + s * 32 * T::ROW;
                fx16 z;
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = 0.0f;
#pragma unroll
                for (int g = 0; g < D / 32; ++g) {
                    fx16 part;
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[i] = 0.0f;
                    part = M::mma32(key_piece(key_at + from, 2 * g, 0), q[2 * g], part);
                    part = M::mma32(key_piece(key_at + from, 2 * g + 1, 0), q[2 * g + 1], part);
                    const h8* sc = reinterpret_cast<const h8*>(&key_scales[buffer][g][32 * s + 16 * half]);
                    const h8 s0 = sc[0], s1 = sc[1];
#pragma unroll
                    for (int i = 0; i < 16; ++i) z[i] = __builtin_fmaf(part[i], (float)(i < 8 ? s0[i] : s1[i - 8]), z[i]);
                }
                u4 w[2] = {}, rest[2];
                raise(z, base + 32 * s, was_lacking >> 2 * s, edge, w);
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const float x0 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i], factor, -m));
                    const float x1 = __builtin_amdgcn_exp2f(__builtin_fmaf(z[i + 1], factor, -m));
                    l += x0 + x1;
                    const h2 high{(_Float16)x0, (_Float16)x1};
                    w[i / 8][i % 8 / 2] = __builtin_bit_cast(uint32_t, high);
                    rest[i / 8][i % 8 / 2] = M::pack(x0 - (float)high.x, x1 - (float)high.y);
                }
                if (IN_TURN && s == 0 && more) {
                    put(0, buffer ^ 1);
                    fetch(1, row, buffer ^ 1);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int t0 = 0; t0 < D / 32; t0 += 2) {
                        const u4 v0 = value_piece(value_at + from, t0, 16 * k * T::ROW);
                        const u4 v1 = value_piece(value_at + from, t0 + 1, 16 * k * T::ROW);
                        o[t0] = M::mma32(v0, w[k], o[t0]);
                        o[t0 + 1] = M::mma32(v1, w[k], o[t0 + 1]);
                        o[t0] = M::mma32(v0, rest[k], o[t0]);
                        o[t0 + 1] = M::mma32(v1, rest[k], o[t0 + 1]);
                    }
            }
            if (more) {
                if (!IN_TURN) put(0, buffer ^ 1);
                put(1, buffer ^ 1, base + T::KEYS, lacking);
            }
        }
    } else {
        // Tile T in steps 2 T and 2 T + 1 of 32 keys.  A step computes the scores of the step after it and the weights of its
        // own beside the product of the weights before it: keys are wanted a tile ahead of values.  The barrier of tile T
        // comes before step 2 T + 1: keys of tile T and values of tile T - 1 are done with, those of T + 1 and T are there.
        uint32_t lacking, next_lacking = (1u << PARTS) - 1;
        look_up(k0);
        int64_t row = locate(k0, lacking);
        fetch(0, row, 0);
        if (IN_TURN) put(0, 0);
        fetch(1, row, 0);
        if (!IN_TURN) put(0, 0);
        put(1, 0);
        look_up(k0 + T::KEYS);
        wait_for_copies();
        __syncthreads();
        fx16 even, uneven;
        u4 w_even[2] = {}, w_odd[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) even[i] = uneven[i] = 0.0f;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
            even = M::mma32(key_piece(key_at, c, 0), q[c], even);
            uneven = M::mma32(key_piece(key_at, c, 32 * T::ROW), q[c], uneven);
        }
        bool edge = lacking != 0 || k0 < all_lo || k0 + T::KEYS > all_hi;
        raise(even, k0, lacking, edge, w_even);
#pragma unroll
        for (int i = 0; i < 16; i += 2) weigh(even, i, w_even);
        if (k0 + T::KEYS < k1) {
            row = locate(k0 + T::KEYS, next_lacking);
            fetch(0, row, 1);
            put(0, 1);
            look_up(k0 + 2 * T::KEYS);
        }
        if constexpr (D == 256) {  // with the sums, where the products read them and nothing else does
#pragma unroll
            for (int c = 0; c < D / 16; ++c) asm volatile("" : "+a"(q[c]));
        }
        int buffer = 0;
        for (int base = k0; base < k1; base += T::KEYS, buffer ^= 1) {
            wait_for_copies();
            asm volatile("" : "+v"(looked_up));  // there now, as far as the compiler's own waits go
            __syncthreads();
            if (__builtin_expect(edge, 0)) clear(base, buffer, lacking);
            const uint32_t was_lacking = lacking;
            lacking = next_lacking;
            next_lacking = (1u << PARTS) - 1;
            if (base + T::KEYS < k1) fetch(1, row, buffer ^ 1);
            if (base + 2 * T::KEYS < k1) {
                row = locate(base + 2 * T::KEYS, next_lacking);
                if (!IN_TURN) fetch(0, row, buffer);
                look_up(base + 3 * T::KEYS);
            }
            asm volatile("" : "+v"(key_at), "+v"(value_at));  // the places along a row are cheaper computed than kept
            const uint32_t here = buffer * 2 * T::BYTES, there = 2 * T::BYTES - here;
            u4 f[AHEAD];
            begin(key_at + there, value_at + here, f);
            raise(uneven, base + 32, was_lacking >> 2, edge, w_even);
            step(key_at + there, value_at + here, f, even, uneven, w_even, w_odd);
            if (IN_TURN && base + T::KEYS < k1) put(1, buffer ^ 1);
            if (IN_TURN && base + 2 * T::KEYS < k1) fetch(0, row, buffer);
            // past the last tile these are scores of whatever lies in LDS, all masked
            edge = lacking != 0 || base + T::KEYS < all_lo || base + 2 * T::KEYS > all_hi;
            begin(key_at + there + 32 * T::ROW, value_at + here + 32 * T::ROW, f);
            raise(even, base + T::KEYS, lacking, edge, w_odd);
            step(key_at + there + 32 * T::ROW, value_at + here + 32 * T::ROW, f, uneven, even, w_odd, w_even);

            if (!IN_TURN && base + T::KEYS < k1) put(1, buffer ^ 1);
            if (base + 2 * T::KEYS < k1) put(0, buffer);
        }
    }

    if (EXACT) odd = __syncthreads_or(odd);
    if (__builtin_expect(odd != 0, 0)) {
        // the values that are not finite reach the rows that see them as infinities (a NaN as both)
        wait_for_copies();
        for (int base = k0; base < k1; base += T::KEYS) {
            look_up(base);
            uint32_t out;
            locate(base, out);
            if (!EXACT && out == 0 && base >= all_lo && base + T::KEYS <= all_hi) continue;
            __syncthreads();
            again(base, 0, out);
            __syncthreads();
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                fx16 plus, minus;
#pragma unroll
                for (int i = 0; i < 16; ++i) plus[i] = minus[i] = 0.0f;
                for (int k = 0; k < T::KEYS / 16; ++k) {
                    const int first = lo - base - 16 * k - 4 * half, end = hi - base - 16 * k - 4 * half;
                    u4 sees;
#pragma unroll
                    for (int p = 0; p < 4; ++p) {
                        const int in = 8 * (p / 2) + 2 * (p % 2);
                        sees[p] = out >> k & 1 ? 0u
                                               : ((in >= first && in < end ? 0xFFFFu : 0u) |
                                                  (in + 1 >= first && in + 1 < end ? 0xFFFF0000u : 0u)) & M::ONES;
                    }
                    const u4 v = value_piece(value_at, t, 16 * k * T::ROW);
                    plus = M::mma32(M::above(v), sees, plus);
                    minus = M::mma32(M::below(v), sees, minus);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (plus[i] > 0.0f) o[t][i] += INFINITY;
                    if (minus[i] > 0.0f) o[t][i] -= INFINITY;
                }
            }
        }
    }
    if (wave0 + n > last) return;
    l = sum_of_halves(l);
    rounded = EXACT ? l : sum_of_halves(rounded);
    const int64_t out = (int64_t)(s.first + token) * a.q_heads + query_head;
    const RowEnd end = row_end(a, s, lo, hi, split);
    if (end == ROW_OUT) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / rounded;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const f4 y = f4{o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]} * inv;
                store4(a.out, out * D + 32 * t + 2 * i + 4 * half, a.out_type, l == 0.0f ? f4{0, 0, 0, 0} : y);
            }
        if (a.lse && half == 0) a.lse[out] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718056f;
    } else if (end == ROW_PART) {
        const int64_t part = (int64_t)split * a.total * a.q_heads + out;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<f4*>(a.part + part * D + 32 * t + 2 * i + 4 * half) =
                    f4{o[t][i], o[t][i + 1], o[t][i + 2], o[t][i + 3]};
        if (half == 0) *reinterpret_cast<float4*>(a.part_ml + 4 * part) = make_float4(m, l, rounded, 0.0f);
    }
}

template <int D>
void launch_types(const AttentionArgs& a, int type, int cache_type, bool exact, dim3 grid, hipStream_t stream) {
    const dim3 block(64 * TILE_WAVES);
    if (cache_type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((tile_attention_kernel<D, _Float16, _Float16, false>), grid, block, 0, stream, a);
    else if (cache_type == IQ4XS_TYPE_BF16)
        hipLaunchKernelGGL((tile_attention_kernel<D, __bf16, __bf16, false>), grid, block, 0, stream, a);
    else if (type == IQ4XS_TYPE_F16 && exact)
        hipLaunchKernelGGL((tile_attention_kernel<D, _Float16, int8_t, true>), grid, block, 0, stream, a);
    else if (type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((tile_attention_kernel<D, _Float16, int8_t, false>), grid, block, 0, stream, a);
    else if (exact)
        hipLaunchKernelGGL((tile_attention_kernel<D, __bf16, int8_t, true>), grid, block, 0, stream, a);
    else
        hipLaunchKernelGGL((tile_attention_kernel<D, __bf16, int8_t, false>), grid, block, 0, stream, a);
}

void launch_tile_attention(const AttentionArgs& a, int head_dim, int type, int cache_type, bool exact, int64_t grid,
                           hipStream_t stream) {
    const dim3 blocks((unsigned)grid);
    if (head_dim == 64)
        launch_types<64>(a, type, cache_type, exact, blocks, stream);
    else if (head_dim == 128)
        launch_types<128>(a, type, cache_type, exact, blocks, stream);
    else
        launch_types<256>(a, type, cache_type, exact, blocks, stream);
}

}  // namespace iq4xs
