// linear_step.hip -- linear attention with a decay for each head, token by token: single tokens and short drafts.
//
//   S <- exp(g) S + k v^T,   o = scale q^T S
//
// Bound by the state's way from memory and back: 8 dk dv bytes for 4 dk dv operations a token.  A wave takes 32 columns
// of a head's state into registers, 4 in each of 8 lanes by dk / 8 rows, so that a row's 32 columns are a whole line of
// 128 bytes; columns do not meet, so waves need no LDS and no barrier.  q and k of the lane's rows and v of its columns are
// fetched a token ahead; what the 8 lanes of a column have of q^T S is added in three exchanges.
// Measured: 64 sequences of 64 heads of 128 x 128, fp32, one token: 99 us, 5.5 TB/s (a large copy 5.1); one sequence 5.0 us
// (5.6 with four waves to a workgroup, 64 of 256 CUs), a chain of dependent loads.
#include "iq4xs_internal.h"
#include "linear_device.h"
#include "linear_launch.h"

namespace iq4xs {

constexpr int STEP_COLUMNS = 32, STEP_WAVES = 4;  // of a workgroup at most

// N consecutive elements as fp32.
template <int N, typename T>
__device__ inline void load_row(const T* p, float (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const f4 w = load4(p + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i + e] = w[e];
    }
}

template <int DK, typename T>
__global__ __launch_bounds__(64 * STEP_WAVES) void linear_step_kernel(LinearArgs a, int dv) {
    constexpr int N = DK / 8;  // rows of a lane
    const int lane = threadIdx.x % 64, column = 4 * (lane % 8), row0 = N * (lane / 8);
    const int tiles = dv / STEP_COLUMNS;
    const int64_t unit = (int64_t)blockIdx.x * (blockDim.x / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    if (unit >= (int64_t)a.seqs * a.heads * tiles) return;
    const int tile = (int)(unit % tiles), head = (int)(unit / tiles % a.heads), seq = (int)(unit / tiles / a.heads);
    const Rows rows = rows_of(a, seq);
    if (rows.count == 0) return;
    const int at = tile * STEP_COLUMNS + column;
    f4 s[N];
    const float* from = state_at(a, a.from_slots, seq, head, DK * dv);
    if (from) {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = load4(from + (row0 + i) * dv + at);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s[i] = f4{0, 0, 0, 0};
    }
    const T* q = static_cast<const T*>(a.q) + (head / a.group) * DK + row0;
    const T* k = static_cast<const T*>(a.k) + (head / a.group) * DK + row0;
    const T* v = static_cast<const T*>(a.v) + head * dv + at;
    float kn[N], qn[N], gn;
    f4 vn;
    auto fetch = [&](int64_t row) {
        load_row<N>(q + row * a.q_stride, qn);
        load_row<N>(k + row * a.k_stride, kn);
        vn = load4(v + row * a.v_stride);
        gn = decay_at(a, row, head);
    };
    fetch(rows.first);
    for (int t = 0; t < rows.count; ++t) {
        const float keep = expf(gn);
        f4 o{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = s[i] * keep + vn * kn[i];
            o += s[i] * qn[i];
        }
        if (t + 1 < rows.count) fetch((int64_t)rows.first + t + 1);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int d = 8; d < 64; d *= 2) o[c] += __shfl_xor(o[c], d);
        if (lane < 8) store4(a.out, ((int64_t)(rows.first + t) * a.heads + head) * dv + at, a.out_type, o * a.scale);
    }
    float* to = state_at(a, a.to_slots, seq, head, DK * dv);
    if (to) {
#pragma unroll
        for (int i = 0; i < N; ++i) *reinterpret_cast<f4*>(to + (row0 + i) * dv + at) = s[i];
    }
}

template <int DK>
static void launch_types(const LinearArgs& a, int dv, int type, dim3 grid, dim3 block, hipStream_t stream) {
    if (type == IQ4XS_TYPE_F32)
        hipLaunchKernelGGL((linear_step_kernel<DK, float>), grid, block, 0, stream, a, dv);
    else if (type == IQ4XS_TYPE_F16)
        hipLaunchKernelGGL((linear_step_kernel<DK, _Float16>), grid, block, 0, stream, a, dv);
    else
        hipLaunchKernelGGL((linear_step_kernel<DK, __bf16>), grid, block, 0, stream, a, dv);
}

void launch_linear_steps(const LinearArgs& a, int dk, int dv, int type, int64_t units, hipStream_t stream) {
    // a wave by itself while that makes no more workgroups than a few to a CU, so that all CUs load
    const int waves = units <= 1024 ? 1 : STEP_WAVES;
    const dim3 blocks((unsigned)((units + waves - 1) / waves)), block(64 * waves);
    if (dk == 64)
        launch_types<64>(a, dv, type, blocks, block, stream);
    else if (dk == 128)
        launch_types<128>(a, dv, type, blocks, block, stream);
    else
        launch_types<256>(a, dv, type, blocks, block, stream);
}

}  // namespace iq4xs
