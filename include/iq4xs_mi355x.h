/*
 * iq4xs_mi355x.h -- C ABI of the MI355X (gfx950) IQ4_XS x Q8_1 mul_mat library
 * (libiq4xs_mi355x.so).
 *
 * Every entry point takes plain device pointers and sizes; `stream` is a
 * hipStream_t passed as void* (NULL = the default stream).  Return values are
 * hipError_t codes as int:
 *   IQ4XS_SUCCESS                 0  hipSuccess
 *   IQ4XS_ERROR_INVALID_VALUE     1  hipErrorInvalidValue  (null pointer, K <= 0,
 *                                    K % 256 != 0, N <= 0, M <= 0, bad layout,
 *                                    workspace too small)
 *   IQ4XS_ERROR_INVALID_CONFIG    9  hipErrorInvalidConfiguration (grid too large)
 *   IQ4XS_ERROR_NOT_SUPPORTED   801  hipErrorNotSupported (e.g. shape not served)
 * or any other hipError_t reported by the runtime.  Arguments are validated
 * before anything is launched; a failing call launches nothing.
 *
 * Reference citations are file:line in the reference repository; "patch"
 * means patches/0001-gfx1100-mul-mat-custom.patch.
 *
 * Data formats (byte-compatible with ggml):
 *   W     : IQ4_XS, row-major [N][K/256] blocks of 136 bytes
 *           (kernels/common/block_iq4_xs.h:10-19)
 *   Q8_1  : 36-byte blocks {uint32 ds = fp16 d | fp16 sum << 16, int8 qs[32]}
 *           (real_stock_dp4a_comparator.hip:22-26); d and sum are encoded with
 *           round-toward-zero as the reference's pack_half2 (:43-62)
 */
#ifndef IQ4XS_MI355X_H
#define IQ4XS_MI355X_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define IQ4XS_SUCCESS 0
#define IQ4XS_ERROR_INVALID_VALUE 1
#define IQ4XS_ERROR_INVALID_CONFIG 9
#define IQ4XS_ERROR_NOT_SUPPORTED 801

#define IQ4XS_QK_K 256
#define IQ4XS_QK8_1 32
#define IQ4XS_BLOCK_BYTES 136
#define IQ4XS_Q8_1_BLOCK_BYTES 36
#define IQ4XS_GGML_TYPE_IQ4_XS 23 /* ggml_type value of GGML_TYPE_IQ4_XS */

/* Activation / output layouts */
#define IQ4XS_LAYOUT_KM 0 /* X[k*M + m], Y[n*M + m]  (standalone kernels/matmul_iq4xs API) */
#define IQ4XS_LAYOUT_MK 1 /* X[m*K + k], Y[m*N + n]  (ggml src1 / dst)                    */

/* Kernel selection for iq4xs_mul_mat_q8_1 / iq4xs_subblock_sums */
#define IQ4XS_PATH_AUTO -1 /* IQ4XS_PATH_GEMV for M <= 8, IQ4XS_PATH_GEMM above */
#define IQ4XS_PATH_GEMV 0  /* streaming GEMV (M <= 8 only)                   */
#define IQ4XS_PATH_GEMM 1  /* matrix-core GEMM (any M); for 8 < M <= 64 the
                            * small-batch matrix-core kernel where it is faster */

/* ===================== standalone API (kernels/matmul_iq4xs) ===================== */

/* Replaces quantize_row_q8_1_gpu, real_stock_dp4a_comparator.hip:266-273.
 * x[K] fp32 -> y[K/32] Q8_1 blocks.  K % 32 == 0. */
int quantize_row_q8_1_gpu(const float* x, void* y, int64_t K, void* stream);

/* Replaces quantize_row_q8_1_batched_gpu, real_stock_dp4a_comparator.hip:308-315.
 * X[k*M + m] -> Y[m*(K/32) + ib].  K % 32 == 0. */
int quantize_row_q8_1_batched_gpu(const float* X, void* Y, int64_t K, int64_t M, void* stream);

/* Replaces gemv_iq4xs_stock_dp4a_gpu, real_stock_dp4a_comparator.hip:480-503:
 * y[N] = W x (x quantised to Q8_1 first).  For K <= 20480 with x 16-byte
 * aligned (K <= 8192 otherwise) the quantisation runs inside the GEMV kernel
 * (one launch, no scratch); otherwise the Q8_1 scratch comes from the
 * library's stream-ordered pool (hipMallocFromPoolAsync/hipFreeAsync on
 * `stream`): no device-wide synchronisation, unlike the reference's
 * hipMalloc/hipFree. */
int gemv_iq4xs_stock_dp4a_gpu(const void* W, const float* x, float* y, int64_t K, int64_t N, void* stream);

/* Replaces the C-linkage gemv_iq4xs_dp4a_coop_gpu, impl_gemv_dp4a_gfx1100.hip:332-341
 * (same contract as gemv_iq4xs_stock_dp4a_gpu). */
int gemv_iq4xs_dp4a_coop_gpu(const void* W, const float* x, float* y, int64_t K, int64_t N, void* stream);

/* Replaces gemv_iq4xs_dp4a_gfx1100_gpu, impl_gemv_dp4a_gfx1100.hip:310-329
 * (same contract as gemv_iq4xs_stock_dp4a_gpu). */
int gemv_iq4xs_dp4a_gfx1100_gpu(const void* W, const float* x, float* y, int64_t K, int64_t N, void* stream);

/* Replaces gemv_iq4xs_dp4a_gfx1100_prequantized_gpu, impl_gemv_dp4a_gfx1100.hip:291-308:
 * y = W * dequant(AQ) for activations already quantised into the reference's
 * 64-byte padded Q8_1 blocks (ds at byte 0, the 32 codes at bytes 16..47;
 * impl_gemv_dp4a_gfx1100.hip:60-66), K/32 of them, 16-byte aligned.  The
 * blocks are copied to a planar workspace from the stream-ordered pool. */
int gemv_iq4xs_dp4a_gfx1100_prequantized_gpu(const void* W, const void* AQ, float* y, int64_t K, int64_t N,
                                             void* stream);

/* Replaces the FP64 comparators gemv_iq4xs_stock_gpu / gemm_iq4xs_stock_gpu,
 * stock_hip_comparator.hip:120-151 (X [K][M], Y [N][M]): per output one double
 * sum of (double)(fp16 d * (ls-32)) * kvalue * (double)x in the loop order of
 * ref_cpu.cpp:12-106, products and sums rounded separately, so the outputs
 * equal the reference's CPU FP64 oracle bit for bit.  One thread per output:
 * a comparator, not a fast path. */
int gemv_iq4xs_stock_gpu(const void* W, const float* x, float* y, int64_t K, int64_t N, void* stream);
int gemm_iq4xs_stock_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M, void* stream);

/* Replaces gemv_iq4xs_gfx1100_gpu, impl_gemv_gfx1100.hip:99-120: the same FP64
 * products, summed as 8 partials per row (one per sub-block index, over all
 * super-blocks) that are then added in index order, as that kernel does. */
int gemv_iq4xs_gfx1100_gpu(const void* W, const float* x, float* y, int64_t K, int64_t N, void* stream);

/* Replace the fp16-WMMA GEMM family and its tiled fallbacks:
 * gemm_iq4xs_wmma_stream_gpu / _wmma_p4_xor_gpu / _wmma_64x64_gpu and
 * gemm_iq4xs_stream_tiled_gpu (impl_gemm_wmma_stream.hip:321-364),
 * gemm_iq4xs_wmma_gpu / gemm_iq4xs_tiled_gpu (impl_gemm_wmma.hip:199-242).
 * Same signature and layout as gemm_iq4xs_stock_dp4a_gpu (X [K][M], Y [N][M]),
 * same argument checks.  They run this library's matrix-core GEMM on Q8_1
 * activations (exact integer sub-block sums, the reference's Q8_1 semantics):
 * the reference's fp16 numerics (dequantised weights x fp16-cast activations)
 * are not reproduced. */
int gemm_iq4xs_wmma_stream_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                               void* stream);
int gemm_iq4xs_wmma_p4_xor_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                               void* stream);
int gemm_iq4xs_wmma_64x64_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                              void* stream);
int gemm_iq4xs_stream_tiled_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                                void* stream);
int gemm_iq4xs_wmma_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M, void* stream);
int gemm_iq4xs_tiled_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M, void* stream);

/* Replaces gemm_iq4xs_lut_gpu, impl_gemm_lut_iq4xs.hip:138-157.  The codebook
 * table LUT is accepted and not read (IQ4_XS fixes it).  Same gate as the
 * reference: hipErrorInvalidConfiguration unless M, N, K are multiples of 16
 * with M >= 512, N >= 32, K >= 32; otherwise as gemm_iq4xs_stock_dp4a_gpu. */
int gemm_iq4xs_lut_gpu(const void* W, const void* LUT, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                       void* stream);

/* Replaces gemm_iq4xs_stock_dp4a_gpu, real_stock_dp4a_comparator.hip:505-548:
 * Y[n*M + m] = sum_k W[n,k] X[k*M + m].  M <= 8 runs the streaming GEMV,
 * larger M the matrix-core GEMM (IQ4XS_PATH_GEMM). */
int gemm_iq4xs_stock_dp4a_gpu(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                              void* stream);

/* Replaces dequant_iq4xs_gpu, kernels/demo_iq4xs_dequant/impl.hip:51-69:
 * n_blocks super-blocks -> 256*n_blocks fp32 weights, bit-identical to the
 * reference's CPU dequantiser (ref_cpu.cpp:6-27).  warp_size is accepted for
 * signature compatibility (32 or 64, anything else is hipErrorInvalidValue);
 * the kernel always runs wave64.  n_blocks == 0 launches nothing and succeeds. */
int dequant_iq4xs_gpu(const void* src, float* dst, int64_t n_blocks, int warp_size, void* stream);

/* ============================ ggml mul_mat boundary ============================ */

/* Replaces custom_gemv_iq4xs_can_handle, patch:274-277.  True for
 * type == GGML_TYPE_IQ4_XS, M == 1 (custom_gemv_iq4xs_dispatch computes one
 * column), K > 0, K % 256 == 0, N > 0 (the reference's K/N whitelist is
 * dropped).  Batches of 2..8 columns are served by custom_gemm_iq4xs_dispatch,
 * which routes them to the small-batch GEMV. */
bool custom_gemv_iq4xs_can_handle(int64_t K, int64_t N, int64_t M, int type);

/* Replaces custom_gemv_iq4xs_dispatch, patch:278-280 (called from the mmvq.cu
 * hook, patch:327-334): y[N] = W x for ggml's src0/src1/dst of one column.
 * Stream-ordered; no host synchronisation (the reference synchronises the
 * stream and refuses graph capture, patch:269-272). */
int custom_gemv_iq4xs_dispatch(const void* W, const float* x, float* y, int64_t K, int64_t N, void* stream);

/* Replaces custom_gemm_iq4xs_can_handle, patch:148-151: type == IQ4_XS,
 * M >= 1, K > 0, K % 256 == 0, N > 0. */
bool custom_gemm_iq4xs_can_handle(int64_t K, int64_t N, int64_t M, int type);

/* Replaces custom_gemm_iq4xs_dispatch, patch:152-154 (mmq.cu hook,
 * patch:299-306): ggml layout X[m*K + k] -> Y[m*N + n]. */
int custom_gemm_iq4xs_dispatch(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M,
                               void* stream);

/* ====================== explicit-workspace API (capture-safe) ======================
 * No counterpart in the reference (which allocates per call, e.g.
 * real_stock_dp4a_comparator.hip:491,501).  For callers that own their memory:
 * the calls below allocate nothing and never synchronise.  The workspace holds
 * Q8_1 activations in planar form: int8 codes [M][K] at offset 0, then the
 * uint32 ds words [M][K/32], then the same codes as fp16 pairs [M][K/32][16]
 * (uint32 word p of a 32-element block = elements p and p + 16), each part at
 * a 256-byte aligned offset: 3 * K * M + K * M / 8 bytes and padding.  Every
 * call that writes a workspace fills all three parts. */

/* Bytes of workspace for M activation columns of length K; 0 for shapes the
 * entry points refuse (K not a positive multiple of 32, M < 1, K or M >= 2^31). */
size_t iq4xs_workspace_bytes(int64_t K, int64_t M);

/* X (layout IQ4XS_LAYOUT_KM or _MK) -> planar Q8_1 in ws. */
int iq4xs_quantize_q8_1(const float* X, int64_t K, int64_t M, int layout, void* ws, size_t ws_bytes,
                        void* stream);

/* Fused producers: the op that writes a mul_mat activation, quantised to
 * planar Q8_1 in ws on the way out (row-major inputs, row m at [m*K]).  They
 * stand for ggml's RMS_NORM + MUL and SWIGLU ahead of the projections
 * (profiled by the reference at benchmarks/profiling/BOTTLENECK-TABLE.md:
 * 24,26,30) and have no kernel counterpart in the reference.  K % 32 == 0.
 *
 * rms norm: h = X + R (R may be NULL), written to H when H is non-NULL
 * (H may be exactly X or R: the in-place residual add); then
 *   mean = (float)(sum (double)(h*h) / K), scale = 1.0f / sqrtf(mean + eps),
 *   y = (h * scale) * gamma[k]       (gamma NULL: y = h * scale)
 * with the sum in a fixed order, so results are reproducible bit for bit.
 * The Qwen-27B-class models use eps = 1e-6
 * (benchmarks/environment/startup-log.txt:128).  X, R, H 16-byte aligned. */
int iq4xs_rms_norm_q8_1(const float* X, const float* R, float* H, const float* gamma, float eps, int64_t K,
                        int64_t M, void* ws, size_t ws_bytes, void* stream);

/* swiglu: y = silu(G) * U, silu(g) = g / (1 + exp(-g)) (exp computed by the
 * library's own Cody-Waite reduction, <= 1 ulp). */
int iq4xs_swiglu_q8_1(const float* G, const float* U, int64_t K, int64_t M, void* ws, size_t ws_bytes,
                      void* stream);

/* RMS norm fused into a grouped bs=1 GEMV: the same result as
 * iq4xs_rms_norm_q8_1(X, R, H, gamma, eps, K, 1, ws) followed by
 * iq4xs_mul_mat_q8_1_group(count, W, Y, N, ws, K, 1, ...) -- Y and H bit for
 * bit -- in one launch and with no workspace: every workgroup of the GEMV
 * runs the norm's passes on the row and quantises it into its own LDS, and
 * workgroup 0 writes H.  For the norm ahead of q/k/v or gate/up at decode.
 * No counterpart in the reference, which runs RMS_NORM, MUL and each
 * projection as separate ggml ops.
 *   - H (may be NULL) must not overlap X or R, and no Y[i] may overlap X, R or H
 *     (in-place forms are rejected with hipErrorInvalidValue);
 *   - X, R, H, gamma 16-byte aligned; K % 256 == 0, eps >= 0;
 *   - hipErrorNotSupported for K < 2048 or K > 8192, or when the row does not
 *     fit the kernel's LDS: use the two calls. */
int iq4xs_rms_norm_mul_mat_group(int count, const void* const* W, float* const* Y, const int64_t* N, const float* X,
                                 const float* R, float* H, const float* gamma, float eps, int64_t K, void* stream);

/* RMS norm, the gate/up pair of a SwiGLU MLP and the SwiGLU itself in one bs=1
 * launch: the same h, gate and up as iq4xs_rms_norm_mul_mat_group(2,
 * {W_gate, W_up}, {Y_gate, Y_up}, {N, N}, X, R, H, gamma, eps, K) -- bit for
 * bit -- and S[n] = silu(gate[n]) * up[n] in fp32 with iq4xs_swiglu_q8_1's
 * arithmetic, so iq4xs_mul_mat(W_down, S, ...) gives the bits of the SwiGLU
 * producer followed by the down GEMV, one launch earlier.  Each workgroup
 * owns the same rows of gate and up.  No counterpart in the reference, which
 * runs RMS_NORM, MUL, the two projections and SWIGLU as separate ggml ops.
 *   - Y_gate, Y_up may be NULL (not written); S must not be NULL;
 *   - H (may be NULL) must not overlap X or R; Y_gate, Y_up and S must not
 *     overlap X, R, H or each other;
 *   - X, R, H, gamma 16-byte aligned; K % 256 == 0, eps >= 0;
 *   - hipErrorNotSupported as iq4xs_rms_norm_mul_mat_group, or when N has no
 *     divisor that makes every workgroup's rows whole steps: use the group
 *     call and iq4xs_swiglu_q8_1. */
int iq4xs_rms_norm_mul_mat_swiglu(const void* W_gate, const void* W_up, int64_t N, const float* X, const float* R,
                                  float* H, const float* gamma, float eps, int64_t K, float* Y_gate, float* Y_up,
                                  float* S, void* stream);

/* Y = W * dequant(ws) from an already quantised workspace; `layout` selects
 * the Y layout; `path` is one of IQ4XS_PATH_*.  The same call gives the same
 * bits every time.  The order in which a row's fp32 terms are added depends on
 * N, K and M: above 64 columns it is one order for every M, below that it
 * changes with the kernel and its split (by steps of 8 columns), so a column's
 * last bits can differ between batch sizes. */
int iq4xs_mul_mat_q8_1(const void* W, const void* ws, float* Y, int64_t K, int64_t N, int64_t M, int layout,
                       int path, void* stream);

/* Several weight matrices (1 <= count <= 4, each N[i] x K) against the same
 * quantised activations in ws: Y[i] = W[i] * dequant(ws), Y[i] laid out as
 * `layout` selects.  For M <= 8 one launch of the streaming GEMV covers
 * every matrix (q/k/v, gate/up of a decode step) and pays the per-launch
 * fixed cost once; the matrices that take the small-batch matrix-core kernel
 * (M >= 4 and N >= 2048, or M == 8 and N >= 1024) share its launches, the
 * others one launch of the streaming GEMV.  For M > 8 the matrices share one
 * GEMM launch, whose small matrices fill the CUs that the big ones' last round
 * of tiles leaves idle, and up to 64 columns those that the small-batch kernel
 * takes (a rule on N, K and M) share its launches instead.  That kernel has
 * one launch per way of splitting K, which follows N, K and M: q/k/v and
 * gate/up are one.  A group with matrices of both kernels pays a launch for
 * each, and the narrow ones do not fill the wide ones' idle CUs: with q above
 * 8192 rows, k and v beside it cost up to 40 % more than in one GEMM launch
 * (12288 + 1536 + 1536 rows, K = 6144, M = 64: 54 against 40 us).  Each output
 * is bit-identical to iq4xs_mul_mat_q8_1 (path AUTO) on its own matrix.  W, Y,
 * N are host arrays of count entries.  No counterpart in the reference, which
 * runs every projection as its own mul_mat. */
int iq4xs_mul_mat_q8_1_group(int count, const void* const* W, float* const* Y, const int64_t* N, const void* ws,
                             int64_t K, int64_t M, int layout, void* stream);

/* Quantise + multiply in one call.  For M == 1 and K <= 20480 with X 16-byte
 * aligned (K <= 8192 otherwise) the quantisation runs inside the GEMV kernel
 * and ws is not written (it is still validated). */
int iq4xs_mul_mat(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M, int layout, void* ws,
                  size_t ws_bytes, void* stream);

/* Largest Q8_1 workspace (iq4xs_workspace_bytes(K, M)) iq4xs_mul_mat_noalloc
 * serves: 128 MiB, e.g. M <= 2460 at K = 17408, M <= 8380 at K = 5120. */
#define IQ4XS_NOALLOC_SCRATCH_BYTES (128u << 20)

/* iq4xs_mul_mat without a workspace argument and without any allocation: the
 * Q8_1 workspace is a static device array of IQ4XS_NOALLOC_SCRATCH_BYTES held
 * by the library (one per GPU, for the life of the process).  The array is part
 * of the library's code object, so every process that runs any kernel of this
 * library on a GPU holds those 128 MiB of that GPU's memory, whether or not it
 * ever calls iq4xs_mul_mat_noalloc.  No counterpart
 * in the reference; for callers that cannot allocate -- code under HIP graph
 * capture, tight serving loops, harnesses that forbid hipMalloc.  Same results
 * as iq4xs_mul_mat bit for bit.  IQ4XS_ERROR_INVALID_VALUE when
 * iq4xs_workspace_bytes(K, M) exceeds IQ4XS_NOALLOC_SCRATCH_BYTES.  Every call
 * on one GPU shares that GPU's scratch: calls that overlap on one GPU (other
 * streams, other host threads) race; serialise them. */
int iq4xs_mul_mat_noalloc(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M, int layout,
                          void* stream);

/* Small-batch (1 <= M <= 8) multiply that quantises X to Q8_1 inside the GEMV
 * kernel (one launch, no workspace).  Same Q8_1 codes and sums as
 * iq4xs_quantize_q8_1 + iq4xs_mul_mat_q8_1.  Returns IQ4XS_ERROR_NOT_SUPPORTED
 * when M*K does not fit the kernel's on-chip activation buffer; the caller then
 * uses the two-step path.  S (may be NULL) receives the per-sub-block int32
 * sums exactly as iq4xs_subblock_sums lays them out. */
int iq4xs_mul_mat_fused(const void* W, const float* X, float* Y, int64_t K, int64_t N, int64_t M, int layout,
                        int32_t* S, void* stream);

/* ===================== the attention half of a layer =====================
 * What runs between the q/k/v projections and o (examples/attention_block.py
 * runs them together): norm and position rotation of
 * queries and keys, a paged key/value cache, and attention over it.  No
 * counterpart in the reference, which leaves these ops to stock ggml.  The
 * calls allocate nothing, never synchronise and may be captured.
 * head_dim is 64, 128 or 256 (IQ4XS_ERROR_NOT_SUPPORTED otherwise); every
 * pointer is 16-byte aligned; token strides are in elements and multiples of 8,
 * a token's heads lie one after another. */

/* Element types */
#define IQ4XS_TYPE_F32 0
#define IQ4XS_TYPE_F16 1
#define IQ4XS_TYPE_BF16 2
#define IQ4XS_TYPE_Q8 3 /* int8 codes, one fp16 scale for each 32 channels; caches only */

/* Which channels turn together: i and i + rot/2, or 2i and 2i + 1 */
#define IQ4XS_ROPE_HALF 0
#define IQ4XS_ROPE_INTERLEAVED 1

/* Key and value pages [pages][heads][page][head_dim] and, for IQ4XS_TYPE_Q8,
 * their scales [pages][heads][page][head_dim/32] (NULL otherwise).  page, the
 * tokens of a page, is a power of two of at least 16; pages * page < 2^31.  The
 * token at slot s lies in page s / page at s % page. */
struct iq4xs_kv_cache {
    void* k;
    void* v;
    void* k_scales;
    void* v_scales;
    int64_t pages;
    int32_t heads;
    int32_t page;
    int32_t head_dim;
    int32_t type; /* IQ4XS_TYPE_F16, _BF16 or _Q8 */
};

struct iq4xs_qk_norm_rope_args {
    const void* q; /* [tokens][q_heads][head_dim], in_type */
    const void* k; /* [tokens][k_heads][head_dim], in_type */
    const void* v; /* as k; iq4xs_qk_norm_rope_append only */
    int64_t q_stride, k_stride, v_stride;
    const int32_t* pos;   /* [tokens] */
    const double* freqs;  /* [rot/2] radians for each position (scaling for long contexts included) */
    const float* q_gamma; /* [head_dim], or NULL */
    const float* k_gamma;
    const int64_t* slots; /* [tokens]; iq4xs_qk_norm_rope_append only */
    void* q_out;          /* [tokens][q_heads][head_dim], out_type */
    void* k_out;          /* as k; iq4xs_qk_norm_rope only */
    int64_t tokens;
    int32_t q_heads, k_heads, head_dim;
    int32_t rot;  /* channels that turn: a multiple of 16, 0 to head_dim */
    int32_t rope; /* IQ4XS_ROPE_* */
    int32_t in_type, out_type;
    float eps;
};

/* For each head of q and k: y = x * rsqrt(mean(x^2) + eps) * gamma, then the
 * first rot channels turned: (a, b) -> (a cos t - b sin t, b cos t + a sin t)
 * with t = pos * freqs[i] for pair i.  fp32 throughout (t in 64 bits), rounded
 * once.  tokens == 0 launches nothing. */
int iq4xs_qk_norm_rope(const struct iq4xs_qk_norm_rope_args* args, void* stream);

/* The same, with k and v (v as it is) written to the cache at slots; a token
 * whose slot is negative or past the cache is not stored.  Two tokens of a call
 * must not share a slot.  IQ4XS_TYPE_Q8: for each 32 channels
 * d = fp16(min(amax / 127, 65504 / 127)), at most 515.5 where fp16 holds amax (127
 * times the next one, 516, is past it), codes = rint(x / d) within +-127; a NaN
 * makes its group's scale NaN. */
int iq4xs_qk_norm_rope_append(const struct iq4xs_qk_norm_rope_args* args, const struct iq4xs_kv_cache* cache,
                              void* stream);

/* Cached tokens as dense rows: row starts[s] + j of k_out and v_out
 * [total][heads][head_dim] (out_type) is token j of sequence s, at page
 * table[s * table_width + j / page].  starts has seqs + 1 entries that never
 * fall.  Rows outside every sequence, and those whose page is past the table or
 * not in the cache, are zero.  Every element of the cache is read as stored,
 * rounded once where out_type is narrower. */
int iq4xs_kv_gather(const struct iq4xs_kv_cache* cache, const int32_t* table, int64_t table_width,
                    const int32_t* starts, int64_t seqs, void* k_out, void* v_out, int64_t total, int out_type,
                    void* stream);

struct iq4xs_paged_attention_args {
    const void* q; /* [total][q_heads][head_dim]; the cache's type, or F16/BF16 for a Q8 cache */
    void* out;     /* [total][q_heads][head_dim], out_type */
    float* lse;    /* [total][q_heads], or NULL */
    const struct iq4xs_kv_cache* cache;
    const int32_t* table;  /* [seqs][table_width] pages of each sequence; entries past its tokens are not read */
    const int32_t* starts; /* [seqs + 1] first row of each sequence in q, never falling, the last at most total */
    const int32_t* kv_len; /* [seqs] cached tokens, the new ones among them */
    int64_t q_stride, table_width, seqs, total;
    int64_t most_q, most_kv; /* at least the new and the cached tokens of any sequence */
    int64_t window;          /* 0: none */
    int32_t q_heads;         /* a multiple of the cache's heads: head h reads cache head h / (q_heads / heads) */
    int32_t type;            /* of q */
    int32_t out_type;        /* F32, F16 or BF16 */
    int32_t causal;
    float scale;
};

/* Bytes of workspace iq4xs_paged_attention needs; 0 also for arguments it refuses
 * (IQ4XS_ERROR_INVALID_CONFIG: total * q_heads, or its workgroups, past 2^31 - 1). */
size_t iq4xs_paged_attention_workspace_bytes(const struct iq4xs_paged_attention_args* args);

/* out = softmax(scale * q k^T over the visible keys) v, lse = log(sum(exp(scale
 * * q k^T))) (natural).  New token i of a sequence stands at p = kv_len - new + i
 * and sees key j < kv_len if j <= p (causal) and j > p - window (window > 0).  A
 * row that sees nothing gives zeros and -Inf.  Keys and values that a row does
 * not see (and all that lies past kv_len) do not reach it, whatever they hold.
 * Scores, statistics and sums are fp32.  For their product with the values,
 * weights are rounded to the cache's 16-bit type (fp16 ones to 2^-32 of the row's
 * largest below 2^-21 of it); the sum they are divided by is that of the rounded
 * ones.  A Q8 cache: values become fp16 (codes times scale past its range an
 * infinity, of the rows that see them), BF16 queries too, with a power of two taken
 * out of each row; keys are exact and weights two fp16 numbers, high and rest.  Only
 * where nothing but BF16 outputs is asked for, of more than 32 rows of a cache head
 * (new tokens times q_heads / heads), keys become fp16, within its range, and weights
 * are one.
 * Tokens on a page that is not in the cache are as masked ones.  Where kv_len is
 * above most_kv, the table or 2^31 - 4096, the first keys count.  A sequence of more
 * new tokens than most_q has its first most_q rows computed, at the places that
 * starts gives them; rows past most_q, and those of no sequence, are not written.
 * The same call gives the same bits. */
int iq4xs_paged_attention(const struct iq4xs_paged_attention_args* args, void* ws, size_t ws_bytes, void* stream);

/* The same with first tokens that stay visible beside the window: new token i also
 * sees key j < sinks (if j <= p, causal).  With no window, or one that hides nothing,
 * sinks change nothing.  The workspace is that of the call without them.  Any number
 * of them is right; one workgroup of a row goes through them all, so that many
 * thousands are slow. */
int iq4xs_paged_attention_sinks(const struct iq4xs_paged_attention_args* args, int64_t sinks, void* ws, size_t ws_bytes,
                                void* stream);

/* Whether shared tokens are gone through once for a group or again for each sequence: AUTO
 * takes what is faster (once for few rows of each sequence over much that is shared). */
#define IQ4XS_SHARED_AUTO 0
#define IQ4XS_SHARED_ONCE 1
#define IQ4XS_SHARED_EACH 2

/* Sequences that begin with the same tokens, on the same pages. */
struct iq4xs_shared_prefix {
    const int32_t* first; /* [groups + 1] first sequence of each group, never falling; NULL: one group of all */
    const int32_t* len;   /* [groups] tokens that the sequences of a group share */
    int64_t groups;
    int64_t most_len;  /* at least the shared tokens of any group, and 1 */
    int64_t most_rows; /* at least the new tokens of a group's sequences together */
    int32_t path;      /* IQ4XS_SHARED_* */
};

/* Bytes of workspace iq4xs_shared_attention needs; 0 also for arguments it refuses. */
size_t iq4xs_shared_attention_workspace_bytes(const struct iq4xs_paged_attention_args* args,
                                              const struct iq4xs_shared_prefix* prefix);

/* iq4xs_paged_attention of a batch whose sequences begin with the same tokens, those
 * read and multiplied once for the rows of all of a group's sequences.  Tables and
 * kv_len are as there, the shared tokens among them: any number of them, with or without
 * the end of a page, of which every table of a group holds the same keys and values (as
 * the same pages do); they are read through one table or another.  A sequence of no group
 * shares none.  args->most_kv is at least the cached tokens of any sequence after its
 * shared ones; args->window is 0 (NOT_SUPPORTED otherwise: a window's calls read little
 * of a prefix).  New tokens come after the shared ones (kv_len - new >= len); what a row
 * before their end sees of them is not specified.  Where len is above most_len, the rest
 * of the shared keys are a sequence's own; rows of a group past most_rows may be left
 * unwritten.  Once, an 8-bit cache's keys of the prefix are rounded as there, by
 * most_rows. */
int iq4xs_shared_attention(const struct iq4xs_paged_attention_args* args, const struct iq4xs_shared_prefix* prefix,
                           void* ws, size_t ws_bytes, void* stream);

/* ================= layers that keep a state in place of a cache =================
 * Linear attention with a decay for each head.  The same conventions as above. */

struct iq4xs_linear_attention_args {
    const void* q;      /* [total][qk_heads][dk], in_type */
    const void* k;      /* as q */
    const void* v;      /* [total][heads][dv], in_type */
    const float* decay; /* natural logarithms: [heads] (decay_stride 0) or [total][heads] */
    const int32_t* starts;     /* [seqs + 1] first row of each sequence, never falling, the last at most total */
    float* states;             /* [slots][heads][dk][dv], or NULL */
    const int64_t* from_slots; /* [seqs] states that sequences go on from, or NULL: all begin at zeros */
    const int64_t* to_slots;   /* [seqs] where their states are left, or NULL: nowhere */
    void* out;                 /* [total][heads][dv], out_type; not the memory of an input */
    int64_t q_stride, k_stride, v_stride, decay_stride; /* of a token, in elements: below 2^23 */
    int64_t slots, seqs, total;
    int64_t most_q; /* at least the tokens of any sequence */
    int32_t heads;  /* a multiple of qk_heads: head h reads q and k of head h / (heads / qk_heads) */
    int32_t qk_heads;
    int32_t dk, dv; /* 64, 128 or 256 each (NOT_SUPPORTED otherwise) */
    int32_t in_type, out_type;
    float scale;
};

/* Bytes of workspace iq4xs_linear_attention needs; 0 also for arguments it refuses
 * (IQ4XS_ERROR_INVALID_CONFIG: launches of more than 2^31 - 1 workgroups). */
size_t iq4xs_linear_attention_workspace_bytes(const struct iq4xs_linear_attention_args* args);

/* Token by token, for each head, from S_0 = the state at from_slots (zeros where the
 * slot is negative or past the states):
 *   S_t = exp(decay_t) S_{t-1} + k_t v_t^T,   o_t = scale q_t^T S_t,
 * and the last S_t goes to to_slots (nowhere where that slot is negative or past the
 * states).  A sequence of no tokens leaves its states as they are.  States and sums are
 * fp32; products of many tokens go through matrix units as sums of 16-bit parts that
 * keep 24 bits of states, updates and fp32 inputs (16 of what makes 16-bit outputs).
 * Sums of products with a query are taken before the decays of up to 31 tokens: with
 * the state that far back and with those tokens' keys they have to fit fp32 as well.
 * Decays above 0 let states grow: within 32 tokens, by less than 2^127.
 * Two sequences must not have one to_slot, nor one's to_slot be another's from_slot;
 * a sequence's own two may be one, and several may begin at one state.
 * A sequence of more than most_q tokens is cut to its first most_q; rows past them and
 * those of no sequence are not written.  What is not finite in a token reaches the
 * outputs and states of its head from that token on (of v, its channel's), as infinities
 * or NaN; others keep their bits.  Decays are taken as -200 at least, exp of which is nothing
 * beside any fp32 number.  The same call gives the same bits. */
int iq4xs_linear_attention(const struct iq4xs_linear_attention_args* args, void* ws, size_t ws_bytes, void* stream);

/* ================================ debug exports ================================
 * No counterpart in the reference; they exist so the Q8_1 blocks and the
 * per-32-element int32 sums can be checked bit for bit. */

/* Planar workspace -> M*(K/32) 36-byte Q8_1 blocks (block (m, ib) at m*(K/32)+ib). */
int iq4xs_q8_1_to_blocks(const void* ws, void* blocks, int64_t K, int64_t M, void* stream);

/* S[(m*N + n)*(K/32) + kb] = sumi * (ls - 32) of sub-block kb, row n, column m,
 * computed by the production kernel selected by `path` (IQ4XS_PATH_GEMV or
 * _GEMM: the same device code as iq4xs_mul_mat_q8_1, with one extra store).
 * The kernel also writes its outputs to Y (M*N floats, layout IQ4XS_LAYOUT_MK). */
int iq4xs_subblock_sums(const void* W, const void* ws, int32_t* S, float* Y, int64_t K, int64_t N, int64_t M,
                        int path, void* stream);

/* One v_mfma_i32_32x32x32_i8 through the operand and result layouts that the
 * small-batch matrix-core GEMV relies on: C[i*32 + j] = sum_k A[i*32 + k] * B[j*32 + k]. */
int iq4xs_probe_mfma_i8(const int8_t* A, const int8_t* B, int32_t* C, void* stream);

/* ============================ synthetic inputs ============================ */

/* n_blocks IQ4_XS blocks made on the device from `seed` (block i is the
 * recipe's block first_block + i). */
int iq4xs_fill_synthetic_weights(void* W, int64_t n_blocks, uint64_t seed, int64_t first_block, void* stream);

/* n fp32 activations ~ N(0,1); outliers != 0 scales 1 % of them x20. */
int iq4xs_fill_synthetic_activations(float* x, int64_t n, uint64_t seed, int outliers, void* stream);

/* Library version string. */
const char* iq4xs_version(void);

#ifdef __cplusplus
}
#endif
#endif
