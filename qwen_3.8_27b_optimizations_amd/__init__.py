"""Python side of the MI355X IQ4_XS mul_mat library.

Loads libiq4xs_mi355x.so (built in this directory by `make`) through ctypes
and exposes the C ABI of include/iq4xs_mi355x.h.  Two layers:

* `Lib` -- one method per extern "C" entry point, raw device pointers (ints)
  and a stream handle; this is the boundary the parity tests call.
* torch helpers (`mul_mat`, `quantize_q8_1`, ...) that take torch tensors on a
  ROCm device, allocate outputs/workspace and pass the current stream.

There is no fallback: if the shared library or a GPU is missing, the calls
raise.  The directory name contains a dot, so load it with
`load_package()` from __graft_entry__ or importlib, not a plain import.
"""
from __future__ import annotations

import ctypes
import os
import struct

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_NAME = "libiq4xs_mi355x.so"
LIB_PATH = os.path.join(HERE, LIB_NAME)

SUCCESS = 0
ERROR_INVALID_VALUE = 1
ERROR_INVALID_CONFIG = 9
ERROR_NOT_SUPPORTED = 801

QK_K = 256
QK8_1 = 32
BLOCK_BYTES = 136
Q8_1_BLOCK_BYTES = 36
GGML_TYPE_IQ4_XS = 23
LAYOUT_KM = 0
LAYOUT_MK = 1
PATH_AUTO = -1
PATH_GEMV = 0
PATH_GEMM = 1
GEMV_MAX_COLS = 8
TYPE_F32 = 0
TYPE_F16 = 1
TYPE_BF16 = 2
TYPE_Q8 = 3
ROPE_HALF = 0
ROPE_INTERLEAVED = 1

# (restype, argtypes) of every exported symbol, in header order
_P = ctypes.c_void_p
_I64 = ctypes.c_int64
_INT = ctypes.c_int
SIGNATURES = {
    "quantize_row_q8_1_gpu": (_INT, [_P, _P, _I64, _P]),
    "quantize_row_q8_1_batched_gpu": (_INT, [_P, _P, _I64, _I64, _P]),
    "gemv_iq4xs_stock_dp4a_gpu": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "gemv_iq4xs_dp4a_coop_gpu": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "gemm_iq4xs_stock_dp4a_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "dequant_iq4xs_gpu": (_INT, [_P, _P, _I64, _INT, _P]),
    "gemv_iq4xs_dp4a_gfx1100_gpu": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "gemv_iq4xs_dp4a_gfx1100_prequantized_gpu": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "gemv_iq4xs_stock_gpu": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "gemm_iq4xs_stock_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemv_iq4xs_gfx1100_gpu": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "gemm_iq4xs_wmma_stream_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemm_iq4xs_wmma_p4_xor_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemm_iq4xs_wmma_64x64_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemm_iq4xs_stream_tiled_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemm_iq4xs_wmma_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemm_iq4xs_tiled_gpu": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "gemm_iq4xs_lut_gpu": (_INT, [_P, _P, _P, _P, _I64, _I64, _I64, _P]),
    "custom_gemv_iq4xs_can_handle": (ctypes.c_bool, [_I64, _I64, _I64, _INT]),
    "custom_gemv_iq4xs_dispatch": (_INT, [_P, _P, _P, _I64, _I64, _P]),
    "custom_gemm_iq4xs_can_handle": (ctypes.c_bool, [_I64, _I64, _I64, _INT]),
    "custom_gemm_iq4xs_dispatch": (_INT, [_P, _P, _P, _I64, _I64, _I64, _P]),
    "iq4xs_workspace_bytes": (ctypes.c_size_t, [_I64, _I64]),
    "iq4xs_quantize_q8_1": (_INT, [_P, _I64, _I64, _INT, _P, ctypes.c_size_t, _P]),
    "iq4xs_mul_mat_q8_1": (_INT, [_P, _P, _P, _I64, _I64, _I64, _INT, _INT, _P]),
    "iq4xs_mul_mat": (_INT, [_P, _P, _P, _I64, _I64, _I64, _INT, _P, ctypes.c_size_t, _P]),
    "iq4xs_mul_mat_noalloc": (_INT, [_P, _P, _P, _I64, _I64, _I64, _INT, _P]),
    "iq4xs_mul_mat_fused": (_INT, [_P, _P, _P, _I64, _I64, _I64, _INT, _P, _P]),
    "iq4xs_mul_mat_q8_1_group": (_INT, [_INT, _P, _P, _P, _P, _I64, _I64, _INT, _P]),
    "iq4xs_rms_norm_q8_1": (_INT, [_P, _P, _P, _P, ctypes.c_float, _I64, _I64, _P, ctypes.c_size_t, _P]),
    "iq4xs_swiglu_q8_1": (_INT, [_P, _P, _I64, _I64, _P, ctypes.c_size_t, _P]),
    "iq4xs_rms_norm_mul_mat_group": (_INT, [_INT, _P, _P, _P, _P, _P, _P, _P, ctypes.c_float, _I64, _P]),
    "iq4xs_rms_norm_mul_mat_swiglu": (_INT, [_P, _P, _I64, _P, _P, _P, _P, ctypes.c_float, _I64, _P, _P, _P, _P]),
    "iq4xs_qk_norm_rope": (_INT, [_P, _P]),
    "iq4xs_qk_norm_rope_append": (_INT, [_P, _P, _P]),
    "iq4xs_kv_gather": (_INT, [_P, _P, _I64, _P, _I64, _P, _P, _I64, _INT, _P]),
    "iq4xs_paged_attention_workspace_bytes": (ctypes.c_size_t, [_P]),
    "iq4xs_paged_attention": (_INT, [_P, _P, ctypes.c_size_t, _P]),
    "iq4xs_q8_1_to_blocks": (_INT, [_P, _P, _I64, _I64, _P]),
    "iq4xs_subblock_sums": (_INT, [_P, _P, _P, _P, _I64, _I64, _I64, _INT, _P]),
    "iq4xs_probe_mfma_i8": (_INT, [_P, _P, _P, _P]),
    "iq4xs_fill_synthetic_weights": (_INT, [_P, _I64, ctypes.c_uint64, _I64, _P]),
    "iq4xs_fill_synthetic_activations": (_INT, [_P, _I64, ctypes.c_uint64, _INT, _P]),
    "iq4xs_version": (ctypes.c_char_p, []),
}


class Iq4xsError(RuntimeError):
    def __init__(self, fn: str, code: int):
        super().__init__(f"{fn} returned hipError {code}")
        self.code = code


class Lib:
    """The C ABI, one attribute per entry point."""

    def __init__(self, path: str = LIB_PATH):
        if not os.path.exists(path):
            raise FileNotFoundError(
                f"{path} is missing: build it with `make -C {HERE}` (or __graft_entry__.build())")
        self.path = path
        self.cdll = ctypes.CDLL(path)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(self.cdll, name)
            fn.restype = res
            fn.argtypes = args
            setattr(self, name, fn)

    def check(self, name: str, *args) -> None:
        code = getattr(self, name)(*args)
        if code != SUCCESS:
            raise Iq4xsError(name, code)


_LIB: Lib | None = None


def lib() -> Lib:
    global _LIB
    if _LIB is None:
        _LIB = Lib()
    return _LIB


# ---------------------------------------------------------------------------
# torch helpers (device memory and streams only)

_TORCH = None  # the module, once a GPU has been seen


def _torch():
    global _TORCH
    if _TORCH is None:
        import torch

        if not torch.cuda.is_available():
            raise RuntimeError("no ROCm GPU visible: the IQ4_XS kernels have no CPU path")
        _TORCH = torch
    return _TORCH


def _stream(torch) -> int:
    # the handle of torch.cuda.current_stream() without building the Stream
    # object: with the availability check made once, 0.4 us of a call's host
    # time against 3.6 (a one-column mul_mat 8.1 -> 5.5 us)
    torch.cuda.init()
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _check_weights(W, K: int, N: int) -> None:
    if W.dtype.itemsize != 1 or W.numel() != N * (K // QK_K) * BLOCK_BYTES or not W.is_contiguous():
        raise ValueError("W must be a contiguous byte tensor of N*(K/256)*136 bytes")


def workspace(K: int, M: int, device=None):
    torch = _torch()
    nbytes = lib().iq4xs_workspace_bytes(K, M)
    if nbytes == 0:
        raise ValueError("bad workspace shape")
    return torch.empty(nbytes, dtype=torch.uint8, device=device or "cuda")


def quantize_q8_1(X, K: int, M: int, layout: int = LAYOUT_MK, ws=None):
    """fp32 activations -> planar Q8_1 workspace (uint8 tensor)."""
    torch = _torch()
    ws = workspace(K, M, X.device) if ws is None else ws
    lib().check("iq4xs_quantize_q8_1", X.data_ptr(), K, M, layout, ws.data_ptr(), ws.numel(), _stream(torch))
    return ws


def rms_norm_q8_1(X, K: int, M: int, residual=None, out_h=None, gamma=None, eps: float = 1e-6, ws=None):
    """h = X (+ residual) -> planar Q8_1 of (h / rms(h)) * gamma.

    out_h receives h when given (it may be X or residual itself: the in-place
    residual add).  Returns the workspace."""
    torch = _torch()
    ws = workspace(K, M, X.device) if ws is None else ws
    ptr = lambda t: None if t is None else t.data_ptr()
    lib().check("iq4xs_rms_norm_q8_1", X.data_ptr(), ptr(residual), ptr(out_h), ptr(gamma), eps, K, M,
                ws.data_ptr(), ws.numel(), _stream(torch))
    return ws


def swiglu_q8_1(G, U, K: int, M: int, ws=None):
    """planar Q8_1 of silu(G) * U; returns the workspace."""
    torch = _torch()
    ws = workspace(K, M, G.device) if ws is None else ws
    lib().check("iq4xs_swiglu_q8_1", G.data_ptr(), U.data_ptr(), K, M, ws.data_ptr(), ws.numel(), _stream(torch))
    return ws


def rms_norm_mul_mat_group(Ws, X, K: int, Ns, residual=None, out_h=None, gamma=None, eps: float = 1e-6, outs=None):
    """RMS norm of one column (h = X + residual, written to out_h) fused into one grouped bs=1 GEMV:
    [W_i * Q8_1((h * scale) * gamma)], bit-identical to rms_norm_q8_1 followed by mul_mat_q8_1_group."""
    torch = _torch()
    n = len(Ws)
    if outs is None:
        outs = [torch.empty(N, dtype=torch.float32, device=X.device) for N in Ns]
    for W, N in zip(Ws, Ns):
        _check_weights(W, K, N)
    wp = (ctypes.c_void_p * n)(*[W.data_ptr() for W in Ws])
    yp = (ctypes.c_void_p * n)(*[y.data_ptr() for y in outs])
    nn = (ctypes.c_int64 * n)(*Ns)
    ptr = lambda t: t.data_ptr() if t is not None else None
    lib().check("iq4xs_rms_norm_mul_mat_group", n, wp, yp, nn, X.data_ptr(), ptr(residual), ptr(out_h), ptr(gamma),
                eps, K, _stream(torch))
    return outs


def rms_norm_mul_mat_swiglu(W_gate, W_up, X, K: int, N: int, residual=None, out_h=None, gamma=None,
                            eps: float = 1e-6, gate_out=None, up_out=None, keep_gate_up: bool = True, out=None):
    """RMS norm + gate/up GEMVs + SwiGLU in one bs=1 launch: returns (S, gate, up) with S = silu(gate) * up
    (fp32, the SwiGLU producer's arithmetic); gate/up bit-identical to rms_norm_mul_mat_group on the pair.
    With keep_gate_up=False gate and up are not written (None is returned for them)."""
    torch = _torch()
    _check_weights(W_gate, K, N)
    _check_weights(W_up, K, N)
    new = lambda: torch.empty(N, dtype=torch.float32, device=X.device)
    S = new() if out is None else out
    g = (new() if gate_out is None else gate_out) if keep_gate_up else None
    u = (new() if up_out is None else up_out) if keep_gate_up else None
    ptr = lambda t: t.data_ptr() if t is not None else None
    lib().check("iq4xs_rms_norm_mul_mat_swiglu", W_gate.data_ptr(), W_up.data_ptr(), N, X.data_ptr(), ptr(residual),
                ptr(out_h), ptr(gamma), eps, K, ptr(g), ptr(u), S.data_ptr(), _stream(torch))
    return S, g, u


def q8_1_blocks(ws, K: int, M: int):
    """Planar workspace -> [M*K/32, 36] uint8 tensor of ggml Q8_1 blocks."""
    torch = _torch()
    out = torch.empty((M * (K // QK8_1), Q8_1_BLOCK_BYTES), dtype=torch.uint8, device=ws.device)
    lib().check("iq4xs_q8_1_to_blocks", ws.data_ptr(), out.data_ptr(), K, M, _stream(torch))
    return out


def mul_mat_q8_1(W, ws, K: int, N: int, M: int, layout: int = LAYOUT_MK, path: int = PATH_AUTO, out=None):
    torch = _torch()
    _check_weights(W, K, N)
    if out is None:
        shape = (M, N) if layout == LAYOUT_MK else (N, M)
        out = torch.empty(shape, dtype=torch.float32, device=W.device)
    lib().check("iq4xs_mul_mat_q8_1", W.data_ptr(), ws.data_ptr(), out.data_ptr(), K, N, M, layout, path,
                _stream(torch))
    return out


def mul_mat_q8_1_group(Ws, ws, K: int, Ns, M: int, layout: int = LAYOUT_MK, outs=None):
    """[W_i * dequant(ws)] for up to 4 matrices sharing the activations, in one launch where one kernel
    takes them all; each output bit-identical to mul_mat_q8_1 on its own matrix."""
    torch = _torch()
    n = len(Ws)
    if not 1 <= n <= 4 or len(Ns) != n:
        raise ValueError("1 to 4 matrices, one N each")
    for W, N in zip(Ws, Ns):
        _check_weights(W, K, N)
    if outs is None:
        outs = [torch.empty((M, N) if layout == LAYOUT_MK else (N, M), dtype=torch.float32, device=Ws[0].device)
                for N in Ns]
    arr_p = ctypes.c_void_p * n
    wp = arr_p(*[W.data_ptr() for W in Ws])
    yp = arr_p(*[Y.data_ptr() for Y in outs])
    nn = (ctypes.c_int64 * n)(*Ns)
    lib().check("iq4xs_mul_mat_q8_1_group", n, wp, yp, nn, ws.data_ptr(), K, M, layout, _stream(torch))
    return outs


def mul_mat(W, X, K: int, N: int, M: int, layout: int = LAYOUT_MK, ws=None, out=None):
    """Y = W * X with X quantised to Q8_1 on the fly (explicit workspace, no allocation in the library)."""
    torch = _torch()
    _check_weights(W, K, N)
    ws = workspace(K, M, W.device) if ws is None else ws
    if out is None:
        shape = (M, N) if layout == LAYOUT_MK else (N, M)
        out = torch.empty(shape, dtype=torch.float32, device=W.device)
    lib().check("iq4xs_mul_mat", W.data_ptr(), X.data_ptr(), out.data_ptr(), K, N, M, layout, ws.data_ptr(),
                ws.numel(), _stream(torch))
    return out


def mul_mat_fused(W, X, K: int, N: int, M: int, layout: int = LAYOUT_MK, out=None, sums: bool = False):
    """Y = W * X for M <= 8 with the Q8_1 quantisation inside the GEMV kernel.

    Raises Iq4xsError with code ERROR_NOT_SUPPORTED when M*K is too large for
    the fused kernel.  With sums=True also returns S[M, N, K/32] (int32)."""
    torch = _torch()
    _check_weights(W, K, N)
    if out is None:
        shape = (M, N) if layout == LAYOUT_MK else (N, M)
        out = torch.empty(shape, dtype=torch.float32, device=W.device)
    S = torch.empty((M, N, K // QK8_1), dtype=torch.int32, device=W.device) if sums else None
    lib().check("iq4xs_mul_mat_fused", W.data_ptr(), X.data_ptr(), out.data_ptr(), K, N, M, layout,
                S.data_ptr() if sums else None, _stream(torch))
    return (out, S) if sums else out


def subblock_sums(W, ws, K: int, N: int, M: int, path: int):
    """(S[M, N, K/32] int32, Y[M, N] fp32) from the production kernel `path`."""
    torch = _torch()
    S = torch.empty((M, N, K // QK8_1), dtype=torch.int32, device=W.device)
    Y = torch.empty((M, N), dtype=torch.float32, device=W.device)
    lib().check("iq4xs_subblock_sums", W.data_ptr(), ws.data_ptr(), S.data_ptr(), Y.data_ptr(), K, N, M, path,
                _stream(torch))
    return S, Y


def dequant(W, n_blocks: int, out=None):
    """IQ4_XS super-blocks -> fp32 weights [n_blocks * 256]."""
    torch = _torch()
    if W.dtype.itemsize != 1 or W.numel() < n_blocks * BLOCK_BYTES:
        raise ValueError("W must hold n_blocks * 136 bytes")
    out = torch.empty(n_blocks * QK_K, dtype=torch.float32, device=W.device) if out is None else out
    lib().check("dequant_iq4xs_gpu", W.data_ptr(), out.data_ptr(), n_blocks, 64, _stream(torch))
    return out


# ---------------------------------------------------------------------------
# the attention half of a layer: argument structs are packed in the header's order

_CACHE = struct.Struct("@PPPPqiiii")
_QK = struct.Struct("@PPPqqqPPPPPPPqiiiiiiif")
_ATTENTION = struct.Struct("@PPPPPPPqqqqqqqiiiif")


_TYPES = {}  # torch dtype -> TYPE_*, filled once a GPU has been seen


def _types(torch):
    if not _TYPES:
        _TYPES.update({torch.float32: TYPE_F32, torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16})
    return _TYPES


def _here(torch, t) -> int:
    """The GPU of a tensor, which must be the current one: the calls launch there.  (A tensor on a GPU says that torch is
    initialised, so the handles below need no checks of their own: 0.3 us of a call's host time against 1.3.)"""
    here = t.get_device()
    if here < 0 or torch._C._cuda_getDevice() != here:
        raise ValueError("tensors must be on the current GPU")
    return here


def _rows(t, name: str):
    """Shape and token stride of [tokens][heads][head] whose heads lie one after another."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head]")
    (tokens, heads, d), (step, between, within) = t.shape, t.stride()
    if within != 1 or (between != d and heads > 1):
        raise ValueError(f"{name}: a token's heads must lie one after another")
    # the stride of a single head or token says nothing
    return tokens, heads, d, step if tokens > 1 else heads * d


def _whole(t, name: str, dtype, shape, here: int) -> int:
    """Address of a contiguous tensor of that type and shape on GPU `here`."""
    if t.dtype != dtype or t.shape != shape or not t.is_contiguous() or t.get_device() != here:
        raise ValueError(f"{name} must be a contiguous {dtype} tensor of shape {list(shape)} on the current GPU")
    return t.data_ptr()


class KVCache:
    """Key and value pages [pages, heads, page, head] in fp16, bf16 or as int8 codes, these with fp16 scales
    [pages, heads, page, head / 32].  Holds the tensors; the calls below read and write them in place.

    page is a power of two of at least 16; head is 64, 128 or 256.  The token at slot s lies in page s // page."""

    def __init__(self, k_pages, v_pages, k_scales=None, v_scales=None):
        torch = _torch()
        if k_pages.dim() != 4:
            raise ValueError("pages must be [pages, heads, page, head]")
        self.pages, self.heads, self.page, self.head_dim = k_pages.shape
        self.type = {torch.float16: TYPE_F16, torch.bfloat16: TYPE_BF16, torch.int8: TYPE_Q8}.get(k_pages.dtype)
        if self.type is None:
            raise ValueError("pages must be float16, bfloat16 or int8")
        if self.head_dim not in (64, 128, 256):
            raise ValueError("head must be 64, 128 or 256")
        if self.page < 16 or self.page & (self.page - 1) or not 0 < self.pages * self.page < 1 << 31:
            raise ValueError("page must be a power of two of at least 16, and the cache hold 1 to 2^31 - 1 tokens")
        self.device = torch.cuda.current_device()
        ptrs = [_whole(t, name, k_pages.dtype, k_pages.shape, self.device)
                for t, name in ((k_pages, "k_pages"), (v_pages, "v_pages"))]
        if (self.type == TYPE_Q8) != (k_scales is not None) or (k_scales is None) != (v_scales is None):
            raise ValueError("int8 pages need k_scales and v_scales, other pages take none")
        if self.type == TYPE_Q8:
            shape = (self.pages, self.heads, self.page, self.head_dim // 32)
            ptrs += [_whole(t, name, torch.float16, shape, self.device)
                     for t, name in ((k_scales, "k_scales"), (v_scales, "v_scales"))]
        else:
            ptrs += [0, 0]
        self.k_pages, self.v_pages, self.k_scales, self.v_scales = k_pages, v_pages, k_scales, v_scales
        self._struct = ctypes.create_string_buffer(
            _CACHE.pack(*ptrs, self.pages, self.heads, self.page, self.head_dim, self.type), _CACHE.size)
        self._address = ctypes.addressof(self._struct)


def _qk(torch, q, k, v, pos, slots, cache, freqs, q_gamma, k_gamma, eps, rope, out_type):
    """Packed arguments and outputs of the two calls below, and their stream."""
    here = _here(torch, q)
    types = _types(torch)
    kind = q.dtype
    out_type = kind if out_type is None else out_type
    if kind not in types or out_type not in types or k.dtype != kind:
        raise ValueError("q and k must have one type and out_type be one: float32, float16 or bfloat16")
    tokens, hq, d, q_stride = _rows(q, "q")
    kt, hk, kd, k_stride = _rows(k, "k")
    if kt != tokens or kd != d or k.get_device() != here:
        raise ValueError("q and k must hold the same tokens and head sizes, on the current GPU")
    if rope not in (ROPE_HALF, ROPE_INTERLEAVED):
        raise ValueError("rope must be ROPE_HALF or ROPE_INTERLEAVED")
    rot = 0 if freqs is None else 2 * freqs.numel()
    if rot > d or rot % 16:
        raise ValueError("freqs must hold a multiple of 8 frequencies, at most one for each two channels")
    fp = _whole(freqs, "freqs", torch.float64, (rot // 2,), here) if rot else 0
    gq = 0 if q_gamma is None else _whole(q_gamma, "q_gamma", torch.float32, (d,), here)
    gk = 0 if k_gamma is None else _whole(k_gamma, "k_gamma", torch.float32, (d,), here)
    q_out = q.new_empty((tokens, hq, d), dtype=out_type)
    k_out, kp, vp, v_stride, sp = None, 0, 0, 0, 0
    if cache is None:
        k_out = q.new_empty((tokens, hk, d), dtype=out_type)
        kp = k_out.data_ptr()
    else:
        if cache.device != here or cache.heads != hk or cache.head_dim != d:
            raise ValueError("the cache must hold k's heads, on the current GPU")
        vt, vh, vd, v_stride = _rows(v, "v")
        if (vt, vh, vd) != (tokens, hk, d) or v.dtype != kind or v.get_device() != here:
            raise ValueError("v must be as k")
        vp, sp = v.data_ptr(), _whole(slots, "slots", torch.int64, (tokens,), here)
    args = _QK.pack(q.data_ptr(), k.data_ptr(), vp, q_stride, k_stride, v_stride,
                    _whole(pos, "pos", torch.int32, (tokens,), here), fp, gq, gk, sp, q_out.data_ptr(), kp, tokens, hq,
                    hk, d, rot, rope, types[kind], types[out_type], eps)
    return args, q_out, k_out, torch._C._cuda_getCurrentRawStream(here)


def qk_norm_rope(q, k, pos, freqs=None, q_gamma=None, k_gamma=None, eps: float = 1e-6, rope: int = ROPE_HALF,
                 out_type=None):
    """RMS norm of each head of q [tokens, q_heads, head] and k [tokens, k_heads, head], then the first
    2 * len(freqs) channels turned by pos * freqs (float64 radians for each position): new q and k in out_type.

    A token's heads lie one after another; tokens may be strided (views of a fused projection)."""
    torch = _torch()
    args, q_out, k_out, stream = _qk(torch, q, k, None, pos, None, None, freqs, q_gamma, k_gamma, eps, rope, out_type)
    lib().check("iq4xs_qk_norm_rope", args, stream)
    return q_out, k_out


def qk_norm_rope_append(q, k, v, pos, slots, cache, freqs=None, q_gamma=None, k_gamma=None, eps: float = 1e-6,
                        rope: int = ROPE_HALF, out_type=None):
    """qk_norm_rope with k and v written to the cache at slots [tokens] (int64; negative or past the cache: the token is
    not stored).  Returns the new q."""
    torch = _torch()
    args, q_out, _, stream = _qk(torch, q, k, v, pos, slots, cache, freqs, q_gamma, k_gamma, eps, rope, out_type)
    lib().check("iq4xs_qk_norm_rope_append", args, cache._address, stream)
    return q_out


def kv_gather(cache, table, starts, total: int, out_type=None):
    """The cached tokens of sequences as dense rows (k, v), each [total, heads, head]: token j of sequence s, at page
    table[s, j // page], is row starts[s] + j.  Rows outside every sequence, and tokens on no page of the cache, are
    zero.  out_type defaults to the cache's, float16 for codes."""
    torch = _torch()
    types = _types(torch)
    if out_type is None:
        out_type = torch.float16 if cache.type == TYPE_Q8 else cache.k_pages.dtype
    if out_type not in types or total < 0:
        raise ValueError("out_type must be float32, float16 or bfloat16, and total not negative")
    here = _here(torch, table)
    seqs = starts.numel() - 1
    width = table.size(1) if table.dim() == 2 else 0
    tp = _whole(table, "table", torch.int32, (seqs, width), here)
    sp = _whole(starts, "starts", torch.int32, (seqs + 1,), here)
    if cache.device != here:
        raise ValueError("the cache must be on the current GPU")
    shape = (total, cache.heads, cache.head_dim)
    k, v = table.new_empty(shape, dtype=out_type), table.new_empty(shape, dtype=out_type)
    lib().check("iq4xs_kv_gather", cache._address, tp, width, sp, seqs, k.data_ptr(), v.data_ptr(), total,
                types[out_type], torch._C._cuda_getCurrentRawStream(here))
    return k, v


def paged_attention(q, cache, table, starts, kv_len, most_q: int, most_kv: int, causal: bool = True, window: int = 0,
                    lse: bool = False, scale: float | None = None, out_type=None):
    """Attention of new tokens q [total, q_heads, head] over the paged cache, which holds their own keys and values too.

    starts [seqs + 1] (int32): first row of each sequence; kv_len [seqs] (int32): its cached tokens, new ones included;
    table [seqs, pages of the longest] (int32).  most_q and most_kv: at least the new and the cached tokens of any
    sequence.  New token i stands at p = kv_len - new + i and sees keys up to p (causal) and after p - window (window >
    0; past every key as good as none).  scale defaults to head ** -0.5, out_type to q's.  Returns out, or (out,
    log-sum-exp of the scores [total, q_heads] in fp32) with lse; a row that sees nothing gives zeros and -inf.  Rows of no
    sequence, and those of a sequence past most_q, are left as they were allocated."""
    torch = _torch()
    here = _here(torch, q)
    types = _types(torch)
    total, hq, d, q_stride = _rows(q, "q")
    out_type = q.dtype if out_type is None else out_type
    kind = types.get(q.dtype, TYPE_F32)
    if kind == TYPE_F32 or (cache.type != TYPE_Q8 and cache.type != kind) or out_type not in types:
        raise ValueError("q must have the cache's type (float16 or bfloat16 for codes), out_type be a float type")
    if d != cache.head_dim or hq % cache.heads or cache.device != here:
        raise ValueError("q must have the cache's head size, a multiple of its heads, and both be on the current GPU")
    seqs = starts.numel() - 1
    width = table.size(1) if table.dim() == 2 else 0
    tp = _whole(table, "table", torch.int32, (seqs, width), here)
    sp = _whole(starts, "starts", torch.int32, (seqs + 1,), here)
    lp = _whole(kv_len, "kv_len", torch.int32, (seqs,), here)
    out = q.new_empty((total, hq, d), dtype=out_type)
    sums = q.new_empty((total, hq), dtype=torch.float32) if lse else None
    args = _ATTENTION.pack(q.data_ptr(), out.data_ptr(), sums.data_ptr() if lse else 0, cache._address, tp, sp, lp,
                           q_stride, width, seqs, total, most_q, most_kv, window, hq, kind, types[out_type],
                           bool(causal), d ** -0.5 if scale is None else scale)
    L = lib()
    nbytes = L.iq4xs_paged_attention_workspace_bytes(args)
    ws = q.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
    L.check("iq4xs_paged_attention", args, ws.data_ptr() if nbytes else 0, nbytes,
            torch._C._cuda_getCurrentRawStream(here))
    return (out, sums) if lse else out


def synthetic_weights(K: int, N: int, seed: int, first_block: int = 0, device=None):
    torch = _torch()
    nblk = N * (K // QK_K)
    W = torch.empty(nblk * BLOCK_BYTES, dtype=torch.uint8, device=device or "cuda")
    lib().check("iq4xs_fill_synthetic_weights", W.data_ptr(), nblk, seed, first_block, _stream(torch))
    return W


def synthetic_activations(n: int, seed: int, outliers: bool = False, device=None):
    torch = _torch()
    x = torch.empty(n, dtype=torch.float32, device=device or "cuda")
    lib().check("iq4xs_fill_synthetic_activations", x.data_ptr(), n, seed, int(outliers), _stream(torch))
    return x
