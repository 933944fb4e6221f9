"""Tensor-level wrappers of the gfx950 kernels (C ABI in include/forgeserve_amd.h).

Each function checks shapes on the host, allocates outputs and workspace with torch's caching
allocator, and launches on torch's current stream. Inputs must already be on the GPU; nothing here
computes on the CPU.

gemm, paged_attention and the acceptance keep one scratch buffer per device from call to call: their calls on several
streams at once are for the caller to order. gemm_e4m3 and the sampling calls take scratch of their own each time.
"""

import math
from typing import Optional, Tuple

import torch

from . import _lib
from ._lib import DTYPE_CODE, STORE_E4M3, KVLayout, check, ptr, require_device, stream_ptr

I32 = torch.int32

def _dt(t: torch.Tensor) -> int:
    try:
        return DTYPE_CODE[t.dtype]
    except KeyError:
        raise ValueError(f"unsupported dtype {t.dtype} (float32, bfloat16, float16)") from None


def _ws(nbytes: int, device) -> torch.Tensor:
    return torch.empty(max(int(nbytes), 256), dtype=torch.uint8, device=device)


_PERSISTENT = {}
_RETIRED = []   # outgrown scratch buffers: a captured HIP graph may still hold their addresses


def _persistent_ws(name: str, nbytes: int, device) -> torch.Tensor:
    """A per-device scratch buffer reused across calls (calls on one stream are ordered, so consecutive
    users never overlap); grown when a call needs more. An outgrown buffer is kept
    alive for the life of the process, since graphs captured earlier launch kernels on it."""
    key = (name, torch.device(device))
    ws = _PERSISTENT.get(key)
    if ws is None or ws.numel() < nbytes:
        if ws is not None:
            _RETIRED.append(ws)
        ws = torch.empty(max(int(nbytes * 1.25), 1 << 20), dtype=torch.uint8, device=key[1])
        _PERSISTENT[key] = ws
    return ws


def _rows(t: torch.Tensor) -> Tuple[int, int]:
    """(rows, row stride) of a 2-D tensor whose last dim is contiguous."""
    if t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"expected a 2-D tensor with a contiguous last dim, got {tuple(t.shape)} {t.stride()}")
    return t.shape[0], t.stride(0)


# ------------------------------------------------------------------------------------------------
# KV pool layout
# ------------------------------------------------------------------------------------------------
def kv_layout(k: torch.Tensor, v: torch.Tensor) -> KVLayout:
    """Layout of one layer: v is a (num_blocks, n_kv_heads, block_size, head_dim) view (any strides); k
    is the same, or (num_blocks, n_kv_heads, block_size, head_dim // 8, 8) with unit stride inside a
    group for keys stored as 8-dim groups (fs_kv_layout.k_group)."""
    if k.dim() == 5 and k.shape[-1] == 8 and k.stride(-1) == 1:
        kb, kh, ks, kg, _ = k.stride()
        k_strides, k_group, kshape = (kb, kh, ks, 1), kg, (*k.shape[:3], 8 * k.shape[3])
    elif k.dim() == 4:
        k_strides, k_group, kshape = k.stride(), 0, tuple(k.shape)
    else:
        raise ValueError(f"k pool view must be 4-D or grouped 5-D (..., head_dim // 8, 8): {tuple(k.shape)}")
    if kshape != tuple(v.shape) or v.dim() != 4 or k.dtype != v.dtype:
        raise ValueError(f"k/v pool views must match: {tuple(k.shape)} vs {tuple(v.shape)}")
    nb, h, bs, d = v.shape
    return KVLayout(k.data_ptr(), v.data_ptr(), *k_strides, *v.stride(), bs, h, d, _dt(k), nb, k_group)


def kv_layout_e4m3(k: torch.Tensor, v: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> KVLayout:
    """Layout of one layer whose keys and values are 8-bit floating point (e4m3 codes, torch.float8_e4m3fn or
    uint8) with one power of two per token, KV head and side as their scale. Every call that takes a layout takes
    this one: the writes encode rows of `dtype`, the gather and the attention decode, with queries and outputs of
    `dtype` (float32, bfloat16, float16).

    k: (num_blocks, n_kv_heads, head_dim // 16, block_size, 16); v: (num_blocks, n_kv_heads, block_size // 4,
    head_dim, 4), the dims of each 64 (or what is left of them) ordered by d % 16 first; scales: uint8
    (num_blocks, n_kv_heads, 2, block_size), the exponent bytes e of the keys', then of the values' scales
    2^(e - 127). The blocks and heads may have any strides; a tile, and a pair of scale rows, is contiguous.
    head_dim is a multiple of 16 and at most 256, block_size a multiple of 4. The scale is the smallest power of
    two that brings a group's largest magnitude to 448 or less (fs_kv_layout says what lies beyond the limits).
    Attention is fast for bfloat16 and float16 with head_dim 64 or 128 and block_size % 16 == 0. A write call
    names a slot once: of two tokens for the same one a mixture may remain."""
    if any(t.dtype not in (torch.uint8, torch.float8_e4m3fn) for t in (k, v)) or scales.dtype != torch.uint8:
        raise ValueError(f"8-bit pool: codes must be float8_e4m3fn or uint8, scales uint8: {k.dtype}, {v.dtype}, "
                         f"{scales.dtype}")
    if k.device != v.device or k.device != scales.device:
        raise ValueError("8-bit pool: codes and scales must be on one device")
    if k.dim() != 5 or v.dim() != 5 or scales.dim() != 4:
        raise ValueError(f"8-bit pool: shapes {tuple(k.shape)}, {tuple(v.shape)}, {tuple(scales.shape)}")
    nb, h, c, bs, w = k.shape
    d = 16 * c
    if (min(nb, h, c, bs) < 1 or w != 16 or v.shape != (nb, h, bs // 4, d, 4) or scales.shape != (nb, h, 2, bs) or bs % 4
            or d > 256):
        raise ValueError(f"8-bit pool: shapes {tuple(k.shape)}, {tuple(v.shape)}, {tuple(scales.shape)} (head_dim a "
                         "multiple of 16 up to 256, block_size a multiple of 4)")
    if not (k[0, 0].is_contiguous() and v[0, 0].is_contiguous() and scales[0, 0].is_contiguous()):
        raise ValueError("8-bit pool: a tile's codes and its scales must be contiguous")
    return KVLayout(k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), scales.stride(0), scales.stride(1), v.stride(0),
                    v.stride(1), 0, 0, bs, h, d, _dt(torch.empty(0, dtype=dtype)) | STORE_E4M3, nb,
                    scales.data_ptr() - k.data_ptr())


def _check_current(what: str, t: torch.Tensor) -> None:
    """A launch goes to the current device's stream."""
    if t.device.type == "cuda" and t.device.index != torch.cuda.current_device():
        raise ValueError(f"{what}: tensors on {t.device}, the current device is cuda:{torch.cuda.current_device()}")


def _check_rows(what: str, t_dtype: torch.dtype, layout: KVLayout) -> None:
    """A pool of codes takes and gives rows of its own dtype only."""
    if layout.dtype & STORE_E4M3 and DTYPE_CODE.get(t_dtype) != layout.dtype & ~STORE_E4M3:
        raise ValueError(f"{what}: {t_dtype} rows and an 8-bit pool of another dtype")


# ------------------------------------------------------------------------------------------------
# dense ops
# ------------------------------------------------------------------------------------------------
def gemm(a: torch.Tensor, w: torch.Tensor, out: Optional[torch.Tensor] = None,
         residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = a @ w.T (+ residual): nn.Linear (model.py:57-60, 88-90, 119) with the residual add fused."""
    require_device(a, w)
    m, lda = _rows(a)
    n, ldb = _rows(w)
    k = a.shape[1]
    if w.shape[1] != k or a.dtype != w.dtype:
        raise ValueError(f"gemm: {tuple(a.shape)} {a.dtype} x {tuple(w.shape)} {w.dtype}")
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _, ldc = _rows(out)
    ldr = 0
    if residual is not None:
        _, ldr = _rows(residual)
        if residual.shape != out.shape or residual.dtype != a.dtype:
            raise ValueError("gemm: residual shape/dtype")
    lib = _lib.load()
    need = lib.fs_gemm_workspace_size(m, n, k, _dt(a))
    ws = _persistent_ws("gemm", need, a.device) if need > 0 else None
    check(lib.fs_gemm(ptr(a), lda, ptr(w), ldb, ptr(out), ldc, ptr(residual), ldr, m, n, k, _dt(a), ptr(ws),
                      ws.numel() if ws is not None else 0, stream_ptr()), "gemm")
    return out


def quantize_e4m3(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x (rows, K) (float32, bfloat16, float16; K a multiple of 128) in 8-bit floating point: (codes, torch.float8_e4m3fn
    (rows, K); scales, uint8 (ceil(K / 512), rows, 4)). Columns 128g .. of row r stand for
    codes * 2^(scales[g // 4, r, g % 4] - 127): the smallest power of two that brings the group's largest magnitude to
    448 or less. A value is kept within 2^-4 of it down to 2^-6 of the scale (at most 2^-13.8 of the group's largest), and
    within 2^-10 of the scale (2^-17.8 of the largest) below that; where the scale is the smallest there is, 2^-117, a
    share of the scale only.
    What is not finite becomes NaN."""
    require_device(x)
    _check_current("quantize_e4m3", x)
    m, ldx = _rows(x)
    k = x.shape[1]
    if k % 128 or k == 0:
        raise ValueError(f"quantize_e4m3: K {k} is not a multiple of 128")
    codes = torch.empty((m, k), dtype=torch.uint8, device=x.device)
    scales = torch.empty((-(-k // 512), m, 4), dtype=torch.uint8, device=x.device)
    if m == 0:
        return codes.view(torch.float8_e4m3fn), scales
    check(_lib.load().fs_quantize_e4m3(ptr(x), ldx, m, k, _dt(x), ptr(codes), k, ptr(scales), stream_ptr()), "quantize_e4m3")
    return codes.view(torch.float8_e4m3fn), scales


def gemm_e4m3(a: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, out: Optional[torch.Tensor] = None,
              residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = a @ w.T (+ residual) with the weight in 8-bit floating point, as quantize_e4m3 leaves it (w (n, k) codes with
    16-byte aligned rows, w_scales (ceil(k / 512), n, 4)), and a (bfloat16 or float16) brought to the same form within
    the call: nn.Linear with half the weight bytes and twice the matrix rate of gemm's (17 to 64 rows of a small weight gain
    little: three launches). Sums are float32 (of each eight
    products the matrix instruction drops what lies more than 13 binary places below the largest); product and residual
    are rounded once, to a's dtype. A row's last bit may depend on how many rows the call has. out may be the
    residual itself, but shares no memory with a or w. linear_e4m3 computes the same product with kernels and an order of its
    own (a last bit may differ), also from rows in codes, and is mostly the faster from about 8 rows to 1000, by up to a third;
    this call is for fewer rows of small weights, by up to a fifth."""
    require_device(a, w, w_scales)
    if not a.device == w.device == w_scales.device or any(t is not None and t.device != a.device for t in (out, residual)):
        raise ValueError("gemm_e4m3: tensors on different devices")
    _check_current("gemm_e4m3", a)
    m, lda = _rows(a)
    n, ldb = _rows(w)
    k = a.shape[1]
    if a.dtype not in (torch.bfloat16, torch.float16):
        raise ValueError(f"gemm_e4m3: rows must be bfloat16 or float16, not {a.dtype}")
    if w.shape[1] != k or w.dtype not in (torch.float8_e4m3fn, torch.uint8):
        raise ValueError(f"gemm_e4m3: {tuple(a.shape)} x {tuple(w.shape)} {w.dtype}")
    if w_scales.dtype != torch.uint8 or w_scales.shape != (-(-k // 512), n, 4) or not w_scales.is_contiguous():
        raise ValueError(f"gemm_e4m3: scales must be contiguous uint8 ({-(-k // 512)}, {n}, 4): {tuple(w_scales.shape)}")
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _, ldc = _rows(out)
    if out.shape != (m, n) or out.dtype != a.dtype:
        raise ValueError("gemm_e4m3: out shape/dtype")
    ldr = 0
    if residual is not None:
        _, ldr = _rows(residual)
        if residual.shape != out.shape or residual.dtype != a.dtype:
            raise ValueError("gemm_e4m3: residual shape/dtype")
    if m == 0 or n == 0:
        return out
    lib = _lib.load()
    ws = _ws(lib.fs_gemm_e4m3_workspace_size(m, n, k), a.device)   # (of the current stream: calls on two do not share it)
    check(lib.fs_gemm_e4m3(ptr(a), lda, ptr(w), ldb, ptr(w_scales), ptr(out), ldc, ptr(residual), ldr, m, n, k, _dt(a), ptr(ws),
                           ws.numel(), stream_ptr()), "gemm_e4m3")
    return out


# The calls on codes below take 5 to 30 us on the GPU: their checks are written so that a good call pays few microseconds.
def _stream_of(what: str, first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """The current stream, with every tensor on the current device (a launch goes to its stream)."""
    index = first.get_device()
    if index >= 0 and index == torch._C._cuda_getDevice():
        for t in others:
            if t is not None and t.get_device() != index:
                break
        else:
            return torch._C._cuda_getCurrentRawStream(index)
    tensors = (first, *others)
    require_device(*tensors)
    if any(t is not None and t.device != first.device for t in tensors):
        raise ValueError(f"{what}: tensors on different devices")
    _check_current(what, first)
    return 0   # (of tensors that are on no GPU: only for checks without one)


def _row_stride(t: torch.Tensor, n: int) -> int:
    """The row stride of a 2-D tensor of n columns whose last dim is contiguous (of a single row: any that holds it)."""
    if t.is_contiguous():
        return n
    strides = t.stride()
    if len(strides) != 2 or (strides[1] != 1 and n > 1):
        raise ValueError(f"expected a 2-D tensor with a contiguous last dim, got {tuple(t.shape)} {strides}")
    return strides[0] if len(t) > 1 else n


_CODES = (torch.float8_e4m3fn, torch.uint8)


def _code_rows(what: str, name: str, codes: torch.Tensor, scales: torch.Tensor, n: int, k: int) -> int:
    """The row stride of (n, k) codes with quantize_e4m3's scales; its rows' alignment is the library's to check."""
    if codes.dtype not in _CODES:
        raise ValueError(f"{what}: {name} must be float8_e4m3fn or uint8 codes, not {codes.dtype}")
    if scales.dtype is not torch.uint8 or scales.shape != ((k + 511) // 512, n, 4) or not scales.is_contiguous():
        raise ValueError(f"{what}: {name}'s scales must be contiguous uint8 ({(k + 511) // 512}, {n}, 4): {tuple(scales.shape)}")
    return _row_stride(codes, k)


def _new_codes(m: int, n: int, device) -> Tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty(m, n, dtype=torch.float8_e4m3fn, device=device),
            torch.empty((n + 511) // 512, m, 4, dtype=torch.uint8, device=device))


def dequantize_e4m3(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The values (rows, K) that codes and scales of quantize_e4m3 (add_rmsnorm_e4m3, linear_e4m3_codes) stand for, rounded
    to dtype: float32 and bfloat16 hold each exactly, float16 what lies in its range (infinite above)."""
    stream = _stream_of("dequantize_e4m3", codes, scales, out)
    m, k = codes.shape if codes.dim() == 2 else (0, 0)
    if k % 128 or k == 0:
        raise ValueError(f"dequantize_e4m3: {tuple(codes.shape)}: K is not a multiple of 128")
    ldc = _code_rows("dequantize_e4m3", "the matrix", codes, scales, m, k)
    code = DTYPE_CODE.get(dtype)
    if code is None:
        raise ValueError(f"dequantize_e4m3: dtype {dtype} (float32, bfloat16, float16)")
    if out is None:
        out, ldo = torch.empty(m, k, dtype=dtype, device=codes.device), k
    elif out.shape != codes.shape or out.dtype is not dtype:
        raise ValueError("dequantize_e4m3: out shape/dtype")
    else:
        ldo = _row_stride(out, k)
    if m:
        check(_lib.load().fs_dequantize_e4m3(codes.data_ptr(), ldc, scales.data_ptr(), m, k, code, out.data_ptr(), ldo, stream),
              "dequantize_e4m3")
    return out


def add_rmsnorm_e4m3(x: torch.Tensor, weight: torch.Tensor, eps: float, delta: Optional[torch.Tensor] = None,
                     x_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """add_rmsnorm with its output in 8-bit floating point, for the product over codes that reads it: (codes, scales) of
    RMSNorm(x [+ delta]) (model.py:29-31), as quantize_e4m3 lays them out; with delta, x + delta is also written to x_out
    (which may be x or delta). N is a multiple of 128. The norm is computed in float32 from the sum as rounded to x's dtype
    (float32, bfloat16, float16), and rounded once, to the code: a value is kept as quantize_e4m3 keeps it. A row whose
    squares' sum passes float32's range has zeros; of one with an infinite or NaN element that element, or all, are NaN."""
    stream = _stream_of("add_rmsnorm_e4m3", x, weight, delta, x_out)
    shape, dtype = x.shape, x.dtype
    m, n = shape if len(shape) == 2 else (0, 0)
    dt = DTYPE_CODE.get(dtype)
    if n % 128 or n == 0 or dt is None:
        raise ValueError(f"add_rmsnorm_e4m3: {tuple(x.shape)} {dtype} (N a multiple of 128; float32, bfloat16, float16)")
    if weight.shape != (n,) or weight.dtype is not dtype or not weight.is_contiguous():
        raise ValueError("add_rmsnorm_e4m3: weight shape/dtype")
    ldx = _row_stride(x, n)
    ldd = ldxo = pd = pxo = 0
    if (delta is None) != (x_out is None):
        raise ValueError("add_rmsnorm_e4m3: delta needs x_out, and x_out delta")
    if delta is not None:
        if delta.shape != shape or x_out.shape != shape or delta.dtype is not dtype or x_out.dtype is not dtype:
            raise ValueError("add_rmsnorm_e4m3: delta or x_out shape/dtype")
        ldd, ldxo, pd, pxo = _row_stride(delta, n), _row_stride(x_out, n), delta.data_ptr(), x_out.data_ptr()
    codes, scales = _new_codes(m, n, x.device)
    if m:
        check(_lib.load().fs_add_rmsnorm_e4m3(x.data_ptr(), ldx, pd, ldd, pxo, ldxo, weight.data_ptr(), codes.data_ptr(), n,
                                              scales.data_ptr(), m, n, eps, dt, stream), "add_rmsnorm_e4m3")
    return codes, scales


ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}   # FS_ACT_*


def _linear_e4m3(what: str, a, w, w_scales, a_scales, bias, activation, gated, residual, out, dtype):
    """Both calls below: (out, None), or with dtype torch.float8_e4m3fn (codes, scales)."""
    stream = _stream_of(what, a, w, w_scales, a_scales, bias, residual, out)
    x_shape, w_shape = a.shape, w.shape
    if len(x_shape) != 2 or len(w_shape) != 2:
        raise ValueError(f"{what}: {tuple(x_shape)} x {tuple(w_shape)}")
    m, k = x_shape
    rows, wk = w_shape
    n = rows // 2 if gated else rows
    if k % 128 or k == 0 or wk != k or n == 0 or (gated and rows % 2):
        raise ValueError(f"{what}: {tuple(a.shape)} x {tuple(w.shape)} (K a multiple of 128, of a gated product an even "
                         "number of rows)")
    ldw = _code_rows(what, "w", w, w_scales, rows, k)
    if a_scales is not None:
        lda, pas, x_dtype = _code_rows(what, "a", a, a_scales, m, k), a_scales.data_ptr(), 0
    else:
        lda, pas, x_dtype = _row_stride(a, k), 0, DTYPE_CODE.get(a.dtype)
        if x_dtype is None:
            raise ValueError(f"{what}: rows of {a.dtype} (codes need a_scales)")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"{what}: activation {activation!r} (one of {', '.join(map(str, ACTIVATIONS))})")
    bias_dtype = pb = ldr = pr = 0
    if bias is not None:
        bias_dtype, pb = DTYPE_CODE.get(bias.dtype), bias.data_ptr()
        if bias.shape != (rows,) or bias_dtype is None or not bias.is_contiguous():
            raise ValueError(f"{what}: bias must be contiguous ({rows},) in float32, bfloat16 or float16")
    scales = None
    if dtype is torch.float8_e4m3fn:
        if n % 128:
            raise ValueError(f"{what}: {n} columns are not a multiple of 128")
        out, scales = _new_codes(m, n, a.device)
        ldo, pos = n, scales.data_ptr()
    else:
        pos = 0
        if out is None:
            out = torch.empty(m, n, dtype=dtype, device=a.device)
            ldo = n
        else:
            if out.shape != (m, n) or out.dtype is not dtype:
                raise ValueError(f"{what}: out shape/dtype")
            ldo = _row_stride(out, n)
        if residual is not None:
            if residual.shape != (m, n) or residual.dtype is not dtype:
                raise ValueError(f"{what}: residual shape/dtype")
            ldr, pr = _row_stride(residual, n), residual.data_ptr()
    if m:
        lib = _lib.load()
        call = _lib.Linear(a.data_ptr(), pas, w.data_ptr(), w_scales.data_ptr(), pb, pr, out.data_ptr(), pos, lda, ldw, ldr, ldo,
                           m, n, k, x_dtype, DTYPE_CODE.get(dtype, 0), bias_dtype, act, 1 if gated else 0, 0)
        need = lib.fs_linear_e4m3_workspace_size(call)
        ws = torch.empty(need, dtype=torch.uint8, device=a.device) if need else None   # (of this stream alone)
        check(lib.fs_linear_e4m3(call, ws.data_ptr() if need else 0, need, stream), what)
    return out, scales


def linear_e4m3(a: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, a_scales: Optional[torch.Tensor] = None,
                bias: Optional[torch.Tensor] = None, activation: Optional[str] = None, gated: bool = False,
                residual: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """act(a @ w.T + bias) + residual over 8-bit floating point, or with a gate, w (2F, K) and bias (2F,) holding the gate's
    rows and then the others', act(gate) * up + residual (nn.Linear, SwiGLU.forward: model.py:57-60, 88-93, with the residual
    add of model.py:105-106). w, w_scales as quantize_e4m3 leaves them; a likewise, with a_scales (from quantize_e4m3,
    add_rmsnorm_e4m3 or linear_e4m3_codes), or rows of float32, bfloat16 or float16, which are encoded within the call.
    activation: None, "relu", "silu", "gelu" (with the normal distribution's function) or "gelu_tanh". bias: float32,
    bfloat16 or float16. The result is bfloat16 or float16: dtype, or out's, the residual's or a's, in that order, or
    bfloat16; the residual has the same. K is a multiple of 128. Sums are float32, but of each eight products the matrix
    instruction drops what lies more than 13 binary places below the largest: 2.5e-5 of a random result's norm. (With every
    product in full: dequantize_e4m3 both to bfloat16, which holds them exactly, and gemm.) The rest is float32, rounded
    once. A row's last bit may depend on how many rows the call has. out may be the residual itself, but shares no memory
    with a or w."""
    if dtype is None:
        dtype = (out.dtype if out is not None else residual.dtype if residual is not None else
                 a.dtype if a.dtype in (torch.bfloat16, torch.float16) else torch.bfloat16)
    if dtype is not torch.bfloat16 and dtype is not torch.float16:
        raise ValueError(f"linear_e4m3: results are bfloat16 or float16, not {dtype}")
    return _linear_e4m3("linear_e4m3", a, w, w_scales, a_scales, bias, activation, gated, residual, out, dtype)[0]


def linear_e4m3_codes(a: torch.Tensor, w: torch.Tensor, w_scales: torch.Tensor, a_scales: Optional[torch.Tensor] = None,
                      bias: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                      gated: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """linear_e4m3 with its result left in 8-bit floating point for the next product: (codes, scales) as quantize_e4m3 lays
    them out, rounded once. The result's columns are a multiple of 128. What the sums drop turns a value next to the middle
    between two codes to the other one: 1e-3 of a random result's norm, where the codes' own rounding is 2.7e-2."""
    return _linear_e4m3("linear_e4m3_codes", a, w, w_scales, a_scales, bias, activation, gated, None, None, torch.float8_e4m3fn)


def gemm_add_rmsnorm(a: torch.Tensor, w: torch.Tensor, residual: torch.Tensor, norm_weight: torch.Tensor,
                     eps: float, x_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """x = a @ w.T + residual (nn.Linear then the residual add, model.py:105-106) and y = RMSNorm(x)
    with norm_weight (model.py:29-31): returns (x, y). When the GEMM splits K into partials, they are
    added by the norm kernel itself (no separate reduction pass); otherwise (no split, or a long batch
    whose workgroups run the splits one after the other) the GEMM adds the residual and the norm runs
    on its output. The results are the same either way. x_out: an (m, n) tensor with unit column stride
    that receives x (returned as x)."""
    require_device(a, w, residual, norm_weight)
    m, lda = _rows(a)
    n, ldb = _rows(w)
    k = a.shape[1]
    lib = _lib.load()
    if (a.dtype in (torch.bfloat16,) and w.dtype == a.dtype and w.shape[1] == k and residual.shape == (m, n)
            and residual.dtype == a.dtype and n % 8 == 0 and n <= 8192 and lib.fs_gemm_splits(n, k, _dt(a)) > 1
            and not lib.fs_gemm_serial(m, n, k, _dt(a))
            and k % 64 == 0 and lda % 8 == 0 and ldb % 8 == 0 and residual.stride(1) == 1
            and residual.stride(0) % 8 == 0 and norm_weight.is_contiguous() and norm_weight.dtype == a.dtype):
        splits = lib.fs_gemm_splits(n, k, _dt(a))
        need = splits * m * n * 4
        ws = _persistent_ws("gemm", need, a.device)
        check(lib.fs_gemm_partials(ptr(a), lda, ptr(w), ldb, m, n, k, _dt(a), ptr(ws), ws.numel(), stream_ptr()),
              "gemm_partials")
        direct = (x_out is not None and x_out.shape == (m, n) and x_out.dtype == a.dtype and x_out.stride(1) == 1
                  and x_out.stride(0) % 8 == 0 and x_out.data_ptr() % 16 == 0)
        x = x_out if direct else torch.empty((m, n), dtype=a.dtype, device=a.device)
        y = torch.empty((m, n), dtype=a.dtype, device=a.device)
        check(lib.fs_splitk_add_rmsnorm(ptr(ws), splits, ptr(residual), residual.stride(0), ptr(x), x.stride(0),
                                        ptr(norm_weight), ptr(y), n, m, n, float(eps), _dt(a), stream_ptr()),
              "splitk_add_rmsnorm")
        if x_out is not None and not direct:
            x = x_out.copy_(x)
        return x, y
    x = gemm(a, w, residual=residual)
    y = add_rmsnorm(x, norm_weight, eps)
    return (x if x_out is None else x_out.copy_(x)), y


def row_stats_parts(m: int, n: int, k: int) -> int:
    """Column blocks per row of gemm_row_stats at this shape (0: the shape has no statistics epilogue)."""
    return int(_lib.load().fs_gemm_row_stats_parts(m, n, k))


def gemm_row_stats(a: torch.Tensor, w: torch.Tensor, temperature: Optional[torch.Tensor],
                   stats: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out = a @ w.T (the LM head, model.py:137-138) and, per row and column block, the softmax
    statistics of the stored logits x at y = x / temperature[row] (a true division, sampling.py:13;
    rows at T = 0 keep only a meaningful argmax). stats: int32
    (M, nparts, 4) records (max, sum, argmax value as float bits, argmax index); rows may be strided."""
    require_device(a, w, stats)
    m, lda = _rows(a)
    n, ldb = _rows(w)
    k = a.shape[1]
    if w.shape[1] != k or a.dtype != w.dtype or a.dtype != torch.bfloat16:
        raise ValueError(f"gemm_row_stats: bf16 {tuple(a.shape)} x {tuple(w.shape)}")
    nparts = row_stats_parts(m, n, k)
    if (stats.dtype != I32 or tuple(stats.shape) != (m, nparts, 4) or stats.stride(2) != 1 or stats.stride(1) != 4
            or stats.stride(0) % 4):
        raise ValueError(f"gemm_row_stats: stats must be int32 ({m}, {nparts}, 4) with whole records per row")
    if temperature is not None and (temperature.dtype != torch.float32 or temperature.shape != (m,)):
        raise ValueError("gemm_row_stats: temperature must be float32 (M,)")
    if out is None:
        out = torch.empty((m, n), dtype=a.dtype, device=a.device)
    _, ldc = _rows(out)
    check(_lib.load().fs_gemm_row_stats(ptr(a), lda, ptr(w), ldb, ptr(out), ldc, m, n, k, ptr(temperature),
                                        ptr(stats), stats.stride(0) // 4, nparts, stream_ptr()), "gemm_row_stats")
    return out


def row_stats_merge(parts: torch.Tensor, out: torch.Tensor, group: int = 1, gstride: int = 1,
                    offset: int = 0) -> torch.Tensor:
    """Merge gemm_row_stats' (M, nparts, 4) records into one per row: row m goes to record
    (m // group) * gstride + m % group + offset of out (int32 (..., 4), contiguous)."""
    require_device(parts, out)
    m, nparts, _ = parts.shape
    if parts.dtype != I32 or out.dtype != I32 or out.shape[-1] != 4 or not out.is_contiguous():
        raise ValueError("row_stats_merge: int32 records of 4")
    if parts.stride(2) != 1 or parts.stride(1) != 4 or parts.stride(0) % 4:
        raise ValueError("row_stats_merge: parts must hold whole records per row")
    last = ((m - 1) // group) * gstride + (m - 1) % group + offset if m else 0
    if last >= out.numel() // 4:
        raise ValueError("row_stats_merge: out is too small for the row mapping")
    check(_lib.load().fs_row_stats_merge(ptr(parts), parts.stride(0) // 4, nparts, m, ptr(out), group, gstride, offset,
                                         stream_ptr()), "row_stats_merge")
    return out


def add_rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float, delta: Optional[torch.Tensor] = None,
                x_out: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y = RMSNorm(x [+ delta]) (model.py:29-31); with delta, x + delta is also written to x_out."""
    require_device(x, weight)
    m, ldx = _rows(x)
    n = x.shape[1]
    if weight.shape != (n,) or weight.dtype != x.dtype:
        raise ValueError("add_rmsnorm: weight shape/dtype")
    ldd = ldxo = 0
    if delta is not None:
        _, ldd = _rows(delta)
        if x_out is None:
            raise ValueError("add_rmsnorm: delta needs x_out")
        _, ldxo = _rows(x_out)
    if y is None:
        y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    _, ldy = _rows(y)
    check(_lib.load().fs_add_rmsnorm(ptr(x), ldx, ptr(delta), ldd, ptr(x_out), ldxo, ptr(weight), ptr(y), ldy, m, n,
                                     float(eps), _dt(x), stream_ptr()), "add_rmsnorm")
    return y


def gemm_swiglu(a: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """silu_mul(gemm(a, w)) for w the [gate; up] weight (2F, K): h (M, F) = silu(a w_gate^T) * (a w_up^T)
    (model.py:93). One kernel when the shape allows it (bf16, no K split), else the two; the results
    are the same either way."""
    require_device(a, w)
    m, lda = _rows(a)
    n2, ldb = _rows(w)
    k = a.shape[1]
    f = n2 // 2
    lib = _lib.load()
    if (a.dtype == torch.bfloat16 and w.dtype == a.dtype and w.shape[1] == k and n2 % 4 == 0 and k % 64 == 0
            and lda % 8 == 0 and ldb % 8 == 0 and lib.fs_gemm_splits(n2, k, _dt(a)) == 1):
        h = torch.empty((m, f), dtype=a.dtype, device=a.device)
        check(lib.fs_gemm_swiglu(ptr(a), lda, ptr(w), ldb, ptr(h), f, m, f, k, _dt(a), stream_ptr()), "gemm_swiglu")
        return h
    return silu_mul(gemm(a, w))


def silu_mul(gu: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """silu(gu[:, :F]) * gu[:, F:] (model.py:93)."""
    require_device(gu)
    m, ld = _rows(gu)
    f = gu.shape[1] // 2
    if out is None:
        out = torch.empty((m, f), dtype=gu.dtype, device=gu.device)
    _, ldh = _rows(out)
    check(_lib.load().fs_silu_mul(ptr(gu), ld, ptr(out), ldh, m, f, _dt(gu), stream_ptr()), "silu_mul")
    return out


def embedding(ids: torch.Tensor, weight: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """weight[ids] for int64 ids of any shape -> (ids.numel(), d) (model.py:134-135)."""
    require_device(ids, weight)
    ids = ids.reshape(-1)
    if ids.dtype != torch.int64:
        ids = ids.long()
    ids = ids.contiguous()
    vocab, d = weight.shape
    if out is None:
        out = torch.empty((ids.numel(), d), dtype=weight.dtype, device=weight.device)
    _, ldo = _rows(out)
    check(_lib.load().fs_embedding(ptr(ids), ids.numel(), ptr(weight.contiguous()), d, vocab, ptr(out), ldo,
                                   _dt(weight), stream_ptr()), "embedding")
    return out


# ------------------------------------------------------------------------------------------------
# KV cache + attention
# ------------------------------------------------------------------------------------------------
def qkv_rope_write(qkv: torch.Tensor, positions: torch.Tensor, T: int, n_heads: int, rope_cos: torch.Tensor,
                   rope_sin: torch.Tensor, tables: torch.Tensor, layout: KVLayout,
                   slots: Optional[torch.Tensor] = None, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotate q and k (model.py:40-45, 67) and write k, v into the pool (paged.py:74-78).

    qkv: (B*T, (n_heads + 2*n_kv_heads) * head_dim); positions/slots: int32 (B*T,);
    tables: int32 (B, max_blocks). Returns the rotated queries (B*T, n_heads * head_dim)."""
    require_device(qkv, positions, tables)
    _check_rows("qkv_rope_write", qkv.dtype, layout)
    m, ld = _rows(qkv)
    d = layout.head_dim
    if q_out is None:
        q_out = torch.empty((m, n_heads * d), dtype=qkv.dtype, device=qkv.device)
    _, ldq = _rows(q_out)
    if positions.dtype != I32 or tables.dtype != I32 or (slots is not None and slots.dtype != I32):
        raise ValueError("qkv_rope_write: positions, slots and tables must be int32")
    check(_lib.load().fs_qkv_rope_write(ptr(qkv), ld, m, T, n_heads, ptr(positions), ptr(slots), ptr(rope_cos),
                                        ptr(rope_sin), rope_cos.shape[0], ptr(tables), tables.stride(0),
                                        tables.shape[1], layout, ptr(q_out), ldq, stream_ptr()), "qkv_rope_write")
    return q_out


def qkv_rope_gemm(h: torch.Tensor, w: torch.Tensor, positions: torch.Tensor, T: int, n_heads: int,
                  rope_cos: torch.Tensor, rope_sin: torch.Tensor, tables: torch.Tensor, layout: KVLayout,
                  slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qkv_rope_write(gemm(h, w), ...): the fused QKV projection (model.py:57-60, 64-66) followed by the
    rotary + pool write. When the projection splits K into partials, the rotary kernel adds them itself
    (no separate reduction pass); the results are the same either way."""
    require_device(h, w, positions, tables)
    m, lda = _rows(h)
    n, ldb = _rows(w)
    k = h.shape[1]
    lib = _lib.load()
    d = layout.head_dim
    if (h.dtype == torch.bfloat16 and w.dtype == h.dtype and w.shape[1] == k and layout.dtype & ~STORE_E4M3 == _dt(h)
            and not (layout.dtype & STORE_E4M3 and d // 16 & (d // 16 - 1))
            and k % 64 == 0 and lda % 8 == 0 and ldb % 8 == 0 and n % 8 == 0 and (d // 2) % 8 == 0
            and lib.fs_gemm_splits(n, k, _dt(h)) > 1 and not lib.fs_gemm_serial(m, n, k, _dt(h))
            and positions.dtype == I32 and tables.dtype == I32
            and (slots is None or slots.dtype == I32)):
        splits = lib.fs_gemm_splits(n, k, _dt(h))
        ws = _persistent_ws("gemm", splits * m * n * 4, h.device)
        check(lib.fs_gemm_partials(ptr(h), lda, ptr(w), ldb, m, n, k, _dt(h), ptr(ws), ws.numel(), stream_ptr()),
              "gemm_partials")
        q_out = torch.empty((m, n_heads * d), dtype=h.dtype, device=h.device)
        check(lib.fs_qkv_rope_write_partials(ptr(ws), splits, m, n, T, n_heads, ptr(positions), ptr(slots),
                                             ptr(rope_cos), ptr(rope_sin), rope_cos.shape[0], ptr(tables),
                                             tables.stride(0), tables.shape[1], layout, ptr(q_out), q_out.stride(0),
                                             stream_ptr()), "qkv_rope_write_partials")
        return q_out
    return qkv_rope_write(gemm(h, w), positions, T, n_heads, rope_cos, rope_sin, tables, layout, slots=slots)


def qkv_rope_write_varlen(qkv: torch.Tensor, positions: torch.Tensor, token_row: torch.Tensor, n_heads: int,
                          rope_cos: torch.Tensor, rope_sin: torch.Tensor, tables: torch.Tensor, layout: KVLayout,
                          q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """qkv_rope_write for packed sequences: token m writes through table row token_row[m].

    qkv: (n_tokens, (n_heads + 2*n_kv_heads) * head_dim); positions, token_row: int32 (n_tokens,);
    tables: int32 (rows, max_blocks). Returns the rotated queries (n_tokens, n_heads * head_dim)."""
    require_device(qkv, positions, token_row, tables)
    _check_rows("qkv_rope_write_varlen", qkv.dtype, layout)
    m, ld = _rows(qkv)
    d = layout.head_dim
    if positions.dtype != I32 or token_row.dtype != I32 or tables.dtype != I32:
        raise ValueError("qkv_rope_write_varlen: positions, token_row and tables must be int32")
    if positions.numel() != m or token_row.numel() != m:
        raise ValueError("qkv_rope_write_varlen: one position and one table row per token")
    if q_out is None:
        q_out = torch.empty((m, n_heads * d), dtype=qkv.dtype, device=qkv.device)
    _, ldq = _rows(q_out)
    check(_lib.load().fs_qkv_rope_write_varlen(ptr(qkv), ld, m, n_heads, ptr(positions.contiguous()),
                                               ptr(token_row.contiguous()), tables.shape[0], ptr(rope_cos),
                                               ptr(rope_sin), rope_cos.shape[0], ptr(tables), tables.stride(0),
                                               tables.shape[1], layout, ptr(q_out), ldq, stream_ptr()),
          "qkv_rope_write_varlen")
    return q_out


def paged_kv_write(k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, tables: torch.Tensor,
                   layout: KVLayout) -> None:
    """Scatter k, v (B, n_kv_heads, T, head_dim) to the pool slots of positions (B, T) (paged.py:74-78)."""
    require_device(k, v, positions, tables)
    _check_rows("paged_kv_write", k.dtype, layout)
    if k.shape != v.shape or k.stride() != v.stride() or k.stride(3) != 1:
        raise ValueError("paged_kv_write: k and v must share shape and strides, head_dim contiguous")
    b, h, t, d = k.shape
    if positions.dtype != I32 or tables.dtype != I32:
        raise ValueError("paged_kv_write: positions and tables must be int32")
    check(_lib.load().fs_paged_kv_write(ptr(k), ptr(v), k.stride(0), k.stride(1), k.stride(2), b, t,
                                        ptr(positions.contiguous()), ptr(tables), tables.stride(0), tables.shape[1],
                                        layout, stream_ptr()), "paged_kv_write")


def paged_gather(layout: KVLayout, tables: torch.Tensor, dtype, device) -> Tuple[torch.Tensor, torch.Tensor]:
    """Every block of every table row, in table order: (B, n_kv_heads, max_blocks*block_size, head_dim)."""
    _check_rows("paged_gather", dtype, layout)
    b, nb = tables.shape
    shape = (b, layout.n_kv_heads, nb * layout.block_size, layout.head_dim)
    k_all = torch.empty(shape, dtype=dtype, device=device)
    v_all = torch.empty(shape, dtype=dtype, device=device)
    check(_lib.load().fs_paged_gather(layout, ptr(tables), tables.stride(0), b, nb, ptr(k_all), ptr(v_all),
                                      stream_ptr()), "paged_gather")
    return k_all, v_all


# The plan key and positions tensor of the last paged-attention call that went through (held, so that no later
# object can share their identities).
_PLAN_KEY = [None, None]


def _reuse_plan(plan_key, positions: torch.Tensor) -> bool:
    """True when the previous paged-attention call carried the same plan key and the same positions
    tensor (the layers of one step)."""
    return plan_key is not None and _PLAN_KEY[0] is plan_key and _PLAN_KEY[1] is positions


def _attended(rc: int, what: str, plan_key, positions: torch.Tensor) -> None:
    """check(rc) of a call that attends, whose plan the next call may reuse only if it went through."""
    if rc != 0:
        _PLAN_KEY[0] = _PLAN_KEY[1] = None
        check(rc, what)
    _PLAN_KEY[0], _PLAN_KEY[1] = plan_key, positions


def paged_attention(q: torch.Tensor, layout: KVLayout, tables: torch.Tensor, positions: torch.Tensor,
                    scale: float, out: Optional[torch.Tensor] = None, plan_key=None) -> torch.Tensor:
    """Causal GQA attention of q (B, T, n_heads, head_dim) over the paged keys (model.py:70-76).

    positions: int32 (B, T); query (b, t) sees the keys at positions 0..positions[b, t].
    plan_key: an object that stands for these positions (the forward step): consecutive calls with the
    same key reuse the work plan of the first (the positions must not change between them)."""
    require_device(q, tables, positions)
    _check_rows("paged_attention", q.dtype, layout)
    b, t, h, d = q.shape
    if q.stride(3) != 1:
        raise ValueError("paged_attention: head_dim must be contiguous")
    if positions.dtype != I32 or tables.dtype != I32 or positions.shape != (b, t):
        raise ValueError("paged_attention: positions (B, T) and tables must be int32")
    positions = positions.contiguous()
    if out is None:
        out = torch.empty((b, t, h, d), dtype=q.dtype, device=q.device)
    nb = tables.shape[1]
    lib = _lib.load()
    need = lib.fs_paged_attention_workspace_size(b, t, h, d, nb, layout.block_size)
    ws = _persistent_ws("attention", need, q.device)
    fn = lib.fs_paged_attention_reuse_plan if _reuse_plan(plan_key, positions) else lib.fs_paged_attention
    _attended(fn(ptr(q), q.stride(0), q.stride(1), q.stride(2), layout, ptr(tables), tables.stride(0), nb, ptr(positions),
                 b, t, h, float(scale), ptr(out), out.stride(0), out.stride(1), out.stride(2), ptr(ws), ws.numel(),
                 stream_ptr()), "paged_attention", plan_key, positions)
    return out


def paged_attention_varlen(q: torch.Tensor, layout: KVLayout, tables: torch.Tensor, positions: torch.Tensor,
                           cu_seqlens: torch.Tensor, scale: float, out: Optional[torch.Tensor] = None,
                           plan_key=None) -> torch.Tensor:
    """paged_attention over packed sequences: q (n_tokens, n_heads, head_dim); sequence s owns tokens
    cu_seqlens[s] .. cu_seqlens[s+1]-1 (int32 (S+1,), on the device; the caller guarantees the bounds:
    cu_seqlens[S] <= n_tokens and no sequence longer than T); positions int32 (S, T), -1 past a
    sequence's tokens; tables int32 (S, max_blocks). Returns out (n_tokens, n_heads, head_dim).
    plan_key: as for paged_attention."""
    require_device(q, tables, positions, cu_seqlens)
    _check_rows("paged_attention_varlen", q.dtype, layout)
    n, h, d = q.shape
    if q.stride(2) != 1:
        raise ValueError("paged_attention_varlen: head_dim must be contiguous")
    s, t = positions.shape
    if (positions.dtype != I32 or tables.dtype != I32 or cu_seqlens.dtype != I32 or cu_seqlens.numel() != s + 1
            or tables.shape[0] != s):
        raise ValueError("paged_attention_varlen: positions (S, T), tables (S, .) and cu_seqlens (S+1,) int32")
    positions = positions.contiguous()
    if out is None:
        out = torch.empty((n, h, d), dtype=q.dtype, device=q.device)
    nb = tables.shape[1]
    lib = _lib.load()
    ws = _persistent_ws("attention", lib.fs_paged_attention_workspace_size(s, t, h, d, nb, layout.block_size), q.device)
    fn = (lib.fs_paged_attention_varlen_reuse_plan if _reuse_plan(plan_key, positions)
          else lib.fs_paged_attention_varlen)
    _attended(fn(ptr(q), q.stride(0), q.stride(1), layout, ptr(tables), tables.stride(0), nb, ptr(positions),
                 ptr(cu_seqlens.contiguous()), s, t, h, float(scale), ptr(out), out.stride(0), out.stride(1), ptr(ws),
                 ws.numel(), stream_ptr()), "paged_attention_varlen", plan_key, positions)
    return out


# ------------------------------------------------------------------------------------------------
# decoder blocks
# ------------------------------------------------------------------------------------------------
def run_blocks(x: torch.Tensor, h: torch.Tensor, b: int, t: int, heads: tuple, ffn: int, positions: torch.Tensor,
               rope_cos: torch.Tensor, rope_sin: torch.Tensor, blocks: list, normed: bool, buffers: dict):
    """Decoder blocks launched by one call (fs_run_blocks): x (B*T, d) and h = the first block's attention norm of
    x, both contiguous; heads: (query heads, KV heads, head_dim). blocks: per block (w_qkv, w_o, w_gate_up,
    w_down, mlp norm weight, its eps, next norm weight or None, its eps, (layout, tables, slots, visible
    positions), plan key), tensors of x's dtype and device with contiguous rows (the caller has checked them).
    buffers: an empty dict, the same for the calls of one forward, which share their workspaces and scratch
    through it. Returns (x, next norm of x or None)."""
    lib = _lib.load()
    m, d = x.shape
    n_heads, nkv, hd = heads
    dt, dev = _dt(x), x.device
    kv_dt = blocks[0][8][0].dtype   # (with the flag of a pool of codes)
    arr = (_lib.Block * len(blocks))()
    sizes = set()
    for e, (wq, wo, wgu, wd, n1, e1, n2, e2, (lay, tab, slots, vis), _) in zip(arr, blocks):
        if (lay.n_kv_heads, lay.head_dim, lay.dtype) != (nkv, hd, kv_dt) or kv_dt & ~STORE_E4M3 != dt:
            raise ValueError("run_blocks: the cache's heads, head_dim or dtype are not the model's")
        if (tab.dtype != I32 or vis.dtype != I32 or vis.shape != (b, t) or not vis.is_contiguous()
                or (slots is not None and (slots.dtype != I32 or slots.numel() != m))):
            raise ValueError("run_blocks: tables, slots and positions (B, T) must be int32")
        require_device(tab, vis, slots)
        e.w_qkv, e.w_o, e.w_gate_up, e.w_down = wq.data_ptr(), wo.data_ptr(), wgu.data_ptr(), wd.data_ptr()
        e.mlp_norm, e.next_norm = n1.data_ptr(), ptr(n2)
        e.kv, e.tables, e.table_stride, e.max_blocks = lay, tab.data_ptr(), tab.stride(0), tab.shape[1]
        e.slots, e.visible, e.mlp_eps, e.next_eps = ptr(slots), vis.data_ptr(), e1, e2
        sizes.add((tab.shape[1], lay.block_size))
    shape = (heads, ffn, kv_dt, frozenset(sizes))
    if shape not in buffers:
        need, attn = (_lib.c_i64 * 3)(), 0
        for nb, bs in sizes:
            check(lib.fs_run_blocks_workspace(b, t, n_heads, nkv, hd, d, ffn, kv_dt, nb, bs, need), "run_blocks_workspace")
            attn = max(attn, need[1])
        buffers[shape] = (_persistent_ws("gemm", need[0], dev) if need[0] > 0 else None,
                          _persistent_ws("attention", attn, dev), _ws(need[2], dev))
    gws, aws, scratch = buffers[shape]
    x_out = torch.empty((m, d), dtype=x.dtype, device=dev)
    y = torch.empty((m, d), dtype=x.dtype, device=dev) if normed else None
    before = _PLAN_KEY
    for e, blk in zip(arr, blocks):   # a block reuses the plan of the one before it: same step, same positions
        key, vis = blk[9], blk[8][3]
        e.reuse_plan = key is not None and before[0] is key and before[1] is vis
        before = key, vis
    rc = lib.fs_run_blocks(arr, len(blocks), b, t, n_heads, d, ffn, kv_dt, positions.data_ptr(), rope_cos.data_ptr(),
                           rope_sin.data_ptr(), rope_cos.shape[0], 1.0 / math.sqrt(hd), x.data_ptr(), h.data_ptr(),
                           x_out.data_ptr(), ptr(y), ptr(gws), 0 if gws is None else gws.numel(), aws.data_ptr(),
                           aws.numel(), scratch.data_ptr(), scratch.numel(), stream_ptr())
    _attended(rc, "run_blocks", *before)
    return x_out, y


# ------------------------------------------------------------------------------------------------
# sampling / acceptance
# ------------------------------------------------------------------------------------------------
def probs_from_logits(logits: torch.Tensor, temperature: float) -> torch.Tensor:
    """softmax(f32(logits) / T), or the one-hot of the argmax in the logits dtype at T == 0 (sampling.py:9-13)."""
    require_device(logits)
    shape = logits.shape
    x = logits.reshape(-1, shape[-1])
    if x.stride(1) != 1:
        x = x.contiguous()
    r, ld = x.shape[0], x.stride(0)
    v = shape[-1]
    out_dtype = torch.float32 if temperature > 0 else logits.dtype
    out = torch.empty((r, v), dtype=out_dtype, device=logits.device)
    lib = _lib.load()
    ws = _ws(lib.fs_sampling_workspace_size(r, v), logits.device)
    check(lib.fs_probs_from_logits(ptr(x), ld, r, v, float(temperature), _dt(x), ptr(out), v, DTYPE_CODE[out_dtype],
                                   ptr(ws), ws.numel(), stream_ptr()), "probs_from_logits")
    return out.reshape(shape)


def sample_logits(logits: torch.Tensor, temperature, noise: Optional[torch.Tensor] = None,
                  out32: Optional[torch.Tensor] = None, out64: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Token ids (int64, logits.shape[:-1]) for logits (..., V) (sampling.py:16-21).

    temperature: a float for every row, or a float32 device tensor with one value per row.
    noise: float32 Exp(1) noise with the logits' shape (the categorical draw is argmax(p / noise));
    None makes every row greedy. out32: optional int32 view that also receives the tokens; out64: an
    optional contiguous int64 tensor of one element per row that receives them as the result does (and
    is returned, reshaped)."""
    require_device(logits)
    shape = logits.shape
    x = logits.reshape(-1, shape[-1])
    if x.stride(1) != 1:
        x = x.contiguous()
    r, ld = x.shape[0], x.stride(0)
    v = shape[-1]
    if out64 is not None and (out64.dtype != torch.int64 or out64.numel() != r or not out64.is_contiguous()):
        raise ValueError("sample_logits: out64 must be a contiguous int64 tensor of one element per row")
    tok = out64.view(-1) if out64 is not None else torch.empty((r,), dtype=torch.int64, device=logits.device)
    t_ptr, t_all = 0, 0.0
    if isinstance(temperature, torch.Tensor):
        require_device(temperature)
        temperature = temperature.to(torch.float32).reshape(-1).contiguous()
        if temperature.numel() != r:
            raise ValueError("sample_logits: one temperature per row")
        t_ptr = ptr(temperature)
    else:
        t_all = float(temperature)
        if t_all < 0:
            raise ValueError("temperature must be >= 0")
    e_ptr, lde = 0, 0
    if noise is not None:
        require_device(noise)
        noise = noise.reshape(-1, v)
        if noise.dtype != torch.float32 or noise.shape[0] != r or noise.stride(1) != 1:
            raise ValueError("sample_logits: noise must be float32 with the logits' shape")
        e_ptr, lde = ptr(noise), noise.stride(0)
    o32, ld32 = 0, 0
    if out32 is not None:
        o32, ld32 = ptr(out32), out32.stride(0) if out32.dim() else 1
    lib = _lib.load()
    ws = _ws(lib.fs_sampling_workspace_size(r, v), logits.device)
    check(lib.fs_sample_logits(ptr(x), ld, r, v, t_ptr, t_all, e_ptr, lde, _dt(x), ptr(tok), o32, ld32, ptr(ws),
                               ws.numel(), stream_ptr()), "sample_logits")
    return tok.reshape(shape[:-1])


def spec_accept(tgt: torch.Tensor, dft: torch.Tensor, draft_tokens: torch.Tensor, k_eff: Optional[torch.Tensor],
                temperature: torch.Tensor, u: torch.Tensor, noise: torch.Tensor,
                seq_len: Optional[torch.Tensor] = None, out_tokens: Optional[torch.Tensor] = None,
                n_accepted: Optional[torch.Tensor] = None,
                row_stats: Optional[torch.Tensor] = None, debug: bool = False):
    """Batched verify_draft from logits (speculative.py:20-33, sampling.py:9-13).

    tgt (B, K+1, V), dft (B, K, V) logits; draft_tokens int32 (B, K); k_eff int32 (B,) or None (= K);
    temperature float32 (B,); u float32 (B, K) uniforms; noise float32 (B, V) Exp(1);
    seq_len int32 (B,) cached lengths, advanced in place by 1 + n_accepted;
    row_stats: int32 (B, 2K+1, 4) softmax statistics of the rows (row_stats_merge of the LM heads'
    gemm_row_stats at the temperatures), which skips the statistics pass.
    Returns out_tokens int32 (B, K+1) (accepted, extra, then -1) and n_accepted int32 (B,); with debug,
    also {"p_x", "q_x": float32 (B, K), p_i(x_i) and q_i(x_i) of the proposals i < k_eff (NaN past it),
    "res_sum": float32 (B,), the residual sum at the first rejection (0: none)}."""
    require_device(tgt, dft, draft_tokens, temperature, u, noise)
    b, k1, v = tgt.shape
    k = k1 - 1
    if dft.shape != (b, k, v) or dft.dtype != tgt.dtype:
        raise ValueError(f"spec_accept: draft logits {tuple(dft.shape)} vs target {tuple(tgt.shape)}")
    if tgt.stride(2) != 1 or dft.stride(2) != 1:
        raise ValueError("spec_accept: vocab dim must be contiguous")
    for name, t, dt, shp in (("draft_tokens", draft_tokens, I32, (b, k)), ("temperature", temperature,
                             torch.float32, (b,)), ("u", u, torch.float32, (b, k)), ("noise", noise, torch.float32,
                             (b, v))):
        if t.dtype != dt or tuple(t.shape) != shp or not t.is_contiguous():
            raise ValueError(f"spec_accept: {name} must be contiguous {dt} {shp}")
    if k_eff is not None and (k_eff.dtype != I32 or k_eff.shape != (b,)):
        raise ValueError("spec_accept: k_eff must be int32 (B,)")
    if out_tokens is None:
        out_tokens = torch.empty((b, k + 1), dtype=I32, device=tgt.device)
    if n_accepted is None:
        n_accepted = torch.empty((b,), dtype=I32, device=tgt.device)
    lib = _lib.load()
    ws = _persistent_ws("accept", lib.fs_spec_accept_workspace_size(b, k, v), tgt.device)
    dbg = None
    if debug:
        dbg = {"p_x": torch.full((b, k), float("nan"), dtype=torch.float32, device=tgt.device),
               "q_x": torch.full((b, k), float("nan"), dtype=torch.float32, device=tgt.device),
               "res_sum": torch.zeros((b,), dtype=torch.float32, device=tgt.device)}
    px, qx, rs = (ptr(dbg["p_x"]), ptr(dbg["q_x"]), ptr(dbg["res_sum"])) if dbg else (0, 0, 0)
    if row_stats is not None:
        if row_stats.dtype != I32 or tuple(row_stats.shape) != (b, 2 * k + 1, 4) or not row_stats.is_contiguous():
            raise ValueError(f"spec_accept: row_stats must be contiguous int32 ({b}, {2 * k + 1}, 4)")
        require_device(row_stats)
        check(lib.fs_spec_accept_stats(ptr(tgt), tgt.stride(0), tgt.stride(1), ptr(dft), dft.stride(0),
                                       dft.stride(1) if k else 0, b, k, v, _dt(tgt), ptr(draft_tokens), ptr(k_eff),
                                       ptr(temperature), ptr(u), ptr(noise), noise.stride(0), ptr(row_stats),
                                       ptr(out_tokens), ptr(n_accepted), ptr(seq_len), px, qx, rs, ptr(ws),
                                       ws.numel(), stream_ptr()), "spec_accept")
    else:
        check(lib.fs_spec_accept(ptr(tgt), tgt.stride(0), tgt.stride(1), ptr(dft), dft.stride(0),
                                 dft.stride(1) if k else 0, b, k, v, _dt(tgt), ptr(draft_tokens), ptr(k_eff),
                                 ptr(temperature), ptr(u), ptr(noise), noise.stride(0), ptr(out_tokens),
                                 ptr(n_accepted), ptr(seq_len), px, qx, rs, ptr(ws), ws.numel(), stream_ptr()),
              "spec_accept")
    return (out_tokens, n_accepted, dbg) if debug else (out_tokens, n_accepted)


def verify_probs(p: torch.Tensor, q: torch.Tensor, draft_tokens: torch.Tensor, u: torch.Tensor,
                 noise: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """verify_draft on probability rows p (K+1, V), q (K, V) (speculative.py:20-33)."""
    require_device(p, q, draft_tokens, u, noise)
    k1, v = p.shape
    k = k1 - 1
    if q.shape != (k, v) or q.dtype != p.dtype or p.stride(1) != 1 or (k and q.stride(1) != 1):
        raise ValueError("verify_probs: p (K+1, V) and q (K, V) of one dtype, contiguous rows")
    if draft_tokens.dtype != I32 or draft_tokens.numel() != k or u.numel() != k or noise.numel() != v:
        raise ValueError("verify_probs: draft_tokens int32 (K,), u (K,), noise (V,)")
    out = torch.empty((k + 1,), dtype=I32, device=p.device)
    n = torch.empty((1,), dtype=I32, device=p.device)
    lib = _lib.load()
    ws = _persistent_ws("accept", lib.fs_spec_accept_workspace_size(1, k, v), p.device)
    check(lib.fs_verify_probs(ptr(p), p.stride(0), ptr(q), q.stride(0) if k else 0, k, v, _dt(p),
                              ptr(draft_tokens.contiguous()), ptr(u.contiguous()), ptr(noise.contiguous()), ptr(out),
                              ptr(n), ptr(ws), ws.numel(), stream_ptr()), "verify_probs")
    return out, n


def spec_advance(res: torch.Tensor, b: int, k: int, first: int, n: torch.Tensor, budget: torch.Tensor,
                 eos: torch.Tensor, done: torch.Tensor, ids: torch.Tensor, last: torch.Tensor, keff: torch.Tensor,
                 pos0: torch.Tensor, posd: torch.Tensor, posv: torch.Tensor) -> None:
    """The next round's inputs from this round's acceptance, in place on the device (the bookkeeping
    of speculative.py:71-85 for b rows): res (b, k+2) int32 from the acceptance; n, budget, eos, done
    int32 (b,); ids int64 (b, 2); last int64 (b,); keff int32 (b,); pos0 int32 (b, 2); posd int32
    (k - first, b); posv int32 (b, k+1)."""
    require_device(res, n, budget, eos, done, ids, last, keff, pos0, posv)
    i32 = (res, n, budget, eos, done, keff, pos0, posd, posv)
    if any(t.dtype != I32 or not t.is_contiguous() for t in i32) or ids.dtype != torch.int64 or last.dtype != torch.int64:
        raise ValueError("spec_advance: int32 rows and positions, int64 ids, contiguous")
    shapes_ok = (res.shape[0] >= b and res.shape[1] >= k + 2 and n.numel() >= b and ids.shape == (b, 2)
                 and posv.shape == (b, k + 1) and pos0.shape == (b, 2) and (k <= first or posd.shape == (k - first, b)))
    if not shapes_ok:
        raise ValueError("spec_advance: shapes")
    check(_lib.load().fs_spec_advance(ptr(res), res.stride(0), b, k, first, ptr(n), ptr(budget), ptr(eos), ptr(done),
                                      ptr(ids), ptr(last), ptr(keff), ptr(pos0), ptr(posd), ptr(posv), stream_ptr()),
          "spec_advance")


RNG_UNIFORM, RNG_EXP = 0, 1


def keyed_noise(keys: torch.Tensor, slot0: int, out: torch.Tensor, kind: int) -> torch.Tensor:
    """Counter-based draws keyed per row: out (n_slots, B, n) or (B, n) float32 (last dim contiguous)
    receives, for slot s and row b, the variates of (keys[b], slot0 + s, column j): uniforms in
    [0, 1) (kind RNG_UNIFORM) or Exp(1) (RNG_EXP). keys: int64 (B,) on the device."""
    require_device(keys, out)
    if keys.dtype != torch.int64 or keys.dim() != 1 or not keys.is_contiguous():
        raise ValueError("keyed_noise: keys must be a contiguous int64 (B,) tensor")
    o = out if out.dim() == 3 else out.unsqueeze(0)
    s, b, n = o.shape
    if o.dtype != torch.float32 or (n > 1 and o.stride(2) != 1) or b != keys.numel():
        raise ValueError("keyed_noise: out must be float32 (n_slots, B, n) with B = len(keys), last dim contiguous")
    check(_lib.load().fs_keyed_noise(ptr(keys), b, slot0, s, n, kind, ptr(o), o.stride(1), o.stride(0), stream_ptr()),
          "keyed_noise")
    return out
