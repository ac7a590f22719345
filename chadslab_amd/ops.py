"""Operator entry points: what a numpy-style LLM runtime's quantized `x @ dequant(W).T` call sites bind to.

Every function runs hand-written HIP kernels from libchadq.so through its C ABI (chadslab_amd/_lib.py) on
torch's current stream.  torch is used for device memory and streams only.  Nothing here computes on the
CPU: tensors must already be on the GPU, and a missing library raises.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Union

import torch

from . import _lib
from .formats import GROUP, QExpertsMXFP4, QWeightInt4G32, QWeightInt4G32Tiles, QWeightInt8, QWeightMXFP4, check_mxfp4

QWeight = Union[QWeightInt4G32, QWeightInt8, QWeightMXFP4]
GEMV_MAX_M = 16  # decode batch sizes served by the bandwidth kernel


def _stream() -> int:
    """The handle of torch's current stream on the current device.  The raw getter: a Stream object made for every call
    (torch.cuda.current_stream()) cost 2.5 us of the 11 that a whole small product took on the host."""
    return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())


def _dev(t: torch.Tensor, name: str, dtype: torch.dtype) -> torch.Tensor:
    if not t.is_cuda:
        raise ValueError("%s must be a GPU tensor (there is no CPU path)" % name)
    if t.dtype is not dtype:  # one object per type
        raise ValueError("%s must be %s, got %s" % (name, dtype, t.dtype))
    return t if t.is_contiguous() else t.contiguous()


def _out(out: Optional[torch.Tensor], shape, dtype: torch.dtype, device) -> torch.Tensor:
    """A caller's result tensor, checked before its address goes to the library; a fresh one if none was given."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not out.is_cuda or out.device != device:
        raise ValueError("out must live on %s, got %s" % (device, out.device))
    if out.dtype != dtype or tuple(out.shape) != tuple(shape) or not out.is_contiguous():
        raise ValueError("out must be a contiguous %s tensor of shape %s, got %s %s" % (dtype, tuple(shape), out.dtype, tuple(out.shape)))
    return out


def unpack_int4(packed: torch.Tensor) -> torch.Tensor:
    """uint8 [..., K/2] -> int8 [..., K] in [-8,7] (low nibble = even k)."""
    p = _dev(packed, "packed", torch.uint8)
    out = torch.empty(*p.shape[:-1], p.shape[-1] * 2, dtype=torch.int8, device=p.device)
    _lib.check(_lib.load().chadq_unpack_i4(p.data_ptr(), out.data_ptr(), p.numel(), _stream()), "chadq_unpack_i4")
    return out


def pack_int4(q: torch.Tensor) -> torch.Tensor:
    """int8 [..., K] in [-8,7] -> uint8 [..., K/2]; inverse of unpack_int4."""
    q = _dev(q, "q", torch.int8)
    if q.shape[-1] % 2:
        raise ValueError("K must be even")
    out = torch.empty(*q.shape[:-1], q.shape[-1] // 2, dtype=torch.uint8, device=q.device)
    _lib.check(_lib.load().chadq_pack_i4(q.data_ptr(), out.data_ptr(), out.numel(), _stream()), "chadq_pack_i4")
    return out


def _launch(device: torch.device, name: str, *args) -> None:
    """Library call `name` on the current stream of `device`, whichever device is current."""
    fn = getattr(_lib.load(), name)
    if device.index == torch._C._cuda_getDevice():
        _lib.check(fn(*args, _stream()), name)
    else:
        with torch.cuda.device(device):
            _lib.check(fn(*args, _stream()), name)


def _arrays(q: Union[QWeightMXFP4, QExpertsMXFP4]):
    """Codes and scales of a container, which may hold other arrays by now than those it was made of: the kernels read as far as the codes' shape
    says, so the scales have to fit it."""
    p, s = q.packed, q.scale
    check_mxfp4(type(q).__name__, p, s, 3 if isinstance(q, QExpertsMXFP4) else 2)
    return p, s


def _mxfp4(p: torch.Tensor, s: torch.Tensor, name: str, device: Optional[torch.device] = None):
    """Codes and scales (of _arrays), checked before their addresses go to the library."""
    p, s = _dev(p, name + ".packed", torch.uint8), _dev(s, name + ".scale", torch.uint8)
    for t in (p, s):
        if t.device != (p.device if device is None else device):
            raise ValueError("%s must live on %s, got %s" % (name, p.device if device is None else device, t.device))
    return p, s


def _int4(qw: Union[QWeightInt4G32, QWeightInt4G32Tiles], name: str = ""):
    """Packed bytes, scales, N and K of an int4 matrix, looked at as _arrays does (no slower than asking the container for N and K)."""
    p, s = qw.packed, qw.scale
    n, kb = p.shape if p.dim() == 2 else (-1, -1)
    if s.shape != (n, kb >> 4):
        raise ValueError("%sscale must be float16 [N,K/32] beside packed [N,K/2], got %s and %s" % (name, tuple(s.shape), tuple(p.shape)))
    return p, s, n, kb * 2


def _int8(qw: QWeightInt8):
    w, s = qw.w, qw.scale
    n, k = w.shape if w.dim() == 2 else (-1, -1)
    if s.shape != (n,):
        raise ValueError("scale must be float32 [N] beside w [N,K], got %s and %s" % (tuple(s.shape), tuple(w.shape)))
    return w, s, n, k


def _rows(x: Union[torch.Tensor, QWeightMXFP4]):
    """The activations of a product on MXFP4 weights: a tensor and None, or codes and scales of one matrix."""
    if isinstance(x, torch.Tensor):
        return x, None
    if not isinstance(x, QWeightMXFP4):
        raise TypeError("x must be a tensor or a QWeightMXFP4 (of activations of more dimensions: quantize_mxfp4(x.flatten(0, -2))), got %r" % type(x))
    return _arrays(x)


_MX_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # chadq_dtype


def quantize_mxfp4(x: torch.Tensor) -> Union[QWeightMXFP4, QExpertsMXFP4]:
    """fp32, bf16 or fp16 [R,K] -> QWeightMXFP4, [E,N,K] -> QExpertsMXFP4; K a multiple of 32.

    Per block of 32 values along K the scale is 2^(floor(log2(largest magnitude)) - 2), at least 2^-127; each value goes to the nearest code,
    ties to the even one, beyond 6 scales to 6.  A block that holds a NaN or an infinity becomes NaN."""
    q = _lib.native().quantize(x)
    if q is not None:
        return q
    if x.dtype not in _MX_TYPES:
        raise ValueError("x must be float32, bfloat16 or float16, got %s" % x.dtype)
    if x.dim() not in (2, 3) or x.size(-1) % GROUP:
        raise ValueError("x must be [R,K] or [E,N,K] with K a multiple of 32, got %s" % (tuple(x.shape),))
    x = _dev(x, "x", x.dtype)
    *lead, k = x.shape
    p = torch.empty(*lead, k // 2, dtype=torch.uint8, device=x.device)
    s = torch.empty(*lead, k // GROUP, dtype=torch.uint8, device=x.device)
    if x.numel():
        _launch(x.device, "chadq_quantize_mxfp4", x.data_ptr(), _MX_TYPES[x.dtype], p.data_ptr(), s.data_ptr(), x.numel() // k, k)
    return QWeightMXFP4(p, s) if len(lead) == 1 else QExpertsMXFP4(p, s)


def dequantize(qw: Union[QWeight, QExpertsMXFP4]) -> torch.Tensor:
    """fp32 [N,K] dequantised weights (exact); [E,N,K] of QExpertsMXFP4."""
    lib = _lib.load()
    if isinstance(qw, (QWeightMXFP4, QExpertsMXFP4)):
        out = _lib.native().dequantize(qw)
        if out is not None:
            return out
        p, s = _mxfp4(*_arrays(qw), "qw")
        k = p.size(-1) * 2
        out = torch.empty(*p.shape[:-1], k, dtype=torch.float32, device=p.device)
        if out.numel():
            _launch(p.device, "chadq_dequant_mxfp4", p.data_ptr(), s.data_ptr(), out.data_ptr(), out.numel() // k, k)
        return out
    if isinstance(qw, QWeightInt4G32):
        p, s, n, k = _int4(qw)
        p, s = _dev(p, "packed", torch.uint8), _dev(s, "scale", torch.float16)
        out = torch.empty(n, k, dtype=torch.float32, device=p.device)
        _lib.check(lib.chadq_dequant_i4g32(p.data_ptr(), s.data_ptr(), out.data_ptr(), n, k, _stream()),
                   "chadq_dequant_i4g32")
        return out
    if isinstance(qw, QWeightInt8):
        w, s, n, k = _int8(qw)
        w, s = _dev(w, "w", torch.int8), _dev(s, "scale", torch.float32)
        out = torch.empty(n, k, dtype=torch.float32, device=w.device)
        _lib.check(lib.chadq_dequant_i8row(w.data_ptr(), s.data_ptr(), out.data_ptr(), n, k, _stream()),
                   "chadq_dequant_i8row")
        return out
    raise TypeError("unknown weight container %r" % type(qw))


def _product_mxfp4(x: Union[torch.Tensor, QWeightMXFP4], qw: QWeightMXFP4, out: Optional[torch.Tensor], y_dtype: torch.dtype) -> torch.Tensor:
    """x (bf16 or MXFP4) [M,K] times MXFP4 weights -> fp32 or bf16 [M,N]."""
    xt, xs = _rows(x)
    x_mx = xs is not None
    p, s = _arrays(qw)
    m, n, k = xt.size(0) if xt.dim() else 0, p.size(0), p.size(1) * 2
    if xt.dim() != 2 or xt.size(1) * (2 if x_mx else 1) != k:
        raise ValueError("x must be [M,%d], got %s" % (k, (m, xt.size(1) * 2) if x_mx else tuple(x.shape)))
    if x_mx:
        xt, xs = _mxfp4(xt, xs, "x")
        xs_ptr = xs.data_ptr()
    else:
        xt, xs_ptr = _dev(x, "x", torch.bfloat16), None
    p, s = _mxfp4(p, s, "weights", xt.device)
    y = _out(out, (m, n), y_dtype, xt.device)
    if m == 0 or n == 0:
        return y
    if k == 0:
        return y.zero_()
    need = _lib.load().chadq_product_mxfp4_workspace_bytes(m, n, k, int(x_mx))
    ws = torch.empty(need, dtype=torch.uint8, device=xt.device) if need else None  # a fresh one per call, as moe_ffn's
    _launch(xt.device, "chadq_product_mxfp4", xt.data_ptr(), xs_ptr, p.data_ptr(), s.data_ptr(), y.data_ptr(), int(y_dtype == torch.bfloat16), m, n, k,
            ws.data_ptr() if need else None, need)
    return y


def _no_mxfp4(x, qw) -> None:
    if isinstance(x, (QWeightMXFP4, QExpertsMXFP4)):
        raise TypeError("MXFP4 activations go with MXFP4 weights, got %r" % type(qw))


def _rows_of(x: torch.Tensor, k: int, qw: QWeight) -> int:
    """M of activations [M,k]."""
    try:
        m, xk = x.shape
    except (AttributeError, ValueError):
        _no_mxfp4(x, qw)
        m, xk = 0, -1
    if xk != k:
        raise ValueError("x must be [M,%d], got %s" % (k, tuple(x.shape)))
    return m


def qgemm_grouped(x: Union[torch.Tensor, QWeightMXFP4], experts: QExpertsMXFP4, offsets: torch.Tensor,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows sorted by expert, each group times its own matrix: y[r] = x[r] @ dequant(experts[e]).T for offsets[e] <= r < offsets[e+1].

    x bf16 [R,K] or QWeightMXFP4 of R rows; offsets int32 [E+1] on the GPU, read there (groups of any size, empty ones too, no host round trip); y bf16
    [R,N], fp32 sums.  Rows in front of offsets[0] and behind offsets[E] are 0 in a fresh result and left as they are in `out`.  Offsets beyond [0, R] count as its ends, one
    that descends as the largest before it."""
    if out is None:
        y = _lib.native().grouped(x, experts, offsets)
        if y is not None:
            return y
    if not isinstance(experts, QExpertsMXFP4):
        raise TypeError("qgemm_grouped wants QExpertsMXFP4, got %r" % type(experts))
    xt, xs = _rows(x)
    x_mx = xs is not None
    p, s = _arrays(experts)
    e, n, k = p.size(0), p.size(1), p.size(2) * 2
    if xt.dim() != 2 or xt.size(1) * (2 if x_mx else 1) != k:
        raise ValueError("x must be [R,%d], got %s" % (k, (xt.size(0), xt.size(1) * 2) if x_mx else tuple(x.shape)))
    if x_mx:
        xt, xs = _mxfp4(xt, xs, "x")
        xs_ptr = xs.data_ptr()
    else:
        xt, xs_ptr = _dev(x, "x", torch.bfloat16), None
    p, s = _mxfp4(p, s, "experts", xt.device)
    offsets = _dev(offsets, "offsets", torch.int32)
    if e < 1 or tuple(offsets.shape) != (e + 1,) or offsets.device != xt.device:
        raise ValueError("offsets must be int32 [%d] on %s, one more than there are experts (at least one), got %s on %s"
                         % (e + 1, xt.device, tuple(offsets.shape), offsets.device))
    y = _out(out, (xt.size(0), n), torch.bfloat16, xt.device)
    if y.numel() == 0:
        return y
    if k == 0:
        raise ValueError("K must be at least 32")
    _launch(xt.device, "chadq_product_mxfp4_grouped", xt.data_ptr(), xs_ptr, p.data_ptr(), s.data_ptr(), offsets.data_ptr(), y.data_ptr(), xt.size(0), e, n, k,
            int(out is None))
    return y


def qgemv(x: Union[torch.Tensor, QWeightMXFP4], qw: QWeight, out: Optional[torch.Tensor] = None, *, fp32_elements: bool = False) -> torch.Tensor:
    """Decode product, fp32 out [M,N], M <= 16.  x is bf16 [M,K] for int4 weights, fp32 [M,K] for int8 weights, bf16 [M,K] or
    QWeightMXFP4 for MXFP4 weights.

    fp32_elements (int8 weights only): fp32 arithmetic on every activation (chadq_gemv_i8row_fp32) instead of the
    matrix-core kernel's per-block fixed point, whose error on a small activation grows with the largest one of its
    2048-k block; the weights are then streamed once per pair of activation rows."""
    return _gemv(x, qw, out, fp32_elements, False)


def _gemv(x: torch.Tensor, qw: QWeight, out: Optional[torch.Tensor], fp32_elements: bool, bf16_out: bool) -> torch.Tensor:
    """qgemv with the sums as fp32 or, bf16_out, rounded to bf16 by the kernel that forms them."""
    lib = _lib.load()
    y_dtype = torch.bfloat16 if bf16_out else torch.float32
    if isinstance(qw, QWeightInt4G32):
        w, s, n, k = _int4(qw)
    elif isinstance(qw, QWeightInt8):
        w, s, n, k = _int8(qw)
    elif isinstance(qw, QWeightMXFP4):
        if fp32_elements:
            raise ValueError("fp32_elements applies to int8 weights (fp32 activations) only")
        xt = _rows(x)[0]
        m = xt.size(0) if xt.dim() == 2 else 0
        if m > GEMV_MAX_M:
            raise ValueError("qgemv takes at most %d rows, got %d" % (GEMV_MAX_M, m))
        return _product_mxfp4(x, qw, out, y_dtype)
    else:
        raise TypeError("unknown weight container %r" % type(qw))
    m = _rows_of(x, k, qw)
    if fp32_elements and not isinstance(qw, QWeightInt8):
        raise ValueError("fp32_elements applies to int8 weights (fp32 activations) only")
    if isinstance(qw, QWeightInt4G32):
        x = _dev(x, "x", torch.bfloat16)
        p, s = _dev(w, "packed", torch.uint8), _dev(s, "scale", torch.float16)
        y = _out(out, (m, n), y_dtype, x.device)
        name = "chadq_gemv_i4g32_bf16" if bf16_out else "chadq_gemv_i4g32"
        need = _lib.native().gemv_bytes(m, n, k, 0)  # as in qgemm
        if need:
            ws = x.new_empty(need, dtype=torch.uint8)
            _lib.check(lib.chadq_gemv_i4g32_ws(x.data_ptr(), p.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, int(bf16_out), ws.data_ptr(), need,
                                               _stream()), name)
            return y
        _lib.check(getattr(lib, name)(x.data_ptr(), p.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, _stream()), name)
        return y
    x = _dev(x, "x", torch.float32)
    w, s = _dev(w, "w", torch.int8), _dev(s, "scale", torch.float32)
    y = _out(out, (m, n), y_dtype, x.device)
    name = "chadq_gemv_i8row_fp32" if fp32_elements else "chadq_gemv_i8row_bf16" if bf16_out else "chadq_gemv_i8row"
    need = 0 if fp32_elements else _lib.native().gemv_bytes(m, n, k, 1)
    if need:
        ws = x.new_empty(need, dtype=torch.uint8)
        _lib.check(lib.chadq_gemv_i8row_ws(x.data_ptr(), w.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, int(bf16_out), ws.data_ptr(), need,
                                           _stream()), name)
        return y
    _lib.check(getattr(lib, name)(x.data_ptr(), w.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, _stream()), name)
    return y


def qgemm(x: Union[torch.Tensor, QWeightMXFP4], qw: QWeight, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Prefill product on the matrix cores: x bf16 [M,K], or QWeightMXFP4 for MXFP4 weights, -> bf16 [M,N], fp32 accumulate."""
    lib = _lib.load()
    if isinstance(qw, QWeightInt4G32):
        w, s, n, k = _int4(qw)
    elif isinstance(qw, QWeightInt8):
        w, s, n, k = _int8(qw)
    elif isinstance(qw, QWeightMXFP4):
        return _product_mxfp4(x, qw, out, torch.bfloat16)
    else:
        raise TypeError("unknown weight container %r" % type(qw))
    m = _rows_of(x, k, qw)
    x = _dev(x, "x", torch.bfloat16)
    y = _out(out, (m, n), torch.bfloat16, x.device)
    # Scratch for the K parts of a product of few tiles (0 bytes where one part is the quicker form): a fresh one per call, as moe_ffn's.
    if isinstance(qw, QWeightInt4G32):
        p, s = _dev(w, "packed", torch.uint8), _dev(s, "scale", torch.float16)
        need = _lib.native().gemm_bytes(m, n, k, 0)
        if need:
            ws = x.new_empty(need, dtype=torch.uint8)
            _lib.check(lib.chadq_gemm_i4g32_bf16_ws(x.data_ptr(), p.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, ws.data_ptr(), need, _stream()),
                       "chadq_gemm_i4g32_bf16")
            return y
        _lib.check(lib.chadq_gemm_i4g32_bf16(x.data_ptr(), p.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, _stream()), "chadq_gemm_i4g32_bf16")
        return y
    w, s = _dev(w, "w", torch.int8), _dev(s, "scale", torch.float32)
    need = _lib.native().gemm_bytes(m, n, k, 1)
    if need:
        ws = x.new_empty(need, dtype=torch.uint8)
        _lib.check(lib.chadq_gemm_i8row_bf16_ws(x.data_ptr(), w.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, ws.data_ptr(), need, _stream()),
                   "chadq_gemm_i8row_bf16")
        return y
    _lib.check(lib.chadq_gemm_i8row_bf16(x.data_ptr(), w.data_ptr(), s.data_ptr(), y.data_ptr(), m, n, k, _stream()), "chadq_gemm_i8row_bf16")
    return y


def qlinear(x: Union[torch.Tensor, QWeightMXFP4], qw: QWeight, *, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """y = x @ dequant(W).T over the last axis of x.

    Up to 16 rows go to the bandwidth-bound GEMV (fp32 result); more rows go to the MFMA GEMM (bf16 result).
    out_dtype picks the result type.  The GEMV writes bf16 itself if that is asked for (the same sums rounded once); any
    other type than the kernel's native one is a cast.  x may be a QWeightMXFP4, [M,K], where the weights are one.
    """
    native = _lib.native()
    y = native.linear(x, qw, out_dtype)
    if y is not None:
        return y
    if not isinstance(x, torch.Tensor):
        y = _qlinear_2d(x, qw, out_dtype if out_dtype == torch.bfloat16 else None)
        return y if out_dtype is None or y.dtype == out_dtype else y.to(out_dtype)
    # more dimensions, strides and a cast at the end are dealt with here, around the native call (8.7 -> 6.2 us of host time for an x of three
    # dimensions, 12.2 -> 9.8 with a cast)
    x2 = (x if x.dim() == 2 else x.reshape(-1, x.shape[-1])).contiguous()
    written = out_dtype if out_dtype == torch.bfloat16 else None
    y = native.linear(x2, qw, written) if x2 is not x or out_dtype is not written else None
    if y is None:
        y = _qlinear_2d(x2, qw, written)
    if out_dtype is not None and y.dtype != out_dtype:
        y = y.to(out_dtype)
    return y if x.dim() == 2 else y.reshape(*x.shape[:-1], qw.N)


def _qlinear_2d(x2: torch.Tensor, qw: QWeight, written: Optional[torch.dtype]) -> torch.Tensor:
    """What the native call leaves: misplaced or strided weights, other types, everything that raises."""
    if isinstance(qw, QWeightMXFP4):  # (no rows at all: an empty result, of the type that few rows have)
        few = _rows(x2)[0].size(0) <= GEMV_MAX_M
        return _product_mxfp4(x2, qw, None, torch.float32 if few and written is None else torch.bfloat16)
    _no_mxfp4(x2, qw)
    m = x2.size(0)
    use_gemv = m <= GEMV_MAX_M and not (isinstance(qw, QWeightInt8) and x2.dtype == torch.bfloat16)
    if isinstance(qw, QWeightInt8) and x2.dtype == torch.float32 and not use_gemv:
        raise ValueError("int8 weights with fp32 activations are served for at most %d rows" % GEMV_MAX_M)
    return _gemv(x2, qw, None, False, written is not None) if use_gemv else qgemm(x2, qw)


def moe_route(logits: torch.Tensor, top_k: int = 2, renorm: bool = True):
    """softmax over experts, top_k by logit (lowest index wins ties) -> (idx int32 [T,top_k], w fp32 [T,top_k])."""
    z = _dev(logits, "logits", torch.float32)
    t, e = z.shape
    idx = torch.empty(t, top_k, dtype=torch.int32, device=z.device)
    w = torch.empty(t, top_k, dtype=torch.float32, device=z.device)
    _lib.check(_lib.load().chadq_moe_route(z.data_ptr(), idx.data_ptr(), w.data_ptr(), t, e, top_k, int(renorm), _stream()),
               "chadq_moe_route")
    return idx, w


def _repack(w, to_tiles: bool):
    lib = _lib.load()
    p, s, n, k = _int4(w)
    p, s = _dev(p, "packed", torch.uint8), _dev(s, "scale", torch.float16)
    if n % 32 or k % 256:
        raise ValueError("tile order needs N %% 32 == 0 and K %% 256 == 0 (N=%d, K=%d)" % (n, k))
    po, so = torch.empty_like(p), torch.empty_like(s)
    fn = lib.chadq_repack_i4g32_tiles if to_tiles else lib.chadq_unrepack_i4g32_tiles
    _lib.check(fn(p.data_ptr(), s.data_ptr(), po.data_ptr(), so.data_ptr(), n, k, _stream()),
               "chadq_repack_i4g32_tiles" if to_tiles else "chadq_unrepack_i4g32_tiles")
    return po, so


def to_tiles(w: QWeightInt4G32) -> QWeightInt4G32Tiles:
    """Row-major int4 group-32 matrix (on the GPU) -> tile order, for the experts of moe_ffn.  Done once at load time."""
    if not isinstance(w, QWeightInt4G32):
        raise TypeError("to_tiles wants a QWeightInt4G32")
    return QWeightInt4G32Tiles(*_repack(w, True))


def to_rows(w: QWeightInt4G32Tiles) -> QWeightInt4G32:
    """The exact inverse of to_tiles."""
    if not isinstance(w, QWeightInt4G32Tiles):
        raise TypeError("to_rows wants a QWeightInt4G32Tiles")
    return QWeightInt4G32(*_repack(w, False))


def moe_ffn(x: torch.Tensor, logits: torch.Tensor, experts, *, top_k: int = 2, renorm: bool = True) -> torch.Tensor:
    """SiLU-gated mixture of experts.  x bf16 [T,H], logits fp32 [T,E]; experts: sequence of (gate, up, down)
    triples with gate/up [F,H] and down [H,F], all QWeightInt4G32 or all QWeightInt4G32Tiles (to_tiles(): faster from
    some 16 tokens on).  Dequantised weights are rounded to bf16 (row order) or fp16 (tile order), so the two orders agree within
    rounding; at most 16 tokens take exact weights in row order and, where the experts hit hold at most 64 MB, in tile order
    too, with the same bits from both.  Or experts is one triple of QExpertsMXFP4, gate and up [E,F,H] and down [E,H,F]: weights multiplied as
    they are.  Returns bf16 [T,H]."""
    several = isinstance(experts, (tuple, list))
    if several and experts and isinstance(experts[0], QExpertsMXFP4):
        return _moe_ffn_mxfp4(x, logits, experts, top_k, renorm)
    y = _lib.native().moe_ffn(x, logits, experts, top_k, renorm)
    if y is not None:
        return y
    if several and any(isinstance(m, QExpertsMXFP4) for m in experts):  # (not a triple: refused there.  Here, as a look at each of 16 experts takes 1 us)
        return _moe_ffn_mxfp4(x, logits, experts, top_k, renorm)
    lib = _lib.load()  # (as in qlinear)
    x = _dev(x, "x", torch.bfloat16)
    z = _dev(logits, "logits", torch.float32)
    t, h = x.shape
    e = len(experts)
    if z.shape != (t, e):
        raise ValueError("logits must be [%d,%d]" % (t, e))
    f = experts[0][0].N
    kinds = {type(m) for tr in experts for m in tr}
    if kinds not in ({QWeightInt4G32}, {QWeightInt4G32Tiles}):
        raise TypeError("the experts' matrices must all be QWeightInt4G32 or all QWeightInt4G32Tiles")
    tiled = kinds == {QWeightInt4G32Tiles}
    arr = (_lib.MoeExpertI4G32 * e)()
    keep = []
    for i, (g, u, d) in enumerate(experts):
        if (g.N, g.K) != (f, h) or (u.N, u.K) != (f, h) or (d.N, d.K) != (h, f):
            raise ValueError("expert %d: gate/up must be [%d,%d] and down [%d,%d]" % (i, f, h, h, f))
        ts = []
        for m, name in ((g, "gate "), (u, "up "), (d, "down ")):
            p, s, _, _ = _int4(m, name)
            ts += [_dev(p, name + "packed", torch.uint8), _dev(s, name + "scale", torch.float16)]
        keep.append(ts)
        arr[i] = _lib.MoeExpertI4G32(*[v.data_ptr() for v in ts])
    need = lib.chadq_moe_ffn_i4g32_workspace_bytes(t, h, f, e, top_k)
    if need == 0:
        raise ValueError("unsupported MoE sizes T=%d H=%d F=%d E=%d top_k=%d" % (t, h, f, e, top_k))
    # The workspace holds the router's output and every intermediate of the call.  A fresh one each time, from torch's
    # allocator: calls in flight on other streams have their own, a later call on this stream may reuse the memory, a
    # captured graph's stays with the graph, and none is kept for a number of tokens that does not come again (480 MiB
    # at 512 tokens, top 4, 4096 x 14336).
    ws = x.new_empty(need, dtype=torch.uint8)
    y = torch.empty(t, h, dtype=torch.bfloat16, device=x.device)
    fn = lib.chadq_moe_ffn_i4g32_tiled if tiled else lib.chadq_moe_ffn_i4g32
    _lib.check(fn(x.data_ptr(), z.data_ptr(), arr, y.data_ptr(), t, h, f, e, top_k, int(renorm), ws.data_ptr(), need, _stream()),
               "chadq_moe_ffn_i4g32_tiled" if tiled else "chadq_moe_ffn_i4g32")
    return y


def _moe_ffn_mxfp4(x: torch.Tensor, logits: torch.Tensor, experts, top_k: int, renorm: bool) -> torch.Tensor:
    y = _lib.native().moe_ffn_mx(x, logits, experts, top_k, renorm)
    if y is not None:
        return y
    if len(experts) != 3 or not all(isinstance(m, QExpertsMXFP4) for m in experts):
        raise TypeError("MXFP4 experts are one (gate, up, down) triple of QExpertsMXFP4")
    arrays = [_arrays(m) for m in experts]
    x, z = _dev(x, "x", torch.bfloat16), _dev(logits, "logits", torch.float32)
    if x.dim() != 2:
        raise ValueError("x must be [T,H], got %s" % (tuple(x.shape),))
    (e, f, kh), up, down = ((p.size(0), p.size(1), p.size(2) * 2) for p, _ in arrays)  # [E,F,H], the same, [E,H,F]
    t, h = x.shape
    if tuple(z.shape) != (t, e) or z.device != x.device:
        raise ValueError("logits must be [%d,%d] on %s" % (t, e, x.device))
    if kh != h or up != (e, f, h) or down != (e, h, f):
        raise ValueError("gate and up must be [%d,%d,%d] and down [%d,%d,%d]" % (e, f, h, e, h, f))
    lib = _lib.load()
    y = torch.empty(t, h, dtype=torch.bfloat16, device=x.device)
    need = lib.chadq_moe_ffn_mxfp4_workspace_bytes(t, h, f, e, top_k)
    if need == 0:
        raise ValueError("unsupported MoE sizes T=%d H=%d F=%d E=%d top_k=%d" % (t, h, f, e, top_k))
    ts = [v for name, ps in zip(("gate", "up", "down"), arrays) for v in _mxfp4(*ps, name, x.device)]
    arr = _lib.MoeMXFP4(*[v.data_ptr() for v in ts])
    ws = torch.empty(need, dtype=torch.uint8, device=x.device)  # as moe_ffn's
    _launch(x.device, "chadq_moe_ffn_mxfp4", x.data_ptr(), z.data_ptr(), ctypes.byref(arr), y.data_ptr(), t, h, f, e, top_k, int(renorm), ws.data_ptr(), need)
    return y
