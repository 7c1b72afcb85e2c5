"""The 8-bit linear layers of a DiT block on B200.

vidax computes its Dense layers in bf16 (WanDiTBlock, src/vidax/models/wan/
wan2_1/dit.py:78-156); this module is this library's 8-bit option for them.
A tensor is held as e4m3 values with a float32 scale for each block of 128
features (`Fp8Tensor`), and three kernels make and use it:

* `quantize_fp8`  -- a bf16 / float32 tensor as an Fp8Tensor;
* `add_norm`      -- the gated residual addition, RMSNorm or LayerNorm,
                     modulation, and the rounding to e4m3 (or bf16) in one
                     pass over the residual stream;
* `linear_fp8`    -- x @ w^T on the tensor cores' 8-bit path, with bias and
                     tanh GELU, its output in bf16, float32 or e4m3 again.

`vidax_b200.wan_dit.quantize_params` gives a whole DiT's weights this form.
Inference only, like the rest of this package: inputs that require a gradient
are refused while gradients are recorded. The operators keep nothing between
calls (no workspace), so any number of them may run at once and in captured
graphs; as with the other kernels, the first call on a device comes before a
capture.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib

BLOCK = 128

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float8_e4m3fn: 2}
_NORMS = {"rms": 0, "layer": 1}
_ACTS = {None: 0, "gelu_tanh": 1}


class QuantizeFp8Args(ctypes.Structure):
    _fields_ = [
        ("src", ctypes.c_void_p), ("dst", ctypes.c_void_p), ("scale", ctypes.c_void_p),
        ("src_stride", ctypes.c_int64), ("dst_stride", ctypes.c_int64),
        ("scale_stride", ctypes.c_int64 * 2),
        ("rows", ctypes.c_int64),
        ("dim", ctypes.c_int32), ("src_type", ctypes.c_int32), ("block_rows", ctypes.c_int32),
    ]


class AddNormArgs(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p), ("y", ctypes.c_void_p), ("sum", ctypes.c_void_p),
        ("gate", ctypes.c_void_p), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p),
        ("scale", ctypes.c_void_p), ("shift", ctypes.c_void_p),
        ("out", ctypes.c_void_p), ("out_scale", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64), ("y_stride", ctypes.c_int64),
        ("sum_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64),
        ("gate_stride", ctypes.c_int64), ("scale_stride", ctypes.c_int64),
        ("shift_stride", ctypes.c_int64),
        ("out_scale_stride", ctypes.c_int64 * 2),
        ("rows", ctypes.c_int64), ("rows_per_batch", ctypes.c_int64),
        ("dim", ctypes.c_int32), ("x_type", ctypes.c_int32), ("out_type", ctypes.c_int32),
        ("norm", ctypes.c_int32), ("eps", ctypes.c_float),
    ]


class LinearFp8Args(ctypes.Structure):
    _fields_ = [
        ("x", ctypes.c_void_p), ("x_scale", ctypes.c_void_p),
        ("w", ctypes.c_void_p), ("w_scale", ctypes.c_void_p),
        ("bias", ctypes.c_void_p), ("out", ctypes.c_void_p), ("out_scale", ctypes.c_void_p),
        ("x_stride", ctypes.c_int64), ("w_stride", ctypes.c_int64), ("out_stride", ctypes.c_int64),
        ("x_scale_stride", ctypes.c_int64 * 2), ("w_scale_stride", ctypes.c_int64 * 2),
        ("out_scale_stride", ctypes.c_int64 * 2),
        ("m", ctypes.c_int32), ("n", ctypes.c_int32), ("k", ctypes.c_int32),
        ("out_type", ctypes.c_int32), ("activation", ctypes.c_int32), ("variant", ctypes.c_int32),
    ]


class Fp8Tensor(NamedTuple):
    """e4m3 values with a float32 scale per block of 128 features.

    data:  (..., K) float8_e4m3fn, features contiguous.
    scale: activations (..., ceil(K / 128)), one scale per row and block;
           weights (N, K): (ceil(N / 128), ceil(K / 128)), one per 128 x 128
           block.
    """
    data: torch.Tensor
    scale: torch.Tensor

    def dequantize(self) -> torch.Tensor:
        """The float32 values this tensor stands for."""
        k = self.data.shape[-1]
        s = self.scale.repeat_interleave(BLOCK, dim=-1)[..., :k]
        if self.scale.shape[:-1] != self.data.shape[:-1]:
            s = s.repeat_interleave(BLOCK, dim=0)[:self.data.shape[0]]
        return self.data.float() * s


_entries = {}

# The argument structs' layouts for struct.pack: a ctypes.Structure takes
# three times as long to fill, a tenth of a small call.
_PACKED = {
    "vx_quantize_fp8": struct.Struct("@3P5q3i4x"),
    "vx_add_norm": struct.Struct("@10P11q4if4x"),
    "vx_linear_fp8": struct.Struct("@7P9q6i"),
}


def _entry(name: str, args=None):
    """The C entry point `name`: for a ctypes.Structure, or for its packed bytes."""
    fn = getattr(_lib.load(), name)
    fn = ctypes.CFUNCTYPE(ctypes.c_int, ctypes.c_char_p if args is None
                          else ctypes.POINTER(type(args)), ctypes.c_void_p)(
        ctypes.cast(fn, ctypes.c_void_p).value)
    if args is None:
        _entries[name] = (fn, _PACKED[name].pack)
    return fn


def _raw_stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# torch's own lookup of the handle, without the Stream object around it (3 us a call)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _raw_stream)


def _launch(name: str, device: torch.device, *args) -> None:
    if name not in _entries:
        _entry(name)
    fn, pack = _entries[name]
    if device.index == torch.cuda.current_device():
        rc = fn(pack(*args), _raw_stream(device.index))
    else:
        with torch.cuda.device(device):
            rc = fn(pack(*args), _raw_stream(device.index))
    if rc:
        _lib.check(rc)


def _check_cuda(name: str, t, dtypes, min_dim: int = 1) -> None:
    if (type(t) is torch.Tensor and t.dtype in dtypes and t.is_cuda and t.dim() >= min_dim
            and not t.requires_grad):
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.dim() < min_dim:
        raise ValueError(f"{name} must have at least {min_dim} dimensions, got shape {tuple(t.shape)}")
    if t.dtype not in dtypes:
        raise NotImplementedError(f"{name}.dtype={t.dtype}: the kernel takes "
                                  + " or ".join(str(d) for d in dtypes))
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this implementation has no CPU path)")
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} requires a gradient: this operator is inference only")


_INT_MAX = 2 ** 31 - 1
_FLT_MAX = (2 - 2 ** -23) * 2.0 ** 127


def _check_sizes(rows: int, *dims: int) -> None:
    """What the entry points' 32-bit sizes hold, and their indices past a row's end."""
    if rows > _INT_MAX or max(dims) > _INT_MAX - 4095:
        raise NotImplementedError(f"sizes {(rows, *dims)}: up to 2^31 - 1 rows of 2^31 - 4096 features are built")


def _row_stride(t: torch.Tensor) -> Optional[int]:
    """Elements between the consecutive rows (..., K) -> (rows, K) of `t`
    without a copy, or None where they are not evenly spaced."""
    k = t.shape[-1]
    if t.is_contiguous():
        return k
    if k > 1 and t.stride(-1) != 1:
        return None
    dims = [(n, s) for n, s in zip(t.shape[:-1], t.stride()[:-1]) if n != 1]
    for (_, s0), (n1, s1) in zip(dims, dims[1:]):
        if s0 != n1 * s1:
            return None
    stride = dims[-1][1] if dims else k
    return stride if stride >= k else None


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """`t` (a copy where its rows are not evenly spaced) and its row stride."""
    s = _row_stride(t)
    if s is None:
        t = t.contiguous()
        s = t.shape[-1]
    return t, s


def _empty_fp8(shape, device) -> Tuple[Fp8Tensor, int, int]:
    """An activation's storage: rows on 16-byte boundaries (the matrix
    product's loads need that), the scales of one block of features side by
    side (a warp of the matrix product reads those of 32 rows at once, the
    quantiser writes those of four). Returns it with the elements between its
    rows and between its blocks of scales."""
    *lead, k = shape
    rows = math.prod(lead)
    ld, ls = -(-k // 16) * 16, -(-rows // 4) * 4
    sd, ss = [ld, 1], [1, ls]
    for n in reversed(lead[1:]):
        sd.insert(0, sd[0] * n)
        ss.insert(0, ss[0] * n)
    data = torch.empty_strided(shape, sd, dtype=torch.float8_e4m3fn, device=device)
    scale = torch.empty_strided((*lead, -(-k // BLOCK)), ss, dtype=torch.float32, device=device)
    return Fp8Tensor(data, scale), ld, ls


def quantize_fp8(x: torch.Tensor, block_rows: int = 1) -> Fp8Tensor:
    """x (..., K) bf16 or float32 as e4m3 with float32 scales, one per row and
    128 features, or with block_rows = 128 (x a weight (N, K)) one per
    128 x 128 block:

        a = max(largest magnitude of the block, 2^-100)
        scale = a / 448,   data = e4m3(x * (448 / a)), round to nearest even

    A NaN stays a NaN in its place; a block with an infinity stands for NaN.
    """
    _check_cuda("x", x, (torch.bfloat16, torch.float32), 2)
    if block_rows not in (1, BLOCK):
        raise NotImplementedError(f"block_rows {block_rows}: 1 and {BLOCK} are built")
    if block_rows == BLOCK and x.dim() != 2:
        raise ValueError(f"a weight is (N, K), got {tuple(x.shape)}")
    if x.shape[-1] < 1:
        raise ValueError("x has no features")
    dev = x.device
    rows, k = math.prod(x.shape[:-1]), x.shape[-1]
    _check_sizes(rows, k)
    out, ld, ls = _empty_fp8(x.shape, dev)
    rs = 1
    if block_rows == BLOCK:
        rs, ls = -(-k // BLOCK), 1
        out = Fp8Tensor(out.data, torch.empty((-(-rows // BLOCK), rs), dtype=torch.float32, device=dev))
    if rows == 0:
        return out
    x, stride = _rows(x)
    _launch("vx_quantize_fp8", dev, x.data_ptr(), out.data.data_ptr(), out.scale.data_ptr(), stride,
            ld, rs, ls, rows, k, _TYPES[x.dtype], block_rows)
    return out


def _vector(name: str, t: Optional[torch.Tensor], shape, device):
    """A float32 vector (dim) or per-batch-item vector (B, dim) / (B, 1, dim)
    in place (converted where its type or layout differs): its address, its
    stride between batch items, and the tensor that holds it."""
    if t is None:
        return 0, 0, None
    if t.__class__ is torch.Tensor and t.dtype is torch.float32 and t.shape == shape \
            and t.device == device and not t.requires_grad and t.is_contiguous():
        return t.data_ptr(), shape[-1], t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} requires a gradient: this operator is inference only")
    if t.device != device:
        raise ValueError(f"{name} must live on x's device")
    if t.dim() == 3 and len(shape) == 2 and t.shape[1] == 1:
        t = t[:, 0]
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != torch.float32:
        t = t.to(torch.float32)
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    return t.data_ptr(), (t.stride(0) if len(shape) == 2 and shape[0] > 1 else 0), t


def add_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None,
             gate: Optional[torch.Tensor] = None, *, norm: str = "rms",
             weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
             scale: Optional[torch.Tensor] = None, shift: Optional[torch.Tensor] = None,
             eps: float = 1e-6, out_dtype: torch.dtype = torch.bfloat16,
             residual_out: Optional[torch.Tensor] = None):
    """The residual addition and the norm that follows it, in one pass:

        h = x + y * gate
        n = (h - m) / sqrt(mean((h - m)^2) + eps) * weight + bias
        out = n * (1 + scale) + shift

    with m = 0 (norm="rms") or mean(h) (norm="layer"). x: the residual stream
    (B, L, dim) or (L, dim), float32 or bf16; y: the sub-layer's output, bf16,
    or None (h = x). weight / bias: (dim); gate / scale / shift: (B, dim) or
    (B, 1, dim) ((1, dim) for a 2-D x). Each may be None. h is rounded to x's
    type and normalised as stored.

    Returns (out, h). out: bf16, or an Fp8Tensor for out_dtype
    torch.float8_e4m3fn. h: written to `residual_out` where that is given (x
    itself for an update in place, or a tensor apart from it; in either case
    apart from y and the five vectors, ValueError otherwise), else to a new
    tensor; x itself without y.
    """
    _check_cuda("x", x, (torch.float32, torch.bfloat16), 2)
    if x.dim() > 3:
        raise ValueError(f"x must be (B, L, dim) or (L, dim), got {tuple(x.shape)}")
    if norm not in _NORMS:
        raise ValueError(f"norm must be 'rms' or 'layer', got {norm!r}")
    if out_dtype not in (torch.bfloat16, torch.float8_e4m3fn):
        raise NotImplementedError(f"out_dtype {out_dtype}: bfloat16 and float8_e4m3fn are built")
    if not 0 <= eps <= _FLT_MAX:
        raise ValueError(f"eps must be >= 0 and finite in float32, got {eps}")
    dim = x.shape[-1]
    batch = x.shape[0] if x.dim() == 3 else 1
    if dim < 1:
        raise ValueError("x has no features")
    _check_sizes(batch * x.shape[-2], dim)
    if y is None:
        if gate is not None or residual_out is not None:
            raise ValueError("gate and residual_out belong to y")
    else:
        _check_cuda("y", y, (torch.bfloat16,))
        if y.shape != x.shape or y.device != x.device:
            raise ValueError(f"y {tuple(y.shape)} must have x's shape {tuple(x.shape)} and device")
    total = x
    if y is not None and residual_out is None:
        total = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    elif y is not None:
        total = residual_out
        if not isinstance(total, torch.Tensor):
            raise TypeError(f"residual_out must be a torch.Tensor, got {type(total).__name__}")
        if total.shape != x.shape or total.dtype != x.dtype or total.device != x.device:
            raise ValueError("residual_out must have x's shape, type and device")
        if _row_stride(total) is None:
            raise ValueError("residual_out must have evenly spaced rows of contiguous features")
        if total.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("residual_out requires a gradient: this operator is inference only")
    dev = x.device
    g, gs, _g = _vector("gate", gate, (batch, dim), dev)
    sc, scs, _sc = _vector("scale", scale, (batch, dim), dev)
    sh, shs, _sh = _vector("shift", shift, (batch, dim), dev)
    w, _, _w = _vector("weight", weight, (dim,), dev)
    b, _, _b = _vector("bias", bias, (dim,), dev)
    if out_dtype == torch.float8_e4m3fn:
        out, ld, ls = _empty_fp8(x.shape, dev)
        o, os = out.data.data_ptr(), out.scale.data_ptr()
    else:
        out = torch.empty(x.shape, dtype=out_dtype, device=dev)
        o, os, ld, ls = out.data_ptr(), 0, dim, 0
    rows = batch * x.shape[-2]
    if rows == 0:
        return out, total
    xr, x_stride = _rows(x)
    yp = sp = 0
    y_stride = s_stride = 0
    if y is not None:
        y, y_stride = _rows(y)
        yp, sp, s_stride = y.data_ptr(), total.data_ptr(), _row_stride(total)
    _launch("vx_add_norm", dev, xr.data_ptr(), yp, sp, g, w, b, sc, sh, o, os, x_stride, y_stride,
            s_stride, ld, gs, scs, shs, 1, ls, rows, x.shape[-2], dim, _TYPES[x.dtype],
            _TYPES[out_dtype], _NORMS[norm], eps)
    return out, total


def _fp8_rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """e4m3 rows on 16-byte boundaries (a padded copy where they are not) and
    their stride."""
    s = _row_stride(t)
    k = t.shape[-1]
    if s is not None and t.data_ptr() % 16 == 0 and (s % 16 == 0 or t.numel() == k):
        return t, -(-s // 16) * 16
    rows, ld = t.numel() // k, -(-k // 16) * 16
    buf = torch.empty((rows, ld), dtype=torch.uint8, device=t.device)
    buf[:, :k] = t.reshape(rows, k).view(torch.uint8)
    return buf, ld


def linear_fp8(x: Fp8Tensor, w: Fp8Tensor, bias: Optional[torch.Tensor] = None, *,
               activation: Optional[str] = None, out_dtype: torch.dtype = torch.bfloat16,
               variant: int = 0):
    """act(x @ w^T + bias) with x (..., K) quantised per row and w (N, K)
    quantised per 128 x 128 block (`quantize_fp8`), summed in float32:

        y[m, n] = sum_b x.scale[m, b] * w.scale[n // 128, b]
                        * sum_{k in block b} x.data[m, k] * w.data[n, k]

    bias: (N) or None; activation: None or "gelu_tanh". Returns (..., N) in
    out_dtype: bfloat16, float32, or (float8_e4m3fn) an Fp8Tensor with a scale
    per row and 128 columns, the next layer's input. Rows of x or w that do
    not lie on 16-byte boundaries are copied first; `quantize_fp8` and
    `add_norm` lay theirs out so. `variant` forces a kernel variant (tuning).
    """
    for name, t in (("x", x), ("w", w)):
        if not isinstance(t, tuple) or len(t) != 2:
            raise TypeError(f"{name} must be an Fp8Tensor, got {type(t).__name__}")
    xd, xs = x
    wd, ws = w
    _check_cuda("x.data", xd, (torch.float8_e4m3fn,), 2)
    _check_cuda("w.data", wd, (torch.float8_e4m3fn,), 2)
    _check_cuda("x.scale", xs, (torch.float32,), 2)
    _check_cuda("w.scale", ws, (torch.float32,), 2)
    if wd.dim() != 2 or wd.shape[0] < 1:
        raise ValueError(f"w.data must be (N, K), got {tuple(wd.shape)}")
    N, K = wd.shape
    if K < 1 or xd.shape[-1] != K:
        raise ValueError(f"x {tuple(xd.shape)} and w {tuple(wd.shape)} disagree on the features")
    kb = -(-K // BLOCK)
    if xs.shape != (*xd.shape[:-1], kb):
        raise ValueError(f"x.scale has shape {tuple(xs.shape)}, expected {(*xd.shape[:-1], kb)}")
    if ws.shape != (-(-N // BLOCK), kb):
        raise ValueError(f"w.scale has shape {tuple(ws.shape)}, expected {(-(-N // BLOCK), kb)}")
    dev = xd.device
    if not (dev == xs.device == wd.device == ws.device):
        raise ValueError("x and w must live on the same device")
    if activation not in _ACTS:
        raise NotImplementedError(f"activation {activation!r}: None and 'gelu_tanh' are built")
    if out_dtype not in _TYPES:
        raise NotImplementedError(f"out_dtype {out_dtype}: bfloat16, float32 and float8_e4m3fn are built")
    if variant not in range(5):
        raise ValueError(f"variant must be 0 to 4, got {variant!r}")
    shape = (*xd.shape[:-1], N)
    m = math.prod(shape[:-1])
    _check_sizes(m, N, K)
    bp, _, _bias = _vector("bias", bias, (N,), dev)
    if out_dtype == torch.float8_e4m3fn:
        out, ld, ls = _empty_fp8(shape, dev)
        o, os = out.data.data_ptr(), out.scale.data_ptr()
    else:
        out = torch.empty(shape, dtype=out_dtype, device=dev)
        o, os, ld, ls = out.data_ptr(), 0, N, 0
    if m == 0:
        return out
    xd, x_stride = _fp8_rows(xd)
    wd, w_stride = _fp8_rows(wd)
    if xs.dim() > 2:
        xs = xs.flatten(0, -2)
    _launch("vx_linear_fp8", dev, xd.data_ptr(), xs.data_ptr(), wd.data_ptr(), ws.data_ptr(), bp, o,
            os, x_stride, w_stride, ld, *xs.stride(), *ws.stride(), 1, ls, m, N, K,
            _TYPES[out_dtype], _ACTS[activation], int(variant))
    return out


def linear_fp8_flops(m: int, n: int, k: int) -> float:
    """FLOPs of one matrix product, 2*m*n*k."""
    return 2.0 * m * n * k
