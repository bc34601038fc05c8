"""The norms around a decoder's blocks, over libdmx_radix.so
(include/dmx_norm.h). No drinkme counterpart: drinkme leaves these to the
model's own code.

  norm(x, weight)                  each row's norm: of tokens, or of every head of q or k
  block_norm(y, residual, weight)  a block's output into the residual stream, with the norm after
                                   the block, its gate and factor, and the norm and modulation in
                                   front of the next block, in one launch

Both norms are root-mean-square ("rms") or layer norms ("layer"):

  rms    v / sqrt(mean(v^2) + eps) * (weight + offset) + bias
  layer  (v - mean(v)) / sqrt(mean((v - mean(v))^2) + eps) * (weight + offset) + bias

Rows and vectors are bf16 or fp32; everything between is fp32 (a sum of squares past
its range is an infinity) and each output is rounded once. Every call launches on torch's
current stream and allocates its outputs with torch. There is no gradient: a call refuses
tensors that ask for one or carry a tangent.
"""

from __future__ import annotations

import ctypes as ct
import math

import torch

from . import _native
from .kv_ops import _MOST, _current, _no_gradient
from .radix_ops import _dtype_code, _stream

KINDS = {"rms": _native.NORM_RMS, "layer": _native.NORM_LAYER}


def _rows_of(x, what, dims):
    """x, bf16 or fp32 on the GPU with adjacent channels, of one of `dims` dimensions."""
    if x.dim() not in dims or x.shape[-1] < 1 or x.shape[-1] > _native.NORM_MAX_DIM:
        raise ValueError(f"{what}: {' or '.join(map(str, dims))} dimensions, rows of 1..{_native.NORM_MAX_DIM}, got {tuple(x.shape)}")
    if x.device.type != "cuda":
        raise ValueError(f"{what} is not on the GPU")
    _dtype_code(x.dtype, what)
    if max(x.shape) >= _MOST:
        raise ValueError(f"{what}: {tuple(x.shape)}, 2^30 or more rows")
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()


def _vectors(v, what, dim, device, rows=(1,)):
    """The dmx_vectors of v [dim] or [n, dim], n one of `rows` (None: any), and what it points into."""
    out = _native.Vectors()
    if v is None:
        return out, None
    shape = tuple(v.shape)
    n = 1 if v.dim() == 1 else shape[0] if v.dim() == 2 else -1
    if n < 0 or shape[-1] != dim or v.device != device or (rows is not None and n not in rows):
        raise ValueError(f"{what}: {'x'.join(map(str, shape))} on {v.device} for rows of {dim} on {device}")
    if n < 1 or n >= _MOST:
        raise ValueError(f"{what}: {n} rows")
    out.dtype = _dtype_code(v.dtype, what)
    v = v.contiguous()
    out.at, out.rows = v.data_ptr(), n
    return out, v


def _form(kind, eps, offset, factor, what):
    if kind not in KINDS:
        raise ValueError(f"{what}: kind {kind!r} is not 'rms' or 'layer'")
    if not (eps >= 0 and math.isfinite(eps) and math.isfinite(offset) and math.isfinite(factor)):
        raise ValueError(f"{what}: eps {eps}, offset {offset}, factor {factor}: finite numbers, eps 0 or more")
    f = _native.NormForm()
    f.kind, f.eps, f.offset, f.factor = KINDS[kind], eps, offset, factor
    return f


def norm(x: torch.Tensor, weight=None, *, bias=None, kind: str = "rms", eps: float = 1e-6, offset: float = 0.0) -> torch.Tensor:
    """Each row of x [T, D] or [T, H, D] (views of a fused product are read in
    place) normed, dense and in x's dtype. weight and bias: [D], or None. `offset`
    is added to the weights (1 where they are kept as their difference from 1)."""
    native = _native.calls()
    if native is not None:  # the plain case in one native call; None: anything else
        out = native.norm(x, weight, bias, KINDS.get(kind, -1), eps, offset, _current(x))
        if out is not None:
            return out
    _no_gradient("norm", x, weight, bias)
    x = _rows_of(x, "norm: x", (2, 3))
    f = _form(kind, eps, offset, 1.0, "norm")
    D = x.shape[-1]
    f.weight, weight = _vectors(weight, "norm: weight", D, x.device)
    f.bias, bias = _vectors(bias, "norm: bias", D, x.device)
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.numel() == 0:
        return out
    r = _native.KvRows()
    r.at, r.token_stride = x.data_ptr(), x.stride(0)
    r.head_stride, r.heads = (x.stride(1), x.shape[1]) if x.dim() == 3 else (0, 1)
    err = _native.error_buffer()
    with torch.cuda.device(x.device):
        st = _native.lib().dmx_norm(ct.byref(r), out.data_ptr(), x.shape[0], D, _dtype_code(x.dtype, "norm"), ct.byref(f),
                                    _stream(x.device), err, len(err))
    _native.check(st, err, "dmx_norm")
    return out


def block_norm(y: torch.Tensor, residual: torch.Tensor, weight=None, *, bias=None, post=None, gate=None, factor: float = 1.0,
               modulate=None, cu=None, kind: str = "rms", eps: float = 1e-6, offset: float = 0.0):
    """A block's output y [T, D] into the residual stream [T, D], and the norm in
    front of the next block:

      residual' = residual + factor * gate * (N(y; post) if post is given else y)
      x         = N(residual'; weight, bias) * (1 + scale) + shift

    -> (residual' in residual's dtype, x in y's dtype), dense. The residual has y's dtype
    or is fp32; it goes into the second norm before its rounding. weight, bias and post: [D]. gate, and
    modulate = (scale, shift): [D] or [n, D], one row for every T / n rows of y one after the
    other, or, with `cu` (int32 [n + 1] on the GPU: offsets of n sequences), one for
    rows cu[i] .. cu[i + 1] - 1 (rows before and behind: the nearest sequence's)."""
    scale, shift = modulate if modulate is not None else (None, None)
    if modulate is not None and (scale is None or shift is None):
        raise ValueError("block_norm: modulate is a scale and a shift")
    native = _native.calls()
    if native is not None:
        outs = native.block_norm(y, residual, weight, bias, post, gate, factor, scale, shift, cu, KINDS.get(kind, -1), eps, offset,
                                 _current(y))
        if outs is not None:
            return outs
    _no_gradient("block_norm", y, residual, weight, bias, post, gate, scale, shift)
    y = _rows_of(y, "block_norm: y", (2,))
    residual = _rows_of(residual, "block_norm: residual", (2,))
    T, D = y.shape
    if residual.shape != y.shape or residual.device != y.device or residual.dtype not in (y.dtype, torch.float32):
        raise ValueError(f"block_norm: a residual {residual.dtype} {tuple(residual.shape)} on {residual.device} beside y {y.dtype} "
                         f"{tuple(y.shape)} on {y.device}")
    f = _form(kind, eps, offset, factor, "block_norm")
    f.weight, weight = _vectors(weight, "block_norm: weight", D, y.device)
    f.bias, bias = _vectors(bias, "block_norm: bias", D, y.device)
    f.post, post = _vectors(post, "block_norm: post", D, y.device)
    f.gate, gate = _vectors(gate, "block_norm: gate", D, y.device, None)
    f.scale, scale = _vectors(scale, "block_norm: scale", D, y.device, None)
    f.shift, shift = _vectors(shift, "block_norm: shift", D, y.device, None)
    if modulate is not None and f.scale.rows != f.shift.rows:
        raise ValueError("block_norm: modulate is a scale and a shift of the same rows")
    batch = None
    if cu is not None:
        if cu.dtype != torch.int32 or cu.dim() != 1 or not 2 <= cu.shape[0] < _MOST or cu.device != y.device:
            raise ValueError(f"block_norm: cu must be int32 [sequences + 1] on {y.device}, got {cu.dtype} {tuple(cu.shape)} on {cu.device}")
        cu = cu.contiguous()
        f.cu, f.batch = cu.data_ptr(), cu.shape[0] - 1
        batch = f.batch
    for what, v in (("gate", f.gate), ("modulate", f.scale)):
        if v.at and v.rows not in (1, batch) and T % v.rows:
            raise ValueError(f"block_norm: {what} of {v.rows} rows for {T}")
    out = torch.empty(y.shape, dtype=y.dtype, device=y.device)
    stream = torch.empty(residual.shape, dtype=residual.dtype, device=y.device)
    err = _native.error_buffer()
    with torch.cuda.device(y.device):
        st = _native.lib().dmx_block_norm(y.data_ptr(), y.stride(0), residual.data_ptr(), residual.stride(0), stream.data_ptr(),
                                          out.data_ptr(), T, D, _dtype_code(y.dtype, "block_norm"),
                                          _dtype_code(residual.dtype, "block_norm"), ct.byref(f), _stream(y.device), err, len(err))
    _native.check(st, err, "dmx_block_norm")
    return stream, out
