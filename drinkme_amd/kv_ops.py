"""What a decoder does between its q/k/v and o projections, over
libdmx_radix.so (include/dmx_kv.h): rotary positions, a paged key/value cache
held in 4 bits, and the attention that reads it. No drinkme counterpart:
drinkme leaves these to the model's own code.

  rotary_table(positions, dim, ...)   the cos/sin table, plain or scaled to a long context
  rotary(q, k, positions, table)      both rotated, one launch
  new_cache(pages, page_size, heads, dim)
                                      an empty cache: a dict of four tensors
  append(cache, k, v, ...)            new tokens into the cache, keys (and q) rotated on the way
  read(cache, ...)                    new tokens as the cache holds them, bf16
  attention(q, cache, ...)            queries against everything cached of their sequences
  cache_bytes(cache)                  device bytes of a cache

The cache holds each token's keys and values, per head, as blocks of 32
channels: an exponent byte and 32 four-bit codes (4.25 bits a value; the format
is in include/dmx_kv.h). Every value it gives back is exactly a bf16 number.

Sequences. A call's new tokens lie one sequence after the other in [T, heads,
dim]. With `cu` None each of the B sequences has T / B of them; else sequence
b has rows cu[b] .. cu[b + 1] - 1. `lengths[b]` counts a sequence's tokens with
the new ones: append, read and attention of one step take the same `block_table`
[B, columns] (the page of each run of page_size positions; unused columns hold
anything), `lengths` and `cu`, int32 on the GPU. Nothing is copied to the host:
what only the GPU can see is checked there (include/dmx_kv.h says how).

Activations are bf16 or fp32. Every call launches on torch's current stream
and allocates its outputs (attention a workspace too) with torch. There is no
gradient: a call refuses tensors that ask for one or carry a tangent.
"""

from __future__ import annotations

import ctypes as ct
import math

import torch
from torch.autograd import forward_ad

from . import _native
from .radix_ops import _dtype_code, _stream

LAYOUTS = {"half": _native.ROTARY_HALF, "interleaved": _native.ROTARY_INTERLEAVED}
HEAD_DIMS = (64, 96, 128, 192, 256)
_MOST = 1 << 30  # positions of a table, tokens of a call: fewer (the C ABI's 32-bit fields hold them and their sums)

# ------------------------------------------------------------------ tables --


def _ramp(dim, base, original, fast, slow):
    """0 where an angle turns more than `fast` times in `original` positions,
    1 where less than `slow`, a line over the indices between."""
    def index(turns):
        return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(math.floor(index(fast)), 0), min(math.ceil(index(slow)), dim - 1)
    i = torch.arange(dim // 2, dtype=torch.float64)
    return ((i - low) / max(high - low, 1e-3)).clamp(0, 1)


def _frequencies(dim, base, scaling):
    """(angles a position, float64 [dim / 2]; the factor on cos and sin)."""
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = base ** (-2.0 * i / dim)
    if scaling is None:
        return f, 1.0
    s = dict(scaling)
    kind = s.pop("kind", None)
    try:
        if kind == "linear":
            f, magnitude = f / float(s.pop("factor")), 1.0
        elif kind == "base":
            f, magnitude = (base * float(s.pop("factor")) ** (dim / (dim - 2))) ** (-2.0 * i / dim), 1.0
        elif kind == "wavelength":
            turns = float(s.pop("original")) * f / (2 * math.pi)
            low, high = float(s.pop("low", 1.0)), float(s.pop("high", 4.0))
            keep = ((turns - low) / (high - low)).clamp(0, 1)
            f, magnitude = keep * f + (1 - keep) * f / float(s.pop("factor")), 1.0
        elif kind == "ramp":
            factor = float(s.pop("factor"))
            r = _ramp(dim, base, float(s.pop("original")), float(s.pop("fast", 32.0)), float(s.pop("slow", 1.0)))
            magnitude = s.pop("magnitude", None)
            magnitude = (0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0) if magnitude is None else float(magnitude)
            f = (1 - r) * f + r * f / factor
        elif kind == "divisors":
            f = f / torch.as_tensor(s.pop("divisors"), dtype=torch.float64).reshape(dim // 2)
            magnitude = float(s.pop("magnitude", 1.0))
        else:
            raise ValueError(f"rotary_table: unknown scaling {kind!r}")
    except KeyError as e:
        raise ValueError(f"rotary_table: {kind} scaling needs {e.args[0]!r}") from None
    if s:
        raise ValueError(f"rotary_table: {kind} scaling does not take {sorted(s)}")
    return f, magnitude


def rotary_table(positions: int, dim: int, base: float = 10000.0, scaling: dict | None = None,
                 device="cuda") -> torch.Tensor:
    """cos and sin of angle i (of dim / 2) at each position: fp32
    [positions, dim / 2, 2], computed in float64. `dim` counts the channels
    that turn, which may be part of the head. `scaling` stretches the
    positions for long contexts:

      {"kind": "linear", "factor"}    every angle / factor
      {"kind": "base", "factor"}      base * factor^(dim / (dim - 2))
      {"kind": "wavelength", "factor", "original", "low": 1, "high": 4}
                                      angles that turn less than `low` times in `original` positions / factor, more
                                      than `high` times kept, between them by the turns
      {"kind": "ramp", "factor", "original", "fast": 32, "slow": 1, "magnitude"}
                                      as above with a line over the angles' indices (YaRN), cos and sin times
                                      magnitude (0.1 ln factor + 1)
      {"kind": "divisors", "divisors", "magnitude": 1}
                                      each angle by its own divisor"""
    positions, dim = int(positions), int(dim)
    if positions < 1 or dim < 2 or dim % 2:
        raise ValueError(f"rotary_table: {positions} positions of {dim} channels (an even number, at least 2)")
    f, magnitude = _frequencies(dim, float(base), scaling)
    t = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * f.to(device)
    return torch.stack([t.cos() * magnitude, t.sin() * magnitude], -1).float()


# ------------------------------------------------------------------ checks --


def _current(x):
    """The handle of the current stream on x's device; 0 off the GPU, where
    the native call takes nothing."""
    return _stream(x.device) if x.is_cuda else 0


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(f"{what} has no gradient: call it under torch.no_grad(), or detach its inputs")
    if forward_ad._current_level >= 0 and torch._C._is_fwd_grad_enabled() and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{what} has no gradient, forward-mode tangents included: unpack its inputs")


def _activation(x, what, heads=None, dim=None, tokens=None, like=None):
    """x [tokens, heads, dim], bf16 or fp32 on the GPU, channels adjacent."""
    if x.dim() != 3:
        raise ValueError(f"{what}: [tokens, heads, dim], got {tuple(x.shape)}")
    if x.device.type != "cuda":
        raise ValueError(f"{what} is not on the GPU")
    _dtype_code(x.dtype, what)
    for name, want, have in (("tokens", tokens, x.shape[0]), ("heads", heads, x.shape[1]), ("channels", dim, x.shape[2])):
        if want is not None and want != have:
            raise ValueError(f"{what}: {have} {name}, not {want}")
    if like is not None and (x.dtype != like.dtype or x.device != like.device):
        raise ValueError(f"{what}: {x.dtype} on {x.device}, not {like.dtype} on {like.device}")
    if max(x.shape) >= _MOST:
        raise ValueError(f"{what}: {tuple(x.shape)}, 2^30 or more tokens, heads or channels")
    return x if x.stride(2) == 1 or x.shape[2] == 1 else x.contiguous()


def _rows(x):
    r = _native.KvRows()
    r.at, r.token_stride, r.head_stride, r.heads = x.data_ptr(), x.stride(0), x.stride(1), x.shape[1]
    return r


def _rotary_of(table, layout, dim, device, what):
    if layout not in LAYOUTS:
        raise ValueError(f"{what}: layout {layout!r} is not 'half' or 'interleaved'")
    if table.dim() != 3 or table.shape[2] != 2 or table.dtype != torch.float32:
        raise ValueError(f"{what}: the table is fp32 [positions, dim / 2, 2] (rotary_table), got {table.dtype} "
                         f"{tuple(table.shape)}")
    if 2 * table.shape[1] > dim:
        raise ValueError(f"{what}: a table of {2 * table.shape[1]} channels for heads of {dim}")
    if table.shape[0] >= _MOST:
        raise ValueError(f"{what}: a table of {table.shape[0]} positions, 2^30 or more")
    if table.device != device:
        raise ValueError(f"{what}: the table is not on {device}")
    table = table.contiguous()
    if table.data_ptr() % 16:  # (rows of an odd number of angles: a slice may begin between)
        table = table.clone()
    t = _native.KvRotaryTable()
    t.at, t.positions, t.dim, t.layout = table.data_ptr(), table.shape[0], 2 * table.shape[1], LAYOUTS[layout]
    return t, table


_CACHE = (("k_codes", torch.int32, 4), ("k_scales", torch.uint8, 4), ("v_codes", torch.int32, 5),
          ("v_scales", torch.uint8, 5))


def _cache_of(cache, what):
    """The dmx_kv_cache of a cache dict, after the checks of its tensors."""
    for name, dtype, dims in _CACHE:
        t = cache[name]
        if t.dtype != dtype or t.dim() != dims or not t.is_contiguous() or t.device.type != "cuda":
            raise ValueError(f"{what}: the cache's {name} must be {dtype}, dense, of {dims} dimensions, on the GPU")
    pages, heads, page, words = cache["k_codes"].shape
    shapes = {"k_scales": (pages, heads, page, words // 4), "v_codes": (pages, heads, page // 8, words, 8),
              "v_scales": (pages, heads, page // 8, words // 4, 8)}
    for name, shape in shapes.items():
        if tuple(cache[name].shape) != shape or cache[name].device != cache["k_codes"].device:
            raise ValueError(f"{what}: the cache's {name} is {tuple(cache[name].shape)}, not {shape} beside its k_codes")
    c = _native.KvCache()
    for name, _, _ in _CACHE:
        setattr(c, name, cache[name].data_ptr())
    c.pages, c.heads, c.page, c.dim = pages, heads, page, 8 * words
    return c


def _seqs_of(block_table, lengths, cu, total, max_tokens, device, what):
    """The dmx_kv_seqs of a call, and the tensors it points into."""
    if total < 0 or total >= _MOST:
        raise ValueError(f"{what}: {total} tokens (0 or more, fewer than 2^30)")
    named = [("block_table", block_table, 2), ("lengths", lengths, 1)] + ([("cu", cu, 1)] if cu is not None else [])
    held = []
    for name, t, dims in named:
        if t.dtype != torch.int32 or t.dim() != dims or t.device != device:
            raise ValueError(f"{what}: {name} must be int32 of {dims} dimension(s) on {device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        if max(t.shape) >= _MOST:
            raise ValueError(f"{what}: {name} is {tuple(t.shape)}, 2^30 or more sequences or columns")
        held.append(t.contiguous())
    batch = lengths.shape[0]
    if block_table.shape[0] != batch or (cu is not None and cu.shape[0] != batch + 1):
        raise ValueError(f"{what}: a block_table of {block_table.shape[0]} rows"
                         + (f" and cu of {cu.shape[0]}" if cu is not None else "") + f" for {batch} lengths")
    if batch == 0 or block_table.shape[1] == 0:
        raise ValueError(f"{what}: no sequences, or a block_table without columns")
    if cu is None and total % batch:
        raise ValueError(f"{what}: {total} tokens are not the same number for each of {batch} sequences, and cu is None")
    s = _native.KvSeqs()
    s.table, s.lengths, s.cu = held[0].data_ptr(), held[1].data_ptr(), held[2].data_ptr() if cu is not None else None
    s.batch, s.table_cols, s.total = batch, block_table.shape[1], total
    s.max_tokens = total // batch if cu is None else total if max_tokens is None else min(max_tokens, total)
    return s, held


# --------------------------------------------------------------- operators --


def rotary(q: torch.Tensor, k, positions: torch.Tensor, table: torch.Tensor, layout: str = "half"):
    """q [T, Hq, D] and k [T, Hk, D] (or None) rotated by `positions` [T]
    (int32 or int64): the pair (a, b) of angle t becomes a cos t - b sin t,
    b cos t + a sin t, in fp32, rounded once to their dtype. Pairs are channels
    (i, i + dim / 2) of the table's dim ("half") or (2 i, 2 i + 1)
    ("interleaved"); channels past the table's dim are copied. Views of a fused
    product are read in place. -> (q', k'), dense. A position outside the table
    gives NaN."""
    native = _native.calls()
    if native is not None:  # the plain case in one native call; None: anything else
        outs = native.rotary(q, k, positions, table, LAYOUTS.get(layout, -1), _current(q))
        if outs is not None:
            return outs
    _no_gradient("rotary", q, k, table)
    q = _activation(q, "rotary: q")
    ins = [q] if k is None else [q, _activation(k, "rotary: k", dim=q.shape[2], tokens=q.shape[0], like=q)]
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != q.shape[:1] or positions.device != q.device:
        raise ValueError(f"rotary: positions must be int32 or int64 [{q.shape[0]}] on {q.device}, got {positions.dtype} "
                         f"{tuple(positions.shape)} on {positions.device}")
    positions = positions.contiguous()
    t, table = _rotary_of(table, layout, q.shape[2], q.device, "rotary")
    outs = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in ins]
    n = len(ins)
    err = _native.error_buffer()
    with torch.cuda.device(q.device):
        st = _native.lib().dmx_rotary((_native.KvRows * n)(*map(_rows, ins)), (_native.KvRows * n)(*map(_rows, outs)), n,
                                      q.shape[0], q.shape[2], _dtype_code(q.dtype, "rotary"), positions.data_ptr(),
                                      positions.dtype == torch.int64, ct.byref(t), _stream(q.device), err, len(err))
    _native.check(st, err, "dmx_rotary")
    return outs[0], outs[1] if k is not None else None


def new_cache(pages: int, page_size: int, heads: int, dim: int, device="cuda") -> dict:
    """An empty cache of `pages` pages of page_size tokens (a power of two,
    8..1024) for `heads` key/value heads of `dim` channels (64, 96, 128, 192
    or 256): k_codes, k_scales, v_codes, v_scales."""
    if page_size < 8 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"new_cache: page_size {page_size} is not a power of two, 8..1024")
    if dim not in HEAD_DIMS:
        raise ValueError(f"new_cache: head dim {dim} is not one of {HEAD_DIMS}")
    if pages < 1 or heads < 1:
        raise ValueError(f"new_cache: {pages} pages of {heads} heads")
    shapes = {"k_codes": (pages, heads, page_size, dim // 8), "k_scales": (pages, heads, page_size, dim // 32),
              "v_codes": (pages, heads, page_size // 8, dim // 8, 8),
              "v_scales": (pages, heads, page_size // 8, dim // 32, 8)}
    return {name: torch.zeros(shapes[name], dtype=dtype, device=device) for name, dtype, _ in _CACHE}


def cache_bytes(cache: dict) -> int:
    """Device bytes of a cache."""
    return sum(cache[name].numel() * cache[name].element_size() for name, _, _ in _CACHE)


def append(cache: dict, k: torch.Tensor, v: torch.Tensor, block_table: torch.Tensor, lengths: torch.Tensor, *,
           cu=None, table=None, layout: str = "half", q=None):
    """The new tokens' k and v [T, H, D] into the cache, in place. With
    `table` (rotary_table's) keys are rotated by their positions, in fp32,
    before they are coded, and q [T, Hq, D], if given, is rotated in the same
    launch -> q' (else None). A token whose position has no page is dropped, and
    one of no sequence (before cu[0], from cu[B] on)."""
    native = _native.calls()
    if native is not None:
        out = native.append(cache, k, v, block_table, lengths, cu, table, LAYOUTS.get(layout, -1), q, _current(k))
        if out is not None:
            return out if q is not None else None
    _no_gradient("append", k, v, q, table)
    c = _cache_of(cache, "append")
    k = _activation(k, "append: k", heads=c.heads, dim=c.dim)
    v = _activation(v, "append: v", heads=c.heads, dim=c.dim, tokens=k.shape[0], like=k)
    if k.device != cache["k_codes"].device:
        raise ValueError("append: k is not on the cache's device")
    s, held = _seqs_of(block_table, lengths, cu, k.shape[0], None, k.device, "append")
    t = out = None
    if table is not None:
        t, table = _rotary_of(table, layout, c.dim, k.device, "append")
    elif q is not None:
        raise ValueError("append: q is rotated, which needs a table")
    if q is not None:
        q = _activation(q, "append: q", dim=c.dim, tokens=k.shape[0], like=k)
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    err = _native.error_buffer()
    with torch.cuda.device(k.device):
        st = _native.lib().dmx_kv_append(ct.byref(c), ct.byref(s), ct.byref(_rows(k)), ct.byref(_rows(v)),
                                         ct.byref(_rows(q)) if q is not None else None,
                                         ct.byref(_rows(out)) if q is not None else None, _dtype_code(k.dtype, "append"),
                                         ct.byref(t) if t is not None else None, _stream(k.device), err, len(err))
    _native.check(st, err, "dmx_kv_append")
    return out


def read(cache: dict, block_table: torch.Tensor, lengths: torch.Tensor, total: int, *, cu=None):
    """The keys and values of the last tokens of each sequence as the cache
    holds them, bf16 [total, H, D] each: `total` / B tokens of each sequence,
    or cu's (the tokens that append writes for the same arguments). A token
    whose position has no page reads NaN, and one of no sequence."""
    native = _native.calls()
    if native is not None:
        outs = native.read(cache, block_table, lengths, total, cu, _current(lengths))
        if outs is not None:
            return outs
    c = _cache_of(cache, "read")
    device = cache["k_codes"].device
    s, held = _seqs_of(block_table, lengths, cu, int(total), None, device, "read")
    k, v = (torch.empty((int(total), c.heads, c.dim), dtype=torch.bfloat16, device=device) for _ in range(2))
    err = _native.error_buffer()
    with torch.cuda.device(device):
        st = _native.lib().dmx_kv_read(ct.byref(c), ct.byref(s), k.data_ptr(), v.data_ptr(), _stream(device), err, len(err))
    _native.check(st, err, "dmx_kv_read")
    return k, v


def attention(q: torch.Tensor, cache: dict, block_table: torch.Tensor, lengths: torch.Tensor, *, cu=None,
              max_tokens: int | None = None, max_length: int | None = None, scale: float | None = None,
              causal: bool = True, window: int | None = None, return_lse: bool = False):
    """softmax(scale q k^T) v of the new tokens' queries q [T, Hq, D] (rotated
    already) over everything cached of their sequences -> [T, Hq, D] in q's
    dtype, and with return_lse each row's log-sum-exp, fp32 [T, Hq]. Hq is a
    multiple of the cache's heads, and query head g reads head g // (Hq / H).
    `scale` defaults to D^-0.5. A query at position p sees the positions of its
    sequence, with `causal` none after p, with `window` the last `window` of
    them (p among them); one that sees nothing gives zeros and -inf. With
    `cu`, max_tokens bounds the new tokens of a sequence (T where not given: the
    launch is shaped for that, many single tokens as for a prompt); a sequence's tokens past it, and tokens of no
    sequence (before cu[0], from cu[B] on), give NaN. `max_length`, a bound on `lengths` where the
    block table is wider than needed, shapes the launch only."""
    native = _native.calls()
    if native is not None:
        outs = native.attention(q, cache, block_table, lengths, cu, max_tokens, max_length or 0, scale, causal, window,
                                return_lse, _current(q))
        if outs is not None:
            return outs
    _no_gradient("attention", q)
    c = _cache_of(cache, "attention")
    q = _activation(q, "attention: q", dim=c.dim)
    if q.device != cache["k_codes"].device:
        raise ValueError("attention: q is not on the cache's device")
    T, Hq = q.shape[:2]
    if Hq == 0 or Hq % c.heads:
        raise ValueError(f"attention: {Hq} query heads over {c.heads} cached ones")
    if window is not None and window < 1:
        raise ValueError(f"attention: a window of {window}")
    if max_tokens is not None and (cu is None or max_tokens < 1):
        raise ValueError("attention: max_tokens, at least 1, goes with cu")
    if max_length is not None and max_length < 0:
        raise ValueError(f"attention: a max_length of {max_length}")
    if window is not None and window >= _MOST:  # past every table: none
        window = None
    max_length = min(max_length or 0, _MOST)
    s, held = _seqs_of(block_table, lengths, cu, T, max_tokens, q.device, "attention")
    out = torch.empty((T, Hq, c.dim), dtype=q.dtype, device=q.device)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    lib, code = _native.lib(), _dtype_code(q.dtype, "attention")
    scale = c.dim ** -0.5 if scale is None else float(scale)
    bytes_ = lib.dmx_kv_attention_workspace(ct.byref(c), ct.byref(s), Hq, code, max_length, window or 0) if T else 0
    ws = torch.empty(bytes_, dtype=torch.uint8, device=q.device) if bytes_ else None
    err = _native.error_buffer()
    with torch.cuda.device(q.device):
        st = lib.dmx_kv_attention(ct.byref(c), ct.byref(s), ct.byref(_rows(q)), code, scale, causal, window or 0,
                                  max_length, out.data_ptr(), lse.data_ptr() if return_lse else None,
                                  ws.data_ptr() if bytes_ else None, bytes_, _stream(q.device), err, len(err))
    _native.check(st, err, "dmx_kv_attention")
    return (out, lse) if return_lse else out
