"""MI355X: the norms around a block (drinkme_amd.norm_ops), against 64 bits within
bounds from their arithmetic."""

import numpy as np
import pytest
import torch

from drinkme_amd import _native, norm_ops
from tests.blocks_reference import standard
from tests.test_gpu_kv import DT, f64

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
# A sum over a row is a chain of 8 * 4 terms a lane and ten sums of lanes and waves: below 64
# roundings of what its absolute terms add up to; a root, a quotient and the factors of an
# element are a few more, of its size.
SUM, FEW = 64, 12


def half(dtype):
    return 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24


def norm_off(v, off, size, kind, eps):
    """How far N(v) may be from 64 bits' where each element of v is off by up to `off` and
    has terms of `size`: the mean's error and the elements' own, against the root; and the root's, of its
    square's sum."""
    n = standard(v, kind, eps)
    if kind == "layer":
        off = off + (off.mean(-1, keepdims=True) + SUM * U * np.abs(v).mean(-1, keepdims=True)) + U * size
        v = v - v.mean(-1, keepdims=True)
    square = (v * v).mean(-1, keepdims=True)
    root = np.sqrt(square + eps)
    d = (2 * np.abs(v) * off + off * off).mean(-1, keepdims=True) + SUM * U * ((np.abs(v) + off) ** 2).mean(-1, keepdims=True)
    ratio = np.minimum(d / (square + eps), 0.5)  # 1 / sqrt(1 - r) - 1 <= r for r up to 1 / 2
    return off / root * (1 + ratio) + np.abs(n) * (ratio + FEW * U)


def check_block(got, y, residual, dtype, rdtype, kind, eps, offset, factor, weight, bias, post, gate, modulate):
    """gate, scale and shift: 64 bits, a row for each row of y (or None)."""
    y, residual = f64(y), f64(residual)
    z, off = y, np.zeros_like(y)
    if post is not None:
        w = f64(post) + offset
        off = norm_off(y, off, np.abs(y), kind, eps) * np.abs(w)
        z = standard(y, kind, eps) * w
        off += FEW * U * np.abs(z)
    if gate is not None:
        z, off = z * gate, off * np.abs(gate) + U * np.abs(z * gate)
    r = residual + factor * z
    off = abs(factor) * off + 2 * U * (np.abs(residual) + np.abs(factor * z))
    bound = off + half(rdtype) * (np.abs(r) + off) + 1e-40
    assert got[0].dtype == DT[rdtype] and got[0].is_contiguous() and (np.abs(f64(got[0]) - r) <= bound).all()
    n, off = standard(r, kind, eps), norm_off(r, off, np.abs(residual) + np.abs(factor * z), kind, eps)
    if weight is not None:
        w = f64(weight) + offset
        n, off = n * w, off * np.abs(w) + FEW * U * np.abs(n * w)
    if bias is not None:
        n = n + f64(bias)
        off = off + U * np.abs(n)
    if modulate is not None:
        scale, shift = modulate
        off = off * np.abs(1 + scale) + FEW * U * (np.abs(n * (1 + scale)) + np.abs(n) + np.abs(shift))
        n = n * (1 + scale) + shift
    bound = off + half(dtype) * (np.abs(n) + off) + 1e-40
    assert got[1].dtype == DT[dtype] and got[1].is_contiguous() and (np.abs(f64(got[1]) - n) <= bound).all()


def randn(rng, shape, dtype, scale=1.0, mean=0.0):
    return torch.from_numpy((mean + scale * rng.standard_normal(shape)).astype(np.float32)).cuda().to(DT[dtype])


def rows_of(v, T):
    return None if v is None else np.repeat(f64(v).reshape(-1, v.shape[-1]), T // (1 if v.dim() == 1 else v.shape[0]), 0)


DIMS = [1, 2, 7, 8, 64, 100, 127, 128, 129, 136, 511, 512, 520, 1000, 1024, 1032, 1536, 2047, 2048, 2056, 4095, 4096, 4104, 5000,
        8192, 8200, 11111, 16384, 16392, 32767, 32768]


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype, rdtype", [("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
def test_block_norm(dim, kind, dtype, rdtype):
    """Every way a row is laid over lanes, whole and ragged, every part on and off."""
    rng = np.random.default_rng(dim)
    for T, full in ((5, True), (6, False), (1, True)):
        y, residual = randn(rng, (T, dim), dtype), randn(rng, (T, dim), rdtype, 4.0, 0.5)
        weight, bias, post = (randn(rng, (dim,), dtype, 0.2, m) for m in (0.0, 0.1, 0.0))
        gate, scale, shift = (randn(rng, (T, dim), dtype, 0.2) for _ in range(3))
        kw = dict(kind=kind, eps=1e-5, offset=1.0, factor=0.37)
        if full:
            got = norm_ops.block_norm(y, residual, weight, bias=bias, post=post, gate=gate, modulate=(scale, shift), **kw)
            check_block(got, y, residual, dtype, rdtype, kind, 1e-5, 1.0, 0.37, weight, bias, post, f64(gate), (f64(scale), f64(shift)))
        else:
            got = norm_ops.block_norm(y, residual, **kw)
            check_block(got, y, residual, dtype, rdtype, kind, 1e-5, 1.0, 0.37, None, None, None, None, None)


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_norm(dim, kind, dtype):
    rng = np.random.default_rng(dim + 1)
    for shape in ((1, dim), (37, dim), (3, 5, dim)):
        x, weight, bias = randn(rng, shape, dtype, 3.0, 1.0), randn(rng, (dim,), dtype, 0.2, 1.0), randn(rng, (dim,), dtype)
        got = norm_ops.norm(x, weight, bias=bias, kind=kind, eps=1e-6)
        v = f64(x)
        n, off = standard(v, kind, 1e-6) * f64(weight), norm_off(v, np.zeros_like(v), np.abs(v), kind, 1e-6) * np.abs(f64(weight))
        want = n + f64(bias)
        off = off + FEW * U * np.abs(n) + U * np.abs(want)
        assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
        assert (np.abs(f64(got) - want) <= off + half(dtype) * (np.abs(want) + off) + 1e-40).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_vectors_of_another_type(dtype):
    """fp32 weights and gates beside bf16 rows, and the other way."""
    rng = np.random.default_rng(2)
    other = "f32" if dtype == "bf16" else "bf16"
    y, residual = randn(rng, (6, 200), dtype), randn(rng, (6, 200), "f32")
    weight, post = randn(rng, (200,), other, 0.1, 1.0), randn(rng, (200,), dtype, 0.1, 1.0)
    gate, scale, shift = randn(rng, (200,), other), randn(rng, (2, 200), other), randn(rng, (2, 200), dtype)
    got = norm_ops.block_norm(y, residual, weight, post=post, gate=gate, modulate=(scale, shift))
    check_block(got, y, residual, dtype, "f32", "rms", 1e-6, 0.0, 1.0, weight, None, post, rows_of(gate, 6),
                (rows_of(scale, 6), rows_of(shift, 6)))


def test_rows_of_gates():
    """One row for all, one each, one for a run of rows, one for the sequences of cu (empty ones among them,
    and rows before the first and behind the last)."""
    rng = np.random.default_rng(3)
    T, D = 12, 264
    y, residual = randn(rng, (T, D), "bf16"), randn(rng, (T, D), "bf16")
    plain = norm_ops.block_norm(y, residual)
    for n in (1, 2, 3, 4, 6, 12):
        gate, scale, shift = (randn(rng, (n, D), "bf16") for _ in range(3))
        got = norm_ops.block_norm(y, residual, gate=gate, modulate=(scale, shift))
        check_block(got, y, residual, "bf16", "bf16", "rms", 1e-6, 0.0, 1.0, None, None, None, rows_of(gate, T),
                    (rows_of(scale, T), rows_of(shift, T)))
    assert not torch.equal(plain[0], got[0])
    for cu in ([0, 3, 3, 7, 12], [2, 3, 5, 9, 10], [0, 0, 0, 0, 12], [-5, 1, 4, 20, 30]):
        gate, scale, shift = (randn(rng, (4, D), "bf16") for _ in range(3))
        at = np.clip(np.searchsorted(np.asarray(cu[:4]), np.arange(T), side="right") - 1, 0, 3)
        got = norm_ops.block_norm(y, residual, gate=gate, modulate=(scale, shift), cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        check_block(got, y, residual, "bf16", "bf16", "rms", 1e-6, 0.0, 1.0, None, None, None, f64(gate)[at], (f64(scale)[at], f64(shift)[at]))
        one = norm_ops.block_norm(y, residual, gate=gate[0], modulate=(scale, shift), cu=torch.tensor(cu, dtype=torch.int32, device="cuda"))
        check_block(one, y, residual, "bf16", "bf16", "rms", 1e-6, 0.0, 1.0, None, None, None, rows_of(gate[0], T), (f64(scale)[at], f64(shift)[at]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_views(dtype):
    """Heads of a fused product, rows of a wider one, odd offsets, shared rows, channels not adjacent."""
    rng = np.random.default_rng(4)
    T, H, D = 11, 6, 96
    fused, odd = randn(rng, (T, H + 3, D), dtype), randn(rng, (T * D * 2 + 5,), dtype)
    weight = randn(rng, (D,), dtype)
    shifted = randn(rng, (D + 1,), dtype)[1:]
    for x in (fused[:, 1:1 + H], fused.transpose(0, 1), fused[:, 2], fused[::2, ::3], odd[5:].view(T, 2, D), odd[1:1 + T * D].view(T, D),
              fused[:1].expand(4, H + 3, D), randn(rng, (T, D, 3), dtype).transpose(1, 2)):
        for w in (weight, shifted):
            assert torch.equal(norm_ops.norm(x, w), norm_ops.norm(x.contiguous(), w.clone()))
    for y in (fused[:, 1], odd[3:3 + T * D].view(T, D), fused[:1, 0].expand(T, D)):
        for r in (fused[:, 2], odd[:T * D * 2].view(T, 2 * D)[:, 7:7 + D]):
            got, want = norm_ops.block_norm(y, r, shifted, gate=shifted), norm_ops.block_norm(y.contiguous(), r.contiguous(), shifted.clone(), gate=shifted.clone())
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_values_that_are_none():
    """A NaN or an infinity stays in its row; a row of zeros is zeros."""
    rng = np.random.default_rng(5)
    y, residual = randn(rng, (6, 700), "bf16"), randn(rng, (6, 700), "f32")
    clean = norm_ops.block_norm(y, residual, post=torch.ones(700, device="cuda"))
    y[1, 3], y[2, 699], residual[4, 0] = float("nan"), float("inf"), float("-inf")
    y[5], residual[5] = 0, 0
    got = norm_ops.block_norm(y, residual, post=torch.ones(700, device="cuda"))
    for a, b in zip(got, clean):
        assert torch.equal(a[[0, 3]], b[[0, 3]]) and not a[5].any()
        assert a[1].isnan().all()
    assert got[0][2].isnan().any() and got[1][4].isnan().any() and got[0][4].isinf().sum() == 1


def test_no_rows_another_stream_and_a_graph():
    rng = np.random.default_rng(6)
    empty = torch.empty((0, 64), device="cuda")
    assert norm_ops.norm(empty).shape == (0, 64) and norm_ops.norm(torch.empty((3, 0, 64), device="cuda")).shape == (3, 0, 64)
    assert [x.shape for x in norm_ops.block_norm(empty, empty)] == [(0, 64)] * 2
    y, residual = randn(rng, (9, 2048), "bf16"), randn(rng, (9, 2048), "f32")
    want = [x.clone() for x in norm_ops.block_norm(y, residual, kind="layer")]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    late = torch.zeros_like(y)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        late.copy_(y)
        got = norm_ops.block_norm(late, residual, kind="layer")
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = norm_ops.block_norm(late, residual, kind="layer")
    for _ in range(3):
        late.copy_(randn(rng, (9, 2048), "bf16"))
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(got, norm_ops.block_norm(late, residual, kind="layer")))


@pytest.mark.parametrize("native", [True, False])
def test_no_rows_beside_vectors_of_several(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_native, "calls", lambda: None)
    empty, some = torch.empty((0, 64), device="cuda"), torch.ones((3, 64), device="cuda")
    cu = torch.zeros(4, dtype=torch.int32, device="cuda")
    for kw in ({"gate": some}, {"modulate": (some, some)}, {"gate": some[:2], "cu": cu}, {"gate": some, "modulate": (some, some), "cu": cu}):
        assert [x.shape for x in norm_ops.block_norm(empty, empty, **kw)] == [(0, 64)] * 2


def test_many_rows():
    """More rows than a launch has at once; each as it is alone."""
    rng = np.random.default_rng(7)
    for shape in ((70001, 64), (5000, 2056)):
        x = randn(rng, shape, "bf16")
        got = norm_ops.norm(x)
        for r in (0, 1, shape[0] // 2, shape[0] - 1):
            assert torch.equal(got[r], norm_ops.norm(x[r:r + 1])[0])


def test_rows_past_a_launch():
    """More rows than one launch has lanes for: each of one channel, x / sqrt(x^2 + eps)."""
    rows = 2 ** 28 + 5
    x = torch.randn((rows, 1), device="cuda").bfloat16()
    weight = torch.tensor([1.5], device="cuda")
    got = norm_ops.norm(x, weight, eps=0.01)
    for at in range(0, rows, 2 ** 26):
        v = x[at:at + 2 ** 26].double()
        want = 1.5 * v / torch.sqrt(v * v + 0.01)
        off = (got[at:at + 2 ** 26].double() - want).abs()
        assert bool((off <= want.abs() * (half("bf16") * (1 + FEW * U) + FEW * U)).all()), at
    del x, got
    y = torch.randn((rows, 1), device="cuda").bfloat16()
    residual, out = norm_ops.block_norm(y, y.flip(0), eps=0.01, gate=torch.tensor([0.5], device="cuda"))
    for at in (0, 2 ** 28 - 40, rows - 40):
        v = y[at:at + 40].double() * 0.5 + y.flip(0)[at:at + 40].double()
        assert bool(((residual[at:at + 40].double() - v).abs() <= v.abs() * half("bf16") + 4 * U).all())
        assert bool(((out[at:at + 40].double() - v / torch.sqrt(v * v + 0.01)).abs() <= half("bf16") * (1 + FEW * U) + 64 * U).all())


def test_refusals():
    y = torch.zeros((4, 64), device="cuda", dtype=torch.bfloat16)
    one = torch.zeros(64, device="cuda")
    cu = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    for kw, match in (({"kind": "other"}, "kind"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"factor": float("inf")}, "factor"),
                      ({"residual": y[:3]}, "residual"), ({"y": y.float()}, "residual"),
                      ({"weight": one[:63]}, "weight"), ({"weight": one.cpu()}, "weight"), ({"post": torch.stack([one] * 4)}, "post"),
                      ({"gate": torch.stack([one] * 3)}, "gate of 3 rows"), ({"gate": one[None, None]}, "gate"),
                      ({"modulate": (one, None)}, "modulate"), ({"modulate": (one, torch.stack([one] * 4))}, "modulate"),
                      ({"gate": torch.stack([one] * 3), "cu": cu}, "gate of 3"), ({"cu": cu.long()}, "cu"), ({"cu": cu[:1]}, "cu"),
                      ({"y": y[0]}, "dimensions"), ({"y": y.cpu(), "residual": y.cpu()}, "GPU"), ({"gate": torch.zeros((0, 64), device="cuda")}, "gate")):
        with pytest.raises(ValueError, match=match):
            norm_ops.block_norm(**{"y": y, "residual": y, "weight": one, **kw})
    for x, match in ((torch.zeros((2, 32769), device="cuda"), "rows of"), (torch.zeros((2, 0), device="cuda"), "rows of"),
                     (torch.zeros(64, device="cuda"), "dimensions")):
        with pytest.raises(ValueError, match=match):
            norm_ops.norm(x)
    for call in (lambda: norm_ops.norm(y.half()), lambda: norm_ops.block_norm(y, y.half()), lambda: norm_ops.norm(y, one.half())):
        with pytest.raises(TypeError, match="not bf16 or fp32"):
            call()
    with pytest.raises(RuntimeError, match="no gradient"):
        norm_ops.norm(y, one.clone().requires_grad_())
    with pytest.raises(RuntimeError, match="no gradient"):
        norm_ops.block_norm(y, y, gate=one.clone().requires_grad_())
    with torch.no_grad():
        norm_ops.norm(y, one.clone().requires_grad_())
