"""MI355X: rotary positions of several axes (kv_ops.rotary(axes=)), against
tests/blocks_reference.py: fp32 roundings exactly, 64 bits within them."""

import numpy as np
import pytest
import torch

from drinkme_amd import kv_ops
from tests import blocks_reference as B
from tests.test_gpu_kv import DT, f64, heads, i32

pytestmark = pytest.mark.gpu


def check(got, x, at, axes, table, layout, dtype):
    exact = B.rotate_axes(f64(x), at, axes, f64(table), layout, np.float32)
    want = torch.from_numpy(exact).to(DT[dtype])
    assert got.is_contiguous() and got.dtype == x.dtype
    assert torch.equal(got.cpu().nan_to_num(nan=99.0), want.nan_to_num(nan=99.0))
    wide = B.rotate_axes(f64(x), at, axes, f64(table), layout)
    ok = ~np.isnan(wide)
    assert (np.isnan(f64(got)) == ~ok).all()
    size = np.nanmax(np.abs(f64(x))) * 2  # three roundings of products and sums that big, and the result's own
    bound = 3 * 2.0 ** -24 * size + (2.0 ** -8 * np.abs(wide) if dtype == "bf16" else 0)
    assert (np.abs(f64(got) - wide)[ok] <= bound[ok] if dtype == "bf16" else np.abs(f64(got) - wide)[ok] <= bound).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("order", ["blocks", "interleaved"])
@pytest.mark.parametrize("D, sections", [(128, (24, 20, 20)), (128, (16, 24, 24)), (128, (64,)), (96, (24, 24)), (96, (5, 0, 19)),
                                         (72, (12, 12, 12)), (256, (1, 40, 40, 47)), (64, (0, 16)), (34, (3, 5, 1)), (2, (0, 0, 0, 1)),
                                         (512, (100, 56, 100))])
def test_rotary_by_axes(D, sections, order, layout, dtype):
    rng = np.random.default_rng(D + sum(sections))
    T, Hq, Hk, A = 37, 5, 2, len(sections)
    axes = kv_ops.rotary_axes(sections, order)
    assert len(axes) == sum(sections) and [axes.count(a) for a in range(A)] == list(sections)
    for own in (None, axes):
        table = kv_ops.rotary_table(300, 2 * len(axes), axes=own)
        q, k = heads(rng, (T, Hq, D), dtype), heads(rng, (T, Hk, D), dtype)
        at = rng.integers(0, 300, (A, T))
        for positions in (i32(at), torch.from_numpy(at).cuda()):
            got = kv_ops.rotary(q, k, positions, table, layout, axes=axes)
            for x, y in zip((q, k), got):
                check(y, x, at, axes, table, layout, dtype)
        one, none = kv_ops.rotary(q, None, i32(at), table, layout, axes=list(axes))
        assert none is None and torch.equal(one, got[0])


def test_equal_positions_are_one_axis():
    """Text: every axis at the same position is the rotation of one axis, bit for bit."""
    rng = np.random.default_rng(1)
    q, k = heads(rng, (50, 8, 128), "bf16"), heads(rng, (50, 2, 128), "bf16")
    table, at = kv_ops.rotary_table(4096, 128, base=1e6), rng.integers(0, 4096, 50)
    want = kv_ops.rotary(q, k, i32(at), table)
    for order in ("blocks", "interleaved"):
        got = kv_ops.rotary(q, k, i32(np.stack([at] * 3)), table, axes=kv_ops.rotary_axes((24, 20, 20), order))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 40])
def test_positions_outside_the_table(D, dtype):
    """Only the channels of the axis that is outside are NaN."""
    rng = np.random.default_rng(2)
    at = np.array([[0, -1, 5, 10, 2 ** 31 - 1], [3, 4, 10, -2 ** 31, 9]])
    q = heads(rng, (5, 3, D), dtype)
    axes = kv_ops.rotary_axes((D // 4 - 3, D // 4 + 3), "interleaved")
    table = kv_ops.rotary_table(10, D)
    for layout in ("half", "interleaved"):
        check(kv_ops.rotary(q, None, i32(at), table, layout, axes=axes)[0], q, at, axes, table, layout, dtype)
    wide = at.astype(np.int64)
    wide[0, 4], wide[1, 3] = 2 ** 40, -2 ** 40
    check(kv_ops.rotary(q, None, torch.from_numpy(wide).cuda(), table, axes=axes)[0], q, wide, axes, table, "half", dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_views(dtype):
    """A fused product's views, an odd offset, shared heads; positions of a transposed grid; a longer
    table's axes left unused."""
    rng = np.random.default_rng(3)
    T, D = 19, 64
    axes, table = kv_ops.rotary_axes((11, 10, 11), "interleaved"), kv_ops.rotary_table(64, D)
    grid = torch.from_numpy(rng.integers(0, 64, (T, 3))).cuda().int()
    fused, odd = heads(rng, (T, 9, D), dtype), heads(rng, (T * 4 * D + 1,), dtype)
    for q, k in ((fused[:, :5], fused[:, 5:7]), (odd[1:].view(T, 4, D), fused[:, 8:]), (fused[:, :1].expand(T, 6, D), fused[:, ::4])):
        got = kv_ops.rotary(q, k, grid.t(), table, axes=axes)
        for x, y in zip((q, k), got):
            check(y, x, grid.t().cpu().numpy(), axes, table, "half", dtype)
    more = torch.cat([grid.t(), grid.t()[:1] + 999])
    assert torch.equal(kv_ops.rotary(q, k, more.contiguous(), table, axes=axes)[0], got[0])


def test_a_large_call():
    """More items than one lane's run of heads, as a long video has."""
    rng = np.random.default_rng(4)
    T = 3000
    q, k = heads(rng, (T, 16, 128), "bf16"), heads(rng, (T, 4, 128), "bf16")
    at, axes, table = rng.integers(0, 60, (3, T)), kv_ops.rotary_axes((16, 24, 24)), kv_ops.rotary_table(60, 128)
    for x, y in zip((q, k), kv_ops.rotary(q, k, i32(at), table, axes=axes)):
        check(y, x, at, axes, table, "half", "bf16")


def test_no_tokens_another_stream_and_a_graph():
    rng = np.random.default_rng(5)
    axes, table = kv_ops.rotary_axes((8, 12, 12)), kv_ops.rotary_table(100, 64)
    empty = torch.empty((0, 2, 64), device="cuda", dtype=torch.bfloat16)
    q, k = kv_ops.rotary(empty, empty, torch.empty((3, 0), dtype=torch.int32, device="cuda"), table, axes=axes)
    assert q.shape == (0, 2, 64) and k.shape == (0, 2, 64)
    x, at = heads(rng, (9, 2, 64), "bf16"), i32(rng.integers(0, 100, (3, 9)))
    want = kv_ops.rotary(x, None, at, table, axes=axes)[0].clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    y = torch.zeros_like(x)
    with torch.cuda.stream(stream):
        torch.cuda._sleep(20_000_000)
        y.copy_(x)
        got = kv_ops.rotary(y, None, at, table, axes=axes)[0]
    stream.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kv_ops.rotary(y, None, at, table, axes=axes)[0]
    for _ in range(3):
        at.copy_(i32(rng.integers(0, 100, (3, 9))))
        graph.replay()
        assert torch.equal(got, kv_ops.rotary(x, None, at, table, axes=axes)[0])


def test_refusals():
    x, at = heads(np.random.default_rng(6), (4, 2, 64), "bf16"), i32(np.zeros((3, 4)))
    table, axes = kv_ops.rotary_table(10, 64), kv_ops.rotary_axes((8, 12, 12))
    for kw, match in (({"axes": (0, 1, 2)}, "axes of 3 angles"), ({"axes": (4,) * 32}, "numbers of 0..3"), ({"axes": (0.0,) * 32}, "numbers"),
                      ({"axes": ()}, "numbers"), ({"positions": at[0]}, "positions"), ({"positions": at[:2]}, "positions"),
                      ({"positions": i32(np.zeros((5, 4)))}, "positions"), ({"positions": at.float()}, "positions"),
                      ({"positions": at[:, :3]}, "positions"), ({"positions": at.cpu()}, "positions"), ({"layout": "other"}, "layout"),
                      ({"table": table.reshape(-1)}, "table")):
        a = {"q": x, "k": x, "positions": at, "table": table, "axes": axes, **kw}
        with pytest.raises(ValueError, match=match):
            kv_ops.rotary(**a)
    with pytest.raises(RuntimeError, match="no gradient"):
        kv_ops.rotary(x.clone().requires_grad_(), None, at, table, axes=axes)
