"""MI355X: rotary positions, the append to the 4-bit paged cache, its read and
the attention over it (drinkme_amd.kv_ops), against tests/kv_reference.py in 64
bits. Codes and rotated keys are compared exactly; the attention within a bound
derived from its arithmetic (kv_reference.bound)."""

import numpy as np
import pytest
import torch

from drinkme_amd import kv_ops
from tests import kv_reference as R

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def f64(t):
    return t.detach().cpu().double().numpy()


def heads(rng, shape, dtype, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * np.float32(scale)).cuda().to(DT[dtype])


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Batch:
    """Sequences of (new tokens, length) in shuffled pages of a cache that
    starts as noise, with spare columns and pages."""

    def __init__(self, rng, sizes, H, D, page, spare=2):
        self.sizes, self.H, self.D, self.page = sizes, H, D, page
        counts = [-(-length // page) for _, length in sizes]
        self.cols = max(1, *counts) + spare
        order = rng.permutation(sum(counts) + 3)
        self.table = np.full((len(sizes), self.cols), -1)
        at = 0
        for b, n in enumerate(counts):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.cache = kv_ops.new_cache(len(order), page, H, D)
        for name, t in self.cache.items():
            noise = rng.integers(0, 256, t.numel() * t.element_size(), dtype=np.uint8)
            t.copy_(torch.from_numpy(noise).view(t.dtype).reshape(t.shape))
        self.total = sum(n for n, _ in sizes)
        self.lengths = i32([length for _, length in sizes])
        self.block_table = i32(self.table)
        uniform = len({n for n, _ in sizes}) == 1
        self.cu = None if uniform else i32(np.concatenate([[0], np.cumsum([n for n, _ in sizes])]))
        self.args = {"cu": self.cu}

    def positions(self):
        return np.concatenate([np.arange(length - n, length) for n, length in self.sizes] or [[]]).astype(np.int64)

    def fill(self, rng, k=None, v=None, scale=1.0):
        """Every position of every sequence written, by append itself; the
        values that the cache then holds: [(k, v) [length, H, D]] in 64 bits."""
        lengths = [length for _, length in self.sizes]
        total = sum(lengths)
        if k is None:
            k, v = (heads(rng, (total, self.H, self.D), "bf16", scale) for _ in range(2))
        cu = i32(np.concatenate([[0], np.cumsum(lengths)]))
        kv_ops.append(self.cache, k, v, self.block_table, self.lengths, cu=cu)
        kk, vv = R.cached(f64(k)), R.cached(f64(v))
        return [(kk[s:e], vv[s:e]) for s, e in zip(cu.tolist(), cu.tolist()[1:])]


def check_attention(batch, held, q, dtype, got, lse=None, causal=True, window=None, scale=None):
    scale = batch.D ** -0.5 if scale is None else scale
    t, worst = 0, 0.0
    out, qq = f64(got), f64(q)
    for (n, length), (k, v) in zip(batch.sizes, held):
        want, l, spread, reach = R.attention(qq[t:t + n], k, v, length - n, scale, causal, window)
        bound = R.bound(want, spread, reach, length, batch.D, dtype == "bf16")
        mine = out[t:t + n]
        assert (np.isnan(mine) == np.isnan(want)).all()
        off = np.abs(mine - want) / bound
        worst = max(worst, np.nanmax(off, initial=0.0))
        if lse is not None:
            le = f64(lse)[t:t + n]
            assert (np.isneginf(le) == np.isneginf(l)).all() and (np.isnan(le) == np.isnan(l)).all()
            ok = np.isfinite(l)
            assert (np.abs(le - l)[ok] <= R.lse_bound(l, reach, length, batch.D)[ok]).all()
        t += n
    assert worst <= 1.0, worst
    return worst


# ------------------------------------------------------------------- rotary --


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D, part", [(128, 128), (96, 48), (64, 16), (80, 20), (256, 64), (34, 6), (2, 2)])
def test_rotary(D, part, layout, dtype):
    rng = np.random.default_rng(D + part)
    T, Hq, Hk = 37, 5, 2
    table = kv_ops.rotary_table(500, part, scaling={"kind": "linear", "factor": 2.0})
    q, k = heads(rng, (T, Hq, D), dtype), heads(rng, (T, Hk, D), dtype)
    at = rng.integers(0, 500, T)
    for positions in (i32(at), torch.from_numpy(at).cuda()):
        got = kv_ops.rotary(q, k, positions, table, layout)
        for x, y in zip((q, k), got):
            want = R.rotate(f64(x), at, f64(table), layout)
            size = np.abs(f64(x)).max() * 2
            assert y.is_contiguous() and y.dtype == x.dtype
            assert (np.abs(f64(y) - want) <= (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0) + 3 * 2.0 ** -24 * size).all()
            exact = torch.from_numpy(R.rotate(f64(x), at, f64(table), layout, np.float32)).to(DT[dtype])
            assert torch.equal(y.cpu(), exact)
    one, none = kv_ops.rotary(q, None, i32(at), table, layout)
    assert none is None and torch.equal(one, got[0])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rotary_reads_views(dtype):
    """A fused product's views, a transposed tensor, an odd offset, shared
    (stride 0) heads, adjacent heads of a reversed order."""
    rng = np.random.default_rng(7)
    T, D = 19, 64
    table = kv_ops.rotary_table(64, D)
    at = i32(np.arange(T))
    fused = heads(rng, (T, 9, D), dtype)
    odd = heads(rng, (T * 6 * D + 3,), dtype)
    forms = [(fused[:, :5], fused[:, 5:7]), (fused.transpose(0, 1).contiguous().transpose(0, 1), fused[:, 8:]),
             (odd[1:1 + T * 4 * D].view(T, 4, D), odd[3:3 + T * D].view(T, 1, D)),
             (fused[:, :1].expand(T, 6, D), fused[::1, ::4]), (heads(rng, (T, D, 3), dtype).transpose(1, 2), fused[:, :1])]
    for q, k in forms:
        got = kv_ops.rotary(q, k, at, table)
        want = kv_ops.rotary(q.contiguous(), k.contiguous(), at, table)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_rotary_positions_outside_the_table():
    rng = np.random.default_rng(1)
    q = heads(rng, (5, 2, 32), "bf16")
    table = kv_ops.rotary_table(10, 16)
    at = torch.tensor([0, -1, 10, 9, 2 ** 40], device="cuda")
    got = f64(kv_ops.rotary(q, None, at, table)[0])
    assert (np.isnan(got[[1, 2, 4]][..., :16])).all() and np.isfinite(got[[0, 3]]).all()
    assert (got[..., 16:] == f64(q)[..., 16:]).all()
    # the pairwise path, too
    got = f64(kv_ops.rotary(q, None, at, kv_ops.rotary_table(10, 6))[0])
    assert (np.isnan(got[[1, 2, 4]][..., :6])).all() and np.isfinite(got[[0, 3]]).all()


def test_rotary_of_no_tokens():
    q = torch.empty(0, 4, 64, dtype=torch.bfloat16, device="cuda")
    assert kv_ops.rotary(q, q[:, :2], i32([]), kv_ops.rotary_table(4, 64))[1].shape == (0, 2, 64)


# ------------------------------------------------------------ append, read --


def stored(batch):
    return kv_ops.read(batch.cache, batch.block_table, batch.lengths, batch.total, **batch.args)


def test_every_bf16_value_is_coded_as_defined():
    """Each pattern once in a block of its own size (32 neighbours), so that
    every scale, tie, overflow, underflow, infinity and NaN is met."""
    bits = np.arange(65536, dtype=np.uint16)
    rng = np.random.default_rng(3)
    order = np.concatenate([bits, rng.permutation(bits)])
    x = torch.from_numpy(order.view(np.int16)).view(torch.bfloat16).cuda().reshape(-1, 1, 128)
    b = Batch(rng, [(x.shape[0], x.shape[0])], 1, 128, 64)
    with np.errstate(invalid="ignore"):
        want = R.cached(f64(x))
    for t in (x, x.float()):
        kv_ops.append(b.cache, t, t.flip(0), b.block_table, b.lengths)
        k, v = stored(b)
        assert np.array_equal(f64(k), want, equal_nan=True)
        assert np.array_equal(f64(v), want[::-1], equal_nan=True)


def test_fp32_values_that_bf16_cannot_hold():
    rng = np.random.default_rng(4)
    x = rng.standard_normal((64, 2, 64)).astype(np.float32) * np.exp2(rng.integers(-149, 127, (64, 2, 1))).astype(np.float32)
    x[0, 0, :8] = [1.75, 1.7499999, 1.7500001, 7, 6.9999995, 0.25, 5e-45, -0.0]
    b = Batch(rng, [(8, 20)] * 8, 2, 64, 16)
    t = torch.from_numpy(x).cuda()
    kv_ops.append(b.cache, t, t, b.block_table, b.lengths)
    k, v = stored(b)
    assert np.array_equal(f64(k), R.cached(x)) and torch.equal(k, v)


SIZES = [[(1, 1)], [(1, 4096)], [(1, n) for n in (1, 7, 8, 9, 64, 65, 1000)], [(5, n) for n in (5, 12, 63, 130)],
         [(70, 70)], [(0, 9), (1, 1), (33, 100), (0, 0), (8, 8), (17, 17)]]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D, part", [(128, 128), (96, 96), (64, 32), (192, 48), (256, 20), (64, 6)])
@pytest.mark.parametrize("sizes", SIZES, ids=str)
def test_append(sizes, D, part, layout, dtype):
    rng = np.random.default_rng(D + part + len(sizes))
    H, Hq = 3, 6
    b = Batch(rng, sizes, H, D, (8, 16, 64)[len(sizes) % 3])
    fused = heads(rng, (b.total, Hq + 2 * H, D), dtype)
    q, k, v = fused[:, :Hq], fused[:, Hq:Hq + H], fused[:, Hq + H:]
    table = kv_ops.rotary_table(4096, part)
    before = {n: t.clone() for n, t in b.cache.items()}
    got = kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, layout=layout, q=q, **b.args)
    at = b.positions()
    turned = [R.rotate(f64(x), at, f64(table), layout, np.float32) for x in (q, k)]
    assert torch.equal(got.cpu(), torch.from_numpy(turned[0]).to(DT[dtype]))
    ck, cv = stored(b)
    assert np.array_equal(f64(ck), R.cached(turned[1])) and np.array_equal(f64(cv), R.cached(f64(v)))
    # nothing else was written: as many bytes differ as the new tokens' at most, and the rest of each page stays
    touched = np.zeros(b.cache["k_codes"].shape[:1] + (b.page,), bool)
    for (n, length), pages in zip(sizes, b.table):
        for p in range(length - n, length):
            touched[pages[p // b.page], p % b.page] = True
    same = torch.from_numpy(~touched).cuda()
    for name in ("k_codes", "k_scales"):
        assert torch.equal(b.cache[name].transpose(1, 2)[same], before[name].transpose(1, 2)[same])
    for name in ("v_codes", "v_scales"):
        now, was = (x[name].permute(0, 2, 4, 1, 3).flatten(1, 2)[same] for x in (b.cache, before))
        assert torch.equal(now, was)
    # keys as they are, without a table
    assert kv_ops.append(b.cache, k, v, b.block_table, b.lengths, **b.args) is None
    assert np.array_equal(f64(stored(b)[0]), R.cached(f64(k)))


def test_append_takes_any_strides():
    rng = np.random.default_rng(9)
    b = Batch(rng, [(11, 30)] * 2, 2, 64, 16)
    table = kv_ops.rotary_table(64, 64)
    buf = heads(rng, (2, 22 * 2 * 64 + 1), "bf16")
    k, v = buf[0, 1:].view(22, 2, 64), buf[1, 1:].view(22, 2, 64)
    q = heads(rng, (22, 64, 4), "bf16").transpose(1, 2)
    got = kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, q=q)
    odd = stored(b)
    want = kv_ops.append(b.cache, k.clone(), v.clone(), b.block_table, b.lengths, table=table, q=q.contiguous())
    assert torch.equal(got, want) and all(torch.equal(x, y) for x, y in zip(odd, stored(b)))


def test_tokens_without_a_page_are_dropped():
    rng = np.random.default_rng(11)
    b = Batch(rng, [(4, 6)] * 3, 1, 64, 8, spare=0)
    b.block_table[0] = -1                  # no page
    b.block_table[1] = 10 ** 9             # not one of the cache's
    lengths = i32([6, 6, 10])              # the last one's tokens 8 and 9 are past the table
    before = {n: t.clone() for n, t in b.cache.items()}
    k = heads(rng, (12, 1, 64), "bf16")
    kv_ops.append(b.cache, k, k, b.block_table, lengths)
    got = [f64(x) for x in kv_ops.read(b.cache, b.block_table, lengths, 12)]
    for x in got:
        assert np.isnan(x[:8]).all() and np.isnan(x[10:]).all() and np.array_equal(x[8:10], R.cached(f64(k))[8:10])
    pages = torch.arange(b.cache["k_codes"].shape[0]).cuda() != b.table[2, 0]
    assert all(torch.equal(b.cache[n][pages], before[n][pages]) for n in before)
    # positions before the first (more new tokens than the length)
    kv_ops.append(b.cache, k, k, i32(b.table), i32([2, 2, 2]))
    got = f64(kv_ops.read(b.cache, i32(b.table), i32([2, 2, 2]), 12)[0]).reshape(3, 4, -1)
    assert np.isnan(got[:, :2]).all() and np.array_equal(got[:, 2:], R.cached(f64(k)).reshape(3, 4, -1)[:, 2:])


# --------------------------------------------------------------- attention --


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", kv_ops.HEAD_DIMS)
@pytest.mark.parametrize("sizes", [[(1, 1)], [(1, n) for n in (1, 31, 32, 33, 500, 1021)], [(5, n) for n in (5, 33, 300)]],
                         ids=str)
@pytest.mark.parametrize("H, Hq", [(1, 1), (2, 8), (2, 22)])
def test_attention_of_few_tokens(sizes, D, H, Hq, dtype):
    rng = np.random.default_rng(D + Hq)
    b = Batch(rng, sizes, H, D, (8, 16, 32, 64)[(D // 32 + Hq) % 4])
    held = b.fill(rng)
    q = heads(rng, (b.total, Hq, D), dtype, 2.0)
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, return_lse=True, **b.args)
    check_attention(b, held, q, dtype, got, lse)
    assert torch.equal(got, kv_ops.attention(q, b.cache, b.block_table, b.lengths, **b.args))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", kv_ops.HEAD_DIMS)
@pytest.mark.parametrize("causal, window", [(True, None), (True, 40), (False, None), (False, 7), (True, 1)])
def test_attention_of_prompts(D, causal, window, dtype):
    rng = np.random.default_rng(D)
    b = Batch(rng, [(70, 70), (0, 40), (1, 1), (33, 161), (0, 0), (64, 64), (19, 83)], 2, D, 16)
    held = b.fill(rng)
    q = heads(rng, (b.total, 6, D), dtype)
    for bound in (70, None):
        got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, causal=causal, window=window, return_lse=True,
                                    max_tokens=bound, **b.args)
        check_attention(b, held, q, dtype, got, lse, causal, window)


@pytest.mark.parametrize("tokens", [2, 3, 4, 6, 8, 9, 16])
@pytest.mark.parametrize("group", [1, 3, 4, 7, 8, 16])
def test_attention_row_tiles(tokens, group):
    """Every count of query rows to a cache head, from one tile to prompts."""
    rng = np.random.default_rng(tokens * group)
    b = Batch(rng, [(tokens, 50), (tokens, tokens), (tokens, 129)], 1, 64, 8)
    held = b.fill(rng)
    q = heads(rng, (b.total, group, 64), "bf16")
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, return_lse=True)
    check_attention(b, held, q, "bf16", got, lse)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("window", [None, 31, 32, 33, 64, 97, 200])
@pytest.mark.parametrize("tokens, length, group", [(330, 330, 4), (150, 700, 3), (600, 600, 1), (8, 500, 4), (5, 1000, 13),
                                                   (1, 777, 16)])
def test_windows_that_begin_anywhere(tokens, length, group, window, dtype):
    """Rows of many workgroups and waves, each with its own first token: on a
    block's edge, inside a block, in a block that another wave takes."""
    rng = np.random.default_rng(tokens + group)
    b = Batch(rng, [(tokens, length)], 1, 64, 32)
    held = b.fill(rng)
    q = heads(rng, (tokens, group, 64), dtype, 1.5)
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, window=window, return_lse=True)
    check_attention(b, held, q, dtype, got, lse, True, window)


@pytest.mark.parametrize("max_length", [None, 1, 700, 10 ** 9])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_over_splits(dtype, max_length):
    """A long axis split over workgroups, some of which get nothing; a wide
    block table; max_length shapes the launch alone."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [(1, 5000), (1, 3), (1, 700)], 1, 128, 64, spare=100)
    held = b.fill(rng)
    q = heads(rng, (3, 2, 128), dtype)
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, return_lse=True, max_length=max_length)
    check_attention(b, held, q, dtype, got, lse)


def test_attention_at_large_scores():
    """Scores far apart (one token takes all) and all equal; scale of its own."""
    rng = np.random.default_rng(6)
    b = Batch(rng, [(4, 200)] * 2, 2, 128, 32)
    held = b.fill(rng, scale=8.0)
    for size, scale in ((30.0, None), (0.0, None), (1.0, 3.0), (1.0, 1e-6)):
        q = heads(rng, (8, 4, 128), "bf16", size)
        got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, scale=scale, return_lse=True)
        check_attention(b, held, q, "bf16", got, lse, scale=scale)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 5, 40])
@pytest.mark.parametrize("shape", ["rise", "steps", "spike", "fall"])
def test_scores_that_leave_their_first_block_behind(shape, tokens, dtype):
    """Scores that grow along the context by more than weights of the first
    block's scale can hold (to hundreds of powers of two), gently, at a step or
    at one token, or that fall away from it."""
    rng = np.random.default_rng(20)
    D, length = 64, 900
    b = Batch(rng, [(tokens, length), (tokens, length - 7)], 1, D, 32)
    total = 2 * length - 7
    at = np.concatenate([np.arange(length), np.arange(length - 7)]) / length
    gain = {"rise": at * 60, "steps": np.floor(at * 8) * 9, "spike": 40.0 * (np.abs(at - 0.6) < 0.5 / length),
            "fall": 60 - 60 * at}[shape]
    direction = np.sign(rng.standard_normal(D))
    k = torch.from_numpy((gain[:, None, None] * direction + rng.standard_normal((total, 1, D))).astype(np.float32)).cuda()
    held = b.fill(rng, k.to(torch.bfloat16), heads(rng, (total, 1, D), "bf16"))
    q = torch.from_numpy((direction * (1 + 0.1 * rng.standard_normal((2 * tokens, 3, D)))).astype(np.float32)).cuda().to(DT[dtype])
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, return_lse=True)
    check_attention(b, held, q, dtype, got, lse)


@pytest.mark.parametrize("tokens", [1, 40])
def test_sums_of_many_weights_above_one(tokens):
    """A long context whose scores lie a little above the first block's: a
    lane's sum passes what the kernels let it grow to, no single weight does."""
    rng = np.random.default_rng(21)
    D, length = 64, 70000
    b = Batch(rng, [(tokens, length)], 1, D, 128)
    direction = np.sign(rng.standard_normal(D))
    gain = np.full(length, 1.0)
    gain[:8192] = 0.0
    k = torch.from_numpy((gain[:, None, None] * direction + 0.2 * rng.standard_normal((length, 1, D))).astype(np.float32)).cuda()
    held = b.fill(rng, k.to(torch.bfloat16), heads(rng, (length, 1, D), "bf16"))
    q = torch.from_numpy((direction * 10.0 / 8 * np.ones((tokens, 1, D))).astype(np.float32)).cuda().to(torch.bfloat16)
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, max_length=512, return_lse=True)  # (one split)
    check_attention(b, held, q, "bf16", got, lse)


def test_rows_that_see_nothing():
    rng = np.random.default_rng(8)
    b = Batch(rng, [(6, 6)] * 2, 1, 64, 8)
    b.fill(rng)
    q = heads(rng, (12, 2, 64), "bf16")
    got, lse = kv_ops.attention(q, b.cache, b.block_table, i32([0, 3]), return_lse=True)
    assert (f64(got)[:9] == 0).all() and np.isneginf(f64(lse)[:9]).all()  # the second's first three are before it
    assert (f64(got)[9:] != 0).any() and np.isfinite(f64(lse)[9:]).all()


@pytest.mark.parametrize("D", [64, 96, 128])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("tokens", [1, 5, 40])
def test_nan_reaches_only_what_sees_it(which, tokens, D):
    """A block that is not finite: every channel of a row that sees its key,
    the block's channels of a row that sees its value, no other row."""
    rng = np.random.default_rng(tokens)
    b = Batch(rng, [(tokens, 90), (tokens, 200)], 2, D, 16)
    k, v = (heads(rng, (290, 2, D), "bf16") for _ in range(2))
    x = k if which == "k" else v
    x[90 - tokens // 2 - 1, 0, 37] = float("inf")  # among the first sequence's new tokens, or just before
    x[90 + 3, 1, 5] = float("nan")                 # early in the second
    held = b.fill(rng, k, v)
    q = heads(rng, (b.total, 4, D), "bf16")
    for causal, window in ((True, None), (True, 20), (False, None), (True, 3)):
        got = kv_ops.attention(q, b.cache, b.block_table, b.lengths, causal=causal, window=window)
        check_attention(b, held, q, "bf16", got, None, causal, window)


def test_positions_without_a_page():
    rng = np.random.default_rng(12)
    b = Batch(rng, [(2, 60)] * 3, 1, 64, 16, spare=0)
    held = b.fill(rng)
    q = heads(rng, (6, 2, 64), "bf16")
    t = b.block_table.clone()
    t[0, 0] = 10 ** 6
    got = f64(kv_ops.attention(q, b.cache, t, b.lengths))
    assert np.isnan(got[:2]).all() and np.isfinite(got[2:]).all()
    got = kv_ops.attention(q, b.cache, t, b.lengths, window=20)  # none of the rows sees it
    check_attention(b, held, q, "bf16", got, None, True, 20)
    got = f64(kv_ops.attention(q, b.cache, b.block_table, i32([60, 2 ** 31 - 1, 65])))  # longer than the table
    # (the third's first row, at position 63, sees the table's 64 positions and no more: the last of them noise here)
    assert np.isfinite(got[:2]).all() and np.isnan(got[[2, 3, 5]]).all()


def test_attention_reads_views():
    rng = np.random.default_rng(13)
    b = Batch(rng, [(3, 100)] * 2, 2, 64, 16)
    b.fill(rng)
    fused = heads(rng, (6, 9, 64), "bf16")
    odd = heads(rng, (6 * 4 * 64 + 1,), "bf16")[1:].view(6, 4, 64)
    for q in (fused[:, 2:6], odd, heads(rng, (6, 64, 4), "bf16").transpose(1, 2), fused[:, :1].expand(6, 4, 64)):
        got = kv_ops.attention(q, b.cache, b.block_table, b.lengths)
        assert torch.equal(got, kv_ops.attention(q.contiguous(), b.cache, b.block_table, b.lengths))


def test_cu_outside_the_call_is_clamped():
    """Offsets that only the GPU can see: no row outside the tensors is read or
    written (the sentinel rows beside the output's own stay)."""
    rng = np.random.default_rng(14)
    b = Batch(rng, [(3, 40)] * 2, 1, 64, 16)
    held = b.fill(rng)
    q = heads(rng, (6, 2, 64), "bf16")
    got = kv_ops.attention(q, b.cache, b.block_table, b.lengths, cu=i32([0, 3, 10 ** 6]), max_tokens=3)
    check_attention(b, held, q, "bf16", got)
    kv_ops.attention(q, b.cache, b.block_table, b.lengths, cu=i32([-5, 10 ** 6, -7]), max_tokens=3)
    torch.cuda.synchronize()


# -------------------------------------------------- long caches, streams --


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes: the pages at its end."""
    rng = np.random.default_rng(15)
    D, page, H = 256, 64, 8
    pages = 2 ** 32 // (H * page * D // 2) + 8
    cache = kv_ops.new_cache(pages, page, H, D)
    k, v = (heads(rng, (100, H, D), "bf16") for _ in range(2))
    for table in ([[pages - 1, pages - 2]], [[pages - 3, 0]]):
        t, n = i32(table), i32([100])
        kv_ops.append(cache, k, v, t, n)
        ck, cv = kv_ops.read(cache, t, n, 100)
        assert np.array_equal(f64(ck), R.cached(f64(k))) and np.array_equal(f64(cv), R.cached(f64(v)))
        q = heads(rng, (1, H, D), "bf16")
        want, _, spread, reach = R.attention(f64(q), f64(ck), f64(cv), 99, D ** -0.5)
        got = f64(kv_ops.attention(q, cache, t, n))
        assert (np.abs(got - want) <= R.bound(want, spread, reach, 100, D, True)).all()


def test_on_another_stream():
    rng = np.random.default_rng(16)
    b = Batch(rng, [(2, 3000)] * 2, 2, 128, 64)
    held = b.fill(rng)
    q = heads(rng, (4, 8, 128), "bf16")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [kv_ops.attention(q, b.cache, b.block_table, b.lengths) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    for got in outs:
        check_attention(b, held, q, "bf16", got)


def test_a_captured_step_replays():
    """append and attention in a graph: each replay on new inputs and lengths
    gives what the eager calls give."""
    rng = np.random.default_rng(17)
    b = Batch(rng, [(1, 600), (1, 90)], 2, 64, 16, spare=4)
    b.fill(rng)
    table = kv_ops.rotary_table(1024, 64)
    q, k, v = (heads(rng, (2, n, 64), "bf16") for n in (8, 2, 2))

    def step():
        turned = kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, q=q)
        return kv_ops.attention(turned, b.cache, b.block_table, b.lengths)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        b.lengths += 0 if n == 0 else 1
        b.block_table[1, 90 // 16 + 1] = b.cache["k_codes"].shape[0] - 1
        for x in (q, k, v):
            x.copy_(heads(rng, x.shape, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, step())
        torch.cuda.synchronize()


def test_calls_of_no_tokens():
    rng = np.random.default_rng(18)
    b = Batch(rng, [(1, 20)] * 2, 2, 64, 16)
    x = torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")
    table = kv_ops.rotary_table(8, 64)
    assert kv_ops.append(b.cache, x, x, b.block_table, b.lengths, table=table, q=x).shape == x.shape
    out, lse = kv_ops.attention(x, b.cache, b.block_table, b.lengths, return_lse=True)
    assert out.shape == x.shape and lse.shape == (0, 2)
    assert kv_ops.read(b.cache, b.block_table, b.lengths, 0)[0].shape == x.shape


def test_the_general_path_gives_the_native_call_s_results(monkeypatch):
    """Every operator without the extension of its per-call path: the same
    kernels through ctypes, the same bits."""
    from drinkme_amd import _native

    rng = np.random.default_rng(19)
    b = Batch(rng, [(5, 70), (1, 33), (0, 4)], 2, 96, 16)
    b.fill(rng)
    table = kv_ops.rotary_table(128, 48)
    q, k, v = (heads(rng, (6, n, 96), "bf16") for n in (4, 2, 2))

    def results():
        out = list(kv_ops.rotary(q, k, b.lengths.repeat(2), table, "interleaved")) + [kv_ops.rotary(q, None, b.lengths.repeat(2), table)[0]]
        out.append(kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, q=q, **b.args))
        out += kv_ops.read(b.cache, b.block_table, b.lengths, 6, **b.args)
        for kw in ({}, {"max_tokens": 5, "scale": 0.5, "window": 9}, {"causal": False, "max_length": 70}):
            out += kv_ops.attention(q, b.cache, b.block_table, b.lengths, return_lse=True, **b.args, **kw)
        out.append(kv_ops.attention(q, b.cache, b.block_table, b.lengths, **b.args))
        assert kv_ops.append(b.cache, k, v, b.block_table, b.lengths, **b.args) is None
        return out

    native = results()
    monkeypatch.setattr(_native, "_calls", None)
    general = results()
    assert len(native) == len(general) and all(torch.equal(x, y) for x, y in zip(native, general))


# ---------------------------------------------------------------- refusals --


def refusing():
    rng = np.random.default_rng(0)
    b = Batch(rng, [(1, 20)] * 2, 2, 64, 16)
    x = {n: heads(rng, (2, h, 64), "bf16") for n, h in (("q", 4), ("k", 2), ("v", 2))}
    return b, x, kv_ops.rotary_table(32, 64)


@pytest.mark.parametrize("case, error, match", [
    (lambda b, x, t: kv_ops.rotary(x["q"].half(), None, b.lengths, t), TypeError, "bf16 or fp32"),
    (lambda b, x, t: kv_ops.rotary(x["q"], x["k"].float(), b.lengths, t), ValueError, "torch.float32"),
    (lambda b, x, t: kv_ops.rotary(x["q"], x["k"], b.lengths.float(), t), ValueError, "positions"),
    (lambda b, x, t: kv_ops.rotary(x["q"], x["k"], b.lengths[:1], t), ValueError, "positions"),
    (lambda b, x, t: kv_ops.rotary(x["q"], x["k"], b.lengths, t, "neox"), ValueError, "layout"),
    (lambda b, x, t: kv_ops.rotary(x["q"], x["k"], b.lengths, t.double()), ValueError, "table"),
    (lambda b, x, t: kv_ops.rotary(x["q"], x["k"], b.lengths, t.cpu()), ValueError, "table is not on"),
    (lambda b, x, t: kv_ops.rotary(x["q"][..., :62], None, b.lengths, t), ValueError, "table of 64 channels"),
    (lambda b, x, t: kv_ops.rotary(x["q"].float().requires_grad_(), None, b.lengths, t), RuntimeError, "no gradient"),
    (lambda b, x, t: kv_ops.append(b.cache, x["q"], x["v"], b.block_table, b.lengths), ValueError, "4 heads, not 2"),
    (lambda b, x, t: kv_ops.append(b.cache, x["k"], x["v"][:1], b.block_table, b.lengths), ValueError, "tokens"),
    (lambda b, x, t: kv_ops.append(b.cache, x["k"], x["v"], b.block_table, b.lengths, q=x["q"]), ValueError, "table"),
    (lambda b, x, t: kv_ops.append(b.cache, x["k"].cpu(), x["v"], b.block_table, b.lengths), ValueError, "GPU"),
    (lambda b, x, t: kv_ops.append(b.cache, x["k"], x["v"], b.block_table.long(), b.lengths), ValueError, "block_table"),
    (lambda b, x, t: kv_ops.append(b.cache, x["k"], x["v"], b.block_table[:1], b.lengths), ValueError, "for 2 lengths"),
    (lambda b, x, t: kv_ops.append({**b.cache, "v_codes": b.cache["v_codes"][..., :4]}, x["k"], x["v"], b.block_table,
                                   b.lengths), ValueError, "v_codes"),
    (lambda b, x, t: kv_ops.append({**b.cache, "k_scales": b.cache["k_scales"][1:]}, x["k"], x["v"], b.block_table,
                                   b.lengths), ValueError, "k_scales"),
    (lambda b, x, t: kv_ops.attention(x["q"][:, :3], b.cache, b.block_table, b.lengths), ValueError, "3 query heads"),
    (lambda b, x, t: kv_ops.attention(x["q"][..., :32], b.cache, b.block_table, b.lengths), ValueError, "channels"),
    (lambda b, x, t: kv_ops.attention(x["q"].double(), b.cache, b.block_table, b.lengths), TypeError, "bf16 or fp32"),
    (lambda b, x, t: kv_ops.attention(x["q"], b.cache, b.block_table, b.lengths, window=0), ValueError, "window"),
    (lambda b, x, t: kv_ops.attention(x["q"], b.cache, b.block_table, b.lengths, max_tokens=2), ValueError, "max_tokens"),
    (lambda b, x, t: kv_ops.attention(x["q"], b.cache, b.block_table, b.lengths, scale=-1.0), RuntimeError, "scale"),
    (lambda b, x, t: kv_ops.attention(x["q"], b.cache, b.block_table, b.lengths, scale=float("nan")), RuntimeError, "scale"),
    (lambda b, x, t: kv_ops.attention(x["q"][:1], b.cache, b.block_table, b.lengths), ValueError, "cu is None"),
    (lambda b, x, t: kv_ops.attention(x["q"], b.cache, b.block_table, b.lengths, cu=b.lengths), ValueError, "cu of 2"),
    (lambda b, x, t: kv_ops.read(b.cache, b.block_table, b.lengths, 3), ValueError, "cu is None"),
])
def test_refusals(case, error, match):
    b, x, t = refusing()
    before = {n: c.clone() for n, c in b.cache.items()}
    with pytest.raises(error, match=match):
        case(b, x, t)
    assert all(torch.equal(before[n], b.cache[n]) for n in before)
