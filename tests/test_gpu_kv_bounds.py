"""MI355X: what must not reach the results of the 4-bit cache's operators
(drinkme_amd.kv_ops): noise behind masks, memory that nothing wrote. Against
tests/kv_reference.py, within its derived bounds."""

import ctypes as ct

import numpy as np
import pytest
import torch

from drinkme_amd import _native, kv_ops
from tests import kv_reference as R
from tests.test_gpu_kv import DT, Batch, check_attention, f64, heads, i32

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------ hidden values --


def spoil(batch, byte):
    """Every token of the cache that no sequence holds becomes the grid's top
    with the exponent `byte`, page 0 all of them (a table's missing pages are
    read there)."""
    table = batch.table
    spare = next(p for p in range(batch.cache["k_codes"].shape[0]) if p not in table)
    table[table == 0] = spare
    batch.block_table.copy_(i32(table))

    def now():
        held = np.zeros((batch.cache["k_codes"].shape[0], batch.page), bool)
        for (_, length), pages in zip(batch.sizes, table):
            at = np.arange(length)
            held[pages[at // batch.page], at % batch.page] = True
        free = torch.from_numpy(~held).cuda()
        for name, value in (("k_codes", 0x77777777), ("v_codes", 0x77777777), ("k_scales", byte), ("v_scales", byte)):
            t = batch.cache[name]
            if name[0] == "k":  # [pages, heads, page, ...]
                t.masked_fill_(free[:, None, :, None].expand_as(t), value)
            else:               # [pages, heads, page / 8, ..., 8]
                t.masked_fill_(free.view(t.shape[0], 1, -1, 1, 8).expand_as(t), value)

    return now


@pytest.mark.parametrize("byte", [253, 254, 255])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 5, 90])
@pytest.mark.parametrize("D", [64, 128, 192, 256])
@pytest.mark.parametrize("page", [8, 16, 64])
def test_no_byte_of_a_hidden_token_reaches_a_row(page, D, tokens, dtype, byte):
    """Exponent bytes past the format's, whose values are infinite: after the
    sequences' ends, and before a window, in pages that the table has lost."""
    rng = np.random.default_rng(page + D + tokens)
    b = Batch(rng, [(tokens, 200), (tokens, 93)], 1, D, page)
    now = spoil(b, byte)
    held = b.fill(rng)
    now()
    q = heads(rng, (b.total, 2, D), dtype)
    for window in (None, 3, 21, 50):
        t = b.block_table.clone()
        if window:
            for s, (n, length) in enumerate(b.sizes):
                t[s, :max(0, length - n + 1 - window) // page] = -1
        got, lse = kv_ops.attention(q, b.cache, t, b.lengths, window=window, return_lse=True)
        check_attention(b, held, q, dtype, got, lse, True, window)


@pytest.mark.parametrize("byte", [253, 254])
@pytest.mark.parametrize("tokens", [6, 40])
def test_a_bad_byte_in_a_new_token_stays_with_the_rows_that_see_it(tokens, byte):
    rng = np.random.default_rng(tokens + byte)
    D, length = 128, 180
    b = Batch(rng, [(tokens, length)], 1, D, 16)
    held = b.fill(rng)
    at = length - tokens + 3  # the fourth new token's values, channels 64 .. 95
    page, slot = b.table[0, at // 16], at % 16
    b.cache["v_scales"][page, 0, slot // 8, 2, slot % 8] = byte
    b.cache["v_codes"][page, 0, slot // 8, 8:12, slot % 8] = 0x77777777
    q = heads(rng, (tokens, 4, D), "bf16")
    got = kv_ops.attention(q, b.cache, b.block_table, b.lengths)
    out = f64(got)
    assert not np.isfinite(out[3:, :, 64:96]).any()
    want, _, spread, reach = R.attention(f64(q), *held[0], length - tokens, D ** -0.5)
    ok = np.abs(out - want) <= R.bound(want, spread, reach, length, D, True)
    assert ok[:3].all() and ok[..., :64].all() and ok[..., 96:].all()


# ------------------------------------------- offsets that only the GPU sees --

GUARD = 5


def through_the_abi(b, q, cu, max_tokens, lengths=None, window=0, max_length=0):
    """dmx_kv_attention into the middle of larger buffers that hold a pattern,
    with a workspace that does, too -> out, lse; the buffers beside them have
    to keep it."""
    T, Hq, D = q.shape
    lib, code = _native.lib(), {torch.bfloat16: 0, torch.float32: 1}[q.dtype]
    c = kv_ops._cache_of(b.cache, "test")
    lengths = b.lengths if lengths is None else lengths
    s = _native.KvSeqs(b.block_table.data_ptr(), lengths.data_ptr(), cu.data_ptr(), len(b.sizes), b.cols, T, max_tokens)
    out = torch.full((T + 2 * GUARD, Hq, D), 7.5, dtype=q.dtype, device="cuda")
    lse = torch.full((T + 2 * GUARD, Hq), 7.5, device="cuda")
    need = lib.dmx_kv_attention_workspace(ct.byref(c), ct.byref(s), Hq, code, max_length, window)
    ws = torch.full((need + 512,), 0x42, dtype=torch.uint8, device="cuda")  # (as floats: 48.6)
    err = _native.error_buffer()
    st = lib.dmx_kv_attention(ct.byref(c), ct.byref(s), ct.byref(kv_ops._rows(q)), code, D ** -0.5, 1, window, max_length,
                              out[GUARD:].data_ptr(), lse[GUARD:].data_ptr(), ws.data_ptr() + 256, need,
                              torch.cuda.current_stream().cuda_stream, err, len(err))
    _native.check(st, err, "dmx_kv_attention")
    for x, value in ((out, 7.5), (lse, 7.5)):
        assert (x[:GUARD] == value).all() and (x[GUARD + T:] == value).all()
    assert (ws[:256] == 0x42).all() and (ws[256 + need:] == 0x42).all()
    return out[GUARD:GUARD + T], lse[GUARD:GUARD + T], need


def expected(b, held, q, cu, max_tokens, dtype, window):
    """(result, bound, lse, its bound) of each token: what its sequence's clamped
    offsets say, NaN past max_tokens and where there is no sequence."""
    T, Hq, D = q.shape
    want, bound = np.full((T, Hq, D), np.nan), np.zeros((T, Hq, D))
    lse, lbound = np.full((T, Hq), np.nan), np.zeros((T, Hq))
    for s, (k, v) in enumerate(held):
        t = min(max(cu[s], 0), T)
        n = min(max(cu[s + 1], t), T) - t
        rows = slice(t, t + min(n, max_tokens))
        if rows.stop > t:
            x, l, spread, reach = R.attention(f64(q)[rows], k, v, len(k) - n, D ** -0.5, True, window or None)
            want[rows], bound[rows] = x, R.bound(x, spread, reach, len(k), D, dtype == "bf16")
            lse[rows], lbound[rows] = l, R.lse_bound(l, reach, len(k), D)
    return want, bound, lse, lbound


# counts of three sequences, max_tokens, offsets: a bound that does not hold; tokens before the first
# sequence, after the last, both; offsets out of range; offsets that decrease
OFFSETS = [(8, 3, [0, 2, 7, 8]), (8, 1, [0, 1, 8, 8]), (8, 8, [3, 5, 6, 8]), (8, 8, [0, 2, 5, 6]), (8, 2, [2, 3, 4, 4]),
           (8, 8, [3, 3, 3, 3]), (8, 3, [-5, 10 ** 6, 10 ** 6, 10 ** 6]), (8, 3, [-7, -5, 10 ** 6, -7]),
           (200, 40, [0, 90, 91, 200]), (200, 200, [30, 100, 101, 150]), (200, 70, [-3, 75, 10 ** 9, 10 ** 9])]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 192, 256])
@pytest.mark.parametrize("length", [260, 1500])
@pytest.mark.parametrize("total, most, cu", OFFSETS, ids=str)
def test_every_row_is_written(total, most, cu, length, D, dtype):
    """Few rows and prompts, split over workgroups (1500) or not: a row is its
    sequence's result, or NaN where it lies past max_tokens or in no sequence."""
    rng = np.random.default_rng(total + D)
    b = Batch(rng, [(1, length), (2, length - 37), (3, length - 200)], 2, D, 16, spare=1)
    held = b.fill(rng)
    q = heads(rng, (total, 4, D), dtype)
    for window in (0, 33):
        got, lse, need = through_the_abi(b, q, i32(cu), most, window=window)
        assert (need > 0) == (length > 512 and not window)
        want, bound, l, lbound = expected(b, held, q, cu, most, dtype, window)
        got, lse = f64(got), f64(lse)
        assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isnan(lse), np.isnan(l))
        assert np.array_equal(np.isneginf(lse), np.isneginf(l))
        ok = ~np.isnan(want)
        assert (np.abs(got - want)[ok] <= bound[ok]).all()
        fin = np.isfinite(l)
        assert (np.abs(lse - l)[fin] <= lbound[fin]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("cu", [[2, 4, 7], [0, 3, 5], [1, 1, 1], [-4, 2, 10 ** 6], [0, 10 ** 6, -3]], ids=str)
def test_tokens_of_no_sequence_are_not_stored(cu, dtype):
    """Before the first offset and after the last one: append leaves the cache
    alone, read gives NaN; q's other rows are as ever, and nothing beside them
    is written."""
    rng = np.random.default_rng(31)
    T, H, Hq, D = 8, 2, 3, 64
    b = Batch(rng, [(3, 40), (5, 23)], H, D, 8, spare=2)
    b.fill(rng)
    spare = next(p for p in range(b.cache["k_codes"].shape[0]) if p not in b.table)
    b.block_table[b.block_table < 0] = spare  # (positions past the sequences' ends have a page, too)
    before = {n: t.clone() for n, t in b.cache.items()}
    table = kv_ops.rotary_table(64, D)
    q, k, v = (heads(rng, (T, n, D), dtype) for n in (Hq, H, H))
    buf = torch.full((T + 2 * GUARD, Hq, D), 7.5, dtype=q.dtype, device="cuda")
    cache, s, err = kv_ops._cache_of(b.cache, "test"), None, _native.error_buffer()
    offsets = i32(cu)
    s = _native.KvSeqs(b.block_table.data_ptr(), b.lengths.data_ptr(), offsets.data_ptr(), 2, b.cols, T, T)
    t, _ = kv_ops._rotary_of(table, "half", D, q.device, "test")
    rows = [ct.byref(kv_ops._rows(x)) for x in (k, v, q, buf[GUARD:GUARD + T])]
    st = _native.lib().dmx_kv_append(ct.byref(cache), ct.byref(s), *rows, {"bf16": 0, "f32": 1}[dtype], ct.byref(t),
                                     torch.cuda.current_stream().cuda_stream, err, len(err))
    _native.check(st, err, "dmx_kv_append")
    assert (buf[:GUARD] == 7.5).all() and (buf[GUARD + T:] == 7.5).all()
    got = [f64(x) for x in kv_ops.read(b.cache, b.block_table, b.lengths, T, cu=offsets)]
    seen = np.zeros(T, bool)
    touched = np.zeros((b.cache["k_codes"].shape[0], 8), bool)
    for n, length in enumerate((40, 23)):
        at = min(max(cu[n], 0), T)
        count = min(max(cu[n + 1], at), T) - at
        if not count:
            continue
        p = np.arange(length - count, length)
        seen[at:at + count] = True
        touched[b.table[n, p // 8], p % 8] = True
        turned = R.rotate(f64(k)[at:at + count], p, f64(table), "half", np.float32)
        assert np.array_equal(got[0][at:at + count], R.cached(turned))
        assert np.array_equal(got[1][at:at + count], R.cached(f64(v)[at:at + count]))
        want = R.rotate(f64(q)[at:at + count], p, f64(table), "half", np.float32)
        assert torch.equal(buf[GUARD + at:GUARD + at + count].cpu(), torch.from_numpy(want).to(DT[dtype]))
    assert all(np.isnan(x[~seen]).all() for x in got)
    same = torch.from_numpy(~touched).cuda()
    for name in ("k_codes", "k_scales"):
        assert torch.equal(b.cache[name].transpose(1, 2)[same], before[name].transpose(1, 2)[same])
    for name in ("v_codes", "v_scales"):
        now, was = (x[name].permute(0, 2, 4, 1, 3).flatten(1, 2)[same] for x in (b.cache, before))
        assert torch.equal(now, was)


# --------------------------------------------------- numbers past 32 bits --


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("over", [2 ** 30, 2 ** 31, 2 ** 32 + 1, 2 ** 64 + 1], ids=str)
def test_bounds_past_32_bits_are_no_bounds(over, native, monkeypatch):
    """A window or a bound longer than any table: every position, every row."""
    rng = np.random.default_rng(33)
    b = Batch(rng, [(70, 90), (3, 60)], 1, 64, 16)
    b.fill(rng)
    q = heads(rng, (73, 2, 64), "bf16")
    want = kv_ops.attention(q, b.cache, b.block_table, b.lengths, **b.args, return_lse=True)
    if not native:
        monkeypatch.setattr(_native, "_calls", None)
    for kw in ({"window": over}, {"max_tokens": over}, {"max_length": over}, {"window": over, "max_tokens": 70, "max_length": 90}):
        got = kv_ops.attention(q, b.cache, b.block_table, b.lengths, **b.args, return_lse=True, **kw)
        assert all(torch.equal(x, y) for x, y in zip(got, want)), kw


def test_too_many_tokens_are_refused():
    table = kv_ops.rotary_table(4, 64)
    many = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda").expand(2 ** 32 + 1, 1, 64)
    few = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    b = Batch(np.random.default_rng(0), [(1, 20)] * 2, 1, 64, 16)
    for call in (lambda: kv_ops.rotary(many, None, b.lengths, table),
                 lambda: kv_ops.append(b.cache, many, many, b.block_table, b.lengths, cu=i32([0, 1, 2])),
                 lambda: kv_ops.attention(many, b.cache, b.block_table, b.lengths, cu=i32([0, 1, 2])),
                 lambda: kv_ops.read(b.cache, b.block_table, b.lengths, 2 ** 32 + 2),
                 lambda: kv_ops.read(b.cache, b.block_table, b.lengths, 2 ** 64 + 2),
                 lambda: kv_ops.read(b.cache, b.block_table, b.lengths, -2)):
        with pytest.raises(ValueError, match="tokens"):
            call()
    with pytest.raises(ValueError, match="max_length"):
        kv_ops.attention(few, b.cache, b.block_table, b.lengths, max_length=-1)


# ---------------------------------------------------------------- gradients --


def test_a_table_that_asks_for_a_gradient_is_refused():
    b = Batch(np.random.default_rng(0), [(1, 20)] * 2, 2, 64, 16)
    q, k, v = (heads(np.random.default_rng(1), (2, n, 64), "bf16") for n in (4, 2, 2))
    table = kv_ops.rotary_table(32, 64).requires_grad_()
    before = {n: t.clone() for n, t in b.cache.items()}
    for call in (lambda: kv_ops.rotary(q, k, b.lengths, table),
                 lambda: kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, q=q)):
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
    assert all(torch.equal(before[n], b.cache[n]) for n in before)
    with torch.no_grad():
        assert torch.equal(kv_ops.rotary(q, None, b.lengths, table)[0], kv_ops.rotary(q, None, b.lengths, table.detach())[0])


@pytest.mark.parametrize("native", [True, False])
def test_tensors_with_a_tangent_are_refused(native, monkeypatch):
    """Forward-mode derivatives have no more of a gradient here than backward ones."""
    from torch.autograd import forward_ad

    if not native:
        monkeypatch.setattr(_native, "_calls", None)
    b = Batch(np.random.default_rng(0), [(1, 20)] * 2, 2, 64, 16)
    q, k, v = (heads(np.random.default_rng(1), (2, n, 64), "bf16") for n in (4, 2, 2))
    table = kv_ops.rotary_table(32, 64)
    before = {n: t.clone() for n, t in b.cache.items()}
    with forward_ad.dual_level():
        dual = lambda x: forward_ad.make_dual(x, torch.ones_like(x))  # noqa: E731
        for call in (lambda: kv_ops.rotary(dual(q), k, b.lengths, table), lambda: kv_ops.rotary(q, dual(k), b.lengths, table),
                     lambda: kv_ops.rotary(q, k, b.lengths, dual(table)),
                     lambda: kv_ops.append(b.cache, dual(k), v, b.block_table, b.lengths),
                     lambda: kv_ops.append(b.cache, k, dual(v), b.block_table, b.lengths),
                     lambda: kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, q=dual(q)),
                     lambda: kv_ops.attention(dual(q), b.cache, b.block_table, b.lengths)):
            with pytest.raises(RuntimeError, match="no gradient"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="no gradient"):  # (which leaves tangents on)
                call()
        assert kv_ops.rotary(q, k, b.lengths, table)[0].shape == q.shape  # plain tensors of the same level are taken
    assert all(torch.equal(before[n], b.cache[n]) for n in before)


# ------------------------------------------------------------------ devices --


def test_the_tensors_device_is_current_for_a_launch(monkeypatch):
    """On the general path each launch is made inside its tensors' device (the
    native call has a guard of its own; with one GPU nothing tells that)."""
    b = Batch(np.random.default_rng(0), [(1, 20)] * 2, 2, 64, 16)
    q, k, v = (heads(np.random.default_rng(1), (2, n, 64), "bf16") for n in (4, 2, 2))
    table = kv_ops.rotary_table(32, 64)
    inside, seen = [], []

    class Device(torch.cuda.device):
        def __enter__(self):
            super().__enter__()
            inside.append(self.idx)

        def __exit__(self, *a):
            inside.pop()
            return super().__exit__(*a)

    class Lib:
        def __getattr__(self, name):
            fn = getattr(real, name)
            if name.endswith("workspace"):
                return fn
            return lambda *a: (seen.append((name, list(inside))), fn(*a))[1]

    real = _native.lib()
    monkeypatch.setattr(_native, "_calls", None)
    monkeypatch.setattr(_native, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "device", Device)
    kv_ops.rotary(q, k, b.lengths, table)
    kv_ops.append(b.cache, k, v, b.block_table, b.lengths)
    kv_ops.read(b.cache, b.block_table, b.lengths, 2)
    kv_ops.attention(q, b.cache, b.block_table, b.lengths)
    assert seen == [(n, [q.device.index]) for n in ("dmx_rotary", "dmx_kv_append", "dmx_kv_read", "dmx_kv_attention")]


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two GPUs")
@pytest.mark.parametrize("native", [True, False])
def test_tensors_of_another_device_than_the_current_one(native, monkeypatch):
    rng = np.random.default_rng(0)
    b = Batch(rng, [(70, 200)] * 2, 2, 128, 16)
    b.fill(rng)
    q = heads(rng, (140, 4, 128), "bf16")
    want = kv_ops.attention(q, b.cache, b.block_table, b.lengths)
    if not native:
        monkeypatch.setattr(_native, "_calls", None)
    there = torch.device("cuda:1")
    cache = {n: t.to(there) for n, t in b.cache.items()}
    got = kv_ops.attention(q.to(there), cache, b.block_table.to(there), b.lengths.to(there))
    assert got.device == there and torch.equal(got.cpu(), want.cpu())


# -------------------------------------------------------------- large values --


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 40])
@pytest.mark.parametrize("shape", ["rise", "steps"])
def test_large_values_under_scores_that_rise(shape, tokens, dtype):
    """Values up to the documented 2^107 / tokens, where weights grow to 2^20
    before their row's reference follows."""
    rng = np.random.default_rng(22)
    D, length = 64, 900
    b = Batch(rng, [(tokens, length)], 1, D, 32)
    at = np.arange(length) / length
    gain = {"rise": at * 60, "steps": np.floor(at * 8) * 9}[shape]
    direction = np.sign(rng.standard_normal(D))
    k = torch.from_numpy((gain[:, None, None] * direction + rng.standard_normal((length, 1, D))).astype(np.float32)).cuda()
    v = rng.standard_normal((length, 1, D)).clip(-4, 4) * 2.0 ** 95  # 4 * 2^95 <= 2^107 / 900
    held = b.fill(rng, k.to(torch.bfloat16), torch.from_numpy(v.astype(np.float32)).cuda().to(torch.bfloat16))
    q = torch.from_numpy((direction * (1 + 0.1 * rng.standard_normal((tokens, 3, D)))).astype(np.float32)).cuda().to(DT[dtype])
    got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, return_lse=True)
    check_attention(b, held, q, dtype, got, lse)


# -------------------------------------------------------------- more forms --


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", kv_ops.HEAD_DIMS)
@pytest.mark.parametrize("window", [None, 70])
@pytest.mark.parametrize("page", [8, 16, 32, 64])
def test_prompts_of_every_head_and_page(page, window, D, dtype):
    """Prompts unsplit and split over workgroups, pages that hold whole blocks
    of 32 and pages that do not, rows that see nothing among them (a prompt
    longer than its sequence's tokens)."""
    rng = np.random.default_rng(D + page)
    for sizes, spare in (([(300, 300), (70, 411), (1, 64), (0, 10)], 0), ([(90, 1500)], 1)):
        b = Batch(rng, sizes, 1, D, page, spare)
        held = b.fill(rng)
        q = heads(rng, (b.total, 2, D), dtype, 1.5)
        got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, window=window, return_lse=True, **b.args)
        check_attention(b, held, q, dtype, got, lse, True, window)
    short = Batch(rng, [(90, 90)], 1, D, page)
    held = short.fill(rng)
    q = heads(rng, (90, 2, D), dtype)
    got, lse = kv_ops.attention(q, short.cache, short.block_table, i32([40]), window=window, return_lse=True)
    out, l = f64(got), f64(lse)
    assert (out[:50] == 0).all() and np.isneginf(l[:50]).all()
    want, wl, spread, reach = R.attention(f64(q), held[0][0][:40], held[0][1][:40], -50, D ** -0.5, True, window)
    assert (np.abs(out - want) <= R.bound(want, spread, reach, 40, D, dtype == "bf16")).all()
    assert (np.abs(l - wl)[50:] <= R.lse_bound(wl, reach, 40, D)[50:]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", kv_ops.HEAD_DIMS)
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("tokens", [1, 8, 50])
@pytest.mark.parametrize("page", [16, 64])
def test_nan_blocks_through_splits(page, tokens, which, D, dtype):
    """A block that is not finite, in every split and beside their edges, alone:
    its channels (a key's: all) of the rows that see it, through the join."""
    rng = np.random.default_rng(tokens + D)
    length = 1500
    b = Batch(rng, [(tokens, length)], 1, D, page, spare=0)
    k, v = (heads(rng, (length, 1, D), "bf16") for _ in range(2))
    q = heads(rng, (tokens, 2, D), dtype)
    for at in (0, 127, 128, 135, 136, 703, 704, 1407, length - tokens // 2 - 1, length - 1):
        x = (k if which == "k" else v).clone()
        x[at, 0, D - 5] = float("nan") if at % 2 else float("inf")
        held = b.fill(rng, *((x, v) if which == "k" else (k, x)))
        for window in (None, 97):
            got, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, window=window, return_lse=True)
            check_attention(b, held, q, dtype, got, lse, True, window)


def test_modes_subclasses_and_vmap():
    """What the native call leaves to the general path gives the same bits; a
    batched tensor, which has no address, is refused."""
    from torch.overrides import TorchFunctionMode
    from torch.utils._python_dispatch import TorchDispatchMode

    made = []

    class Function(TorchFunctionMode):
        def __torch_function__(self, func, types, args=(), kwargs=None):
            made.append(getattr(func, "__name__", str(func)))
            return func(*args, **(kwargs or {}))

    class Dispatch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            made.append(str(func))
            return func(*args, **(kwargs or {}))

    class Sub(torch.Tensor):
        pass

    rng = np.random.default_rng(41)
    b = Batch(rng, [(3, 600), (2, 33)], 2, 64, 16)
    b.fill(rng)
    table = kv_ops.rotary_table(1024, 64)
    q, k, v = (heads(rng, (5, n, 64), "bf16") for n in (4, 2, 2))
    at = i32(range(5))

    calls = {"rotary": lambda q: kv_ops.rotary(q, k, at, table)[0],
             "append": lambda q: kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=table, q=q, **b.args),
             "attention": lambda q: kv_ops.attention(q, b.cache, b.block_table, b.lengths, **b.args)}
    for name, call in calls.items():
        want = call(q)
        for mode in (Function, Dispatch):
            made.clear()
            with mode():
                got = call(q)
            assert torch.equal(got, want) and any("empty" in n for n in made), name
        assert torch.equal(call(q.as_subclass(Sub)).as_subclass(torch.Tensor), want), name
        with pytest.raises(RuntimeError):
            torch.vmap(call)(q[None])


def test_threads_with_a_stream_each():
    """Inputs made late on each thread's stream, outputs read there."""
    import threading

    rng = np.random.default_rng(42)
    b = Batch(rng, [(1, 3000)] * 2, 2, 64, 16)
    b.fill(rng)
    xs = [heads(rng, (2, 8, 64), "bf16") for _ in range(4)]
    table = kv_ops.rotary_table(4096, 64)
    at = i32([2999, 2999])

    def call(x):
        return kv_ops.attention(kv_ops.rotary(x, None, at, table)[0], b.cache, b.block_table, b.lengths)

    want = [call(x) for x in xs]
    torch.cuda.synchronize()
    good, errors = [False] * 4, []

    def work(i):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    x = torch.zeros_like(xs[i])
                    big = torch.randn(1024, 1024, device="cuda")
                    for _ in range(4):
                        big = big @ big * 1e-2
                    x.copy_(xs[i])  # (after the products: a launch on another stream would read zeros)
                    if not torch.equal(call(x), want[i]):
                        raise AssertionError(f"thread {i} read another stream's data")
                torch.cuda.current_stream().synchronize()
            good[i] = True
        except BaseException as e:  # noqa: BLE001 (handed to the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]
    assert all(good)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("part, first", [(6, 1), (6, 2), (34, 3), (64, 1)])
def test_a_slice_of_a_table_is_a_table(part, first, native, monkeypatch):
    """Also where it begins at an address that is not a multiple of 16."""
    if not native:
        monkeypatch.setattr(_native, "_calls", None)
    rng = np.random.default_rng(part)
    b = Batch(rng, [(3, 20)] * 2, 2, 64, 16)
    q, k, v = (heads(rng, (6, n, 64), "bf16") for n in (4, 2, 2))
    at, whole = i32([0, 5, 9, 1, 1, 30]), kv_ops.rotary_table(40, part)
    sliced = whole[first:]
    got = kv_ops.rotary(q, k, at, sliced)
    assert all(torch.equal(x, y) for x, y in zip(got, kv_ops.rotary(q, k, at + first, whole)))
    got = kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=sliced, q=q)
    assert torch.equal(got, kv_ops.append(b.cache, k, v, b.block_table, b.lengths, table=sliced.clone(), q=q))
