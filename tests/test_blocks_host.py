"""CPU: the C ABI of the pages, the axes, the selection and the norms
(include/dmx_kv.h, include/dmx_norm.h) is exported with the bindings' signatures
and structures, and refuses bad arguments by name before any device call; tables of several axes against
their formula; refusals of the Python surface that need no GPU; and the tests' oracle against itself."""

import ctypes as ct
import os
import re

import numpy as np
import pytest
import torch

from drinkme_amd import _native, kv_ops, norm_ops
from tests import blocks_reference as B
from tests.test_kv_host import FAKE, SHARED, _cache, _refused, _rows, _seqs, _table, cpu_only

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def header(name):
    return re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", name)).read(), flags=re.S)


def test_the_norm_header_is_bound_and_exported():
    declared = sorted(set(re.findall(r"\b(dmx_\w+)\s*\(", header("dmx_norm.h"))))
    assert declared == sorted(_native.NORM_SIGNATURES)
    lib = ct.CDLL(_native.LIB)
    assert all(hasattr(lib, name) for name in declared)


@pytest.mark.parametrize("struct, name, file", [
    (_native.KvRotaryAxes, "dmx_rotary_axes", "dmx_kv.h"), (_native.KvPool, "dmx_kv_pool", "dmx_kv.h"),
    (_native.KvSummaries, "dmx_kv_summaries", "dmx_kv.h"), (_native.Vectors, "dmx_vectors", "dmx_norm.h"),
    (_native.NormForm, "dmx_norm_form", "dmx_norm.h")])
def test_structures_have_the_header_s_fields_in_order(struct, name, file):
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, header(file), re.S).group(1)
    assert re.findall(r"(\w+)(?:\[\d+\])?\s*;", body) == [f[0] for f in struct._fields_]


def test_constants_are_the_header_s():
    assert re.search(r"DMX_KV_MAX_COLUMNS (\d+)", header("dmx_kv.h")).group(1) == str(_native.KV_MAX_COLUMNS)
    text = header("dmx_norm.h")
    for name in ("NORM_RMS", "NORM_LAYER", "NORM_MAX_DIM"):
        assert re.search(r"DMX_%s (\d+)" % name, text).group(1) == str(getattr(_native, name))


# ------------------------------------------------------------------ refusals --


def _pool(**kw):
    p = _native.KvPool(FAKE, FAKE, FAKE, 12)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"pool": None}, b"null pool"), ({"pool": _pool(free=None)}, b"null pool"), ({"pool": _pool(lacking=None)}, b"null pool"),
    ({"pool": _pool(pages=0)}, b"pool of no pages"), ({"pool": _pool(pages=1 << 30)}, b"too many"), ({"table": None}, b"null block table"),
    ({"lengths": None}, b"lengths"), ({"batch": 0}, b"no sequences"), ({"cols": 0}, b"without columns"), ({"batch": 65536}, b"too many sequences"),
    ({"page": 24}, b"power of two"), ({"page": 2048}, b"power of two"), ({"cols": 1 << 24}, b"2\\^30 positions")])
def test_bad_pages_are_refused(change, match):
    a = {"pool": _pool(), "table": FAKE, "lengths": FAKE, "given": FAKE, "batch": 2, "cols": 3, "page": 64}
    a.update(change)
    a = list(a.values())
    assert re.search(match, _refused("dmx_kv_reserve", *a, 4, FAKE, FAKE, FAKE))
    assert re.search(match, _refused("dmx_kv_trim", *a))


@cpu_only
def test_bad_reservations_are_refused():
    a = [_pool(), FAKE, FAKE, FAKE, 2, 3, 64]
    assert b"too many tokens" in _refused("dmx_kv_reserve", *a, 1 << 30, FAKE, FAKE, FAKE)
    for outs in ((None, FAKE, FAKE), (FAKE, None, FAKE), (FAKE, FAKE, None)):
        assert b"null offsets" in _refused("dmx_kv_reserve", *a, 4, *outs)
    a[3] = None
    assert b"not a multiple" in _refused("dmx_kv_reserve", *a, 5, FAKE, FAKE, FAKE)
    assert b"keep" in _refused("dmx_kv_trim", *a)


def _axes(*of, count=3):
    x = _native.KvRotaryAxes()
    x.count = count
    for i, a in enumerate(of):
        x.of[i // 16] |= a << (2 * (i % 16))
    return x


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"axes": None}, b"null axes"), ({"axes": _axes(count=0)}, b"no axes"), ({"axes": _axes(count=5)}, b"more than 4"),
    ({"axes": _axes(0, 1, 3)}, b"axis that there is not"), ({"table": _table(dim=514), "dim": 514}, b"256 angles"),
    ({"positions": None}, b"null positions"), ({"in": None}, b"null rows"), ({"n": 3}, b"one or two"), ({"dtype": 7}, b"dtype"),
    ({"dim": 127}, b"head dim odd"), ({"tokens": 1 << 30}, b"too many tokens"), ({"out": _rows(heads=3)}, b"as many out")])
def test_bad_rotations_are_refused(change, match):
    a = {"in": _rows(), "out": _rows(), "n": 1, "tokens": 4, "dim": 128, "dtype": 0, "positions": FAKE, "wide": 0,
         "axes": _axes(0, 1, 2), "table": _table()}
    a.update(change)
    assert re.search(match, _refused("dmx_rotary_by_axes", *a.values()))


def _summaries(**kw):
    s = _native.KvSummaries(FAKE, FAKE)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@cpu_only
@pytest.mark.parametrize("cache, seqs, match", SHARED)
def test_bad_caches_and_sequences_are_refused(cache, seqs, match):
    c = None if cache is None else _cache(**cache)
    s = None if seqs is None else _seqs(**seqs)
    said = [_refused("dmx_kv_summarize", c, _summaries(), s), _refused("dmx_kv_select", c, _summaries(), s, _rows(), 0, 2, 1, 1, 1, FAKE, None, 0),
            _refused("dmx_kv_attention_blocks", c, s, _rows(), 0, 1.0, 1, FAKE, 2, 0, FAKE, None, None, 0)]
    assert all(re.search(match, x) for x in said), said
    c, s = ct.byref(c) if c else None, ct.byref(s) if s else None
    assert _native.lib().dmx_kv_attention_blocks_workspace(c, s, 4, 0, 2, 0) == 0 == _native.lib().dmx_kv_select_workspace(c, s, 4)


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"summaries": None}, b"null summaries"), ({"summaries": _summaries(scales=None)}, b"null summaries"),
    ({"summaries": _summaries(bounds=FAKE + 8)}, b"not 16-byte"), ({"q": None}, b"null queries"), ({"q": _rows(heads=3)}, b"query heads"),
    ({"dtype": 2}, b"dtype"), ({"count": 0}, b"no columns"), ({"count": 16385}, b"16384"), ({"first": 3}, b"more than count"),
    ({"first": 2 ** 32 - 1, "last": 2}, b"more than count"), ({"seqs": _seqs(table_cols=16385)}, b"16384"), ({"blocks": None}, b"lists"),
    ({"q": _rows(at=None)}, b"null queries"), ({"ws": None}, b"workspace"), ({"ws": FAKE + 8}, b"workspace"), ({"bytes": 64}, b"workspace")])
def test_bad_selections_are_refused(change, match):
    a = {"cache": _cache(), "summaries": _summaries(), "seqs": _seqs(table_cols=4000), "q": _rows(), "dtype": 0, "count": 2, "first": 1,
         "last": 1, "causal": 1, "blocks": FAKE, "ws": FAKE, "bytes": 1 << 30}
    need = _native.lib().dmx_kv_select_workspace(ct.byref(a["cache"]), ct.byref(a["seqs"]), 2)
    assert 64 < need < 1 << 30
    a.update(change)
    assert re.search(match, _refused("dmx_kv_select", *a.values()))


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"q": None}, b"null queries"), ({"q": _rows(heads=3)}, b"query heads"), ({"scale": 0.0}, b"scale"), ({"scale": float("nan")}, b"scale"),
    ({"scale": 3e38}, b"scale"), ({"blocks": None}, b"lists"), ({"count": 0}, b"no columns"), ({"count": 16385}, b"16384"), ({"out": None}, b"output"),
    ({"seqs": _seqs(table_cols=16385)}, b"16384"), ({"dtype": 3}, b"dtype"), ({"ws": None}, b"workspace"), ({"ws": FAKE + 8}, b"workspace"),
    ({"bytes": 64}, b"workspace"), ({"seqs": _seqs(cu=FAKE, max_tokens=0)}, b"max_tokens is 0")])
def test_bad_attentions_are_refused(change, match):
    a = {"cache": _cache(), "seqs": _seqs(table_cols=64), "q": _rows(heads=8), "dtype": 0, "scale": 1.0, "causal": 1, "blocks": FAKE,
         "count": 64, "max_length": 0, "out": FAKE, "lse": None, "ws": FAKE, "bytes": 1 << 30}
    need = _native.lib().dmx_kv_attention_blocks_workspace(ct.byref(a["cache"]), ct.byref(a["seqs"]), 8, 0, 64, 0)
    assert 64 < need < 1 << 30
    a.update(change)
    assert re.search(match, _refused("dmx_kv_attention_blocks", *a.values()))


@cpu_only
@pytest.mark.parametrize("total, q_heads, heads, seqs", [
    (131071, 64, 8, {}), (131072, 64, 8, {}), (262144, 32, 8, {}), (300000, 32, 8, {"batch": 4, "cu": FAKE, "max_tokens": 300000}),
    (65535 * 16, 2, 2, {}), (65535 * 16 + 1, 2, 2, {}), (2 ** 30 - 1, 2, 2, {}), (32767, 65535, 1, {})])
def test_attentions_over_long_prompts_pass_the_checks(total, q_heads, heads, seqs):
    """What the attention over everything takes, the one over lists takes, too: it comes as far as the device."""
    c, s, q = _cache(heads=heads), _seqs(**{"batch": 1, "table_cols": 16384, "total": total, **seqs}), _rows(heads=q_heads)
    assert _refused("dmx_kv_attention_blocks", c, s, q, 0, 1.0, 1, FAKE, 32, 0, FAKE, None, FAKE, 1 << 60) == b"no current device"


@cpu_only
def test_rows_past_31_bits_are_refused():
    for total, q_heads in ((2 ** 30 - 1, 3), (2 ** 25, 64), (2 ** 30 - 1, 65535)):
        s = _seqs(batch=1, table_cols=16384, total=total)
        assert b"too many query rows" in _refused("dmx_kv_attention_blocks", _cache(heads=1), s, _rows(heads=q_heads), 0, 1.0, 1, FAKE, 32, 0, FAKE, None,
                                                  FAKE, 1 << 60)


def _form(**kw):
    f = _native.NormForm(0, 1e-6, 0.0, 1.0)
    for k, v in kw.items():
        setattr(f, k, _native.Vectors(*v) if isinstance(v, tuple) else v)
    return f


NORM_SHARED = [({"kind": 2}, b"kind"), ({"eps": -1.0}, b"eps"), ({"eps": float("nan")}, b"eps"), ({"eps": float("inf")}, b"eps"),
               ({"offset": float("nan")}, b"offset"), ({"weight": (FAKE, 0, 2)}, b"one row"), ({"bias": (FAKE, 5, 1)}, b"bias: dtype")]


@cpu_only
@pytest.mark.parametrize("form, match", NORM_SHARED + [(None, b"null form")])
def test_bad_norms_are_refused(form, match):
    f = None if form is None else _form(**form)
    assert re.search(match, _refused("dmx_norm", _rows(), FAKE, 4, 128, 0, f))
    assert re.search(match, _refused("dmx_block_norm", FAKE, 128, FAKE, 128, FAKE, FAKE, 4, 128, 0, 0, f))


@cpu_only
def test_bad_rows_of_norms_are_refused():
    for args, match in (((None, FAKE, 4, 128, 0), b"null rows"), ((_rows(at=None), FAKE, 4, 128, 0), b"null rows"), ((_rows(), None, 4, 128, 0), b"null rows"),
                        ((_rows(), FAKE, 4, 0, 0), b"no channels"), ((_rows(), FAKE, 4, 32769, 0), b"32768"), ((_rows(heads=0), FAKE, 4, 128, 0), b"no heads"),
                        ((_rows(heads=65535), FAKE, 1 << 20, 128, 0), b"too many rows"), ((_rows(), FAKE, 4, 128, 9), b"dtype")):
        assert re.search(match, _refused("dmx_norm", *args, _form()))
    good = dict(y=FAKE, ys=128, r=FAKE, rs=128, ro=FAKE, out=FAKE, rows=4, dim=128, dtype=0, rdtype=0, form=_form())
    for kw, match in (({"y": None}, b"null rows"), ({"ro": None}, b"null rows"), ({"dtype": 1}, b"bf16 residual"), ({"rdtype": 4}, b"dtype"),
                      ({"rows": 1 << 31}, b"too many rows"), ({"form": _form(factor=float("inf"))}, b"factor"),
                      ({"form": _form(post=(FAKE, 0, 4))}, b"one row"), ({"form": _form(gate=(FAKE, 0, 3))}, b"gate: 3 rows"),
                      ({"form": _form(gate=(FAKE, 0, 0))}, b"gate: 0 rows"), ({"form": _form(scale=(FAKE, 0, 1))}, b"without a shift"),
                      ({"form": _form(shift=(FAKE, 0, 1))}, b"without a scale"), ({"form": _form(scale=(FAKE, 0, 1), shift=(FAKE, 0, 4))}, b"different rows"),
                      ({"form": _form(cu=FAKE, batch=0)}, b"no sequences"), ({"form": _form(cu=FAKE, batch=2, gate=(FAKE, 0, 3))}, b"gate: 3 rows")):
        assert re.search(match, _refused("dmx_block_norm", *{**good, **kw}.values()))


def test_workspaces_of_too_many_heads_are_none():
    """As for any call that is refused; the query returns, whatever it is asked."""
    s = ct.byref(_seqs(table_cols=4000))
    for heads, q_heads in ((1, 2 ** 32 - 1), (1, 2 ** 31 + 1), (2, 2 ** 32 - 2), (1, 65536), (65535, 65535 * 65537)):
        c = ct.byref(_cache(heads=heads))
        assert _native.lib().dmx_kv_select_workspace(c, s, q_heads) == 0, q_heads
    assert _native.lib().dmx_kv_select_workspace(ct.byref(_cache(heads=1)), s, 65535) > 0


@cpu_only
def test_norms_of_no_rows_return():
    """With vectors of several rows, too: no row divides them."""
    err = _native.error_buffer()
    for kw in ({}, {"gate": (FAKE, 0, 2)}, {"scale": (FAKE, 0, 3), "shift": (FAKE, 1, 3)}, {"cu": FAKE, "batch": 4, "gate": (FAKE, 0, 2)},
               {"cu": FAKE, "batch": 4, "gate": (FAKE, 0, 4)}, {"gate": (FAKE, 0, 2 ** 32 - 1)}):
        f = _form(**kw)
        assert _native.lib().dmx_block_norm(FAKE, 128, FAKE, 128, FAKE, FAKE, 0, 128, 0, 0, ct.byref(f), None, err, len(err)) == 0, kw
    f = _form()
    assert _native.lib().dmx_norm(ct.byref(_rows()), FAKE, 0, 128, 0, ct.byref(f), None, err, len(err)) == 0
    assert b"gate: 0 rows" in _refused("dmx_block_norm", FAKE, 128, FAKE, 128, FAKE, FAKE, 0, 128, 0, 0, _form(gate=(FAKE, 0, 0)))


def test_calls_off_the_gpu_are_refused():
    x = torch.zeros((2, 2, 64))
    cache = kv_ops.new_cache(2, 16, 2, 64, device="cpu")
    pool, one = kv_ops.new_pool(4, device="cpu"), torch.ones(2, dtype=torch.int32)
    table, s = one[:, None].contiguous(), kv_ops.new_summaries(cache)
    for call in (lambda: kv_ops.reserve(pool, table, one, 16, 2), lambda: kv_ops.trim(pool, table, one, 16, one),
                 lambda: kv_ops.rotary(x, None, torch.zeros((2, 2), dtype=torch.int32), kv_ops.rotary_table(4, 64, device="cpu"), axes=(0, 1) * 16),
                 lambda: kv_ops.summarize(cache, s, table, one, 2), lambda: kv_ops.select(x, cache, s, table, one, 1, last=0),
                 lambda: norm_ops.norm(x), lambda: norm_ops.block_norm(x[0], x[0])):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_a_modulation_without_its_parts_is_refused(monkeypatch):
    """Before any path is taken: the native call sees no modulation in it."""
    y, one = torch.zeros((2, 64)), torch.ones(64)

    class Native:
        def block_norm(self, *args):
            return y, y

    monkeypatch.setattr(_native, "calls", Native)
    for modulate in ((None, None), (one, None), (None, one)):
        with pytest.raises(ValueError, match="modulate"):
            norm_ops.block_norm(y, y, modulate=modulate)


# -------------------------------------------------------------------- tables --


def test_pools_and_summaries_as_they_begin():
    p = kv_ops.new_pool(5, device="cpu")
    assert p["free"].tolist() == [4, 3, 2, 1, 0] and p["count"].tolist() == [5] and p["lacking"].tolist() == [0]
    for pages in (0, -1, 1 << 30):
        with pytest.raises(ValueError, match="pages"):
            kv_ops.new_pool(pages, device="cpu")
    s = kv_ops.new_summaries(kv_ops.new_cache(3, 16, 2, 96, device="cpu"))
    assert s["bounds"].shape == (3, 2, 2, 96) and s["scales"].shape == (3, 2)


def test_axes_are_dealt_as_said():
    assert kv_ops.rotary_axes((2, 3, 1)) == (0, 0, 1, 1, 1, 2)
    assert kv_ops.rotary_axes((2, 3, 1), "interleaved") == (0, 1, 2, 0, 1, 1)
    assert kv_ops.rotary_axes((0, 2), "interleaved") == (1, 1)
    for sections in ((), (0, 0), (1, -1), (1,) * 5, (200, 57)):
        with pytest.raises(ValueError, match="sections"):
            kv_ops.rotary_axes(sections)
    with pytest.raises(ValueError, match="order"):
        kv_ops.rotary_axes((1,), "other")


def test_axes_are_whole_numbers_every_time():
    """Whatever was asked for before: what equals an axis without being a whole number is refused, too."""
    kv_ops._packed_axes.cache_clear()
    for _ in range(2):
        for axes in ((1.0, 0.0, 2.0), (0, 4), (-1,), (0.5,), ("0",), (None,), (256,), (), (0,) * 257, 3):
            with pytest.raises(ValueError, match="numbers of 0..3"):
                kv_ops._axes_of(axes)
        for axes in ((1, 0, 2), [1, 0, 2], (np.int64(1), False, np.uint8(2))):
            x = kv_ops._axes_of(axes)
            assert (x.count, x.angles, x.of[0]) == (3, 3, 1 | 2 << 4)


def test_tables_of_several_axes():
    axes = kv_ops.rotary_axes((3, 5, 2), "interleaved")
    table = kv_ops.rotary_table(40, 20, base=1e4, device="cpu", axes=axes).double()
    at = np.arange(40.0)
    for a, n in enumerate((3, 5, 2)):
        mine = [i for i, x in enumerate(axes) if x == a]
        for j, i in enumerate(mine):
            angle = at * 1e4 ** (-j / n)
            assert np.abs(table[:, i, 0].numpy() - np.cos(angle)).max() < 1e-7 and np.abs(table[:, i, 1].numpy() - np.sin(angle)).max() < 1e-7
    one = kv_ops.rotary_table(40, 20, device="cpu", axes=(0,) * 10, scaling={"kind": "linear", "factor": 2.0})
    assert torch.equal(one, kv_ops.rotary_table(40, 20, device="cpu", scaling={"kind": "linear", "factor": 2.0}))
    for kw, match in (({"axes": axes[:9]}, "9 angles"), ({"axes": axes, "scaling": {"kind": "divisors", "divisors": [1.0] * 10}}, "divisors"),
                      ({"axes": (0,) * 9 + (1,), "scaling": {"kind": "base", "factor": 2.0}}, "one angle")):
        with pytest.raises(ValueError, match=match):
            kv_ops.rotary_table(40, 20, device="cpu", **kw)


# -------------------------------------------------------------------- oracle --


def test_the_oracle_s_summaries_bound_their_keys():
    rng = np.random.default_rng(0)
    for scale in (1e-30, 1.0, 1e20):
        k = rng.standard_normal((9, 64)) * scale
        bounds, e = B.summary(k)
        unit = 2.0 ** (e - 127)
        assert (bounds[0] * unit >= k.max(0)).all() and (bounds[1] * unit <= k.min(0)).all() and np.abs(bounds).max() in range(64, 128)
        q = rng.standard_normal((3, 64))
        w = B.whole_queries(q)
        assert np.abs(w).max() in range(64, 128)
        assert B.score(q, bounds, e) >= (w @ k.T).max() * (1 - 1e-6)


def test_the_oracle_sees_planted_mistakes():
    free, table, lengths = [3, 1, 2, 0], [[5, -1], [-1, -1]], [8, 0]
    cu, positions, slots, count, lacking = B.reserve(free, 4, table, lengths, [1, 3], 8, 5, 9)
    assert (cu, positions, slots, count, lacking) == ([0, 1, 4], [8, 0, 1, 2, -1], [0, 16, 17, 18, -1], 2, 0)
    assert B.trim(free, count, table, lengths, [8, 0], 8) == 4 and free == [3, 1, 2, 0] and table == [[5, -1], [-1, -1]]
    bounds = np.zeros((4, 2, 64), np.int64)
    bounds[2, 0], bounds[3, 0] = 1, 1
    q, scales = np.ones((1, 64)), np.full(4, 127)
    assert B.select(q, bounds, scales, [0, 1, 2, 3], 4, 2, 0, 0) == [2, 3]
    assert B.select(q, bounds, scales, [0, 1, 2, 3], 4, 2, 1, 0) == [0, 2]
    assert B.select(q, bounds, scales, [3, 1, 2, 9], 4, 2, 0, 1) == [0, 3]
    assert B.select(q, bounds, scales, [9, 1, 2, 9], 4, 3, 0, 0) == [0, 1, 2]
    assert B.select(q, bounds, scales, [0], 1, 2, 0, 0) == [0, -1]
