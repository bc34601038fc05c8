"""CPU: the key/value cache's C ABI (include/dmx_kv.h) is exported with the
bindings' signatures and refuses bad arguments by name before any device call;
rotary tables against their formulas; the Python surface's refusals that need
no GPU; and the tests' oracle against itself (a planted mistake is seen)."""

import ctypes as ct
import math
import os
import re

import numpy as np
import pytest
import torch

from drinkme_amd import _native, kv_ops
from tests import kv_reference as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "dmx_kv.h")


def test_the_header_is_bound_and_exported():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = sorted(set(re.findall(r"\b(dmx_\w+)\s*\(", text)))
    assert declared == sorted(_native.KV_SIGNATURES)
    lib = ct.CDLL(_native.LIB)
    assert all(hasattr(lib, name) for name in declared)


@pytest.mark.parametrize("struct, name", [(_native.KvCache, "dmx_kv_cache"), (_native.KvSeqs, "dmx_kv_seqs"),
                                          (_native.KvRows, "dmx_rows"), (_native.KvRotaryTable, "dmx_rotary_table")])
def test_structures_have_the_header_s_fields_in_order(struct, name):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\}" % name, text, re.S).group(1)
    fields = re.findall(r"(\w+)\s*;", body)
    assert fields == [f[0] for f in struct._fields_]


# ------------------------------------------------------------------ refusals --

FAKE = 0x10000  # never dereferenced: every case is refused first


def _cache(**kw):
    c = _native.KvCache(FAKE, FAKE, FAKE, FAKE, 4, 2, 64, 128)
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def _seqs(**kw):
    s = _native.KvSeqs(FAKE, FAKE, None, 2, 3, 4, 2)
    for k, v in kw.items():
        setattr(s, k, v)
    return s


def _rows(**kw):
    r = _native.KvRows(FAKE, 1024, 128, 2)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def _table(**kw):
    t = _native.KvRotaryTable(FAKE, 64, 128, 0)
    for k, v in kw.items():
        setattr(t, k, v)
    return t


def _refused(name, *args):
    err = _native.error_buffer()
    args = [ct.byref(a) if isinstance(a, ct.Structure) else a for a in args]
    assert getattr(_native.lib(), name)(*args, None, err, len(err)) == 1
    return err.value


SHARED = [
    (None, {}, b"null cache"),
    ({"k_codes": None}, {}, b"null cache buffer"),
    ({"v_codes": FAKE + 4}, {}, b"not aligned"),
    ({"k_scales": FAKE + 4}, {}, b"not aligned"),
    ({"pages": 0}, {}, b"empty cache"),
    ({"heads": 0}, {}, b"empty cache"),
    ({"pages": 1 << 31}, {}, b"too many pages"),
    ({"page": 48}, {}, b"power of two"),
    ({"page": 4}, {}, b"power of two"),
    ({"page": 2048}, {}, b"power of two"),
    ({"dim": 80}, {}, b"head dim"),
    ({}, None, b"null sequences"),
    ({}, {"table": None}, b"null block table"),
    ({}, {"lengths": None}, b"null block table or lengths"),
    ({}, {"batch": 0}, b"no sequences"),
    ({}, {"table_cols": 0}, b"without columns"),
    ({}, {"batch": 65536, "total": 65536}, b"too many sequences"),
    ({}, {"total": 1 << 30}, b"too many sequences or tokens"),
    ({}, {"table_cols": 1 << 26}, b"2\\^30 positions"),
    ({}, {"total": 5}, b"not a multiple"),
]
cpu_only = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="stand-in device pointers: CPU only")


@cpu_only
@pytest.mark.parametrize("cache, seqs, match", SHARED)
def test_bad_caches_and_sequences_are_refused(cache, seqs, match):
    c = None if cache is None else _cache(**cache)
    s = None if seqs is None else _seqs(**seqs)
    k = _rows()
    said = [_refused("dmx_kv_append", c, s, k, k, None, None, 0, None), _refused("dmx_kv_read", c, s, FAKE, FAKE),
            _refused("dmx_kv_attention", c, s, k, 0, 1.0, 1, 0, 0, FAKE, None, None, 0)]
    assert all(re.search(match, x) for x in said), said
    assert _native.lib().dmx_kv_attention_workspace(ct.byref(c) if c else None, ct.byref(s) if s else None, 4, 0, 0, 0) == 0


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"dtype": 5}, b"dtype"), ({"k": None}, b"null keys"), ({"q": None}, b"without their output"),
    ({"table": None}, b"without a rotary table"), ({"k": _rows(heads=3)}, b"other heads"),
    ({"q_out": _rows(heads=3)}, b"query heads"), ({"v": _rows(at=None)}, b"null rows"),
    ({"table": _table(at=None)}, b"null rotary table"), ({"table": _table(at=FAKE + 8)}, b"16-byte"),
    ({"table": _table(dim=130)}, b"rotary dim"), ({"table": _table(dim=7)}, b"rotary dim"),
    ({"table": _table(positions=0)}, b"without positions"), ({"table": _table(layout=2)}, b"layout"),
])
def test_bad_appends_are_refused(change, match):
    a = {"k": _rows(), "v": _rows(), "q": _rows(), "q_out": _rows(), "dtype": 0, "table": _table(), **change}
    assert re.search(match, _refused("dmx_kv_append", _cache(), _seqs(), *a.values()))


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"q": None}, b"null queries"), ({"q": _rows(heads=3)}, b"multiple of the cache's"),
    ({"q": _rows(at=None)}, b"null queries or output"), ({"out": None}, b"null queries or output"),
    ({"dtype": 2}, b"dtype"), ({"scale": 0.0}, b"scale"), ({"scale": float("inf")}, b"scale"),
    ({"window": 1 << 30}, b"window"), ({"workspace": None}, b"workspace"), ({"bytes": 64}, b"workspace"),
    ({"workspace": FAKE + 8}, b"workspace"),
])
def test_bad_attentions_are_refused(change, match):
    a = {"q": _rows(heads=8), "dtype": 0, "scale": 1.0, "causal": 1, "window": 0, "max_length": 0, "out": FAKE,
         "lse": None, "workspace": FAKE, "bytes": 1 << 40, **change}
    seqs = _seqs(table_cols=1000)  # (long enough to be split, which takes a workspace)
    need = _native.lib().dmx_kv_attention_workspace(ct.byref(_cache()), ct.byref(seqs), 8, 0, 0, 0)
    assert need > 64
    assert re.search(match, _refused("dmx_kv_attention", _cache(), seqs, *a.values()))


@cpu_only
@pytest.mark.parametrize("change, match", [
    ({"x": None}, b"null rows"), ({"n": 3}, b"one or two"), ({"dim": 7}, b"head dim"), ({"dim": 0}, b"head dim"),
    ({"positions": None}, b"null positions"), ({"x": _rows(heads=0)}, b"no heads"), ({"dtype": 9}, b"dtype"),
    ({"tokens": 1 << 30}, b"too many tokens"), ({"table": None}, b"null rows or table"),
])
def test_bad_rotations_are_refused(change, match):
    a = {"x": _rows(), "out": _rows(), "n": 1, "tokens": 4, "dim": 128, "dtype": 0, "positions": FAKE, "wide": 0,
         "table": _table(), **change}
    assert re.search(match, _refused("dmx_rotary", *a.values()))


def test_the_python_surface_refuses_what_is_not_on_the_gpu():
    x = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    ones = torch.ones(2, dtype=torch.int32)
    cache = kv_ops.new_cache(2, 16, 2, 64, device="cpu")
    table = kv_ops.rotary_table(4, 64, device="cpu")
    for call in (lambda: kv_ops.rotary(x, x, ones, table), lambda: kv_ops.append(cache, x, x, ones[:, None], ones),
                 lambda: kv_ops.attention(x, cache, ones[:, None], ones), lambda: kv_ops.read(cache, ones[:, None], ones, 2)):
        with pytest.raises(ValueError, match="GPU"):
            call()


@pytest.mark.parametrize("args, match", [((0, 16, 2, 64), "0 pages"), ((2, 12, 2, 64), "page_size 12"),
                                         ((2, 2048, 2, 64), "page_size"), ((2, 16, 2, 80), "head dim 80"),
                                         ((2, 16, 0, 64), "0 heads")])
def test_new_cache_refuses(args, match):
    with pytest.raises(ValueError, match=match):
        kv_ops.new_cache(*args, device="cpu")


def test_cache_bytes():
    c = kv_ops.new_cache(3, 16, 2, 96, device="cpu")
    assert kv_ops.cache_bytes(c) == 3 * 16 * 2 * 2 * 96 * 17 // 32


# -------------------------------------------------------------------- tables --


def _angles(t, magnitude=1.0):
    """The angles of position 1, which are below pi for base >= 1."""
    c, s = t[1, :, 0].double() / magnitude, t[1, :, 1].double() / magnitude
    assert torch.allclose(c * c + s * s, torch.ones_like(c), atol=1e-6)
    return torch.atan2(s, c).numpy()


def _plain(dim, base=10000.0):
    return np.array([base ** (-2 * i / dim) for i in range(dim // 2)])


def test_tables():
    make = lambda s=None, dim=64, **kw: kv_ops.rotary_table(300, dim, scaling=s, device="cpu", **kw)  # noqa: E731
    t = make()
    assert t.shape == (300, 32, 2) and t.dtype == torch.float32
    want = np.arange(300)[:, None] * _plain(64)
    assert np.abs(t[..., 0].numpy() - np.cos(want)).max() < 1e-7 and np.abs(t[..., 1].numpy() - np.sin(want)).max() < 1e-7
    close = lambda a, b: np.allclose(a, b, rtol=2e-6, atol=2e-9)  # noqa: E731
    assert close(_angles(make(base=500.0, dim=6)), _plain(6, 500.0))
    assert close(_angles(make({"kind": "linear", "factor": 4})), _plain(64) / 4)
    assert close(_angles(make({"kind": "base", "factor": 2.0})), _plain(64, 10000.0 * 2 ** (64 / 62)))
    got = _angles(make({"kind": "wavelength", "factor": 8, "original": 8192}))
    for f, g in zip(_plain(64), got):
        turns = 8192 * f / (2 * math.pi)
        want = f if turns > 4 else f / 8 if turns < 1 else f / 8 + (f - f / 8) * (turns - 1) / 3
        assert close(g, want)
    m = 0.1 * math.log(16) + 1
    got = _angles(make({"kind": "ramp", "factor": 16, "original": 4096}), m)
    index = lambda turns: 64 * math.log(4096 / (2 * math.pi * turns)) / (2 * math.log(10000))  # noqa: E731
    low, high = math.floor(index(32)), math.ceil(index(1))
    for i, (f, g) in enumerate(zip(_plain(64), got)):
        r = min(max((i - low) / (high - low), 0), 1)
        assert close(g, f * (1 - r) + f / 16 * r)
    d = np.linspace(1, 9, 32)
    assert close(_angles(make({"kind": "divisors", "divisors": d.tolist(), "magnitude": 1.5}), 1.5), _plain(64) / d)


@pytest.mark.parametrize("args, match", [
    ((0, 64), "0 positions"), ((4, 7), "7 channels"), ((4, 64, 1e4, {"kind": "bent"}), "unknown scaling"),
    ((4, 64, 1e4, {"kind": "linear"}), "needs 'factor'"), ((4, 64, 1e4, {"kind": "linear", "factor": 2, "low": 1}), "low"),
])
def test_tables_refuse(args, match):
    with pytest.raises(ValueError, match=match):
        kv_ops.rotary_table(*args, device="cpu")


# -------------------------------------------------------------------- oracle --


def test_the_oracle_s_codes_are_nearest():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * np.exp2(rng.integers(-100, 100, (200, 1)))
    code, e = R.encode(x)
    unit = np.exp2(e.astype(float) - 127).repeat(32, -1)
    top = np.abs(x.reshape(200, 2, 32)).max(-1)
    assert (top < 7 * np.exp2(e.astype(float) - 127)).all() and (top >= 3.5 * np.exp2(e.astype(float) - 127)).all()
    grid = np.concatenate([R.GRID, -R.GRID])
    best = np.abs(x[..., None] / unit[..., None] - grid).min(-1)
    assert np.array_equal(np.abs(x - R.decode(code, e)) / unit, best)


def test_the_bound_sees_planted_mistakes():
    """In the oracle: a token left out, a neighbouring position's key, a scale
    byte off by one, a weight not divided by the sum."""
    rng = np.random.default_rng(1)
    k, v = R.cached(rng.standard_normal((40, 1, 64))), R.cached(rng.standard_normal((40, 1, 64)))
    q = rng.standard_normal((1, 2, 64))
    out, _, spread, reach = R.attention(q, k, v, 39, 0.125)
    bound = R.bound(out, spread, reach, 40, 64, True)
    more = v.copy()
    more[20, 0, :32] *= 2
    for kk, vv in ((k[:-1], v[:-1]), (np.roll(k, 1, 0), v), (k, more)):
        wrong = R.attention(q, kk, vv, len(kk) - 1, 0.125)[0]
        assert (np.abs(wrong - out) > bound).any()
    assert (np.abs(out * 1.02 - out) > bound).any()
