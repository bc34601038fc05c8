"""MI355X: what must not reach the results of the 4-bit cache's operators
(drinkme_amd.kv_ops): noise behind masks. Against tests/kv_reference.py, within
its derived bounds."""

import numpy as np
import pytest
import torch

from drinkme_amd import kv_ops
from tests import kv_reference as R
from tests.test_gpu_kv import Batch, check_attention, f64, heads, i32

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
