"""MI355X: the attention over selected pages (kv_ops.summarize, select,
attention(blocks=)): summaries and selections exactly against
tests/blocks_reference.py, the attention within kv_reference's derived bound."""

import numpy as np
import pytest
import torch

from drinkme_amd import kv_ops
from tests import blocks_reference as B
from tests import kv_reference as R
from tests.test_gpu_kv import Batch, f64, heads, i32

pytestmark = pytest.mark.gpu


def noisy_summaries(rng, cache):
    s = kv_ops.new_summaries(cache)
    s["bounds"].copy_(torch.from_numpy(rng.integers(-128, 128, s["bounds"].shape, dtype=np.int8)))
    s["scales"].copy_(torch.from_numpy(rng.integers(0, 256, s["scales"].shape, dtype=np.uint8)))
    return s


def want_summaries(batch, held, before, new=None):
    """The summaries after a call for the batch's new tokens (or new[b] of them)."""
    bounds, scales = before["bounds"].cpu().numpy().copy(), before["scales"].cpu().numpy().copy()
    for b, ((n, length), (k, _)) in enumerate(zip(batch.sizes, held)):
        n = n if new is None else new[b]
        if n:
            for col in range((length - n) // batch.page, (length - 1) // batch.page + 1):
                page = batch.table[b][col]
                for h in range(batch.H):
                    bounds[page, h], scales[page, h] = B.summary(k[col * batch.page:(col + 1) * batch.page, h])
    return bounds, scales


def summarized(rng, batch, held):
    """Summaries of all that is cached."""
    s = noisy_summaries(rng, batch.cache)
    lengths = [length for _, length in batch.sizes]
    cu = i32(np.concatenate([[0], np.cumsum(lengths)]))
    kv_ops.summarize(batch.cache, s, batch.block_table, batch.lengths, sum(lengths), cu=cu)
    return s


def want_blocks(batch, q, s, count, first, last, causal=True):
    bounds, scales = s["bounds"].cpu().numpy(), s["scales"].cpu().numpy()
    q, out = f64(q), []
    group = q.shape[1] // batch.H
    t = 0
    for b, (n, length) in enumerate(batch.sizes):
        for m in range(n):
            p = length - n + m if causal else length - 1
            pages = min(p // batch.page + 1, batch.cols)
            out.append([B.select(q[t, h * group:(h + 1) * group], bounds[:, h], scales[:, h], batch.block_table[b].tolist(), pages,
                                 count, first, last) for h in range(batch.H)])
            t += 1
    return np.array(out).reshape(t, batch.H, count)


def check_listed(batch, held, q, blocks, got, dtype, lse=None, causal=True, scale=None):
    scale = batch.D ** -0.5 if scale is None else scale
    t, out, qq, blocks = 0, f64(got), f64(q), blocks.cpu().numpy()
    for (n, length), (k, v) in zip(batch.sizes, held):
        want, l, spread, reach = B.listed_attention(qq[t:t + n], k, v, length - n, scale, blocks[t:t + n], batch.page, causal)
        bound = R.bound(want, spread, reach, length, batch.D, dtype == "bf16")
        assert (np.isnan(out[t:t + n]) == np.isnan(want)).all()
        assert np.nanmax(np.abs(out[t:t + n] - want) / bound, initial=0.0) <= 1.0
        if lse is not None:
            le = f64(lse)[t:t + n]
            assert (np.isneginf(le) == np.isneginf(l)).all() and (np.isnan(le) == np.isnan(l)).all()
            ok = np.isfinite(l)
            assert (np.abs(le - l)[ok] <= R.lse_bound(l, reach, length, batch.D)[ok]).all()
        t += n


# ---------------------------------------------------------------- summaries --


@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("sizes", [[(1, 1)], [(1, 300), (1, 65), (1, 64), (1, 257)], [(5, 66), (5, 5), (5, 200)],
                                   [(70, 70), (0, 33), (1, 129), (300, 420), (0, 0)]])
def test_summaries(sizes, page, D):
    rng = np.random.default_rng(page + D + len(sizes))
    b = Batch(rng, sizes, 3, D, page)
    total = sum(length for _, length in sizes)
    k, v = heads(rng, (total, 3, D), "bf16", 3.0), heads(rng, (total, 3, D), "bf16")
    k *= torch.exp2(torch.randint(-20, 20, (total, 3, 1), device="cuda"))  # (blocks of very different sizes)
    k[::5] = k[::5].abs()  # (tokens all of one sign)
    if total > 40:
        k[7, 1, 3], k[30, 0, 40], k[31, :, :32] = float("nan"), float("inf"), 0.0
        k[33:33 + 2 * page, 2, :32] = float("nan")  # (a page whose channels are no numbers)
    held = b.fill(rng, k, v)
    s = noisy_summaries(rng, b.cache)
    want = want_summaries(b, held, s)
    kv_ops.summarize(b.cache, s, b.block_table, b.lengths, b.total, **b.args)
    assert (s["bounds"].cpu().numpy() == want[0]).all() and (s["scales"].cpu().numpy() == want[1]).all()


def test_summaries_of_extreme_keys():
    """The smallest and the largest keys that the cache holds, alone and together."""
    rng = np.random.default_rng(1)
    b = Batch(rng, [(48, 48)], 1, 64, 8)
    k = torch.zeros((48, 1, 64), device="cuda")
    k[8:16, 0, :32], k[8:16, 0, 32:] = 2.0 ** -126, -2.0 ** -126
    k[16:24, 0, :32], k[16:24, 0, 32:] = 1.5 * 2.0 ** 127, -2.0 ** -126
    k[24:32, 0, :32], k[24:32, 0, 32:] = -1.5 * 2.0 ** 127, 2.0 ** -126
    k[32:40] = torch.exp2(torch.arange(8, device="cuda") - 4.0)[:, None, None]
    k[40:48, 0] = torch.linspace(-127, 127, 64, device="cuda")
    held = b.fill(rng, k, torch.zeros_like(k))
    s = noisy_summaries(rng, b.cache)
    want = want_summaries(b, held, s)
    kv_ops.summarize(b.cache, s, b.block_table, b.lengths, 48)
    assert (s["bounds"].cpu().numpy() == want[0]).all() and (s["scales"].cpu().numpy() == want[1]).all()


def test_summaries_of_tokens_without_a_page_or_a_sequence():
    rng = np.random.default_rng(2)
    b = Batch(rng, [(9, 40), (5, 30)], 2, 64, 8)
    held = b.fill(rng)
    b.block_table[0, 4], b.block_table[1, 3] = -1, 10 ** 6
    s = noisy_summaries(rng, b.cache)
    keep = {n: t.clone() for n, t in s.items()}
    b.table[0][4] = b.table[1][3] = 0
    want = want_summaries(b, held, s)
    for name, w in zip(("bounds", "scales"), want):  # (page 0 stands for the lost ones: as it was)
        w[0] = keep[name].cpu().numpy()[0]
    used = {b.table[0][3], b.table[1][3]}
    cu = i32([2, 11, 16])  # rows before and behind: of no sequence
    kv_ops.summarize(b.cache, s, b.block_table, b.lengths, 20, cu=cu)
    if 0 in b.table[0][:4] or 0 in b.table[1][:3]:
        used.add(0)
    assert used and (s["bounds"].cpu().numpy() == want[0])[1:].all() and (s["scales"].cpu().numpy() == want[1])[1:].all()
    again = {n: t.clone() for n, t in s.items()}
    kv_ops.summarize(b.cache, s, b.block_table, i32([0, -7]), 4)  # positions below 0
    assert all(torch.equal(again[n], s[n]) for n in s)


@pytest.mark.parametrize("D, page, batch, cols, pages, most", [
    (64, 8, 2, 2, 2, 16), (128, 64, 40, 2, 6, 3), (256, 16, 300, 3, 20, 1), (96, 16, 300, 1, 4, 1), (192, 8, 33, 40, 60, 320), (128, 8, 700, 4, 1500, 5)])
def test_summaries_of_shared_pages(D, page, batch, cols, pages, most):
    """Sequences share pages, one has a page twice, and each holds another number of tokens there: the summary
    is of the most. Many workgroups meet at a page; every byte is one's."""
    rng = np.random.default_rng(D + batch)
    b = Batch(rng, [(page * pages, page * pages)], 2, D, page, spare=0)
    (k, _), = b.fill(rng)
    column = {int(p): c for c, p in enumerate(b.table[0])}  # (where a page's keys are held)
    shared = 0
    for turn in range(4):
        table = rng.choice(b.table[0], (batch, cols))
        lengths = rng.integers(0, cols * page + 1, batch)
        if turn == 3:
            lengths[:] = rng.integers(1, page, batch)  # (all within a page)
        new = np.minimum(rng.integers(0, most + 1, batch), lengths) if turn % 2 else np.full(batch, min(most, cols * page))
        lengths = np.maximum(lengths, new)
        before, pad = int(rng.integers(0, 4)) * (turn % 2), int(rng.integers(0, 5)) * (turn % 2)
        cu = i32(before + np.concatenate([[0], np.cumsum(new)])) if turn % 2 else None
        s = noisy_summaries(rng, b.cache)
        bounds, scales = s["bounds"].cpu().numpy().copy(), s["scales"].cpu().numpy().copy()
        held = {}
        for n, length, row in zip(new, lengths, table):
            for col in range((length - n) // page, -(-length // page)) if n else ():
                held[int(row[col])] = max(held.get(int(row[col]), 0), int(min(page, length - col * page)))
        shared += sum(-(-length // page) - (length - n) // page for n, length in zip(new, lengths) if n) - len(held)
        for p, n in held.items():
            at = column[p] * page
            for h in range(2):
                bounds[p, h], scales[p, h] = B.summary(k[at:at + n, h])
        for _ in range(3):
            kv_ops.summarize(b.cache, s, i32(table), i32(lengths), before + int(new.sum()) + pad, cu=cu)
            assert (s["bounds"].cpu().numpy() == bounds).all() and (s["scales"].cpu().numpy() == scales).all()
    assert shared > 0


# ---------------------------------------------------------------- selection --


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("sizes, page, H, Hq, count, first, last", [
    ([(1, 1)], 8, 2, 2, 1, 0, 0), ([(1, 900), (1, 8), (1, 1)], 8, 2, 8, 9, 1, 2), ([(1, 2000)], 8, 1, 5, 64, 2, 1),
    ([(5, 700), (5, 5), (5, 331)], 16, 2, 6, 7, 0, 1), ([(40, 333), (0, 50), (1, 1000)], 8, 2, 2, 12, 3, 4),
    ([(3, 4100)], 8, 1, 16, 100, 1, 1), ([(2, 1500)], 16, 1, 37, 5, 1, 0)])
def test_selection(sizes, page, H, Hq, count, first, last, D, dtype):
    rng = np.random.default_rng(D + len(sizes) + count)
    b = Batch(rng, sizes, H, D, page)
    held = b.fill(rng, scale=2.0)
    s = summarized(rng, b, held)
    q = heads(rng, (b.total, Hq, D), dtype)
    got = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, count, first=first, last=last, **b.args)
    assert got.dtype == torch.int32 and got.is_contiguous()
    assert (got.cpu().numpy() == want_blocks(b, q, s, count, first, last)).all()
    got = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, count, first=first, last=last, causal=False, **b.args)
    assert (got.cpu().numpy() == want_blocks(b, q, s, count, first, last, False)).all()


def summaries_at_random(rng, b, few=False):
    """Bounds and scales drawn, not summarized: `few` values, so that most scores tie."""
    s = kv_ops.new_summaries(b.cache)
    lo, hi = (-1, 2) if few else (-127, 128)
    s["bounds"].copy_(torch.from_numpy(rng.integers(lo, hi, s["bounds"].shape, dtype=np.int8)))
    s["scales"].copy_(torch.from_numpy(rng.integers(126, 128 if few else 131, s["scales"].shape, dtype=np.uint8)))
    return s


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("tokens, batch, length, heads_, count", [
    (1, 1, 8 * 16000, 2, 700), (1, 1, 8 * 16384, 1, 16383), (1, 2, 8 * 4099, 1, 33), (1, 3, 8 * 513, 2, 511), (2, 1, 8 * 512, 2, 77), (1, 1, 8 * 4096, 1, 1),
    (600, 1, 8 * 700, 1, 20), (1100, 1, 8 * 400, 2, 16), (512, 1, 8 * 4096, 1, 30)])
def test_selection_over_every_team(tokens, batch, length, heads_, count, few):
    """Each number of waves to a token, at its most columns; ties in plenty, which go to
    the lower column."""
    rng = np.random.default_rng(length + count + few)
    b = Batch(rng, [(tokens, length)] * batch, heads_, 64, 8, spare=0)
    s = summaries_at_random(rng, b, few)
    q = heads(rng, (b.total, heads_, 64), "f32")
    if few:
        q = q.sign()
    got = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, count, first=0, last=1).cpu().numpy()
    bounds, scales = s["bounds"].cpu().numpy().astype(np.int64), s["scales"].cpu().numpy().astype(np.int64)
    qq = f64(q)
    for t in sorted({0, 1, b.total // 2, b.total - 1} & set(range(b.total))):
        seq = t // tokens
        n = (length - tokens + t % tokens) // 8 + 1
        pages = b.table[seq][:n]
        for h in range(heads_):
            w = B.whole_queries(qq[t, h:h + 1])[0]
            score = (np.where(w > 0, w, 0) * bounds[pages, h, 0]).sum(-1) + (np.where(w < 0, w, 0) * bounds[pages, h, 1]).sum(-1)
            key = np.ldexp(score.astype(np.float64), scales[pages, h] - 127)
            key[n - 1] = np.inf
            best = np.sort(np.argsort(-key, kind="stable")[:count])
            assert (got[t, h, :len(best)] == best).all() and (got[t, h, len(best):] == -1).all()


@pytest.mark.parametrize("few", [False, True])
@pytest.mark.parametrize("tokens, batch, columns, count, first, last", [
    (1, 70, 1100, 40, 1, 2), (1, 70, 1024, 40, 0, 0), (300, 1, 5000, 33, 0, 1), (1, 1, 2000, 3, 1, 2), (1, 70, 1100, 3, 1, 2), (40, 1, 300, 3, 1, 2),
    (1, 3, 100, 3, 1, 2), (1, 3, 400, 4, 4, 0), (1, 3, 385, 384, 0, 384), (20, 2, 4096, 4095, 2, 3), (1, 65, 2000, 1999, 0, 1), (1, 65, 1026, 1, 0, 0)])
def test_selection_on_every_path(tokens, batch, columns, count, first, last, few):
    """Many rows and few, over more columns than a wave takes and fewer, prompts past the columns that they share; forced
    columns alone, all columns but one. (The sequences share their pages, which the scores do not mind.)"""
    rng = np.random.default_rng(columns + count + few)
    b = Batch(rng, [(tokens, 8 * columns)], 2, 64, 8, spare=0)
    s = summaries_at_random(rng, b, few)
    table, lengths = b.block_table.expand(batch, columns).contiguous(), b.lengths.expand(batch).contiguous()
    q = heads(rng, (tokens * batch, 4, 64), "f32")
    if few:
        q = q.sign()
    got = kv_ops.select(q, b.cache, s, table, lengths, count, first=first, last=last).cpu().numpy()
    bounds, scales = s["bounds"].cpu().numpy().astype(np.int64), s["scales"].cpu().numpy().astype(np.int64)
    qq = f64(q)
    for t in sorted({0, 1, tokens * batch // 2, tokens * batch - 1} & set(range(tokens * batch))):
        n = (8 * columns - tokens + t % tokens) // 8 + 1
        pages = b.table[0][:n]
        for h in range(2):
            w = B.whole_queries(qq[t, 2 * h:2 * h + 2])
            score = (np.where(w > 0, w, 0) @ bounds[pages, h, 0].T + np.where(w < 0, w, 0) @ bounds[pages, h, 1].T).max(0)
            key = np.ldexp(score.astype(np.float64), scales[pages, h] - 127)
            key[:first], key[n - last:] = np.inf, np.inf
            best = np.sort(np.argsort(-key, kind="stable")[:count])
            assert (got[t, h, :len(best)] == best).all() and (got[t, h, len(best):] == -1).all()


def test_selection_of_queries_that_are_none():
    """NaN and infinities in a query count as 0; a query of zeros takes the lowest columns; the smallest and the largest
    queries; columns without a page come last, forced or not."""
    rng = np.random.default_rng(5)
    b = Batch(rng, [(8, 400)], 1, 64, 8)
    s = summarized(rng, b, b.fill(rng))
    q = heads(rng, (8, 2, 64), "f32")
    q[0, 0, 3], q[0, 1, 9], q[1] = float("nan"), float("inf"), 0.0
    q[2], q[3], q[4] = q[2] * 2.0 ** -126, q[3] * 2.0 ** -140, q[4] * 2.0 ** 125
    q[5] = torch.linspace(-127.5, 127.5, 128, device="cuda").view(2, 64)
    q[6] = 2.0 ** 127
    b.block_table[0, 5:30] = -1
    b.block_table[0, 49] = 12345
    for first, last, count in ((0, 0, 9), (6, 2, 20), (1, 1, 30), (0, 0, 49)):
        got = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, count, first=first, last=last)
        assert (got.cpu().numpy() == want_blocks(b, q, s, count, first, last)).all()


def test_scores_past_fp32_are_ties():
    rng = np.random.default_rng(6)
    b = Batch(rng, [(1, 200)], 1, 64, 8)
    s = summaries_at_random(rng, b)
    s["scales"].fill_(248)
    q = heads(rng, (1, 1, 64), "f32")
    got = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, 6)
    assert (got.cpu().numpy() == want_blocks(b, q, s, 6, 1, 1)).all()


def test_selection_of_tokens_of_no_sequence():
    rng = np.random.default_rng(7)
    b = Batch(rng, [(4, 100), (3, 50)], 2, 64, 8)
    s = summarized(rng, b, b.fill(rng))
    q = heads(rng, (12, 2, 64), "bf16")
    got = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, 5, cu=i32([2, 6, 9])).cpu()
    assert (got[:2] == -1).all() and (got[9:] == -1).all()
    assert (got[2:9].numpy() == want_blocks(b, q[2:9], s, 5, 1, 1)).all()
    got = kv_ops.select(q[:4], b.cache, s, b.block_table, i32([1, 2]), 5).cpu()  # first positions below 0
    assert (got[0] == -1).all() and got[1, :, 0].eq(0).all() and got[2, :, 0].eq(0).all()


# ---------------------------------------------------------------- attention --


def random_lists(rng, batch, count, near=False):
    """Lists of columns in any order, some twice, some of none; `near`: neighbours' alike."""
    out = []
    for n, length in batch.sizes:
        cols = max(1, -(-length // batch.page))
        base = rng.integers(-1, cols, (1, batch.H, count)) if near else None
        for m in range(n):
            x = rng.integers(-2, cols + 1, (batch.H, count))
            if near:
                x = np.where(rng.random(x.shape) < 0.8, base[0], x)
            out.append(np.minimum(x, cols - 1))
    return i32(np.array(out).reshape(-1, batch.H, count))


SHAPES = [([(1, 1)], 1), ([(1, 300), (1, 65), (1, 8)], 3), ([(1, 2100)], 40), ([(5, 600), (5, 5), (5, 77)], 6), ([(8, 1030)] * 2, 30),
          ([(33, 333), (0, 50), (1, 200), (70, 70)], 4)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
@pytest.mark.parametrize("page", [8, 16, 32, 128])
@pytest.mark.parametrize("sizes, count", SHAPES)
def test_attention_over_lists(sizes, count, page, D, dtype):
    rng = np.random.default_rng(page + D + count)
    H, Hq = (2, 6) if len(sizes) % 2 else (1, 4)
    b = Batch(rng, sizes, H, D, page)
    held = b.fill(rng)
    q = heads(rng, (b.total, Hq, D), dtype)
    for near, causal in ((False, True), (True, True), (False, False)):
        blocks = random_lists(rng, b, count, near)
        out, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, return_lse=True, causal=causal, **b.args)
        check_listed(b, held, q, blocks, out, dtype, lse, causal)
        again = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, causal=causal, max_length=max(n for _, n in sizes), **b.args)
        check_listed(b, held, q, blocks, again, dtype, None, causal)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("sizes", [[(1, 700), (1, 130)], [(6, 500)], [(90, 333), (7, 40)]])
@pytest.mark.parametrize("group", [1, 2, 3, 8, 16, 40])
def test_every_column_listed_is_the_whole_attention(group, sizes, dtype):
    """Against the definition and, to two bounds, against the attention over everything."""
    rng = np.random.default_rng(group + len(sizes))
    b = Batch(rng, sizes, 2, 64, 16)
    held = b.fill(rng)
    q = heads(rng, (b.total, 2 * group, 64), dtype)
    blocks = torch.arange(b.cols, device="cuda", dtype=torch.int32).flip(0).expand(b.total, 2, b.cols)
    out, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, return_lse=True, scale=0.3, **b.args)
    check_listed(b, held, q, blocks, out, dtype, lse, scale=0.3)


def test_lists_that_show_nothing():
    """Rows of no columns, of later ones, of a sequence's empty part: zeros and -inf."""
    rng = np.random.default_rng(9)
    b = Batch(rng, [(6, 100), (6, 6)], 2, 128, 8)
    held = b.fill(rng)
    q = heads(rng, (12, 4, 128), "bf16")
    blocks = torch.full((12, 2, 5), -1, dtype=torch.int32, device="cuda")
    blocks[2:4], blocks[5, 0, 3] = 13, 2 ** 31 - 1  # (past the token's column, and far past)
    blocks[4, 1] = torch.tensor([-2 ** 31, 3, 3, -1, 3], device="cuda")
    out, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, return_lse=True)
    check_listed(b, held, q, blocks, out, "bf16", lse)
    assert not out[0].any() and lse[0].isneginf().all() and lse[4, 2:].isfinite().all()
    assert not kv_ops.attention(q[:2], b.cache, b.block_table, i32([0, 0]), blocks=blocks[:2]).any()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [1, 4, 40])
@pytest.mark.parametrize("page", [8, 64])
def test_noise_behind_lists_stays_there(page, tokens, dtype):
    """Unlisted pages, positions after a token's and tokens behind the sequence's end hold NaN and
    infinite blocks; a listed one gives NaN to who lists and sees it alone."""
    rng = np.random.default_rng(page + tokens)
    b = Batch(rng, [(tokens, 500), (tokens, 67)], 2, 128, page)
    k, v = (heads(rng, (567, 2, 128), "bf16") for _ in range(2))
    bad = rng.permutation(500)[:30]
    k[bad[:15], 0, 5], v[bad[15:], 1, 77] = float("nan"), float("inf")
    held = b.fill(rng, k, v)
    q = heads(rng, (b.total, 4, 128), dtype)
    blocks = random_lists(rng, b, 6)
    out, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, return_lse=True)
    want = []
    t = 0
    for (n, length), (kk, vv) in zip(b.sizes, held):  # NaN values reach their own channels alone: the plain result, channel by channel
        got = B.listed_attention(f64(q)[t:t + n], kk, np.where(np.isnan(vv), 0, vv), length - n, 128 ** -0.5, blocks[t:t + n].cpu().numpy(), page)
        hit = B.listed_attention(np.zeros_like(f64(q)[t:t + n]), np.zeros_like(kk), np.isnan(vv) * 1.0, length - n, 1.0, blocks[t:t + n].cpu().numpy(), page)
        o = np.where((hit[0] > 0) & ~np.isnan(got[0]), np.nan, got[0])
        bound = R.bound(got[0], got[2], got[3], length, 128, dtype == "bf16")
        mine = f64(out)[t:t + n]
        assert (np.isnan(mine) == np.isnan(o)).all()
        assert np.nanmax(np.abs(mine - o) / bound, initial=0.0) <= 1
        want.append(np.isnan(o).any())
        t += n
    assert any(want) or tokens == 1


def test_listed_columns_without_a_page():
    """Seen and listed: NaN. Not listed, or not seen: nothing."""
    rng = np.random.default_rng(10)
    b = Batch(rng, [(3, 60)], 1, 64, 8, spare=0)
    held = b.fill(rng)
    q = heads(rng, (3, 4, 64), "bf16")
    b.block_table[0, 2] = -1
    blocks = i32([[[0, 1, 3, 7]], [[0, 2, 3, 7]], [[5, 5, 0, 7]]])
    out = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks)
    assert out[1].isnan().all() and not out[[0, 2]].isnan().any()
    more = i32([72])  # positions 69..71: the eighth column is not in the table
    out = kv_ops.attention(q, b.cache, b.block_table, more, blocks=i32([[[0, 1]], [[0, 8]], [[9, 0]]]))
    assert out[1].isnan().all() and not out[[0, 2]].isnan().any()
    out, lse = kv_ops.attention(q, b.cache, b.block_table, i32([2 ** 31 - 1]), blocks=i32([[[0, 1]], [[0, 2 ** 28 - 1]], [[6, 2 ** 28]]]), return_lse=True)  # (the seventh is full: behind the sixtieth token lies noise)
    assert out[1].isnan().all() and lse[1].isnan().all() and not out[[0, 2]].isnan().any()


def test_tokens_past_max_tokens_and_of_no_sequence():
    rng = np.random.default_rng(11)
    b = Batch(rng, [(4, 100), (6, 50)], 2, 64, 16)
    b.fill(rng)
    q = heads(rng, (14, 4, 64), "bf16")
    blocks = i32(rng.integers(0, 4, (14, 2, 3)))
    for length in (100, 5000):
        table = torch.cat([b.block_table, b.block_table.new_full((2, length // 16), -1)], 1)
        out, lse = kv_ops.attention(q, b.cache, table, b.lengths, cu=i32([2, 6, 12]), max_tokens=5, blocks=blocks, return_lse=True)
        gone = [0, 1, 11, 12, 13]
        assert out[gone].isnan().all() and lse[gone].isnan().all()
        assert out[2:11].isfinite().all()


def test_lists_of_every_size():
    """Counts past a workgroup's lanes, all columns that a table may have."""
    rng = np.random.default_rng(12)
    b = Batch(rng, [(2, 8 * 900)], 1, 64, 8, spare=16384 - 900)
    held = b.fill(rng)
    q = heads(rng, (2, 2, 64), "bf16")
    for count in (257, 900, 16384):
        blocks = i32(rng.integers(-1, 900, (2, 1, count)))
        out, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, return_lse=True)
        check_listed(b, held, q, blocks, out, "bf16", lse)
    q = heads(rng, (2, 2, 64), "f32")
    check_listed(b, held, q, blocks, kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks), "f32")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_prompts_of_more_rows_than_a_launch_has(dtype):
    """Over 65535 tiles of 16 rows: tokens on both sides of the border against the definition, all of them against
    calls of a part each, and offsets of two sequences with tokens of none behind them."""
    rng = np.random.default_rng(19)
    T, group, D = 16389, 64, 64  # (the border is within token 16383)
    b = Batch(rng, [(T, T + 100)], 1, D, 64)
    (k, v), = b.fill(rng)
    q = heads(rng, (T, group, D), dtype)
    blocks = i32(rng.integers(-1, b.cols, (T, 1, 3)))
    out, lse = kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks, return_lse=True)
    for t in (0, 1, 8191, 16382, 16383, 16384, T - 1):
        want, l, spread, reach = B.listed_attention(f64(q[t:t + 1]), k, v, 100 + t, D ** -0.5, blocks[t:t + 1].cpu().numpy(), 64)
        assert (np.abs(f64(out[t:t + 1]) - want) <= R.bound(want, spread, reach, T + 100, D, dtype == "bf16")).all()
        seen = np.isfinite(l)
        assert (np.isneginf(f64(lse[t:t + 1])) == ~seen).all()
        assert (np.abs(f64(lse[t:t + 1])[seen] - l[seen]) <= R.lse_bound(l, reach, T + 100, D)[seen]).all()
    for t0, t1 in ((0, 6000), (6000, T)):
        part, sums = kv_ops.attention(q[t0:t1], b.cache, b.block_table, i32([100 + t1]), blocks=blocks[t0:t1], return_lse=True)
        assert torch.equal(part, out[t0:t1]) and torch.equal(sums, lse[t0:t1])
    again = kv_ops.attention(q, b.cache, b.block_table.expand(2, -1), i32([107, T + 97]), cu=i32([0, 7, T - 3]), blocks=blocks)
    assert torch.equal(again[:T - 3], out[:T - 3]) and bool(again[T - 3:].isnan().all())


def test_large_heads_and_tables_at_once():
    rng = np.random.default_rng(13)
    b = Batch(rng, [(9, 900)], 1, 256, 8, spare=16384 - 113)
    held = b.fill(rng)
    for dtype in ("bf16", "f32"):
        q = heads(rng, (9, 4, 256), dtype)
        blocks = i32(rng.integers(-1, 113, (9, 1, 20)))
        check_listed(b, held, q, blocks, kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks), dtype)


def test_views_and_the_same_bits_every_time():
    rng = np.random.default_rng(14)
    b = Batch(rng, [(1, 3000), (1, 2000)], 2, 128, 16)
    held = b.fill(rng)
    s = summarized(rng, b, held)
    fused = heads(rng, (2, 12, 128), "bf16")
    q = fused[:, 1:9]
    odd = torch.empty(q.numel() + 1, dtype=torch.bfloat16, device="cuda")[1:].view(q.shape).copy_(q)
    want = kv_ops.select(q.contiguous(), b.cache, s, b.block_table, b.lengths, 20)
    out = kv_ops.attention(q.contiguous(), b.cache, b.block_table, b.lengths, blocks=want)
    for x in (q, odd, q.transpose(0, 1).contiguous().transpose(0, 1)):
        for _ in range(3):
            blocks = kv_ops.select(x, b.cache, s, b.block_table, b.lengths, 20)
            assert torch.equal(blocks, want)
            assert torch.equal(kv_ops.attention(x, b.cache, b.block_table, b.lengths, blocks=blocks), out)
            assert torch.equal(kv_ops.attention(x, b.cache, b.block_table, b.lengths, blocks=blocks.transpose(0, 2).contiguous().transpose(0, 2).flip(-1)), out)


def test_offsets_past_32_bits():
    """A cache of more than 2^32 bytes of codes: its last pages, their summaries, and lists of them."""
    rng = np.random.default_rng(15)
    H, D, page = 8, 256, 1024
    pages = 2200  # 2.3e9 bytes of key codes, 4.6e9 of summaries' cache indexes
    cache = {"k_codes": torch.empty((pages, H, page, D // 8), dtype=torch.int32, device="cuda"),
             "k_scales": torch.empty((pages, H, page, D // 32), dtype=torch.uint8, device="cuda"),
             "v_codes": torch.empty((pages, H, page // 8, D // 8, 8), dtype=torch.int32, device="cuda"),
             "v_scales": torch.empty((pages, H, page // 8, D // 32, 8), dtype=torch.uint8, device="cuda")}
    length = 1500
    k, v = (heads(rng, (length, H, D), "bf16") for _ in range(2))
    table, lengths = i32([[pages - 1, pages - 2]]), i32([length])
    small = kv_ops.new_cache(2, page, H, D)
    s, t = kv_ops.new_summaries(cache), kv_ops.new_summaries(small)
    q = heads(rng, (1, 16, D), "bf16")
    outs = []
    for c, x, tab in ((cache, s, table), (small, t, i32([[0, 1]]))):
        kv_ops.append(c, k, v, tab, lengths)
        kv_ops.summarize(c, x, tab, lengths, length)
        blocks = kv_ops.select(q, c, x, tab, lengths, 1, first=0, last=0)
        outs.append((x["bounds"][tab[0].long()], x["scales"][tab[0].long()], blocks, kv_ops.attention(q, c, tab, lengths, blocks=blocks)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_on_another_stream_and_in_a_graph():
    """A step's summaries, selection and attention in a graph, replayed with new queries, keys and lengths."""
    rng = np.random.default_rng(16)
    b = Batch(rng, [(1, 1500), (1, 900)], 2, 64, 8, spare=30)
    b.fill(rng)
    spare = [p for p in range(b.cache["k_codes"].shape[0]) if p not in b.table]
    b.block_table[0, 188], b.block_table[1, 113] = spare[0], spare[1]
    s = summarized(rng, b, None)
    q, k, v = heads(rng, (2, 4, 64), "bf16"), heads(rng, (2, 2, 64), "bf16"), heads(rng, (2, 2, 64), "bf16")

    def step():
        kv_ops.append(b.cache, k, v, b.block_table, b.lengths)
        kv_ops.summarize(b.cache, s, b.block_table, b.lengths, 2)
        blocks = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, 16)
        return s["bounds"].clone(), blocks, kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for n in range(4):
        b.lengths.add_(1)
        for x in (q, k, v):
            x.copy_(heads(rng, x.shape, "bf16"))
        graph.replay()
        torch.cuda.synchronize()
        first = [x.clone() for x in got]
        assert all(torch.equal(a, c) for a, c in zip(first, step()))


def test_no_tokens():
    rng = np.random.default_rng(17)
    b = Batch(rng, [(1, 20)], 2, 64, 8)
    s = noisy_summaries(rng, b.cache)
    q = torch.empty((0, 4, 64), device="cuda")
    kv_ops.summarize(b.cache, s, b.block_table, b.lengths, 0)
    blocks = kv_ops.select(q, b.cache, s, b.block_table, b.lengths, 3)
    assert blocks.shape == (0, 2, 3)
    assert kv_ops.attention(q, b.cache, b.block_table, b.lengths, blocks=blocks).shape == (0, 4, 64)


def test_as_many_tokens_as_a_launch_takes():
    """A token of many selects what a call of the last ones alone does; those before the sequence's first position
    list nothing; one more is refused."""
    rng = np.random.default_rng(17)
    columns, most = 4100, 2 ** 23 - 1
    b = Batch(rng, [(1, 8 * columns)], 1, 64, 8, spare=0)
    s = summaries_at_random(rng, b)
    q = heads(rng, (1, 1, 64), "bf16")
    got = kv_ops.select(q.expand(most, 1, 64), b.cache, s, b.block_table, b.lengths, 4)
    for n in (1, 3000):
        want = kv_ops.select(q.expand(n, 1, 64), b.cache, s, b.block_table, b.lengths, 4)
        assert torch.equal(got[most - n:], want) and bool((want >= 0).all())
    assert bool((got[:most - 8 * columns] == -1).all())
    assert got[most - 8 * columns].tolist() == [[0, -1, -1, -1]]
    with pytest.raises(RuntimeError, match="too many tokens"):
        kv_ops.select(q.expand(most + 1, 1, 64), b.cache, s, b.block_table, b.lengths, 4)


def test_refusals():
    rng = np.random.default_rng(18)
    b = Batch(rng, [(2, 20)], 2, 64, 8)
    s = noisy_summaries(rng, b.cache)
    q, blocks = heads(rng, (2, 4, 64), "bf16"), i32(np.zeros((2, 2, 3)))
    wide = torch.zeros((1, 16385), dtype=torch.int32, device="cuda")
    for kw, match in (({"count": 0}, "0 columns"), ({"count": 16385}, "16385 columns"), ({"count": 2, "first": 1, "last": 2}, "more than"),
                      ({"first": -1}, "first -1"), ({"block_table": wide}, "16385 columns"), ({"q": q[:, :3]}, "query heads"),
                      ({"q": q[..., :32]}, "channels"), ({"summaries": {**s, "scales": s["scales"][:1]}}, "scales"),
                      ({"summaries": {**s, "bounds": s["bounds"].float()}}, "bounds"), ({"q": q.cpu()}, "GPU")):
        a = {"q": q, "cache": b.cache, "summaries": s, "block_table": b.block_table, "lengths": b.lengths, "count": 3, **kw}
        with pytest.raises(ValueError, match=match):
            kv_ops.select(**a)
    for kw, match in (({"blocks": blocks.long()}, "int32"), ({"blocks": blocks[:1]}, r"\[2, 2, n\]"), ({"blocks": blocks[:, :1]}, r"\[2, 2, n\]"),
                      ({"blocks": blocks[..., :0]}, "0 columns"), ({"blocks": blocks.cpu()}, "blocks"), ({"window": 5}, "window"),
                      ({"block_table": wide}, "16385 columns"), ({"blocks": blocks[0]}, r"\[2, 2, n\]")):
        a = {"q": q, "cache": b.cache, "block_table": b.block_table, "lengths": b.lengths, "blocks": blocks, **kw}
        with pytest.raises(ValueError, match=match):
            kv_ops.attention(**a)
    with pytest.raises(ValueError, match="scales"):
        kv_ops.summarize(b.cache, {**s, "scales": s["scales"].int()}, b.block_table, b.lengths, 2)
    with pytest.raises(ValueError, match="not the same number"):
        kv_ops.summarize(b.cache, s, b.block_table.expand(2, -1), b.lengths.expand(2), 3)
    with pytest.raises(RuntimeError, match="no gradient"):
        kv_ops.select(q.clone().requires_grad_(), b.cache, s, b.block_table, b.lengths, 3)
