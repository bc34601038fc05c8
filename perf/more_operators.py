"""What a decoder's step does around the paged 4-bit cache and between its
blocks, as a list of measured cases: pages handed out and given back, rotary
positions of several axes, norms fused with their residual, and attention over
the pages that a cheap score selects for each query.

A case is one pass of one of them:

  pages   a step's new tokens get their pages, offsets, positions and slots;
          then the sequences are cut back to what they held (drafts that were
          not accepted, requests that end), which returns the pages
  axes    queries and keys rotated by positions of several axes
  norm    a block's output into the residual stream, and the norm in front of
          the next block; or the norm of each head of a fused product
  sparse  summaries of the pages that new tokens lie in, then of each new token
          the pages that score highest, then the attention over those

The pool of pages is a stack: free[0 .. count - 1]; the next page is the last.
The cache holds, of each token and key/value head, blocks of 32 channels: an
exponent byte e (the block's scale 2^(e - 127)) and 32 four-bit codes (sign,
then 0 .5 1 1.5 2 3 4 6):

  k_codes   int32 [pages, H, P, D/8]      nibble n of a word: channel 8 w + n
  k_scales  uint8 [pages, H, P, D/32]
  v_codes   int32 [pages, H, P/8, D/8, 8] eight tokens' words side by side
  v_scales  uint8 [pages, H, P/8, D/32, 8]

A page's summary, for each head: of every channel the largest and the smallest
cached key, as whole numbers of a power of two E, at most 127 of them (the
least E that allows it, -126 or more), the largest rounded up and the smallest
down; exponent byte E + 127.

  bounds    int8 [pages, H, 2, D]
  scales    uint8 [pages, H]

A query's score of a page bounds its product with every key there: with q as
whole numbers of a power of two (to the nearest, at most 127, one power for the
query heads that share a cache head) the sum over channels of q times the
largest where q > 0 and times the smallest where q < 0, of those heads the
largest sum, times 2^E. Sums are whole numbers below 2^24.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pages(name, batch, tokens, length, page, form="even", pool=1.0, pad=0):
    return {"name": name, "kind": "pages", "batch": batch, "tokens": tokens, "length": length, "page": page,
            "form": form, "pool": pool, "pad": pad}


def _axes(name, t, heads, kv_heads, dim, sections, order, layout="half", x="bf16", spectrum="shared", fused=False):
    return {"name": name, "kind": "axes", "t": t, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "sections": sections, "order": order, "layout": layout, "x": x, "spectrum": spectrum, "fused": fused}


def _norm(name, t, dim, x="bf16", residual="bf16", norm="rms", post=False, gate="none", modulate=False, batch=1,
          offset=0.0, factor=1.0, form="block", heads=1):
    return {"name": name, "kind": "norm", "form": form, "t": t, "heads": heads, "dim": dim, "x": x,
            "residual": residual, "norm": norm, "post": post, "gate": gate, "modulate": modulate, "batch": batch,
            "offset": offset, "factor": factor}


def _sparse(name, batch, tokens, length, heads, kv_heads, dim, page, count, x="bf16", ragged=False, first=1, last=2,
            lse=False):
    return {"name": name, "kind": "sparse", "batch": batch, "tokens": tokens, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "count": count, "x": x, "ragged": ragged, "first": first,
            "last": last, "lse": lse}


def listed():
    return [
        # a verify step of a busy server: one accepted and four draft rows a sequence, none of the drafts accepted
        _pages("pages-step", 32, 5, 8192, 64),
        # a batch of prompts of different lengths in small pages, its rows padded to a round number
        _pages("pages-prompts", 64, 2048, 4096, 16, form="ragged", pad=4096),
        # a decode step's one token, three axes dealt in turn (time, height, width)
        _axes("axes-step", 1, 32, 8, 128, "24,20,20", "interleaved"),
        # a video of 16 frames of 24 x 21 patches, axes in blocks, out of a fused q/k/v product
        _axes("axes-video", 8064, 32, 8, 128, "16,24,24", "blocks", fused=True),
        # an image of odd sides, two axes with a spectrum each, pairs side by side, fp32
        _axes("axes-image-f32", 1147, 16, 16, 96, "24,24", "blocks", layout="interleaved", x="f32", spectrum="own"),
        # a decode step's one token: the residual, and the norm in front of the next block
        _norm("norm-step", 1, 4096),
        # a prompt: norms after and before, an fp32 residual stream, weights kept as 1 + w
        _norm("norm-prompt", 8192, 4096, residual="f32", post=True, offset=1.0),
        # an image model's block: layer norm, gate, scale and shift by the image
        _norm("norm-image", 4 * 1021, 1536, norm="layer", gate="sequence", modulate=True, batch=4),
        # one sequence, one token, a context of ordinary length
        _sparse("sparse-one", 1, 1, 8190, 32, 8, 128, 64, 16),
        # a decode step of a busy server over long contexts
        _sparse("sparse-batch", 32, 1, 16384, 32, 8, 128, 64, 32, ragged=True),
        # verify rows, fp32 activations, small pages
        _sparse("sparse-verify-f32", 8, 5, 8193, 16, 4, 96, 16, 64, x="f32", ragged=True, lse=True),
        # a chunk of a long prompt
        _sparse("sparse-chunk", 1, 1024, 32768, 32, 8, 128, 64, 32),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    u = rng.random()
    x = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if u < 0.2:
        page, batch = rng.choice([8, 16, 32, 64, 128]), _log_between(rng, 1, 256)
        tokens = _log_between(rng, 1, 4096)
        tokens = max(1, min(tokens, 131072 // batch))
        length = _log_between(rng, 1, min(32768, 4096 * page * 16 // batch))
        c = _pages("", batch, tokens, length, page, rng.choice(["even", "ragged", "ragged"]),
                   rng.choice([1.0, 1.0, 0.6]), rng.choice([0, 0, 64]))
    elif u < 0.4:
        dim, axes = rng.choice([64, 72, 96, 128, 128, 256]), rng.choice([1, 2, 3, 3, 4])
        angles = rng.choice([dim // 2, dim // 2, dim // 4])
        cuts = sorted(rng.randrange(angles + 1) for _ in range(axes - 1))
        sections = [b - a for a, b in zip([0] + cuts, cuts + [angles])]
        kv = rng.choice([1, 2, 4, 8, 16])
        heads = kv * rng.choice([1, 2, 4, 5, 8])
        t = max(1, min(_log_between(rng, 1, 8192),
                       8064 * 40 * 128 // ((heads + kv) * dim * (2 if x == "f32" else 1))))
        c = _axes("", t, heads, kv, dim, ",".join(map(str, sections)), rng.choice(["blocks", "interleaved"]),
                  rng.choice(["half", "interleaved"]), x, rng.choice(["shared", "own"]), rng.random() < 0.5)
    elif u < 0.6:
        if rng.random() < 0.3:
            heads, dim = rng.choice([1, 4, 8, 32, 40]), rng.choice([64, 96, 128, 128, 256])
            t = max(1, min(_log_between(rng, 1, 16384), (1 << 25) // (heads * dim)))
            c = _norm("", t, dim, x, x, rng.choice(["rms", "rms", "layer"]), offset=rng.choice([0.0, 1.0]),
                      form="heads", heads=heads)
        else:
            dim = _log_between(rng, 64, 16384)
            dim = dim if rng.random() < 0.2 else max(8, dim // 8 * 8)
            batch = rng.choice([1, 1, 2, 4, 7])
            residual = "f32" if x == "f32" else rng.choice(["bf16", "f32"])
            t = max(1, min(_log_between(rng, 1, 16384), (1 << 25) // dim // (2 if x == "f32" else 1)))
            t = max(batch, t // batch * batch)
            c = _norm("", t, dim, x, residual, rng.choice(["rms", "rms", "layer"]), rng.random() < 0.5,
                      rng.choice(["none", "channel", "token", "sequence"]), rng.random() < 0.4, batch,
                      rng.choice([0.0, 1.0]), rng.choice([1.0, 0.22]))
    else:
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 4, 5, 8])
        dim, page = rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([8, 16, 32, 64, 64, 128])
        few = rng.random() < 0.65
        tokens = rng.choice([1, 1, 1, 2, 5, 8]) if few else _log_between(rng, 9, 1024)
        length = max(tokens, min(_log_between(rng, 16, 131072 if few else 32768), 4096 * page))
        first, last = rng.choice([0, 1, 1, 2]), rng.choice([1, 2, 2, 4])
        count = max(first + last, _log_between(rng, 2, 64))
        batch = _log_between(rng, 1, 48 if few else 6)
        # (values cached, bytes selected, products: no more than the listed ones')
        one = heads * dim * (count * page + length // page) * (3 if x == "f32" else 1)
        most = 1024 * 32 * 128 * (32 * 64 + 512)
        batch = max(1, min(batch, 32 * 16384 * 8 * 128 // 2 // (length * kv * dim), most // (tokens * one),
                           300000000 // (count * page * kv * dim)))
        tokens = max(1, min(tokens, most // one))
        c = _sparse("", batch, tokens, length, heads, kv, dim, page, count, x, rng.random() < 0.6, first, last,
                    rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs --


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _sizes(case):
    """(new tokens, tokens in all) of each sequence: where ragged, contexts and
    prompts shrink to half, the second prompt is empty and the third one token."""
    out = []
    for b in range(case["batch"]):
        n, length = case["tokens"], case["length"]
        if case["ragged"] and b:
            f = 1 - 0.5 * ((b * 0.618034) % 1.0)
            cached = int((length - n) * f)
            if n > 8:
                n = 0 if b == 1 else 1 if b == 2 else max(1, int(n * f))
            length = cached + n
        out.append((n, length))
    return out


def _counts(case):
    """(new tokens, tokens before) of each sequence of a pages case."""
    ragged = case["form"] == "ragged"
    out = []
    for b in range(case["batch"]):
        f = 1 - 0.9 * ((b * 0.618034) % 1.0)
        n = 0 if ragged and b % 7 == 3 else max(1, int(case["tokens"] * f)) if ragged else case["tokens"]
        out.append((n, 0 if ragged and b % 5 == 1 else int(case["length"] * (1 - 0.5 * ((b * 0.381966) % 1.0)))))
    return out


def _total(case):
    total = sum(n for n, _ in _counts(case))
    return -(-total // case["pad"]) * case["pad"] if case["pad"] else total


def _prepare_pages(case, gen, state):
    P, sizes = case["page"], _counts(case)
    held = [-(-length // P) for _, length in sizes]
    need = [-(-(length + n) // P) for n, length in sizes]
    wanted = sum(need) - sum(held)
    spare = int(case["pool"] * wanted) + (8 if case["pool"] >= 1 else 0)
    order = torch.randperm(sum(held) + spare, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(sizes), max(1, max(need)) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
    free = torch.full_like(order, -1)
    free[:spare] = order[at:]
    state["pool"] = {"free": free, "count": _i32([spare]), "lacking": _i32([0])}
    state["block_table"], state["lengths"] = table, _i32([length for _, length in sizes])
    state["new"] = None if case["form"] == "even" and not case["pad"] else _i32([n for n, _ in sizes])
    state["keep"] = state["lengths"].clone()
    state["total"] = _total(case)


def _axis_of(case):
    """The axis of each angle: in blocks, or dealt in turn until an axis has its share."""
    left = [int(n) for n in case["sections"].split(",")]
    if case["order"] == "blocks":
        return tuple(a for a, n in enumerate(left) for _ in range(n))
    out = []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return tuple(out)


def _frequencies(case, device="cuda"):
    """Of each angle, base 10000: one spectrum over all of them, or one for each axis's own."""
    axis = _axis_of(case)
    place = [axis[:i].count(a) for i, a in enumerate(axis)] if case["spectrum"] == "own" else range(len(axis))
    of = [axis.count(a) for a in axis] if case["spectrum"] == "own" else [len(axis)] * len(axis)
    share = torch.tensor([i / n for i, n in zip(place, of)], dtype=torch.float64, device=device)
    return 10000.0 ** -share


def _grid(case, gen):
    """Positions [axes, T] of a grid as square as its size allows, its last axes
    the fastest, counted from a random first position on each."""
    A, T = case["sections"].count(",") + 1, case["t"]
    side = max(1, math.ceil(T ** (1 / A)))
    t = torch.arange(T, device="cuda")
    at = torch.stack([t // side ** (A - 1 - a) % (side if a else T) for a in range(A)])
    return (at + torch.randint(0, 64, (A, 1), generator=gen, device="cuda")).to(torch.int32), side


def _prepare_axes(case, gen, state):
    T, Hq, H, D, dtype = case["t"], case["heads"], case["kv_heads"], case["dim"], DTYPES[case["x"]]
    if case["fused"]:
        qkv = _randn(gen, (T, Hq + 2 * H, D), dtype)
        state["q"], state["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + H]
    else:
        state["q"], state["k"] = _randn(gen, (T, Hq, D), dtype), _randn(gen, (T, H, D), dtype)
    state["positions"], side = _grid(case, gen)
    state["axes"] = _axis_of(case)
    f = _frequencies(case)
    angle = torch.arange(max(T, side) + 64, dtype=torch.float64, device="cuda")[:, None] * f
    state["table"] = torch.stack([angle.cos(), angle.sin()], -1).float()


def _prepare_norm(case, gen, state):
    T, D, x, r = case["t"], case["dim"], DTYPES[case["x"]], DTYPES[case["residual"]]

    def near(mean, *shape):  # trained weights, gates and shifts
        return (mean + 0.2 * torch.randn(shape, generator=gen, device="cuda")).to(x)

    one = 1.0 - case["offset"]
    state["weight"] = near(one, D)
    state["bias"] = near(0.0, D) if case["norm"] == "layer" else None
    if case["form"] == "heads":
        fused = _randn(gen, (T, case["heads"] + 2, D), x)
        state["y"] = fused[:, 1:1 + case["heads"]]
        return
    state["y"] = _randn(gen, (T, D), x)
    # a residual stream: larger than what a block adds, with a few channels far larger
    gain = 3 + 40 * (torch.rand(D, generator=gen, device="cuda") < 0.004).float()
    state["residual"] = (torch.randn(T, D, generator=gen, device="cuda") * gain).to(r)
    state["post"] = near(one, D) if case["post"] else None
    groups = {"channel": 1, "token": T, "sequence": case["batch"]}
    state["gate"] = near(0.5, groups[case["gate"]], D) if case["gate"] != "none" else None
    state["modulate"] = (near(0.0, case["batch"], D), near(0.0, case["batch"], D)) if case["modulate"] else None


def _power(e):
    """2^e in fp32, e in -126..127."""
    return ((e + 127) << 23).view(torch.float32)


def _code(x):
    """x [..., 32 n] fp32, finite -> codes uint8 [..., 32 n] and exponent bytes
    uint8 [..., n]: the smallest exponent whose grid's top, 6, the block's
    largest value rounds to (or below); then to the nearest value of the grid,
    ties to the even code."""
    y = x.unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    e = ((top.view(torch.int32) + 0x200000) >> 23).sub_(2).clamp_(2, 252)
    y = y * _power(127 - e)
    a = y.abs()
    step = 0.5 + 0.5 * (a >= 2) + (a >= 4)
    a = (torch.round(a / step) * step).clamp_(max=6.0)
    code = (2 * a).clamp(max=4) + (a - 2).clamp(0, 2) + ((a - 4) / 2).clamp(0, 1)
    code = code.to(torch.uint8) + (y < 0).to(torch.uint8) * 8
    return code.flatten(-2), e.squeeze(-1).to(torch.uint8)


def _words(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous().view(torch.int32)


def _prepare_sparse(case, gen, state):
    """The sequences in shuffled pages of a cache that is noise elsewhere. Keys
    of a page share a topic, and a run of queries looks for some of them."""
    H, Hq, D, P = case["kv_heads"], case["heads"], case["dim"], case["page"]
    sizes = _sizes(case)
    counts = [-(-length // P) for _, length in sizes]
    total = sum(counts) + 2
    order = torch.randperm(total, generator=gen, device="cuda")

    def noise(shape, lo, hi, dtype):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=dtype)

    kc, vc = noise((total, H, P, D // 8), -2 ** 31, 2 ** 31, torch.int32), \
        noise((total, H, P // 8, D // 8, 8), -2 ** 31, 2 ** 31, torch.int32)
    ks, vs = noise((total, H, P, D // 32), 0, 256, torch.uint8), noise((total, H, P // 8, D // 32, 8), 0, 256, torch.uint8)
    bounds, scales = noise((total, H, 2, D), -128, 128, torch.int8), noise((total, H), 0, 256, torch.uint8)
    table = torch.full((len(sizes), max(1, *counts)), -1, dtype=torch.int32, device="cuda")
    gain = 1 + 3 * (torch.rand(H, 1, D, generator=gen, device="cuda") < 0.03).float()
    topics = torch.randn(H, 32, D, generator=gen, device="cuda")
    at = 0
    for b, (n, length) in enumerate(sizes):
        table[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
        step = max(1, (1 << 25) // (H * D * P)) * P
        for t0 in range(0, length, step):
            m = min(step, length - t0)
            where = torch.arange(t0, t0 + m, device="cuda")
            page, slot = table[b, where // P].long()[:, None], (where % P)[:, None]
            head = torch.arange(H, device="cuda")[None]
            topic = torch.randint(0, 32, (m // P + 2,), generator=gen, device="cuda")[(where - t0) // P]
            k = 0.7 * topics[:, topic] + 0.7 * torch.randn(H, m, D, generator=gen, device="cuda")
            codes, e = _code(k * gain)
            kc[page, head, slot], ks[page, head, slot] = _words(codes).transpose(0, 1), e.transpose(0, 1)
            codes, e = _code(torch.randn(H, m, D, generator=gen, device="cuda"))
            vc[page, head, slot // 8, :, slot % 8] = _words(codes).transpose(0, 1)
            vs[page, head, slot // 8, :, slot % 8] = e.transpose(0, 1)
        held = (length - n) // P if n else counts[b]  # (the pages that the new tokens do not touch)
        for c0 in range(0, held, max(1, (1 << 25) // (H * D * P))):
            page = table[b, c0:min(held, c0 + max(1, (1 << 25) // (H * D * P)))].long()
            c = torch.arange(c0, c0 + page.shape[0], device="cuda")
            bounds[page], scales[page] = _bounds(kc, ks, page, (length - c * P).clamp(max=P))
    state["cache"] = {"k_codes": kc, "k_scales": ks, "v_codes": vc, "v_scales": vs}
    state["summaries"] = {"bounds": bounds, "scales": scales}
    state["block_table"], state["lengths"] = table, _i32([length for _, length in sizes])
    state["cu"] = None
    T = sum(n for n, _ in sizes)
    if len({n for n, _ in sizes}) > 1:
        ends = [0]
        for n, _ in sizes:
            ends.append(ends[-1] + n)
        state["cu"] = _i32(ends)
    run = torch.arange(T, device="cuda") // 64
    topic = torch.randint(0, 32, (T // 64 + 1, H), generator=gen, device="cuda")[run]
    look = topics[torch.arange(H, device="cuda"), topic][:, :, None].expand(T, H, Hq // H, D)
    q = 0.5 * look.reshape(T, Hq, D) + torch.randn(T, Hq, D, generator=gen, device="cuda")
    state["q"] = q.to(DTYPES[case["x"]])


PREPARE = {"pages": _prepare_pages, "axes": _prepare_axes, "norm": _prepare_norm, "sparse": _prepare_sparse}


def prepare(case, seed):
    state = {"case": case, "kind": case["kind"]}
    PREPARE[case["kind"]](case, _gen(seed), state)
    return state


# -------------------------------------------------------------- plain forms --


def _plain_pages(state):
    P, T, table, lengths, pool = state["case"]["page"], state["total"], state["block_table"], state["lengths"], state["pool"]
    B, cols = table.shape
    free, count = pool["free"], pool["count"]
    new = torch.full_like(lengths, T // B) if state["new"] is None else state["new"]
    cu = torch.zeros(B + 1, dtype=torch.int32, device="cuda")
    cu[1:] = new.clamp(min=0).long().cumsum(0).clamp(max=T)
    n = cu.diff()
    have, want = (lengths + P - 1) // P, ((lengths + n + P - 1) // P).clamp(max=cols)
    need = (want - have).clamp(min=0)
    col = torch.arange(cols, device="cuda")
    rank = (need.cumsum(0) - need)[:, None] + col - have[:, None]
    taken = count - 1 - rank
    page = torch.where(taken >= 0, free[taken.clamp(min=0, max=free.shape[0] - 1)], -1)
    table.copy_(torch.where((col >= have[:, None]) & (col < want[:, None]), page, table))
    pool["lacking"].copy_((need.sum() - count).clamp(min=0))
    count.copy_((count - need.sum()).clamp(min=0))
    t = torch.arange(T, device="cuda")
    seq = torch.searchsorted(cu[1:], t.int(), right=True).clamp(max=B - 1)
    at = lengths[seq] + t - cu[seq]
    inside = t < cu[-1]
    page = table[seq, (at // P).clamp(max=cols - 1)].long()
    ok = inside & (at // P < cols) & (page >= 0) & (page < free.shape[0])
    slots = torch.where(ok, page * P + at % P, -1)
    positions = torch.where(inside, at, -1).int()
    lengths += n
    # cut back
    keep = torch.minimum(state["keep"].clamp(min=0), lengths)
    gone = (col >= ((keep + P - 1) // P)[:, None]) & (col < ((lengths + P - 1) // P)[:, None])
    back = (gone & (table >= 0) & (table < free.shape[0])).flatten()
    order = back.cumsum(0)
    to = torch.where(back, count + order[-1] - order, free.shape[0])
    longer = torch.cat([free, free[:1]])
    longer[to] = table.flatten()
    free.copy_(longer[:-1])
    count.add_(order[-1])
    table.masked_fill_(gone, -1)
    lengths.copy_(keep)
    return [cu, positions, slots, table, lengths, free, count, pool["lacking"]]


def _plain_axes(state):
    c = state["case"]
    axis = torch.tensor(state["axes"], device="cuda")
    angle = torch.arange(len(state["axes"]), device="cuda")
    cs = state["table"][state["positions"].long()[axis].t(), angle]  # [T, angles, 2]
    cos, sin = cs[:, None, :, 0], cs[:, None, :, 1]
    n, out = len(state["axes"]), []
    for x in (state["q"], state["k"]):
        y = x.float()
        if c["layout"] == "half":
            a, b = y[..., :n], y[..., n:2 * n]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = y[..., 0:2 * n:2], y[..., 1:2 * n:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        out.append(torch.cat([r, y[..., 2 * n:]], -1).to(x.dtype))
    return out


EPS = 1e-6


def _plain_one(v, kind, weight, bias, offset):
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS) * (weight.float() + offset)
    return v if bias is None else v + bias.float()


def _by_row(v, t):
    """[groups, D] for t rows, each group's the same number of them."""
    return v.float().repeat_interleave(t // v.shape[0], 0, output_size=t)


def _plain_norm(state):
    c, y = state["case"], state["y"]
    if c["form"] == "heads":
        return _plain_one(y.float(), c["norm"], state["weight"], state["bias"], c["offset"]).to(y.dtype)
    z = y.float()
    if state["post"] is not None:
        z = _plain_one(z, c["norm"], state["post"], None, c["offset"])
    if state["gate"] is not None:
        z = z * _by_row(state["gate"], c["t"])
    r = state["residual"].float() + c["factor"] * z
    x = _plain_one(r, c["norm"], state["weight"], state["bias"], c["offset"])
    if state["modulate"] is not None:
        scale, shift = state["modulate"]
        x = x * (1 + _by_row(scale, c["t"])) + _by_row(shift, c["t"])
    return [r.to(state["residual"].dtype), x.to(y.dtype)]


def _values(codes, e):
    """codes [..., D], exponent bytes [..., D/32] -> fp32 values."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    scale = torch.where(e == 255, math.nan, _power(e.int().clamp(1, 254) - 127))
    return (grid[codes.long()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _nibbles(words):
    b = words.contiguous().view(torch.uint8)
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _bounds(kc, ks, page, tokens):
    """The summaries of pages [N], of which `tokens` [N] tokens count: int8 [N, H, 2, D], uint8 [N, H]."""
    k = _values(_nibbles(kc[page]), ks[page])  # [N, H, P, D]
    out = (torch.arange(k.shape[2], device="cuda") >= tokens[:, None])[:, None, :, None] | k.isnan()
    hi, lo = k.masked_fill(out, -math.inf).amax(2), k.masked_fill(out, math.inf).amin(2)
    hi, lo = torch.where(hi == -math.inf, 0.0, hi), torch.where(lo == math.inf, 0.0, lo)
    top = torch.maximum(hi.abs(), lo.abs()).amax(-1).double()
    m, x = torch.frexp(top)
    e = torch.where(top > 0, x - 7 + (m > 127 / 128), -126).clamp(min=-126)
    unit = torch.exp2(e.double())[..., None]
    return torch.stack([torch.ceil(hi / unit), torch.floor(lo / unit)], 2).to(torch.int8), (e + 127).to(torch.uint8)


def _where(state):
    """Of each new token: its sequence, its place there and its position."""
    T, B = state["q"].shape[0], state["lengths"].shape[0]
    t = torch.arange(T, device="cuda")
    if state["cu"] is None:
        n = T // B
        seq, m, count = t // n, t % n, torch.full((B,), n, device="cuda")
    else:
        seq = torch.searchsorted(state["cu"][1:].long(), t, right=True)
        m, count = t - state["cu"].long()[seq], state["cu"].diff()
    return seq, m, state["lengths"].long()[seq] - count[seq] + m, count


def _plain_summarize(state, count):
    """The pages of the new tokens, all sequences as many columns as the longest
    can have; past a sequence's last one, and where it has none, the first
    sequence's last one again."""
    c, lengths, P = state["case"], state["lengths"].long(), state["case"]["page"]
    col = ((lengths - count) // P)[:, None] + torch.arange((c["tokens"] + P - 2) // P + 1, device="cuda")
    last = (lengths - 1) // P
    in_ = (col <= last[:, None]) & (count > 0)[:, None]
    col = torch.where(in_, col, last[0])
    seq = torch.where(in_, torch.arange(len(lengths), device="cuda")[:, None], 0)
    page = state["block_table"].long()[seq, col]
    held = (lengths[seq] - col * P).clamp(max=P).flatten()
    page = page.flatten()
    bounds, scales = _bounds(state["cache"]["k_codes"], state["cache"]["k_scales"], page, held)
    state["summaries"]["bounds"][page] = bounds
    state["summaries"]["scales"][page] = scales


def _plain_select(state, seq, at):
    """-> columns [T, H, count], ascending, -1 behind."""
    c, q, table = state["case"], state["q"].float(), state["block_table"].long()
    T, (B, cols), H, D, P, count = q.shape[0], table.shape, c["kv_heads"], c["dim"], c["page"], c["count"]
    q = q.view(T, H, -1, D)
    top = q.abs().amax((2, 3), keepdim=True)
    m, x = torch.frexp(top)
    e = torch.where(top > 0, x - 7 + (m >= 127.5 / 128).int(), -126).clamp(min=-126)
    q = torch.round(q * _power(-e))
    sides = torch.cat([q.clamp(min=0), q.clamp(max=0)], -1)  # [T, H, group, 2 D]
    column = torch.arange(cols, device="cuda")
    out = []
    step = max(1, (1 << 27) // (H * cols * max(sides.shape[2], 2 * D)))
    if B == 1:  # one sequence: its summaries laid out once
        page = table[0].clamp(min=0)
        one = state["summaries"]["bounds"][page].float().permute(1, 2, 3, 0).reshape(1, H, 2 * D, cols)
        unit = _power(state["summaries"]["scales"][page].int() - 127).t()[None]
        step = max(1, (1 << 27) // (H * cols * sides.shape[2]))
    for t0 in range(0, T, step):
        b, p = seq[t0:t0 + step], at[t0:t0 + step]
        if B == 1:
            s = torch.matmul(sides[t0:t0 + step].transpose(0, 1).flatten(1, 2), one[0])
            s = s.view(H, -1, sides.shape[2], cols).transpose(0, 1).amax(2) * unit
        else:
            page = table[b].clamp(min=0)
            bounds = state["summaries"]["bounds"][page].float()  # [t, cols, H, 2, D]
            bounds = bounds.permute(0, 2, 3, 4, 1).reshape(-1, H, 2 * D, cols)
            s = torch.matmul(sides[t0:t0 + step], bounds).amax(2)
            s = s * _power(state["summaries"]["scales"][page].int() - 127).transpose(1, 2)
        seen = column * P <= p[:, None]
        kept = seen & ((column < c["first"]) | (column > (p // P)[:, None] - c["last"]))
        key = torch.where(kept[:, None], math.inf, s.double())
        key = torch.where(seen[:, None], key, -math.inf)
        key, best = key.sort(dim=-1, descending=True, stable=True)
        best = torch.where(key > -math.inf, best, cols)[..., :count].sort(-1).values
        best = torch.where(best < cols, best, -1).int()
        out.append(torch.nn.functional.pad(best, (0, count - best.shape[-1]), value=-1))
    return torch.cat(out)


def _plain_listed(state, blocks, seq, at):
    """Softmax over the positions of the listed columns up to each query's own."""
    c, q, cache = state["case"], state["q"], state["cache"]
    T, Hq, D = q.shape
    H, P = c["kv_heads"], c["page"]
    head, slot = torch.arange(H, device="cuda")[:, None], torch.arange(P, device="cuda")
    outs, lses = [], []
    step = max(1, (1 << 26) // (H * c["count"] * P * D))
    for t0 in range(0, T, step):
        list_, p = blocks[t0:t0 + step].long(), at[t0:t0 + step]
        page = state["block_table"][seq[t0:t0 + step, None, None], list_.clamp(min=0)].long()
        k = _values(_nibbles(cache["k_codes"][page, head]), cache["k_scales"][page, head]).flatten(2, 3)
        v = _values(_nibbles(cache["v_codes"][page, head].transpose(-1, -2)),
                    cache["v_scales"][page, head].transpose(-1, -2)).flatten(2, 4)  # [t, H, count P, D]
        place = list_[..., None] * P + slot
        seen = ((place <= p[:, None, None, None]) & (list_ >= 0)[..., None]).flatten(2)[:, :, None]
        rows = q[t0:t0 + step].float().view(-1, H, Hq // H, D)
        s = torch.matmul(rows, k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        w = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
        total = w.sum(-1, keepdim=True)
        o = torch.matmul(w, torch.where(seen.transpose(-1, -2), v, 0.0)) / torch.where(total == 0, 1.0, total)
        outs.append(o.reshape(-1, Hq, D).to(q.dtype))
        lses.append((top + total.log()).reshape(-1, Hq))
    return torch.cat(outs), torch.cat(lses)


def _plain_sparse(state):
    seq, _, at, count = _where(state)
    _plain_summarize(state, count)
    blocks = _plain_select(state, seq, at)
    out, lse = _plain_listed(state, blocks, seq, at)
    sums = state["summaries"]
    return [sums["bounds"], sums["scales"], blocks, out] + ([lse] if state["case"]["lse"] else [])


PLAIN = {"pages": _plain_pages, "axes": _plain_axes, "norm": _plain_norm, "sparse": _plain_sparse}


# -------------------------------------------------------------------- cases --


@torch.no_grad()
def run(state):
    if not own:
        return PLAIN[state["kind"]](state)
    from drinkme_amd import kv_ops, norm_ops

    c = state["case"]
    if c["kind"] == "pages":
        pool, table, lengths = state["pool"], state["block_table"], state["lengths"]
        cu, positions, slots = kv_ops.reserve(pool, table, lengths, c["page"], state["total"], new=state["new"])
        kv_ops.trim(pool, table, lengths, c["page"], state["keep"])
        return [cu, positions, slots, table, lengths, pool["free"], pool["count"], pool["lacking"]]
    if c["kind"] == "axes":
        return list(kv_ops.rotary(state["q"], state["k"], state["positions"], state["table"], layout=c["layout"],
                                  axes=state["axes"]))
    if c["kind"] == "norm":
        if c["form"] == "heads":
            return norm_ops.norm(state["y"], state["weight"], bias=state["bias"], kind=c["norm"], eps=EPS,
                                 offset=c["offset"])
        return list(norm_ops.block_norm(state["y"], state["residual"], state["weight"], bias=state["bias"],
                                        post=state["post"], gate=state["gate"], factor=c["factor"],
                                        modulate=state["modulate"], kind=c["norm"], eps=EPS, offset=c["offset"]))
    cache, sums, table, lengths, cu = (state[x] for x in ("cache", "summaries", "block_table", "lengths", "cu"))
    most = c["tokens"] if cu is not None else None
    kv_ops.summarize(cache, sums, table, lengths, state["q"].shape[0], cu=cu)
    blocks = kv_ops.select(state["q"], cache, sums, table, lengths, c["count"], cu=cu, first=c["first"], last=c["last"])
    out = kv_ops.attention(state["q"], cache, table, lengths, cu=cu, max_tokens=most, blocks=blocks, return_lse=c["lse"])
    return [sums["bounds"], sums["scales"], blocks] + (list(out) if c["lse"] else [out])


def work(case):
    if case["kind"] == "pages":
        P, sizes = case["page"], _counts(case)
        handed = sum(-(-(length + n) // P) - -(-length // P) for n, length in sizes)
        touched = sum(-(-(length + n) // P) - length // P for n, length in sizes if n)  # table entries that slots need
        return {"bytes": 24 * len(sizes) + 16 * handed + 4 * touched + 12 * _total(case),
                "flops": 4 * _total(case) + 8 * len(sizes)}
    if case["kind"] == "axes":
        T, heads, size = case["t"], case["heads"] + case["kv_heads"], DTYPES[case["x"]].itemsize
        part = 2 * len(_axis_of(case))
        return {"bytes": 2 * T * heads * case["dim"] * size + T * (4 * part + 4 * (case["sections"].count(",") + 1)),
                "flops": 3 * T * heads * part}
    if case["kind"] == "norm":
        n, size = case["t"] * case["heads"] * case["dim"], DTYPES[case["x"]].itemsize
        if case["form"] == "heads":
            return {"bytes": 2 * n * size, "flops": 5 * n}
        side = {"none": 0, "channel": 1, "token": case["t"], "sequence": case["batch"]}[case["gate"]]
        side += 1 + case["post"] + (case["norm"] == "layer") + 2 * case["batch"] * case["modulate"]
        return {"bytes": n * 2 * (size + DTYPES[case["residual"]].itemsize) + side * case["dim"] * size,
                "flops": n * (7 + 4 * case["post"] + (case["gate"] != "none") + 2 * case["modulate"])}
    H, Hq, D, P, size = case["kv_heads"], case["heads"], case["dim"], case["page"], DTYPES[case["x"]].itemsize
    bytes_ = flops = tokens = 0
    for n, length in _sizes(case):
        if not n:
            continue
        first = length - n
        touched, pages = (length - 1) // P - first // P + 1, -(-length // P)
        bytes_ += touched * H * (min(P, length) * D * 17 / 32 + 2 * D + 1)  # summaries of the new tokens' pages
        bytes_ += pages * (H * (2 * D + 1) + 4)  # all summaries, for the scores
        seen = [(m // P + 1, m % P + 1) for m in range(first, length)]
        bytes_ += min(max(min(s, case["count"]) for s, _ in seen) * (1 if n <= 8 else n / 8), pages) * P * H * D * 17 / 16
        pairs = sum((min(s, case["count"]) - 1) * P + own_ for s, own_ in seen)
        flops += 4 * pairs * Hq * D + 4 * sum(s for s, _ in seen) * Hq * D
        tokens += n
    return {"bytes": bytes_ + tokens * (Hq * (2 * D * size + (4 if case["lse"] else 0)) + 4 * H * case["count"]),
            "flops": flops}


# ------------------------------------------------------------ in 64 bits --


def _exact_pages(case, state):
    P = case["page"]
    free, count = state["pool"]["free"].tolist(), state["pool"]["count"].item()
    table, lengths = state["block_table"].tolist(), state["lengths"].tolist()
    cols, T, pages = len(table[0]), state["total"], len(free)
    new = [T // len(lengths)] * len(lengths) if state["new"] is None else state["new"].tolist()
    cu, positions, slots, short = [0], [-1] * T, [-1] * T, 0
    for b, n in enumerate(new):
        n = min(n, T - cu[-1])
        for col in range(-(-lengths[b] // P), min(cols, -(-(lengths[b] + n) // P))):
            if count:
                count -= 1
                table[b][col] = free[count]
            else:
                table[b][col], short = -1, short + 1
        for m in range(n):
            p, t = lengths[b] + m, cu[-1] + m
            positions[t] = p
            if p // P < cols and 0 <= table[b][p // P] < pages:
                slots[t] = table[b][p // P] * P + p % P
        lengths[b] += n
        cu.append(cu[-1] + n)
    back = []
    for b, keep in enumerate(state["keep"].tolist()):
        keep = min(keep, lengths[b])
        for col in range(-(-keep // P), min(cols, -(-lengths[b] // P))):
            if table[b][col] >= 0:
                back.append(table[b][col])
            table[b][col] = -1
        lengths[b] = keep
    for page in reversed(back):
        free[count] = page
        count += 1
    return [torch.tensor(x, dtype=d, device="cuda") for x, d in
            ((cu, torch.int32), (positions, torch.int32), (slots, torch.int64), (table, torch.int32),
             (lengths, torch.int32), (free, torch.int32), ([count], torch.int32), ([short], torch.int32))]


def _exact_axes(case, state):
    n = len(state["axes"])
    # (the table's own roundings are part of the inputs: what it says is turned)
    cs = state["table"].double()
    turn = torch.zeros(case["t"], n, dtype=torch.complex128, device="cuda")
    for i, a in enumerate(state["axes"]):
        turn[:, i] = torch.view_as_complex(cs[:, i].contiguous())[state["positions"][a].long()]
    out = []
    for x in (state["q"], state["k"]):
        x = x.double()
        part = x[..., :2 * n]
        z = part.unflatten(-1, (2, n)).transpose(-1, -2) if case["layout"] == "half" else part.unflatten(-1, (n, 2))
        z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[:, None])
        z = z.transpose(-1, -2) if case["layout"] == "half" else z
        out.append(torch.cat([z.flatten(-2), x[..., 2 * n:]], -1))
    return out


def _exact_norm(case, state):
    def norm(v, weight, bias):
        scale = weight.double() + case["offset"]
        if case["norm"] == "layer":
            v = (v - v.mean(-1, keepdim=True)) / (v.var(-1, keepdim=True, correction=0) + EPS).sqrt() * scale
        else:
            v = v / (v.square().mean(-1, keepdim=True) + EPS).sqrt() * scale
        return v + bias.double() if bias is not None else v

    y = state["y"].double()
    if case["form"] == "heads":
        return norm(y, state["weight"], state["bias"])
    if state["post"] is not None:
        y = norm(y, state["post"], None)

    def rows(v):
        return v.double()[torch.arange(case["t"], device="cuda") // (case["t"] // v.shape[0])]

    if state["gate"] is not None:
        y = rows(state["gate"]) * y
    r = state["residual"].double() + case["factor"] * y
    x = norm(r, state["weight"], state["bias"])
    if state["modulate"] is not None:
        x = x + rows(state["modulate"][0]) * x + rows(state["modulate"][1])
    return [r, x]


def _exact_sparse(case, state):
    H, D, P, group = case["kv_heads"], case["dim"], case["page"], case["heads"] // case["kv_heads"]
    cache, grid = state["cache"], torch.tensor(GRID, dtype=torch.float64, device="cuda")
    shifts = 4 * torch.arange(8, device="cuda")
    bounds, scales = state["summaries"]["bounds"].clone(), state["summaries"]["scales"].clone()
    q = state["q"].double()
    T = q.shape[0]
    blocks = torch.full((T, H, case["count"]), -1, dtype=torch.int32, device="cuda")
    out, lse = torch.zeros_like(q), torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")

    def values(words, e):  # words [n, D/8], e [n, D/32]
        code = ((words.long()[..., None] >> shifts) & 15).flatten(1)
        return grid[code & 7] * torch.where(code > 7, -1.0, 1.0) * torch.exp2(e.double() - 127).repeat_interleave(32, 1)

    t0 = 0
    for b, (n, length) in enumerate(_sizes(case)):
        if not n:
            continue
        t = torch.arange(length, device="cuda")
        page, slot = state["block_table"][b].long()[t // P], t % P
        used = state["block_table"][b, :-(-length // P)].long()
        at = torch.arange(length - n, length, device="cuda")
        for h in range(H):
            k = values(cache["k_codes"][page, h, slot], cache["k_scales"][page, h, slot])
            v = values(cache["v_codes"][page, h, slot // 8, :, slot % 8], cache["v_scales"][page, h, slot // 8, :, slot % 8])
            c = torch.arange(len(used), device="cuda")
            whole = torch.nn.functional.pad(k, (0, 0, 0, len(used) * P - length), value=math.nan).view(-1, P, D)
            hi = whole.nan_to_num(nan=-math.inf).amax(1)
            lo = whole.nan_to_num(nan=math.inf).amin(1)
            top = torch.maximum(hi.abs(), lo.abs()).amax(1)
            e = torch.ceil(torch.log2(top.clamp(min=2.0 ** -140) / 127)).clamp(min=-126)  # then to the border itself
            e = torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e)
            e = torch.where(127 * torch.exp2(e) < top, e + 1, e).clamp(min=-126)
            up, down = torch.ceil(hi / torch.exp2(e)[:, None]), torch.floor(lo / torch.exp2(e)[:, None])
            new = c >= (length - n) // P
            bounds[used[new], h, 0], bounds[used[new], h, 1] = up[new].to(torch.int8), down[new].to(torch.int8)
            scales[used[new], h] = (e[new] + 127).to(torch.uint8)
            mine = q[t0:t0 + n, h * group:(h + 1) * group]  # [n, group, D]
            most = mine.abs().amax((1, 2)).clamp(min=2.0 ** -140)
            f = torch.ceil(torch.log2(most / 127.5)).clamp(min=-126)
            f = torch.where(127.5 * torch.exp2(f - 1) > most, f - 1, f)
            f = torch.where(127.5 * torch.exp2(f) <= most, f + 1, f).clamp(min=-126)
            whole_q = torch.round(mine / torch.exp2(f)[:, None, None])
            score = torch.where(whole_q > 0, whole_q, 0) @ up.t() + torch.where(whole_q < 0, whole_q, 0) @ down.t()
            score = score.amax(1) * torch.exp2(e)  # [n, columns]
            last = (at // P)[:, None]
            score = torch.where((c < case["first"]) | (c > last - case["last"]), math.inf, score)
            # the rank of a column: those that beat it, and of its equals those before it
            order = torch.argsort(torch.where(c <= last, -score, math.inf), dim=1, stable=True)
            take = torch.zeros(n, len(used), dtype=torch.bool, device="cuda")
            take.scatter_(1, order[:, :case["count"]], True)
            take &= c <= last
            place = take.cumsum(1) - 1
            row = torch.arange(n, device="cuda")[:, None].expand_as(take)
            blocks[t0 + row[take], h, place[take]] = c.expand_as(take)[take].int()
            seen = take[:, t // P] & (t <= at[:, None])
            for g in range(h * group, (h + 1) * group):
                s = torch.where(seen, q[t0:t0 + n, g] @ k.t() / math.sqrt(D), -math.inf)
                lse[t0:t0 + n, g] = torch.logsumexp(s, -1)
                out[t0:t0 + n, g] = torch.softmax(s, -1) @ v
        t0 += n
    return [bounds, scales, blocks, out] + ([lse] if case["lse"] else [])


EXACT = {"pages": _exact_pages, "axes": _exact_axes, "norm": _exact_norm, "sparse": _exact_sparse}


@torch.no_grad()
def exact(case, seed):
    return EXACT[case["kind"]](case, prepare(case, seed))
