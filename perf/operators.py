"""The operators between a decoder's q/k/v and o projections, as a list of
measured cases: rotary positions, the append to a paged key/value cache held
in 4 bits, and the attention that reads it.

A case is one pass of one of them:

  rotary  the queries and keys of t tokens rotated by their positions
  append  the new tokens' queries rotated, their keys rotated and coded into
          the cache, their values coded; then those tokens read back from it
  attend  the new tokens' queries against everything cached of their
          sequences: one token a sequence (a decode step), 2..8 (the verify
          rows of speculative decoding) or prompts of many

The cache holds, of each token and key/value head, blocks of 32 channels: an
exponent byte e (the block's scale 2^(e - 127); 255 where the block held a
value that is not finite) and 32 four-bit codes (sign, then 0 .5 1 1.5 2 3 4 6).
With H heads of D channels and pages of P tokens it is

  k_codes   int32 [pages, H, P, D/8]      nibble n of a word: channel 8 w + n
  k_scales  uint8 [pages, H, P, D/32]
  v_codes   int32 [pages, H, P/8, D/8, 8] eight tokens' words side by side
  v_scales  uint8 [pages, H, P/8, D/32, 8]

Token m of the n new ones of a sequence sits at position lengths - n + m, in
page block_table[sequence, position / P]. Keys and values are N(0, 1), keys
with a few channels four times as large, as trained models have; what the
pages hold past a sequence's end is noise.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _rotary(name, t, heads, kv_heads, dim, part, layout="half", x="bf16", scaling="none", positions=8192, fused=False):
    return {"name": name, "kind": "rotary", "t": t, "heads": heads, "kv_heads": kv_heads, "dim": dim, "part": part,
            "layout": layout, "x": x, "scaling": scaling, "positions": positions, "fused": fused}


def _append(name, batch, tokens, length, heads, kv_heads, dim, part, page, layout="half", x="bf16", ragged=False):
    return {"name": name, "kind": "append", "batch": batch, "tokens": tokens, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "part": part, "page": page, "layout": layout, "x": x, "ragged": ragged}


def _attend(name, batch, tokens, length, heads, kv_heads, dim, page, x="bf16", ragged=False, window=0, causal=True,
            lse=False):
    return {"name": name, "kind": "attend", "batch": batch, "tokens": tokens, "length": length, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "x": x, "ragged": ragged, "window": window,
            "causal": causal, "lse": lse}


def listed():
    return [
        # a decode step's one token (32 query and 8 key heads of 128, as 4096 and 1024 rows of q and k)
        _rotary("rotary-step", 1, 32, 8, 128, 128),
        # a prompt, out of a fused q/k/v product, by a table scaled to a long context
        _rotary("rotary-prompt", 8192, 32, 8, 128, 128, scaling="wavelength", positions=131072, fused=True),
        # half of an odd-sized head, pairs side by side, fp32 activations, an odd count of tokens
        _rotary("rotary-part-f32", 1021, 16, 2, 96, 48, layout="interleaved", x="f32", scaling="linear"),
        # a decode step of 32 sequences: a token each
        _append("append-step", 32, 1, 4096, 32, 8, 128, 128, 64, ragged=True),
        # a batch of prompts of different lengths
        _append("append-prompts", 6, 2048, 2048, 32, 8, 128, 128, 64, ragged=True),
        # the smallest attention of a server: one sequence, a short context
        _attend("attend-one", 1, 1, 1021, 32, 8, 128, 64),
        # a decode step of a busy server
        _attend("attend-batch", 32, 1, 8192, 32, 8, 128, 64, ragged=True),
        # one sequence of a very long context (64 query heads, as 8192 rows of q)
        _attend("attend-long", 1, 1, 131072, 64, 8, 128, 128),
        # speculative decoding: one accepted and four draft rows, small pages
        _attend("attend-verify", 8, 5, 4097, 32, 8, 128, 16, ragged=True, lse=True),
        # a chunk of a long prompt after what is already cached
        _attend("attend-chunk", 1, 2048, 10240, 32, 8, 128, 64),
        # a batch of prompts (one of a single token, one empty), a sliding window, small heads
        _attend("attend-prompts-window", 6, 2048, 2048, 16, 4, 64, 32, ragged=True, window=512),
        # fp32 activations, one key head for all, wide heads
        _attend("attend-f32", 4, 1, 4097, 8, 1, 256, 64, x="f32", ragged=True, lse=True),
    ]


def _log_between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    u = rng.random()
    kv = rng.choice([1, 2, 4, 8, 8, 16])
    heads = kv * rng.choice([1, 2, 3, 4, 4, 5, 8])
    x = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if u < 0.25:
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        part = rng.choice([dim, dim, dim // 2, dim // 4])
        t = max(1, min(_log_between(rng, 1, 8192), 8192 * 40 * 128 // ((heads + kv) * dim * (2 if x == "f32" else 1))))
        c = _rotary("", t, heads, kv, dim, part, rng.choice(["half", "interleaved"]), x,
                    rng.choice(["none", "linear", "wavelength"]), _log_between(rng, 8192, 131072), rng.random() < 0.5)
    else:
        dim, page = rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([16, 32, 64, 64, 128])
        ragged = rng.random() < 0.6
        if u < 0.45:
            tokens = rng.choice([1, 1, 2, 5, 8, 0])
            tokens = tokens or _log_between(rng, 9, 2048)
            batch = _log_between(rng, 1, 64)
            batch = max(1, min(batch, 8192 * 48 * 128 // (tokens * (heads + 2 * kv) * dim * 2)))
            c = _append("", batch, tokens, tokens + _log_between(rng, 1, 4096), heads, kv, dim,
                        rng.choice([dim, dim, dim // 2]), page, rng.choice(["half", "interleaved"]), x, ragged)
        else:
            few = u < 0.75
            tokens = rng.choice([1, 1, 1, 2, 3, 4, 5, 8]) if few else _log_between(rng, 9, 2048)
            length = max(tokens, _log_between(rng, 16, 131072 if few else 8192))
            cost = length * kv * dim if few else length * tokens * heads * dim * (6 if x == "f32" else 1)
            most = 32 * 8192 * 8 * 128 // 2 if few else 10240 * 2048 * 32 * 128 // 2
            batch = max(1, min(_log_between(rng, 1, 64 if few else 8), most // cost))
            if cost > most:
                length = max(tokens, length * most // cost)
            c = _attend("", batch, tokens, length, heads, kv, dim, page, x, ragged,
                        rng.choice([0, 0, 0, _log_between(rng, 16, 4096)]), rng.random() < 0.9, rng.random() < 0.3)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs --


def _sizes(case):
    """(new tokens, cached tokens) of each sequence: where ragged, prompts and
    contexts shrink to half, the second prompt is empty and the third one
    token."""
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


def _uneven(case):
    return case["ragged"] and case["tokens"] > 8


def _frequencies(dim, scaling):
    """The rotary frequencies of `dim` channels, base 10000: divided by 4
    ("linear"), or by 8 where the wavelength passes 8192 positions and by
    less down to 2048 ("wavelength")."""
    i = torch.arange(dim // 2, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-2.0 * i / dim)
    if scaling == "linear":
        return f / 4
    if scaling == "wavelength":
        turns = 8192.0 * f / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        return keep * f + (1 - keep) * f / 8
    return f


def _table(dim, positions, scaling="none"):
    t = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * _frequencies(dim, scaling)
    return torch.stack([t.cos(), t.sin()], -1).float()


def _heads(gen, t, heads, dim, dtype):
    return torch.randn(t, heads, dim, generator=gen, device="cuda").to(dtype)


def _power(e):
    """2^e in fp32, e in -126..127."""
    return ((e + 127) << 23).view(torch.float32)


def _code(x):
    """x [..., 32 n] fp32 -> codes uint8 [..., 32 n] and exponent bytes
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
    return code.flatten(-2), torch.where(torch.isfinite(top), e, 255).squeeze(-1).to(torch.uint8)


def _words(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).contiguous().view(torch.int32)


def _pages(case, gen):
    """A cache that holds the case's sequences in shuffled pages, their table
    (-1 past a sequence's end) and lengths."""
    H, D, P = case["kv_heads"], case["dim"], case["page"]
    sizes = _sizes(case)
    counts = [-(-length // P) for _, length in sizes]
    total = sum(counts) + 2
    order = torch.randperm(total, generator=gen, device="cuda")
    kc = torch.randint(-2 ** 31, 2 ** 31, (total, H, P, D // 8), generator=gen, device="cuda", dtype=torch.int32)
    vc = torch.randint(-2 ** 31, 2 ** 31, (total, H, P // 8, D // 8, 8), generator=gen, device="cuda",
                       dtype=torch.int32)
    ks = torch.randint(0, 256, (total, H, P, D // 32), generator=gen, device="cuda", dtype=torch.uint8)
    vs = torch.randint(0, 256, (total, H, P // 8, D // 32, 8), generator=gen, device="cuda", dtype=torch.uint8)
    table = torch.full((len(sizes), max(1, *counts)), -1, dtype=torch.int32, device="cuda")
    gain = 1 + 3 * (torch.rand(H, 1, D, generator=gen, device="cuda") < 0.03).float()
    at = 0
    for b, (_, length) in enumerate(sizes):
        table[b, :counts[b]] = order[at:at + counts[b]]
        at += counts[b]
        if case["kind"] == "append":
            continue
        step = max(1, (1 << 26) // (H * D * P)) * P
        for t0 in range(0, length, step):
            n = min(step, length - t0)
            where = torch.arange(t0, t0 + n, device="cuda")
            page, slot = table[b, where // P].long()[:, None], (where % P)[:, None]
            head = torch.arange(H, device="cuda")[None]
            codes, e = _code(torch.randn(H, n, D, generator=gen, device="cuda") * gain)
            kc[page, head, slot], ks[page, head, slot] = _words(codes).transpose(0, 1), e.transpose(0, 1)
            codes, e = _code(torch.randn(H, n, D, generator=gen, device="cuda"))
            vc[page, head, slot // 8, :, slot % 8] = _words(codes).transpose(0, 1)
            vs[page, head, slot // 8, :, slot % 8] = e.transpose(0, 1)
    cache = {"k_codes": kc, "k_scales": ks, "v_codes": vc, "v_scales": vs}
    return cache, table, torch.tensor([length for _, length in sizes], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, H, D = DTYPES[case["x"]], case["kv_heads"], case["dim"]
    state = {"case": case, "kind": case["kind"]}
    if case["kind"] == "rotary":
        T, Hq = case["t"], case["heads"]
        if case["fused"]:
            qkv = _heads(gen, T, Hq + 2 * H, D, dtype)
            state["q"], state["k"] = qkv[:, :Hq], qkv[:, Hq:Hq + H]
        else:
            state["q"], state["k"] = _heads(gen, T, Hq, D, dtype), _heads(gen, T, H, D, dtype)
        first = torch.randint(0, case["positions"] - T + 1, (1,), generator=gen, device="cuda")
        state["positions"] = (first + torch.arange(T, device="cuda")).to(torch.int32)
        state["table"] = _table(case["part"], case["positions"], case["scaling"])
        return state
    sizes = _sizes(case)
    T = sum(n for n, _ in sizes)
    state["cache"], state["block_table"], state["lengths"] = _pages(case, gen)
    state["cu"] = None
    if _uneven(case):
        ends = [0]
        for n, _ in sizes:
            ends.append(ends[-1] + n)
        state["cu"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
    state["q"] = _heads(gen, T, case["heads"], D, dtype)
    if case["kind"] == "append":
        state["k"], state["v"] = _heads(gen, T, H, D, dtype), _heads(gen, T, H, D, dtype)
        state["table"] = _table(case["part"], case["length"])
    return state


# -------------------------------------------------------------- plain forms --


def _rotate(x, cos, sin, part, layout):
    """x [T, H, D] fp32 by cos, sin [T, part / 2]."""
    c, s, r = cos[:, None], sin[:, None], x[..., :part]
    if layout == "half":
        a, b = r[..., :part // 2], r[..., part // 2:]
        r = torch.cat([a * c - b * s, b * c + a * s], -1)
    else:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    return torch.cat([r, x[..., part:]], -1)


def _rounded_to_cache(x):
    codes, e = _code(x)
    return _values(codes, e).to(torch.bfloat16)


def _values(codes, e):
    """codes [..., D], exponent bytes [..., D/32] -> fp32 values."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    scale = torch.where(e == 255, math.nan, _power(e.int().clamp(1, 254) - 127))
    return (grid[codes.long()].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


def _nibbles(words):
    b = words.contiguous().view(torch.uint8)
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


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
    return seq, m, state["lengths"].long()[seq] - count[seq] + m


def _plain_rotary(state):
    c = state["case"]
    cs = state["table"][state["positions"].long()]
    return [_rotate(x.float(), cs[..., 0], cs[..., 1], c["part"], c["layout"]).to(x.dtype)
            for x in (state["q"], state["k"])]


def _plain_append(state):
    c = state["case"]
    cs = state["table"][_where(state)[2]]
    q, k = (_rotate(x.float(), cs[..., 0], cs[..., 1], c["part"], c["layout"]) for x in (state["q"], state["k"]))
    return [q.to(state["q"].dtype), _rounded_to_cache(k), _rounded_to_cache(state["v"].float())]


def _plain_attend(state):
    c, q, cache = state["case"], state["q"], state["cache"]
    B, H, D, L = c["batch"], c["kv_heads"], c["dim"], state["block_table"].shape[1] * c["page"]
    pages = state["block_table"].clamp(min=0).long()
    k = _values(_nibbles(cache["k_codes"][pages]), cache["k_scales"][pages])  # [B, pages, H, P, D]
    vw = cache["v_codes"][pages].transpose(-1, -2)
    v = _values(_nibbles(vw), cache["v_scales"][pages].transpose(-1, -2)).flatten(3, 4)
    k, v = (x.transpose(1, 2).reshape(B, H, L, D) for x in (k, v))
    seq, m, at = _where(state)
    M, group = c["tokens"], c["heads"] // H
    rows = torch.zeros(B, M, c["heads"], D, device="cuda").index_put_((seq, m), q.float())
    place = torch.full((B, M), -1, device="cuda").index_put_((seq, m), at)
    rows = rows.reshape(B, M, H, group, D).permute(0, 2, 3, 1, 4).reshape(B, H, group * M, D)
    t = torch.arange(L, device="cuda")
    seen = (t < state["lengths"][:, None])[:, None] & (place >= 0)[..., None]  # [B, M, L]
    if c["causal"]:
        seen = seen & (t <= place[..., None])
    if c["window"]:
        seen = seen & (t > place[..., None] - c["window"])
    seen = seen[:, None, None].expand(B, 1, group, M, L).reshape(B, 1, group * M, L)
    v = torch.where((t < state["lengths"][:, None])[:, None, :, None], v, 0.0)
    s = torch.matmul(rows, k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    o = o.reshape(B, H, group, M, D).permute(0, 3, 1, 2, 4).reshape(B, M, c["heads"], D)[seq, m].to(q.dtype)
    if not c["lse"]:
        return o
    lse = (top + total.log()).reshape(B, H, group, M).permute(0, 3, 1, 2).reshape(B, M, c["heads"])
    return [o, lse[seq, m]]


PLAIN = {"rotary": _plain_rotary, "append": _plain_append, "attend": _plain_attend}


# -------------------------------------------------------------------- cases --


@torch.no_grad()
def run(state):
    if not own:
        return PLAIN[state["kind"]](state)
    from drinkme_amd import kv_ops

    c = state["case"]
    if c["kind"] == "rotary":
        return list(kv_ops.rotary(state["q"], state["k"], state["positions"], state["table"], layout=c["layout"]))
    cache, table, lengths, cu = state["cache"], state["block_table"], state["lengths"], state["cu"]
    if c["kind"] == "append":
        q = kv_ops.append(cache, state["k"], state["v"], table, lengths, cu=cu, table=state["table"],
                          layout=c["layout"], q=state["q"])
        return [q, *kv_ops.read(cache, table, lengths, state["q"].shape[0], cu=cu)]
    return kv_ops.attention(state["q"], cache, table, lengths, cu=cu, max_tokens=c["tokens"] if cu is not None else None,
                            causal=c["causal"], window=c["window"] or None, return_lse=c["lse"])


def work(case):
    size, D, H, Hq = DTYPES[case["x"]].itemsize, case["dim"], case["kv_heads"], case["heads"]
    if case["kind"] == "rotary":
        T = case["t"]
        return {"bytes": 2 * T * (Hq + H) * D * size + T * (4 * case["part"] + 4), "flops": 3 * T * (Hq + H) * case["part"]}
    sizes = _sizes(case)
    T = sum(n for n, _ in sizes)
    coded = 2 * H * D * 17 / 32  # of one token, keys and values
    if case["kind"] == "append":
        values = 2 * Hq * D * size + 2 * H * D * size
        return {"bytes": T * (values + 4 * case["part"] + 2 * coded + 2 * H * D * 2), "flops": 3 * T * (Hq + H) * case["part"]}
    tokens = pairs = 0
    for n, length in sizes:
        first = length - n
        spans = []
        for m in range(n):
            hi = first + m + 1 if case["causal"] else length
            lo = max(0, first + m + 1 - case["window"]) if case["window"] else 0
            spans.append((lo, hi))
        pairs += sum(hi - lo for lo, hi in spans)
        tokens += max((hi for _, hi in spans), default=0) - min((lo for lo, _ in spans), default=0)
    return {"bytes": tokens * coded + T * Hq * (2 * D * size + (4 if case["lse"] else 0)), "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------ in 64 bits --


def _exact_turn(x, positions, case, scaling):
    """x [T, H, D] turned, channel by channel: a complex number times
    exp(i * position * frequency)."""
    part = case["part"]
    angle = positions.double()[:, None] * _frequencies(part, scaling)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    x = x.double()
    pairs = x[..., :part].unflatten(-1, (2, part // 2)).transpose(-1, -2) if case["layout"] == "half" else \
        x[..., :part].unflatten(-1, (part // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    z = z.transpose(-1, -2) if case["layout"] == "half" else z
    return torch.cat([z.flatten(-2), x[..., part:]], -1)


def _exact_cached(x):
    """The values that the cache holds of x (64 bits): per 32 channels, the
    grid times the power of two, by the grid's midpoints."""
    y = x.unflatten(-1, (-1, 32))
    top = y.abs().amax(-1, keepdim=True)
    m, x = torch.frexp(top)  # top = m 2^x, m in [1/2, 1): the smallest e with top < 7 2^e
    e = torch.where(top > 0, x - 3 + (m >= 0.875), -125).clamp(-125, 125)
    unit = ((e.long() + 1023) << 52).view(torch.float64)
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    mids = (grid[1:] + grid[:-1]) / 2
    a = (y / unit).abs()
    up = torch.searchsorted(mids, a.contiguous(), right=True)
    down = torch.searchsorted(mids, a.contiguous(), right=False)
    code = torch.where(up == down, up, up - up % 2)  # a tie: the even one of the two
    return (grid[code] * unit * torch.sign(y)).flatten(-2)


def _exact_rows(case, state):
    """(sequence, position) of every new token, in order."""
    out = []
    for b, (n, length) in enumerate(_sizes(case)):
        out += [(b, length - n + m) for m in range(n)]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "rotary":
        return [_exact_turn(state[x], state["positions"], case, case["scaling"]) for x in ("q", "k")]
    if case["kind"] == "append":
        at = torch.tensor([p for _, p in _exact_rows(case, state)], device="cuda")
        q, k = (_exact_turn(state[x], at, case, "none") for x in ("q", "k"))
        return [q, _exact_cached(k), _exact_cached(state["v"].double())]
    H, D, P, group = case["kv_heads"], case["dim"], case["page"], case["heads"] // case["kv_heads"]
    cache, grid = state["cache"], torch.tensor(GRID, dtype=torch.float64, device="cuda")
    shifts = 4 * torch.arange(8, device="cuda")
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(state["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")

    def values(words, e):  # words [n, D/8], e [n, D/32]
        code = ((words.long()[..., None] >> shifts) & 15).flatten(1)
        v = grid[code & 7] * torch.where(code > 7, -1.0, 1.0)
        return v * torch.exp2(e.double() - 127).repeat_interleave(32, 1)

    t0 = 0
    for b, (n, length) in enumerate(_sizes(case)):
        if n:
            t = torch.arange(length, device="cuda")
            page, slot = state["block_table"][b].long()[t // P], t % P
            at = torch.arange(length - n, length, device="cuda")[:, None]
            seen = (t <= at) if case["causal"] else torch.ones(n, length, dtype=torch.bool, device="cuda")
            if case["window"]:
                seen = seen & (at - t < case["window"])
            for h in range(H):
                k = values(cache["k_codes"][page, h, slot], cache["k_scales"][page, h, slot])
                v = values(cache["v_codes"][page, h, slot // 8, :, slot % 8],
                           cache["v_scales"][page, h, slot // 8, :, slot % 8])
                for g in range(h * group, (h + 1) * group):
                    s = state["q"][t0:t0 + n, g].double() @ k.t() / math.sqrt(D)
                    s = torch.where(seen, s, -math.inf)
                    lse[t0:t0 + n, g] = torch.logsumexp(s, -1)
                    out[t0:t0 + n, g] = torch.softmax(s, -1) @ v
        t0 += n
    return [out, lse] if case["lse"] else out
