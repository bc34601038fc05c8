"""The attention of a decoder block over packed weights and a 4-bit cache, as a
serving loop calls it: three prompts of different lengths at once, then single
tokens, then the verify rows of speculative decoding.

    python examples/attention_block.py [--steps N]

q and o are radix-packed Linears, k and v raw ones (fewer than 1024 rows), all
of synthetic weights. Each pass hands out the pages that its tokens need, norms the heads of q and
k, appends to the cache (keys rotated on the way), attends to it, and adds its output to the residual
stream in front of the next block's norm; at the end the keys and values are read back from the cache
and the last pass is compared with a plain attention over them in fp32."""

from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch

from drinkme_amd import kv_ops, norm_ops, radix_pack, swap, synth

HIDDEN, HEADS, KV_HEADS, DIM = 2048, 16, 4, 128
PAGE = 64


class AttentionBlock(torch.nn.Module):
    """q, k, v, their norms, rotary positions, cache, attention, o, residual and norm.
    `pages` are the cache's, in all; a sequence takes a free one when it outgrows its own."""

    def __init__(self, sequences: int, pages: int, positions: int):
        super().__init__()
        for name, rows, cols in (("q_proj", HEADS * DIM, HIDDEN), ("k_proj", KV_HEADS * DIM, HIDDEN),
                                 ("v_proj", KV_HEADS * DIM, HIDDEN), ("o_proj", HIDDEN, HEADS * DIM)):
            bits = synth.weight("attention-block", 0, name, rows, cols)
            if rows >= 1024:
                module = swap.make_module(radix_pack.pack_weight_radix(bits, "sip"))
            else:
                module = torch.nn.Linear(cols, rows, bias=False, device="meta")
                weight = swap.to_device_raw({"R": rows, "C": cols, "raw_bits": bits})["weight"]
                module.weight = torch.nn.Parameter(weight, requires_grad=False)
            self.add_module(name, module)
        swap.install_narrow(self, "cuda")
        self.table = kv_ops.rotary_table(positions, DIM, scaling={"kind": "wavelength", "factor": 8.0, "original": 8192})
        self.cache = kv_ops.new_cache(pages, PAGE, KV_HEADS, DIM)
        self.block_table = torch.full((sequences, -(-positions // PAGE)), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")
        self.pool = kv_ops.new_pool(pages)
        self.held = [0] * sequences  # tokens, as the host counts them
        ones = lambda n: torch.ones(n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.q_norm, self.k_norm, self.next_norm = ones(DIM), ones(DIM), ones(HIDDEN)

    @torch.no_grad()
    def forward(self, x, residual, counts):
        """x [T, HIDDEN], the new tokens of the sequences one after the other,
        counts[b] of them each, and the residual stream [T, HIDDEN] -> both for the next block."""
        new = torch.tensor(counts, dtype=torch.int32, device="cuda")
        cu, _, _ = kv_ops.reserve(self.pool, self.block_table, self.lengths, PAGE, sum(counts), new=new)
        self.held = [held + n for held, n in zip(self.held, counts)]
        even = len(set(counts)) == 1
        cu = None if even else cu
        q = norm_ops.norm(self.q_proj(x).view(-1, HEADS, DIM), self.q_norm)
        k, v = (proj(x).view(-1, KV_HEADS, DIM) for proj in (self.k_proj, self.v_proj))
        k = norm_ops.norm(k, self.k_norm)
        q = kv_ops.append(self.cache, k, v, self.block_table, self.lengths, cu=cu, table=self.table, q=q)
        out = kv_ops.attention(q, self.cache, self.block_table, self.lengths, cu=cu,
                               max_tokens=None if even else max(counts), max_length=max(self.held))
        self.last = q, out  # (for the comparison below)
        residual, x = norm_ops.block_norm(self.o_proj(out.view(-1, HEADS * DIM)), residual, self.next_norm)
        return x, residual


def plain(block, counts):
    """The last pass's attention from the cache read back, fp32."""
    q = block.last[0].float()
    cu = torch.tensor([sum(block.held[:b]) for b in range(len(counts) + 1)], dtype=torch.int32, device="cuda")
    keys, values = (x.float() for x in kv_ops.read(block.cache, block.block_table, block.lengths, sum(block.held), cu=cu))
    out, t, s = [], 0, 0
    for n, length in zip(counts, block.held):
        k, v = (x[s:s + length].repeat_interleave(HEADS // KV_HEADS, 1).transpose(0, 1).contiguous() for x in (keys, values))
        scores = q[t:t + n].transpose(0, 1).contiguous() @ k.transpose(1, 2).contiguous() * DIM ** -0.5
        later = torch.arange(length, device="cuda") > torch.arange(length - n, length, device="cuda")[:, None]
        out.append((scores.masked_fill(later, float("-inf")).softmax(-1) @ v).transpose(0, 1))
        t, s = t + n, s + length
    return torch.cat(out)


def main(steps: int) -> float:
    prompts = [200, 33, 1]
    block = AttentionBlock(len(prompts), pages=32, positions=1024)
    x = lambda n: torch.randn(n, HIDDEN, device="cuda").to(torch.bfloat16)  # noqa: E731
    torch.manual_seed(0)
    worst = 0.0
    for name, counts, times in (("prompts", prompts, 1), ("tokens", [1, 1, 1], steps), ("verify", [4, 4, 4], 1)):
        for _ in range(times):
            y, _ = block(x(sum(counts)), x(sum(counts)), counts)
        want = plain(block, counts)
        off = ((block.last[1].float() - want).norm() / want.norm()).item()
        worst = max(worst, off)
        print(f"{name}: {tuple(y.shape)}, {block.held} tokens held, attention {off:.2e} from plain fp32", flush=True)
    raw = sum(block.held) * KV_HEADS * DIM * 2 * 2
    print(f"cache: {kv_ops.cache_bytes(block.cache)} bytes for {32 * PAGE} tokens; {raw} bytes in bf16 for the "
          f"{sum(block.held)} held, {raw * 17 // 64} here")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--steps", type=int, default=70)
    main(ap.parse_args().steps)
