"""MI355X: the operators of a decoder's step run together, as a server runs
them: pages reserved, heads normed, turned by three axes, appended, summarized,
selected, attended to, added to the residual; prompts, single tokens, verify
rows whose drafts are dropped, requests that end; also from a captured graph, from another
thread's stream, and without the native calls."""

import numpy as np
import pytest
import torch

from drinkme_amd import _native, kv_ops, norm_ops
from tests import blocks_reference as B
from tests import kv_reference as R
from tests.test_gpu_kv import DT, f64, heads, i32

pytestmark = pytest.mark.gpu

H, HQ, D, PAGE, COUNT, WIDTH = 2, 6, 64, 8, 7, 256


class Server:
    """State on the GPU, and the same as the definitions have it."""

    def __init__(self, rng, batch, cols, pages):
        self.rng, self.batch = rng, batch
        self.cache = kv_ops.new_cache(pages, PAGE, H, D)
        self.sums, self.pool = kv_ops.new_summaries(self.cache), kv_ops.new_pool(pages)
        self.table = torch.full((batch, cols), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")
        self.axes = kv_ops.rotary_axes((12, 10, 10), "interleaved")
        self.angles = kv_ops.rotary_table(4 * cols * PAGE, D)
        self.q_norm, self.k_norm, self.norm, self.post = (1 + 0.1 * heads(rng, (1, 1, n), "bf16")[0, 0] for n in (D, D, WIDTH, WIDTH))
        self.gate = heads(rng, (1, batch, WIDTH), "bf16")[0]
        self.free, self.count = self.pool["free"].tolist(), pages
        self.held_table, self.held_lengths = self.table.tolist(), [0] * batch
        self.keys = [np.zeros((0, H, D)) for _ in range(batch)]
        self.values = [np.zeros((0, H, D)) for _ in range(batch)]

    def inputs(self, total):
        fused = heads(self.rng, (total, HQ + 2 * H, D), "bf16")
        y, residual = heads(self.rng, (1, total, WIDTH), "bf16")[0], heads(self.rng, (1, total, WIDTH), "f32")[0]
        return fused, y, residual

    def run(self, fused, y, residual, new, most):
        total = fused.shape[0]
        cu, positions, slots = kv_ops.reserve(self.pool, self.table, self.lengths, PAGE, total, new=new)
        seqs = {"cu": cu} if new is not None else {}
        q = norm_ops.norm(fused[:, :HQ], self.q_norm)
        k = norm_ops.norm(fused[:, HQ:HQ + H], self.k_norm)
        at = torch.stack([positions, 2 * positions, 3 * positions + 1])  # (any grid's)
        q2, k2 = kv_ops.rotary(q, k, at, self.angles, axes=self.axes)
        kv_ops.append(self.cache, k2, fused[:, HQ + H:], self.table, self.lengths, **seqs)
        kv_ops.summarize(self.cache, self.sums, self.table, self.lengths, total, **seqs)
        blocks = kv_ops.select(q2, self.cache, self.sums, self.table, self.lengths, COUNT, first=1, last=2, **seqs)
        more = {"max_tokens": most} if new is not None else {}
        out, lse = kv_ops.attention(q2, self.cache, self.table, self.lengths, blocks=blocks, return_lse=True, **seqs, **more)
        kw = {"cu": cu} if new is not None else {}
        stream, x = norm_ops.block_norm(y, residual, self.norm, post=self.post, gate=self.gate, **kw)
        return {"cu": cu, "positions": positions, "slots": slots, "q": q, "k": k, "at": at, "q2": q2, "k2": k2, "blocks": blocks, "out": out,
                "lse": lse, "stream": stream, "x": x}

    def check(self, got, fused, counts):
        """Every result of a pass against its definition on the pass's own inputs."""
        total = fused.shape[0]
        cu, positions, slots, self.count, _ = B.reserve(self.free, self.count, self.held_table, self.held_lengths, counts, PAGE, total,
                                                        len(self.free))
        assert (got["cu"].tolist(), got["positions"].tolist(), got["slots"].tolist()) == (cu, positions, slots)
        assert self.table.tolist() == self.held_table and self.lengths.tolist() == self.held_lengths
        live = cu[-1]
        for name, x, w in (("q", fused[:, :HQ], self.q_norm), ("k", fused[:, HQ:HQ + H], self.k_norm)):
            want = B.standard(f64(x), "rms", 1e-6) * f64(w)
            assert (np.abs(f64(got[name]) - want) <= (2.0 ** -8 + 2.0 ** -17) * np.abs(want) + 1e-30).all()
            turned = B.rotate_axes(f64(got[name]), got["at"].cpu().numpy(), self.axes, f64(self.angles), "half", np.float32)
            have = torch.from_numpy(turned).to(torch.bfloat16)
            assert torch.equal(got[name + "2"].cpu().nan_to_num(nan=9.0), have.nan_to_num(nan=9.0))
        k, v = R.cached(f64(got["k2"][:live])), R.cached(f64(fused[:live, HQ + H:]))
        bounds, scales = self.sums["bounds"].cpu().numpy(), self.sums["scales"].cpu().numpy()
        q, out, lse, blocks = (x.cpu() for x in (got["q2"], got["out"], got["lse"], got["blocks"]))
        for b, n in enumerate(counts):
            rows = slice(cu[b], cu[b + 1])
            self.keys[b], self.values[b] = np.concatenate([self.keys[b], k[rows]]), np.concatenate([self.values[b], v[rows]])
            length = self.held_lengths[b]
            assert len(self.keys[b]) == length
            for col in range(-(-length // PAGE)):
                page = self.held_table[b][col]
                for h in range(H):
                    want, e = B.summary(self.keys[b][col * PAGE:(col + 1) * PAGE, h])
                    assert (bounds[page, h] == want).all() and scales[page, h] == e
            for m in range(n):
                cols = (length - n + m) // PAGE + 1
                for h in range(H):
                    mine = f64(q[cu[b] + m, h * HQ // H:(h + 1) * HQ // H])
                    want = B.select(mine, bounds[:, h], scales[:, h], self.held_table[b], cols, COUNT, 1, 2)
                    assert blocks[cu[b] + m, h].tolist() == want
            if n:
                want, l, spread, reach = B.listed_attention(f64(q[rows]), self.keys[b], self.values[b], length - n, D ** -0.5,
                                                            blocks[rows].numpy(), PAGE)
                assert (np.abs(f64(out[rows]) - want) <= R.bound(want, spread, reach, length, D, True)).all()
                assert (np.abs(f64(lse[rows]) - l) <= R.lse_bound(l, reach, length, D)).all()
        assert out[live:].isnan().all() and (blocks[live:] == -1).all()
        assert got["stream"].isfinite().all() and got["x"].isfinite().all()

    def trim(self, keep):
        kv_ops.trim(self.pool, self.table, self.lengths, PAGE, i32(keep))
        self.count = B.trim(self.free, self.count, self.held_table, self.held_lengths, keep, PAGE)
        self.keys = [k[:n] for k, n in zip(self.keys, self.held_lengths)]
        self.values = [v[:n] for v, n in zip(self.values, self.held_lengths)]
        assert self.table.tolist() == self.held_table and self.lengths.tolist() == self.held_lengths
        assert self.pool["free"].tolist() == self.free and self.pool["count"].item() == self.count

    def step(self, counts, pad=0):
        total = sum(counts) + pad
        even = len(set(counts)) == 1 and not pad
        fused, y, residual = self.inputs(total)
        self.check(self.run(fused, y, residual, None if even else i32(counts), max(counts)), fused, counts)


@pytest.mark.parametrize("native", [True, False])
def test_a_server_s_life(native, monkeypatch):
    if not native:
        monkeypatch.setattr(_native, "_calls", None)
    s = Server(np.random.default_rng(1 + native), batch=4, cols=30, pages=70)
    s.step([90, 0, 33, 1])           # prompts, one request waiting
    s.step([1, 121, 1, 0], pad=5)    # one of them arrives beside single tokens, in a padded batch
    for _ in range(3):
        s.step([1, 1, 1, 1])
    s.step([4, 4, 4, 4])             # verify rows
    s.trim([n - d for n, d in zip(s.held_lengths, (3, 0, 1, 2))])  # of which drafts are dropped
    s.step([2, 1, 3, 1])
    s.trim([s.held_lengths[0], 0, s.held_lengths[2], 0])           # two requests end
    s.step([1, 60, 1, 8])            # others take their pages
    s.step([1, 1, 1, 1])


def test_a_captured_step():
    """Single tokens from a graph: reserve moves the lengths on, and each replay is the next step."""
    s = Server(np.random.default_rng(3), batch=3, cols=30, pages=80)
    s.step([70, 41, 8])
    fused, y, residual = s.inputs(3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        s.check(s.run(fused, y, residual, None, 1), fused, [1, 1, 1])
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = s.run(fused, y, residual, None, 1)
    for _ in range(12):
        for x, z in zip((fused, y, residual), s.inputs(3)):
            x.copy_(z)
        graph.replay()
        torch.cuda.synchronize()
        s.check(got, fused, [1, 1, 1])
        torch.empty(1 << 20, device="cuda").normal_().sum().item()


def test_an_empty_pool():
    """Tokens that get no page are counted, read NaN and give NaN to who lists them; the rest is as ever."""
    s = Server(np.random.default_rng(4), batch=2, cols=6, pages=3)
    fused, y, residual = s.inputs(30)
    got = s.run(fused, y, residual, i32([14, 16]), 16)
    assert s.pool["lacking"].item() == 1 and s.table.tolist() == [[0, 1, -1, -1, -1, -1], [2, -1, -1, -1, -1, -1]]
    assert got["slots"][22:].eq(-1).all() and got["out"][:22].isfinite().all() and got["out"][22:].isnan().all()
    kv_ops.trim(s.pool, s.table, s.lengths, PAGE, i32([0, 8]))
    assert s.pool["count"].item() == 2 and s.table[1].tolist() == [2, -1, -1, -1, -1, -1]


def test_threads_with_a_stream_each():
    import threading

    servers = [Server(np.random.default_rng(5 + i), batch=2, cols=20, pages=50) for i in range(4)]
    errors = []

    def work(s):
        try:
            with torch.no_grad(), torch.cuda.stream(torch.cuda.Stream()):
                for counts in ([50, 9], [1, 1], [3, 3], [1, 2]):
                    s.step(counts)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 (handed to the main thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in servers]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors[0]


def calls_of(rng):
    """Each operator as a call of its floating-point tensor (or of no such tensor)."""
    s = Server(rng, batch=2, cols=12, pages=30)
    s.step([40, 25])
    q = heads(rng, (2, HQ, D), "bf16")
    blocks = i32(rng.integers(0, 5, (2, H, 3)))
    y = heads(rng, (1, 2, WIDTH), "bf16")[0]
    return s, q, {
        "rotary": lambda q: kv_ops.rotary(q, None, i32([[0, 1], [2, 3], [4, 5]]), s.angles, axes=s.axes)[0],
        "select": lambda q: kv_ops.select(q, s.cache, s.sums, s.table, s.lengths, 3),
        "attention": lambda q: kv_ops.attention(q, s.cache, s.table, s.lengths, blocks=blocks),
        "norm": lambda q: norm_ops.norm(q, s.q_norm, kind="layer"),
        "block_norm": lambda q: norm_ops.block_norm(q.reshape(2, -1)[:, :WIDTH], y, s.norm, post=s.post, gate=s.gate, factor=0.5)[1]}


def test_modes_subclasses_and_vmap():
    """What the native calls leave to the general path gives the same bits; a batched tensor, which has no address, is refused."""
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

    _, q, calls = calls_of(np.random.default_rng(6))
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


def test_gradients_and_tangents_are_refused(monkeypatch):
    from torch.autograd import forward_ad

    _, q, calls = calls_of(np.random.default_rng(7))
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_native, "_calls", None)
        for name, call in calls.items():
            with pytest.raises(RuntimeError, match="no gradient"):
                call(q.clone().requires_grad_())
            with torch.no_grad():
                assert torch.equal(call(q.clone().requires_grad_()), call(q)), name
            with forward_ad.dual_level(), pytest.raises(RuntimeError, match="no gradient"):
                call(forward_ad.make_dual(q, torch.ones_like(q)))


def test_the_general_path_gives_the_native_calls_results(monkeypatch):
    """Strided tensors, absent arguments and every type, through ctypes and without: the same bits."""
    outs = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(_native, "_calls", None)
        rng = np.random.default_rng(8)
        s, q, calls = calls_of(rng)
        got = [call(q) for call in calls.values()]
        wide = heads(rng, (2, HQ, 2 * D), "f32")[..., :D]
        got += [norm_ops.norm(wide), norm_ops.norm(wide[:, 0], s.q_norm, bias=s.k_norm, kind="layer", offset=1.0)]
        y, r = heads(rng, (1, 6, WIDTH), "bf16")[0], heads(rng, (1, 6, 2 * WIDTH), "f32")[0][:, 5:5 + WIDTH]
        vectors = heads(rng, (3, 3, WIDTH), "f32")
        got += norm_ops.block_norm(y, r, bias=s.norm, gate=vectors[0], modulate=(vectors[1], vectors[2]), cu=i32([0, 1, 5, 6]))
        got += norm_ops.block_norm(y, y, s.norm, modulate=(vectors[1, 0], vectors[2, 0]), kind="layer")
        got += kv_ops.rotary(wide, wide[:, :2], torch.zeros((2, 2), dtype=torch.int64, device="cuda"), kv_ops.rotary_table(9, 32), "interleaved",
                             axes=kv_ops.rotary_axes((9, 7)))
        got.append(kv_ops.select(wide, s.cache, s.sums, s.table, s.lengths, 2, cu=i32([0, 0, 2]), first=0, last=2, causal=False))
        got += kv_ops.attention(wide, s.cache, s.table, s.lengths, cu=i32([0, 0, 2]), max_tokens=2, max_length=90, scale=0.2, causal=False,
                                blocks=got[-1], return_lse=True)
        got += kv_ops.reserve(s.pool, s.table, s.lengths, PAGE, 9, new=i32([3, 4]))
        kv_ops.trim(s.pool, s.table, s.lengths, PAGE, i32([41, 0]))
        kv_ops.summarize(s.cache, s.sums, s.table, s.lengths, 3, cu=i32([0, 2, 3]))
        got += [s.table, s.lengths, *s.pool.values(), *s.sums.values()]
        outs.append([x.clone() for x in got])
    assert len(outs[0]) == len(outs[1])
    assert all(a.dtype == b.dtype and torch.equal(a.nan_to_num(nan=7.0) if a.is_floating_point() else a,
                                                  b.nan_to_num(nan=7.0) if b.is_floating_point() else b) for a, b in zip(*outs))
