"""The paged-cache operators together: steps of serving, eagerly and as
replayed graphs, against the oracle.

Every step's plan is compared with the oracle's, the cache rows with the
float64 rotation of the raw keys (bounds of test_gpu_rotary.py), and the
outputs with float64 attention over the caches as they are (bounds of
tree_util.py)."""

import numpy as np
import pytest

import flashlite_amd as fl
from flashlite_amd import kernel_driver
from oracle import paged
from test_gpu_cache_plan import i32
from test_gpu_rotary import assert_rotated
from tree_util import check

pytestmark = pytest.mark.gpu


class Server:
    """Requests over one layer's paged cache: the device state, and beside it
    the oracle's plan and the raw keys and values of every stored token."""

    def __init__(self, dev, seed, dtype, b, h, hk, d, block, most, pool):
        import torch

        self.rs = np.random.RandomState(seed)
        self.dev, self.dtype, self.t = dev, dtype, getattr(torch, dtype)
        self.b, self.h, self.hk, self.d, self.block = b, h, hk, d, block
        self.host = [np.full((b, most), -1).tolist(), [0] * b, self.rs.permutation(pool).tolist(),
                     [int(self.rs.randint(pool)), pool]]
        self.tables, self.held, self.ring, self.state = (i32(x, dev) for x in self.host)
        self.lengths = torch.zeros(b, dtype=torch.int32, device=dev)
        self.k_cache, self.v_cache = (
            torch.full((pool, block, hk, d), float("nan"), dtype=self.t, device=dev).transpose(1, 2)
            for _ in range(2))
        self.freqs, self.scale = fl.rotary_frequencies(d, device=dev)
        self.raw = [{} for _ in range(b)]  # place in the request -> (k, v, position)

    def tensors(self, n):
        """Projections as a layer leaves them: [B, n, (H + 2 H_k) D] slices."""
        import torch

        x = torch.from_numpy(self.rs.standard_normal(
            (self.b, n, self.h + 2 * self.hk, self.d)).astype(np.float32)).to(self.dev, self.t)
        x = x.transpose(1, 2)
        return x[:, :self.h], x[:, self.h:self.h + self.hk], x[:, self.h + self.hk:]

    def step(self, counts, n, parents=None, check_all=True):
        """Plans, stores and attends n new tokens of each request (counts of
        them there); returns the outputs."""
        before = self.lengths.tolist()
        q, k, v = self.tensors(n)
        there = i32(counts, self.dev)
        positions, slots, info = fl.plan_cache(self.lengths, there, self.tables, self.held,
                                               self.ring, self.state, self.block, n)
        *self.host, want_pos, want_slots, want_info = paged.plan_cache(
            before, counts, *self.host, self.block, n)
        self.host = list(self.host)
        for got, want in zip((self.tables, self.held, self.ring, self.state, positions, slots, info),
                             self.host + [want_pos, want_slots, want_info]):
            assert got.tolist() == want
        mask = seen = None
        if parents is not None:
            mask, positions = fl.plan_tree(i32(parents, self.dev), self.lengths, there)
            seen, want_pos = paged.plan_tree(parents, before, counts)
            assert positions.tolist() == want_pos
        turned = fl.rotary_to_cache(q, k, v, positions, slots, self.freqs, self.k_cache,
                                    self.v_cache, scale=self.scale)
        out, lse = fl.forward_tree(turned, self.k_cache, self.v_cache, self.tables, self.lengths,
                                   mask, there, return_lse=True)
        kk, vv = k.double().cpu().numpy(), v.double().cpu().numpy()
        for b in range(self.b):
            for i in range(min(max(counts[b], 0), n)):
                if want_slots[b][i] >= 0:
                    self.raw[b][before[b] + i] = (kk[b, :, i], vv[b, :, i], want_pos[b][i])
        if check_all:
            self.check_cache()
            self.check_out(turned, out, lse, before, counts, seen, n)
        return out

    def check_cache(self):
        """Every stored row is the rotation of its raw key, or its raw value."""
        import torch

        for b in range(self.b):
            if not self.raw[b]:
                continue
            at = np.array(sorted(self.raw[b]))
            ids = torch.from_numpy(np.asarray(self.host[0][b])[at // self.block]).to(self.dev)
            rows = torch.from_numpy(at % self.block).to(self.dev)
            k = np.stack([self.raw[b][t][0] for t in at], 1)[None]
            v = np.stack([self.raw[b][t][1] for t in at], 1)
            pos = np.array([self.raw[b][t][2] for t in at])[None]
            got = self.k_cache[ids, :, rows].transpose(0, 1)[None]
            freqs = self.freqs.cpu().numpy()
            want = paged.rotary(k, pos, freqs, scale=self.scale)
            assert_rotated(got, k, want, self.dtype, len(freqs), False, self.scale)
            got = self.v_cache[ids, :, rows].transpose(0, 1)
            assert np.array_equal(got.double().cpu().numpy(), v)

    def check_out(self, turned, out, lse, before, counts, seen, n):
        class View:  # what tree_util.check asks of a problem
            pass

        p = View()
        p.counts, p.n, p.d, p.dtype = np.asarray(counts), n, self.d, self.dtype
        p.lengths = np.asarray(before)
        as64 = lambda x: x.double().cpu().numpy()  # noqa: E731
        ref = paged.tree_attention(as64(turned), as64(self.k_cache), as64(self.v_cache),
                                   np.asarray(self.host[0]), p.lengths, seen, p.counts)
        check(out, lse, p, ref)

    def keep(self, accepted):
        """The first accepted[b] of the step's tokens stay."""
        self.lengths += i32(accepted, self.dev)
        for b, n in enumerate(self.lengths.tolist()):
            self.raw[b] = {t: x for t, x in self.raw[b].items() if t < n}

    def end(self, gone):
        """The requests in `gone` give their blocks back."""
        self.step([-1 if b in gone else 0 for b in range(self.b)], 1, check_all=False)
        for b in gone:
            self.raw[b] = {}
        self.lengths *= i32([b not in gone for b in range(self.b)], self.dev)


@pytest.mark.parametrize("dtype,d,h,hk,block", [
    ("float16", 64, 4, 2, 16), ("bfloat16", 64, 3, 1, 20), ("float16", 128, 2, 2, 16),
    ("bfloat16", 128, 8, 2, 64)])
def test_prompts_drafts_and_ends(cuda, dtype, d, h, hk, block):
    """Prompts in chunks, decode steps, verified drafts of which some stay,
    requests that end and whose blocks others take."""
    rs = np.random.RandomState(d + h)
    b, most = 4, -(-260 // block)
    s = Server(cuda, 7, dtype, b, h, hk, d, block, most, b * most)
    for n, counts in ((70, [70, 3, 0, 41]), (70, [11, 0, 70, 1])):  # prompts
        s.step(counts, n)
        s.keep(counts)
    for _ in range(3):  # a token a step
        s.step([1, 1, 1, 0], 1)
        s.keep([1, 1, 1, 0])
    for n in (7, 20):  # drafts: a chain of the first ones, and branches
        stay = rs.randint(0, 5, b)
        parents = [[i - 1 if i < stay[r] else int(rs.randint(-1, i)) for i in range(n)]
                   for r in range(b)]
        s.step([n, n - 2, 5, n], n, parents)
        s.keep(np.minimum(stay, [n, n - 2, 5, n]).tolist())
    s.end([1, 2])
    s.step([0, 90, 50, 6], 90)
    s.keep([0, 90, 50, 6])
    s.step([1] * b, 1)


def test_steps_equal_attention_over_the_whole_sequence(cuda):
    """Prompt, chunk and decode steps give what forward_flash2_ex gives over the
    rotated sequence at once."""
    import torch

    b, h, d, total = 2, 4, 64, 150
    s = Server(cuda, 9, "float16", b, h, h, d, 16, 10, 25)
    outs, qs, ks, vs = [], [], [], []
    draw = s.tensors
    s.tensors = lambda n: [y.append(x) or x for x, y in zip(draw(n), (qs, ks, vs))]
    for n in (97, 40, 1, 1, 11):
        outs.append(s.step([n] * b, n, check_all=False))
        s.keep([n] * b)
    q, k, v = (torch.cat(x, 2).contiguous() for x in (qs, ks, vs))
    positions = torch.arange(total, dtype=torch.int32, device=cuda)[None].expand(b, total)
    q, k = fl.forward_rotary(q, k, positions, s.freqs)
    want = fl.forward_flash2_ex(q, k, v, is_causal=True)
    assert float((torch.cat(outs, 2).float() - want.float()).abs().max()) <= 2e-3


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("n,h,hk,d,dtype", [(1, 8, 2, 128, "bfloat16"), (12, 4, 2, 64, "float16"),
                                            (40, 4, 1, 128, "float16")])
def test_captured_steps(cuda, n, h, hk, d, dtype, long):
    """Two captured steps, each with what it allocates, replayed in turn with
    eager calls between: every replay equals the eager step on the same state.
    `long`: tables with room for many more tokens, which split the keys."""
    import torch

    b, block, most = 5, 16, 4000 if long else 40
    rs = np.random.RandomState(3)

    def state():
        r = np.random.RandomState(5)
        pool = 200
        return dict(tables=i32(np.full((b, most), -1), cuda), held=i32([0] * b, cuda),
                    ring=i32(r.permutation(pool), cuda), state=i32([17, pool], cuda),
                    lengths=i32([0] * b, cuda),
                    k=torch.full((pool, hk, block, d), float("nan"), dtype=getattr(torch, dtype),
                                 device=cuda),
                    v=torch.full((pool, hk, block, d), float("nan"), dtype=getattr(torch, dtype),
                                 device=cuda))

    freqs, _ = fl.rotary_frequencies(d, device=cuda)
    parents = i32(np.floor(rs.rand(b, n) * (np.arange(n) + 1)).astype(int) - 1, cuda)
    q, k, v = (torch.zeros((b, x, n, d), dtype=getattr(torch, dtype), device=cuda)
               for x in (h, hk, hk))
    counts = i32([n] * b, cuda)

    def step(s):
        positions, slots, info = fl.plan_cache(s["lengths"], counts, s["tables"], s["held"],
                                               s["ring"], s["state"], block, n)
        mask, positions = fl.plan_tree(parents, s["lengths"], counts)
        turned = fl.rotary_to_cache(q, k, v, positions, slots, freqs, s["k"], s["v"])
        out, lse = fl.forward_tree(turned, s["k"], s["v"], s["tables"], s["lengths"], mask, counts,
                                   return_lse=True)
        s["lengths"] += counts.clamp(min=0)
        s["lengths"] *= counts >= 0  # an ended request has no tokens
        return out, lse, info

    eager, first, second = state(), state(), state()
    step(state())  # everything is loaded before a capture
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(s))
        graphs.append(g)
    for i in range(5):
        for x in (q, k, v):
            x.copy_(torch.from_numpy(rs.standard_normal(tuple(x.shape)).astype(np.float32)))
        counts.copy_(i32([n, max(n - 3, 0), 0, n, -1 if i == 3 else 1], cuda))
        want = step(eager)
        torch.cuda.synchronize()
        for g, got, s in zip(graphs, outs, (first, second)):
            g.replay()
            junk = torch.randn(1 << 20, device=cuda).sum()  # eager work between the replays
            there = torch.arange(n, device=cuda)[None] < counts[:, None]
            there = there[:, None].expand(b, h, n)
            assert torch.equal(got[0][there], want[0][there])
            assert torch.equal(got[1][there], want[1][there])
            assert torch.equal(got[2], want[2])
            for name in ("tables", "held", "ring", "state", "lengths"):
                assert torch.equal(s[name], eager[name]), name
            assert torch.isfinite(junk)
        assert bool(torch.isfinite(want[0][there]).all())


def test_steps_on_two_streams(cuda):
    """Two servers on streams of their own, at once, each as if alone."""
    import torch

    def run(seed, stream):
        s = Server(cuda, seed, "float16", 3, 4, 2, 64, 16, 300, 200)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            outs = []
            for n in (50, 1, 9, 1):
                outs.append(s.step([n, n // 2, n], n, check_all=False))
                s.lengths += i32([n, n // 2, n], cuda)
        return outs

    main = torch.cuda.current_stream()
    alone = [run(seed, main) for seed in (1, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    both = [run(seed, s) for seed, s in zip((1, 2), streams)]
    torch.cuda.synchronize()
    for a, b in zip(alone, both):
        for i, (x, y) in enumerate(zip(a, b)):
            n = (50, 1, 9, 1)[i]
            assert torch.equal(x[::2], y[::2])
            assert torch.equal(x[1, :, :n // 2], y[1, :, :n // 2])


@pytest.mark.parametrize("args", [
    ["--serve", "3", "4", "2", "100"],
    ["--serve", "2", "8", "2", "65", "--drafts", "9", "--head-dim", "128", "--dtype", "bf16"],
    ["--serve", "1", "4", "4", "20", "--drafts", "40", "--chain", "--block", "32"],
])
def test_the_driver_serves(cuda, capsys, args):
    kernel_driver.main(args + ["--iters", "2"])
    text = capsys.readouterr().out
    tree = "--drafts" in args and "--chain" not in args
    for name in ("plan_cache", "rotary_to_cache", "forward_tree", "us replayed"):
        assert name in text
    assert ("plan_tree" in text) == tree


def test_the_driver_turns(cuda, capsys):
    kernel_driver.main(["--rotary", "2", "4", "2", "100", "--dtype", "bf16", "--iters", "2"])
    text = capsys.readouterr().out
    assert "forward_rotary B2 H4/2 N100" in text and "backward_rotary" in text
