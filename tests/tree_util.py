"""Problems of forward_tree and the bound of its outputs.

The kernel's errors against 64 bits, u half a step of the element type
(2^-11 fp16, 2^-8 bf16):
- scores: D products summed in 32 bits, off by at most (D + 8) 2^-24 sum |q k|
  |scale| (`reach`), and 2^-22 of the exponential itself: delta, relative on p;
- p rounded to the element type before the product with V: u of each p, so u of
  sum p |v| / sum p (`weight`); fp16's smallest steps, 2^-25 a key against a
  largest p of at least 1, add 2^-25 sum |v|;
- 32-bit sums over the keys: (keys + 64) 2^-24 of `weight`;
- the output's own rounding, u of it.
The log-sum-exp is ln of the unrounded sum: delta, the sum's error, and 2^-21
of its size for the logarithm and the stabiliser's product.
"""

import numpy as np

from oracle import paged

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


class Problem:
    """Seeded q, a paged cache in random block order (blocks of nobody hold
    NaN), lengths, drafts and masks."""

    def __init__(self, seed, dtype, b, h, hk, n, d, block, lengths, tree=None, ragged=False,
                 rows_first=True, scale=0.0, q_scale=1.0, table_pad=0):
        import torch

        rs = self.rs = np.random.RandomState(seed)
        self.dtype, self.d, self.n, self.scale = dtype, d, n, scale
        t = getattr(torch, dtype)
        self.lengths = np.asarray(lengths, dtype=np.int64)
        need = -(-(self.lengths + n) // block)
        m = max(1, int(need.max())) + table_pad
        blocks = int(need.sum()) + 3
        ids = rs.permutation(blocks)
        self.tables = np.full((b, m), -1, dtype=np.int64)
        at = 0
        for i in range(b):
            self.tables[i, :need[i]] = ids[at:at + need[i]]
            at += need[i]
        shape = (blocks, block, hk, d) if rows_first else (blocks, hk, block, d)
        caches = []
        for _ in range(2):
            c = torch.from_numpy(rs.standard_normal(shape).astype(np.float32)).to(t)
            c = c.transpose(1, 2) if rows_first else c
            c[torch.from_numpy(ids[at:].copy())] = float("nan")
            caches.append(c)
        self.k, self.v = caches
        q = torch.from_numpy((rs.standard_normal((b, n, h, d)) * q_scale).astype(np.float32)).to(t)
        self.q = q.transpose(1, 2)
        self.counts = rs.randint(0, n + 1, b) if ragged else None
        self.seen = None
        if tree == "tree":
            parents = np.floor(rs.rand(b, n) * (np.arange(n) + 1)).astype(int) - 1
            self.seen = paged.plan_tree(parents.tolist(), self.lengths, None)[0]
        elif tree == "any":  # arbitrary bits, rows that see no draft among them
            self.seen = [[set(np.flatnonzero(rs.rand(n) < p).tolist())
                          for p in rs.choice([0.0, 0.1, 0.5, 1.0], n)] for _ in range(b)]

    def mask(self):
        if self.seen is None:
            return None
        return np.stack([paged.words(s, self.n) for s in self.seen])

    def reference(self):
        as64 = lambda x: x.double().numpy()  # noqa: E731
        return paged.tree_attention(as64(self.q), as64(self.k), as64(self.v), self.tables,
                                    self.lengths, self.seen, self.counts, self.scale)

    def device(self, dev):
        """Arguments of forward_tree on `dev`."""
        import torch

        def i32(x):
            return None if x is None else torch.tensor(x, dtype=torch.int32, device=dev)

        m = self.mask()
        return dict(q=self.q.to(dev), k_cache=self.k.to(dev), v_cache=self.v.to(dev),
                    block_tables=i32(self.tables), lengths=i32(self.lengths),
                    mask=None if m is None else torch.from_numpy(m).to(dev),
                    counts=i32(self.counts), sm_scale=self.scale)


def check(got, got_lse, problem, ref=None):
    """`got` and `got_lse` (or None) within the bound; NaN where the oracle has
    NaN; rows of drafts that are not there are not compared."""
    out, lse, weight, reach = problem.reference() if ref is None else ref
    there = np.ones(out.shape[:3], bool)
    if problem.counts is not None:
        there &= (np.arange(problem.n) < problem.counts[:, None])[:, None]
    got = got.double().cpu().numpy()
    x, want = got[there], out[there]
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(x), np.isnan(want)), "NaN pattern"
    assert np.array_equal(x[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    u = HALF_STEP[problem.dtype]
    keys = int(problem.lengths.max()) + problem.n
    delta = ((problem.d + 8) * 2.0 ** -24 * reach[there] + 2.0 ** -22)[:, None]
    sums = (keys + 64) * 2.0 ** -24
    with np.errstate(invalid="ignore"):
        bound = (u * np.abs(want) + (u + 2 * delta + sums) * weight[there]
                 + 2.0 ** -25 * keys * 4.0 * (problem.dtype == "float16") + 2.0 ** -25)
        err = np.abs(x - want)
        worst = (err[finite] / bound[finite]).max() if finite.any() else 0.0
    assert worst <= 1.0, f"out: {worst:.3g} of the bound"
    if got_lse is not None:
        y, want = got_lse.double().cpu().numpy()[there], lse[there]
        assert np.array_equal(np.isnan(y), np.isnan(want)), "NaN pattern of the log-sum-exp"
        same = np.isneginf(want)
        assert np.array_equal(np.isneginf(y), same)
        fin = np.isfinite(want)
        bound = (delta[:, 0] + sums + 2.0 ** -21 * (np.abs(want) + reach[there] + 1))[fin]
        assert (np.abs(y[fin] - want[fin]) <= bound).all(), "log-sum-exp"
