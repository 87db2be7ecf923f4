"""Attention whose every sum is exact: q is 0, so each visible key has p = 1, and
V holds whole numbers of at most 8, whose sums 32 bits hold up to 2^21 keys.

An output is then A / n with exact A and n: off by the reciprocal's and the
product's rounding, together at most 2^-21 of it, and half a step of its type.
The log-sum-exp is ln n: off by at most 2^-21 (ln n + 1).  At 40000 keys that is
6e-6, where one key more or less changes it by 2.5e-5: a lost or doubled tile of
any size shows."""

import numpy as np

from oracle import paged

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}
MOST = 8


class Counted:
    """Seeded whole numbers V in a paged cache in random block order."""

    def __init__(self, seed, dtype, b, h, hk, n, d, block, lengths, tree=None, rows_first=True,
                 room=0):
        rs = np.random.RandomState(seed)
        self.dtype, self.h, self.hk, self.n, self.d, self.block = dtype, h, hk, n, d, block
        self.lengths, self.rows_first = np.asarray(lengths), rows_first
        need = -(-(self.lengths + n) // block)
        self.blocks = int(need.sum()) + 1
        ids = rs.permutation(self.blocks)
        self.tables = np.full((b, int(need.max()) + room), -1)
        ends = np.cumsum(need)
        for i in range(b):
            self.tables[i, :need[i]] = ids[ends[i] - need[i]:ends[i]]
        self.v = rs.randint(-MOST, MOST + 1, (self.blocks, hk, block, d))  # [., heads, rows, .]
        self.seen = None
        if tree:
            parents = np.floor(rs.rand(b, n) * (np.arange(n) + 1)).astype(int) - 1
            self.seen = paged.plan_tree(parents.tolist(), self.lengths, None)[0]

    def rows(self, i):
        """Request i's values in order, [hk, length + n, d]."""
        at = np.arange(self.lengths[i] + self.n)
        x = self.v[self.tables[i, at // self.block], :, at % self.block]
        return x.transpose(1, 0, 2)

    def visible(self, i):
        """[n, n]: whether draft j sees draft k."""
        if self.seen is None:
            return np.tri(self.n, dtype=np.int64)
        out = np.zeros((self.n, self.n), dtype=np.int64)
        for j, s in enumerate(self.seen[i]):
            out[j, sorted(s)] = 1
        return out

    def sums(self):
        """Exact (A [b, h, n, d], n [b, n])."""
        b = len(self.lengths)
        a = np.zeros((b, self.h, self.n, self.d), dtype=np.int64)
        keys = np.zeros((b, self.n), dtype=np.int64)
        for i, length in enumerate(self.lengths):
            x, vis = self.rows(i), self.visible(i)
            total = x[:, :length].sum(1)[:, None] + np.einsum("jk,hkd->hjd", vis, x[:, length:])
            a[i] = np.repeat(total, self.h // self.hk, 0)
            keys[i] = length + vis.sum(1)
        return a, keys

    def device(self, dev):
        import torch

        t = getattr(torch, self.dtype)
        v = torch.from_numpy(self.v.astype(np.float32)).to(dev).to(t)
        k = torch.randn(v.shape, device=dev).to(t)
        if self.rows_first:
            k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
        b = len(self.lengths)
        mask = None
        if self.seen is not None:
            mask = torch.from_numpy(np.stack([paged.words(s, self.n) for s in self.seen])).to(dev)
        q = torch.zeros((b, self.n, self.h, self.d), dtype=t, device=dev).transpose(1, 2)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        return dict(q=q, k_cache=k, v_cache=v, block_tables=i32(self.tables),
                    lengths=i32(self.lengths), mask=mask)


def out_errors(got, a, keys, dtype):
    """[b, h, n, d]: whether an output is out of its bound."""
    want = a / keys[:, None, :, None]
    return np.abs(got - want) > (HALF_STEP[dtype] + 2.0 ** -21) * np.abs(want) + 2.0 ** -25


def lse_errors(got, keys):
    """[b, h, n]: whether a log-sum-exp is."""
    want = np.log(keys.astype(np.float64))[:, None]
    return np.abs(got - want) > 2.0 ** -21 * (want + 1)
