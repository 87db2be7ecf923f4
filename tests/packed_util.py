"""Problems of forward_packed and backward_packed and the bounds of their outputs.

u is half a step of the element type (2^-11 fp16, 2^-8 bf16), 2^-24 that of fp32.

Forward:
- scores: D products summed in 32 bits, off by at most (D + 8) 2^-24 sum |q k
  scale| (`reach`), and 2^-22 of the exponential itself: delta, relative on p;
- p rounded to the element type before the product with V, and (head dim 64)
  summed so for the row sum: u of each p twice over, so 2 u of sum p |v| / sum p
  (`weight`); fp16's smallest steps, 2^-25 a key against a largest p of at least
  2^-8 (the stabiliser lags by at most 8 in base 2): 2^-17 a key, seldom more
  than 16 of them count, as they are at most 2^-17 of the largest each;
- 32-bit sums over the keys: (keys + 64) 2^-24 of `weight`;
- the output's own rounding, u of it.
The log-sum-exp: delta, the sums, 2 u of rounded p in the row sum, 2^-21 of its
size for the logarithm and the stabiliser's product.

Backward, from out and lse as they are given:
- p: (D + 8) 2^-24 (sum |q k scale| + |lse| + 1), relative (`reach`);
- dout v' and dout . out: (D + 8) 2^-24 of their absolute sums, on ds with the
  weight p (`ds`);
- p and ds rounded for their products, u of each term (`terms`), fp16's smallest
  step 2^-25 of each times the other factor (`other`; ds without the scale, so
  times |scale|);
- 32-bit sums over the rows: (count + 64) 2^-24 of `terms`;
- the result's own rounding, u of it, and 2^-25.
"""

import numpy as np

from oracle import packed

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


class Problem:
    """Seeded tensors of packed sequences: `lengths` and `keys` (None: the
    same), rows of nobody NaN (`gap` of them before the first sequence and
    behind the last)."""

    def __init__(self, seed, dtype, d, h, hk, lengths, keys=None, causal=True, layout="rows",
                 gap=0, scale=0.0, q_scale=1.0):
        import torch

        rs = np.random.RandomState(seed)
        self.dtype, self.d, self.h, self.hk, self.causal = dtype, d, h, hk, causal
        self.sm_scale = scale
        self.scale = scale if scale != 0.0 else 1.0 / np.sqrt(d)
        self.starts = gap + np.concatenate([[0], np.cumsum(lengths)]).astype(int)
        self.key_starts = (self.starts if keys is None
                           else gap + np.concatenate([[0], np.cumsum(keys)]).astype(int))
        self.shared = keys is None
        self.rows, self.key_rows = self.starts[-1] + gap, self.key_starts[-1] + gap
        t = getattr(torch, dtype)

        def tensor(heads, rows, starts, size=1.0):
            x = torch.from_numpy((rs.standard_normal((heads, rows, d)) * size).astype(np.float32))
            x[:, :starts[0]] = x[:, starts[-1]:] = float("nan")
            return x.to(t)

        self.q = tensor(h, self.rows, self.starts, q_scale)
        self.k = tensor(hk, self.key_rows, self.key_starts)
        self.v = tensor(hk, self.key_rows, self.key_starts)
        self.dout = tensor(h, self.rows, self.starts)
        self.layout = layout

    def view(self, x, dev):
        """x [heads, rows, d] as [1, heads, rows, d] on dev, stored as the layout says."""
        x = x.to(dev)
        if self.layout == "rows":
            x = x.transpose(0, 1).contiguous().transpose(0, 1)
        return x[None]

    def device(self, dev):
        import torch

        if self.layout == "qkv":
            assert self.shared
            x = torch.cat([self.q, self.k, self.v]).transpose(0, 1).contiguous().to(dev)
            x = x.transpose(0, 1)[None]
            q, k, v = x[:, :self.h], x[:, self.h:self.h + self.hk], x[:, self.h + self.hk:]
        else:
            q, k, v = (self.view(x, dev) for x in (self.q, self.k, self.v))
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        return dict(q=q, k=k, v=v, starts=i32(self.starts),
                    key_starts=None if self.shared else i32(self.key_starts),
                    sm_scale=self.sm_scale, is_causal=self.causal)

    def arrays(self):
        return [x.double().numpy() for x in (self.q, self.k, self.v)]

    def reference(self):
        return packed.attention(*self.arrays(), self.starts, self.key_starts, self.causal,
                                self.scale)

    def inside(self, key=False):
        s = self.key_starts if key else self.starts
        there = np.zeros(self.key_rows if key else self.rows, bool)
        there[s[0]:s[-1]] = True
        return there


def patterns(got, want, what):
    """The same NaN and infinities; where both are finite."""
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"{what}: NaN pattern"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities"
    return np.isfinite(want)


def check(got, got_lse, p, ref=None):
    out, lse, weight, reach = p.reference() if ref is None else ref
    there = p.inside()
    got = got[0].double().cpu().numpy()[:, there]
    want, weight, reach, lse = out[:, there], weight[:, there], reach[:, there], lse[:, there]
    u = HALF_STEP[p.dtype]
    keys = int(np.diff(p.key_starts).max(initial=0))
    delta = (p.d + 8) * 2.0 ** -24 * reach + 2.0 ** -22
    sums = (keys + 64) * 2.0 ** -24
    fin = patterns(got, want, "out")
    with np.errstate(invalid="ignore"):
        bound = (u * np.abs(want) + (2 * u + 2 * delta[..., None] + sums) * weight
                 + 2.0 ** -17 * 16 * (p.dtype == "float16") * 2.0 ** -8 + 2.0 ** -25)
        ratio = (np.abs(got - want) / bound)[fin]
    assert ratio.size == 0 or ratio.max() <= 1.0, f"out: {ratio.max():.3g} of the bound"
    if got_lse is not None:
        y = got_lse[0].double().cpu().numpy()[:, there]
        fin = patterns(y, lse, "lse")
        bound = delta + sums + 2 * u + 2.0 ** -21 * (np.abs(lse) + reach + 1)
        assert (np.abs(y[fin] - lse[fin]) <= bound[fin]).all(), "log-sum-exp"


def check_gradients(got, p, out, lse, ref=None):
    """got: (dq, dk, dv) tensors [1, heads, rows, d]; out and lse: what the
    gradients were taken from."""
    a = [x[0].double().cpu().numpy() for x in (out, lse)]
    g = (packed.gradients(*p.arrays(), *a, p.dout.double().numpy(), p.starts, p.key_starts,
                          p.causal, p.scale) if ref is None else ref)
    u = HALF_STEP[p.dtype]
    e = (p.d + 8) * 2.0 ** -24
    for name, t in zip(("dq", "dk", "dv"), got):
        there = p.inside(name != "dq")
        w = {k: x[:, there] for k, x in g[name].items()}
        x = t[0].double().cpu().numpy()[:, there]
        fin = patterns(x, w["value"], name)
        small = 2.0 ** -25 * (p.dtype == "float16")
        with np.errstate(invalid="ignore"):
            bound = (u * np.abs(w["value"]) + (u + 2.0 ** -21 + (w["count"] + 64) * 2.0 ** -24)
                     * w["terms"] + e * (w["reach"] + 2 * w["ds"])
                     + small * w["other"] * max(1.0, abs(p.scale)) + 2.0 ** -25)
            ratio = (np.abs(x - w["value"]) / bound)[fin]
        assert ratio.size == 0 or ratio.max() <= 1.0, f"{name}: {ratio.max():.3g} of the bound"
