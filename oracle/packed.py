"""CPU oracle of attention over packed sequences with its gradients, and of the
norms with the rotary positions (test infrastructure only): float64 numpy, one
head and query row at a time.

No counterpart in the reference; the definitions are the comments of
``include/flashlite_attn.h``.  Beside each result stands the size that its
rounding errors follow.
"""

from __future__ import annotations

import numpy as np

from .paged import rotary


def rows_seen(nq, nk, i, causal):
    """The number of keys, from the first on, that query i of nq sees."""
    return min(max(i + nk - nq + 1, 0), nk) if causal else nk


def _walk(starts, key_starts, causal, heads, kv_heads):
    for a, b, c, e in zip(starts, starts[1:], key_starts, key_starts[1:]):
        for h in range(heads):
            for i in range(b - a):
                yield h, h // (heads // kv_heads), a + i, c, rows_seen(b - a, e - c, i, causal)


def attention(q, k, v, starts, key_starts, causal, scale):
    """(out, lse, weight, reach) over q [H, T, D] and k, v [H_k, T_k, D]: weight
    is sum_j p_j |v_j| a value, reach the largest sum |q k scale| a row.  Rows
    of no sequence are NaN."""
    out = np.full(q.shape, np.nan)
    lse, reach, weight = np.full(q.shape[:2], np.nan), np.zeros(q.shape[:2]), np.zeros(q.shape)
    with np.errstate(invalid="ignore", over="ignore"):
        for h, j, t, c, seen in _walk(starts, key_starts, causal, q.shape[0], k.shape[0]):
            out[h, t], lse[h, t] = 0.0, -np.inf
            if seen == 0:
                continue
            kk, vv = k[j, c:c + seen], v[j, c:c + seen]
            s = kk @ q[h, t] * scale
            top = s.max()
            p = np.exp(s - top)
            total = p.sum()
            out[h, t], lse[h, t] = p @ vv / total, top + np.log(total)
            weight[h, t] = p @ np.abs(vv) / total
            reach[h, t] = (np.abs(kk) @ np.abs(q[h, t])).max() * abs(scale)
    return out, lse, weight, reach


def gradients(q, k, v, out, lse, dout, starts, key_starts, causal, scale):
    """{name: (value, spread)} of dq, dk and dv from out and lse as they are
    given.  spread [...] holds what errors follow, for each value: "terms" the
    sum of the absolute terms, "ds" that of the products with ds's own sizes:
    |p| (sum |dout v| + sum |dout out|), "p" the same with |p|'s, "reach" with
    |ds| sum |q k scale|, "count" the terms, "other" the sum of the other
    factor's sizes."""
    names = {"dq": q.shape, "dk": k.shape, "dv": v.shape}
    keys = ("value", "terms", "ds", "reach", "count", "other")
    g = {n: {x: np.zeros(s) for x in keys} for n, s in names.items()}
    mag = np.abs
    with np.errstate(invalid="ignore", over="ignore"):
        for h, j, t, c, seen in _walk(starts, key_starts, causal, q.shape[0], k.shape[0]):
            if seen == 0:
                continue
            at = slice(c, c + seen)
            kk, vv, do = k[j, at], v[j, at], dout[h, t]
            p = np.exp(kk @ q[h, t] * scale - lse[h, t])
            reach = mag(kk) @ mag(q[h, t]) * abs(scale) + mag(lse[h, t]) + 1.0
            size = mag(vv) @ mag(do) + mag(do) @ mag(out[h, t])
            ds = p * (vv @ do - do @ out[h, t]) * scale
            for n, where, w, other in (("dv", (j, at), p, do[None]), ("dk", (j, at), ds, q[h, t][None]),
                                       ("dq", (h, t), ds, kk)):
                def put(x, y):
                    y = y[:, None] * mag(other) if x != "value" else y[:, None] * other
                    g[n][x][where] += y if n != "dq" else y.sum(0)
                put("value", w)
                put("terms", mag(w))
                put("reach", mag(w) * reach)
                put("other", np.ones(seen))
                if n != "dv":
                    put("ds", p * size * abs(scale))
                g[n]["count"][where] += 1 if n != "dq" else seen
    return g


def norm_rotary(x, weight, positions, freqs, axes=None, eps=1e-6, interleaved=False, scale=1.0):
    """R(x r w) over x [B, H, N, D]; weight None: no norm.  positions [B, N], or
    [A, B, N] with axes."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    return turn(x, positions, freqs, axes, interleaved, scale)


def turn(x, positions, freqs, axes=None, interleaved=False, scale=1.0, transpose=False):
    """The rotation alone, pair by pair where the positions have axes."""
    if axes is None:
        return rotary(x, positions, freqs, interleaved, scale, transpose)
    out = np.array(x, np.float64)
    for j, (f, a) in enumerate(zip(freqs, axes)):
        a = min(max(int(a), 0), len(positions) - 1)
        cols = [2 * j, 2 * j + 1] if interleaved else [j, j + len(freqs)]
        out[..., cols] = rotary(x[..., cols], positions[a], [f], True, scale, transpose)
    return out


def norm_rotary_gradients(x, dy, weight, positions, freqs, axes=None, eps=1e-6, interleaved=False,
                          scale=1.0):
    """(dx, dw, g, spread): g = R' dy, spread the size of dx's terms."""
    x = np.asarray(x, np.float64)
    g = turn(np.asarray(dy, np.float64), positions, freqs, axes, interleaved, scale, True)
    if weight is None:
        return g, None, g, np.abs(g)
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    dw = (g * x * r).sum((0, 1, 2))
    gw = g * weight
    along = (gw * x).mean(-1, keepdims=True) * r * r
    spread = r * (np.abs(gw) + np.abs(x) * r * r * np.abs(gw * x).mean(-1, keepdims=True))
    return r * (gw - x * along), dw, g, spread
