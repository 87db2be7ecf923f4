"""Rotary positions in 32 bits keep the accuracy of their type: sine and cosine
times the scale are rounded once from 64 bits.

The angle itself is position * freq in 64 bits, here and in the oracle: off by
at most 2^-52 of its size (two roundings of the kernel's turns, one of the
oracle's).  A rotated value a cos - b sin then counts half a step, 2^-24, for
each factor, for one product and for the sum."""

import numpy as np
import pytest

import flashlite_amd as fl

pytestmark = pytest.mark.gpu

STEP = 2.0 ** -24


def turns(n, pairs, first, seed):
    """positions [1, n], freqs, and the exact sines and cosines [n, pairs]."""
    rs = np.random.RandomState(seed)
    positions = (first + rs.permutation(4 * n)[:n])[None]
    freqs = 10000.0 ** (-np.arange(pairs) / pairs)
    angle = np.multiply.outer(positions[0].astype(np.float64), freqs)
    return positions, freqs, np.cos(angle), np.sin(angle), 2.0 ** -51 * angle


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("first,scale,pairs", [(0, 1.0, 32), (4096, 1.2, 32), (1 << 20, 1.0, 5),
                                               (131072, 0.7, 64)])
def test_sine_and_cosine(cuda, inter, first, scale, pairs):
    """Pairs (1, 0) become (scale cos, scale sin)."""
    import torch

    n, d = 2000, 128
    positions, freqs, cos, sin, far = turns(n, pairs, first, 3)
    a, b = ((slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if inter
            else (slice(0, pairs), slice(pairs, 2 * pairs)))
    q = torch.zeros((1, 1, n, d), device=cuda)
    q[..., a] = 1.0
    pos, f = torch.from_numpy(positions).to(cuda), torch.from_numpy(freqs).to(cuda)
    for turn, sign in ((fl.forward_rotary, 1.0), (fl.backward_rotary, -1.0)):
        out = turn(q, None, pos, f, inter, scale)[0, 0].double().cpu().numpy()
        for got, want in ((out[:, a], scale * cos), (out[:, b], sign * scale * sin)):
            assert (np.abs(got - want) <= STEP * np.abs(want) + scale * far + 2.0 ** -50).all()


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("heads,first,scale", [(1, 0, 1.0), (24, 70000, 1.2)])
def test_values(cuda, inter, heads, first, scale):
    import torch

    n, d, pairs = 501, 64, 32
    positions, freqs, cos, sin, far = turns(n, pairs, first, 4)
    x = np.random.RandomState(5).standard_normal((1, heads, n, d)).astype(np.float32)
    pos, f = torch.from_numpy(positions).to(cuda), torch.from_numpy(freqs).to(cuda)
    out = fl.forward_rotary(torch.from_numpy(x).to(cuda), None, pos, f, inter, scale)
    out, x = out.double().cpu().numpy(), x.astype(np.float64)
    a, b = ((x[..., 0::2], x[..., 1::2]) if inter else (x[..., :pairs], x[..., pairs:]))
    got = ((out[..., 0::2], out[..., 1::2]) if inter else (out[..., :pairs], out[..., pairs:]))
    for y, (u, v) in zip(got, ((a * cos, -b * sin), (a * sin, b * cos))):
        u, v = scale * u, scale * v
        bound = (STEP * (np.abs(u) + np.abs(v) + np.maximum(np.abs(u), np.abs(v)) + np.abs(u + v))
                 * (1 + 4 * STEP) + scale * far * (np.abs(a) + np.abs(b)) + 2.0 ** -48)
        assert (np.abs(y - (u + v)) <= bound).all()
