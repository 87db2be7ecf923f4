"""Seeded random shapes through the paged-cache operators (bounds in
tree_util.py and test_gpu_rotary.py)."""

import numpy as np
import pytest

import flashlite_amd as fl
from oracle import paged
from test_gpu_cache_plan import check as check_plan
from test_gpu_cache_plan import make
from test_gpu_rotary import assert_rotated, draw, views
from test_gpu_tree import run
from tree_util import Problem, check

pytestmark = pytest.mark.gpu


def spread(rs, low, high):
    """A whole number, even over the logarithm."""
    return int(round(np.exp(rs.uniform(np.log(low), np.log(high)))))


@pytest.mark.parametrize("seed", range(60))
def test_tree(cuda, seed):
    rs = np.random.RandomState(1000 + seed)
    dtype, d = [("float16", 64), ("bfloat16", 64), ("float16", 128), ("bfloat16", 128)][seed % 4]
    group, hk = spread(rs, 1, 9), spread(rs, 1, 9)
    n = 1 if rs.rand() < 0.3 else spread(rs, 1, 150)
    b = spread(rs, 1, 5) if rs.rand() < 0.8 or group * hk * n > 60 else spread(rs, 60, 90)
    lengths = [0 if rs.rand() < 0.2 else spread(rs, 1, 2000 if b < 10 else 200) for _ in range(b)]
    tree = None if n == 1 else [None, "tree", "any"][rs.randint(3)]
    p = Problem(seed, dtype, b, group * hk, hk, n, d, int(rs.choice([1, 8, 16, 20, 64, 257])),
                lengths, tree, ragged=rs.rand() < 0.5, rows_first=rs.rand() < 0.5,
                scale=float(rs.choice([0.0, 0.2, -0.1])), q_scale=float(rs.choice([1.0, 8.0])),
                table_pad=int(rs.choice([0, 1, 37, 3000])))
    if rs.rand() < 0.5:  # some pages nobody has
        p.tables[rs.rand(*p.tables.shape) < 0.1] = rs.choice([-1, p.k.shape[0], 2 ** 31 - 1])
    check(*run(p, cuda, lse=rs.rand() < 0.7), p)


@pytest.mark.parametrize("seed", range(30))
def test_rotary(cuda, seed):
    import torch

    rs = np.random.RandomState(2000 + seed)
    dtype = ["float16", "bfloat16", "float32"][seed % 3]
    d = int(rs.choice([64, 128]))
    b, h, hk, n = (spread(rs, 1, x) for x in (4, 20, 9, 300))
    pairs, inter = int(rs.randint(0, d // 2 + 1)), bool(rs.randint(2))
    scale = float(rs.choice([1.0, 1.3]))
    q, q64 = draw(rs, (b, h, n, d), dtype, cuda)
    k, k64 = draw(rs, (b, hk, n, d), dtype, cuda)
    positions = rs.randint(0, spread(rs, 10, 10 ** 7), (b, n))
    freqs = 10000.0 ** (-np.arange(pairs) / max(pairs, 1))
    layout = ["bhnd", "bnhd"][rs.randint(2)]
    turn, back = [(fl.forward_rotary, False), (fl.backward_rotary, True)][rs.randint(2)]
    got = turn(views(q, layout), views(k, layout), torch.from_numpy(positions).to(cuda),
               torch.from_numpy(freqs).to(cuda), inter, scale)
    for g, x in zip(got, (q64, k64)):
        want = paged.rotary(x, positions, freqs, inter, scale, back)
        assert_rotated(g, x, want, dtype, pairs, inter, scale)


@pytest.mark.parametrize("seed", range(30))
def test_plan(cuda, seed):
    rs = np.random.RandomState(3000 + seed)
    b, width, block, m = (spread(rs, *x) for x in ((1, 2600), (1, 900), (1, 300), (1, 30)))
    b = min(b, max(1, 200000 // width))
    args = make(seed, b, width, block, m, ended=rs.uniform(0, 0.5),
                free=None if rs.rand() < 0.6 else int(rs.randint(0, 50)))
    check_plan(args, block, width, cuda, in_place=bool(rs.randint(2)), table_pad=int(rs.randint(3)))
