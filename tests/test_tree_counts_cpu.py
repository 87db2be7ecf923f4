"""The bounds of tests/tree_counts.py tell: results with any one tile of keys left
out, or counted twice, are out of them, the outputs' and the log-sum-exps' alike."""

import numpy as np
import pytest

from tree_counts import Counted, lse_errors, out_errors


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,tile", [(64, 64), (128, 32)])
@pytest.mark.parametrize("length", [700, 9000, 40000])
@pytest.mark.parametrize("times", [0, 2])
def test_a_lost_or_doubled_tile_shows(dtype, d, tile, length, times):
    p = Counted(5, dtype, 1, 1, 1, 1, d, 16, [length])
    a, keys = p.sums()
    assert not out_errors(a / keys[:, None, :, None], a, keys, dtype).any()
    x = p.rows(0)[0]
    for at in range(0, length + 1, tile):
        part = x[at:at + tile]
        wrong = a + (times - 1) * part.sum(0)
        count = keys + (times - 1) * len(part)
        assert out_errors(wrong / count[:, None, :, None], a, keys, dtype).any(), at
        assert lse_errors(np.log(count.astype(float))[:, None], keys).any(), at


def test_one_lost_key_shows():
    p = Counted(6, "float16", 1, 1, 1, 1, 64, 16, [40000])
    _, keys = p.sums()
    assert lse_errors(np.log(keys - 1.0)[:, None], keys).all()


def test_sums_by_hand():
    p = Counted(7, "float16", 2, 4, 2, 3, 64, 4, [5, 0], "tree")
    a, keys = p.sums()
    for i in range(2):
        for h in range(4):
            x = p.rows(i)[h // 2]
            for j in range(3):
                at = list(range(p.lengths[i])) + [p.lengths[i] + k for k in p.seen[i][j]]
                assert keys[i, j] == len(at)
                assert np.array_equal(a[i, h, j], x[at].sum(0))
