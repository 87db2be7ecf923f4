"""forward_tree counts every key once: whole numbers, exact sums, and bounds that
one lost or doubled tile breaks (tests/tree_counts.py), over the launches of
test_gpu_tree_split.py."""

import pytest

import flashlite_amd as fl
from tree_counts import Counted, lse_errors, out_errors

pytestmark = pytest.mark.gpu

KINDS = [("float16", 64), ("bfloat16", 64), ("float16", 128), ("bfloat16", 128)]
# heads of one KV head and drafts: 1, 12, 48, 120 and 150 rows
ROWS = [(1, 1), (4, 3), (4, 12), (4, 30), (1, 150)]


def counted(p, cuda):
    a, keys = p.sums()
    out, lse = fl.forward_tree(return_lse=True, **p.device(cuda))
    wrong = out_errors(out.double().cpu().numpy(), a, keys, p.dtype)
    assert not wrong.any(), f"{int(wrong.sum())} outputs"
    wrong = lse_errors(lse.double().cpu().numpy(), keys)
    assert not wrong.any(), f"{int(wrong.sum())} log-sum-exps"


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("length", [700, 9000, 40000])
def test_one_request(cuda, dtype, d, group, n, length):
    """All parts of one unit, or of a few."""
    counted(Counted(n + length, dtype, 1, group, 1, n, d, 16, [length]), cuda)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("rows_first", [False, True])
def test_unlike_requests(cuda, dtype, d, group, n, tree, rows_first):
    """Long ones among short and empty ones, 4 heads side by side among them."""
    lengths = [9000, 1, 0, 5000, 63, 64, 65, 40000, 31, 700]
    counted(Counted(n, dtype, len(lengths), 4 * group, 4, n, d, 16, lengths, tree, rows_first),
            cuda)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("block", [7, 64, 257])
def test_many_units_and_blocks(cuda, dtype, d, group, n, block):
    lengths = [(37 * i * i) % 1500 for i in range(70)]
    counted(Counted(n, dtype, len(lengths), 4 * group, 4, n, d, block, lengths, room=40), cuda)
