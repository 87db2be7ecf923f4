"""forward_tree over more requests than 65535 (what some launches allow along a
dimension), and over part of a table's columns."""

import math

import pytest

import flashlite_amd as fl
from tree_util import Problem, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows_first", [True, False])
def test_more_than_65535_requests(cuda, rows_first):
    """One token over up to 11 keys each, in tables with room for 4800, so that
    the longest walk that the launch has to allow for is a long one."""
    import torch

    b, h, d, block, blocks, m = 65600, 4, 64, 16, 300, 300
    g = torch.Generator(device=cuda)
    g.manual_seed(5)
    rand = lambda *s: torch.randn(s, generator=g, device=cuda).half()  # noqa: E731
    q = rand(b, h, 1, d)
    k, v = ((rand(blocks, block, h, d).transpose(1, 2) if rows_first
             else rand(blocks, h, block, d)) for _ in range(2))
    lengths = torch.randint(0, 11, (b,), generator=g, device=cuda).int()
    ids = torch.randint(0, blocks, (b,), generator=g, device=cuda)
    tables = torch.full((b, m), -1, dtype=torch.int32, device=cuda)
    tables[:, 0] = ids.int()
    out, lse = fl.forward_tree(q, k, v, tables, lengths, return_lse=True)

    worst = 0.0
    for i in range(0, b, 8200):  # 8 parts
        at = ids[i:i + 8200]
        kd, vd = k[at].double(), v[at].double()  # [., h, block, d]
        s = (q[i:i + 8200].double() * kd).sum(-1) / math.sqrt(d)
        reach = (q[i:i + 8200].double() * kd).abs().sum(-1).amax(-1) / math.sqrt(d)
        hidden = torch.arange(block, device=cuda) > lengths[i:i + 8200, None]
        s = s.masked_fill(hidden[:, None], -math.inf)
        p = torch.softmax(s, -1)[..., None]
        want, weight = (p * vd).sum(2), (p * vd.abs()).sum(2)
        # scores: d products and sums of 2^-24 and the exponential's 2^-22, relative on p;
        # p and the output rounded to fp16: half steps of 2^-11; fp16's smallest
        # steps, 2^-25 of each of 16 keys' p |v| < 6 and of the output
        delta = ((d + 8) * 2.0 ** -24 * reach + 2.0 ** -22)[..., None]
        bound = (2.0 ** -11 * want.abs() + (2.0 ** -11 + 2 * delta + 80 * 2.0 ** -24) * weight
                 + (16 * 6 + 1) * 2.0 ** -25)
        err = (out[i:i + 8200, :, 0].double() - want).abs()
        worst = max(worst, float((err / bound).max()))
        logs = torch.logsumexp(s, -1)
        off = (lse[i:i + 8200, :, 0].double() - logs).abs()
        assert bool((off <= delta[..., 0] + 80 * 2.0 ** -24
                     + 2.0 ** -21 * (logs.abs() + reach + 1)).all())
    assert worst <= 1.0


@pytest.mark.parametrize("n,tree", [(1, None), (30, "tree")])
def test_the_first_columns_of_a_wide_table(cuda, n, tree):
    """A caller that knows its longest request hands over fewer columns."""
    p = Problem(95, "bfloat16", 3, 8, 2, n, 128, 16, [600, 0, 333], tree, table_pad=3000)
    args = p.device(cuda)
    ref = p.reference()
    for m in (args["block_tables"].shape[1], -(-(600 + n) // 16)):
        out, lse = fl.forward_tree(return_lse=True,
                                   **{**args, "block_tables": args["block_tables"][:, :m]})
        check(out, lse, p, ref)
