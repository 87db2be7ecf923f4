"""forward_tree (attention of drafted tokens over a paged cache) against the
float64 oracle; bounds in tree_util.py."""

import numpy as np
import pytest

import flashlite_amd as fl
from tree_util import Problem, check

pytestmark = pytest.mark.gpu

FILL = 7.0


def run(p, dev, lse=True, **kw):
    """One call into outputs that hold FILL; rows that are not there keep it."""
    import torch

    args = p.device(dev)
    out = torch.full_like(args["q"], FILL)
    ls = torch.full(args["q"].shape[:3], FILL, device=dev) if lse else None
    args.update(out=out, return_lse=lse, lse=ls)
    args.update(kw)
    got = fl.forward_tree(**args)
    torch.cuda.synchronize(dev)
    assert (got[0] if lse else got).data_ptr() == out.data_ptr()
    if p.counts is not None:
        gone = torch.from_numpy(np.arange(p.n) >= p.counts[:, None]).to(dev)
        gone = gone[:, None].expand(out.shape[:3])
        assert bool((out[gone] == FILL).all()), "a row that is not there was written"
        assert ls is None or bool((ls[gone] == FILL).all())
    return out, ls


KINDS = [("float16", 64), ("bfloat16", 64), ("float16", 128), ("bfloat16", 128)]


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("b,h,hk,n,block,lengths,tree", [
    (1, 1, 1, 1, 16, [0], None),                    # a first token
    (1, 1, 1, 1, 16, [1], None),
    (3, 4, 4, 1, 16, [5, 64, 63], None),
    (2, 8, 2, 1, 20, [100, 333], None),             # pages that end inside a tile
    (2, 3, 1, 1, 1, [70, 9], None),                 # a page a key
    (1, 8, 1, 4, 257, [1000], "tree"),              # 32 rows
    (2, 2, 2, 5, 16, [0, 31], "tree"),
    (2, 6, 2, 33, 8, [40, 130], "tree"),            # 99 rows
    (1, 7, 1, 19, 16, [200], "any"),                # 133 rows
    (2, 4, 4, 70, 16, [10, 0], "any"),              # masks of two words
    (1, 2, 1, 130, 64, [0], "any"),                 # drafts only, three words
    (1, 4, 2, 200, 32, [77], None),                 # a prompt's chunk
    (5, 2, 1, 3, 16, [0, 1, 15, 16, 17], "tree"),
])
def test_shapes(cuda, dtype, d, b, h, hk, n, block, lengths, tree):
    p = Problem(b + n, dtype, b, h, hk, n, d, block, lengths, tree)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("b,h,hk,n,block,lengths,tree", [
    (6, 4, 2, 9, 16, [0, 5, 100, 33, 64, 1], "tree"),
    (4, 4, 2, 1, 16, [7, 0, 100, 33], None),
    (3, 8, 2, 40, 16, [130, 0, 40], "any"),
    (3, 2, 2, 90, 20, [0, 11, 70], None),
])
def test_ragged_drafts(cuda, dtype, d, b, h, hk, n, block, lengths, tree):
    p = Problem(17 + n, dtype, b, h, hk, n, d, block, lengths, tree, ragged=True, rows_first=False,
                table_pad=2)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("b,h,hk,n,block,lengths,tree", [
    (1, 4, 1, 1, 16, [9000], None),
    (2, 4, 2, 12, 64, [4000, 2500], "tree"),
    (3, 2, 1, 2, 16, [6000, 3, 900], None),
    (1, 8, 2, 20, 128, [3001], "any"),
    (2, 16, 2, 16, 16, [1500, 700], "tree"),
])
def test_long_caches(cuda, dtype, d, b, h, hk, n, block, lengths, tree):
    p = Problem(23 + n, dtype, b, h, hk, n, d, block, lengths, tree)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("scale,q_scale", [(-0.3, 1.0), (0.7, 1.0), (0.125, 30.0), (1.0 / 1.4426950408889634, 1.0)])
def test_scales(cuda, dtype, d, scale, q_scale):
    """Signs, sharp rows (later tiles far above the first), a factor of one."""
    p = Problem(31, dtype, 2, 4, 2, 7, d, 16, [700, 90], "tree", scale=scale, q_scale=q_scale)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
def test_first_visible_key_far_below_zero(cuda, dtype, d):
    """Drafts only, whose visible keys start in a late tile with scores far
    below 0: a stabiliser of 0 would lose them."""
    n = 200
    p = Problem(37, dtype, 1, 2, 1, n, d, 16, [0], "any", scale=1.0)
    p.seen = [[{j for j in (150, 170, i) if j <= max(i, 150) and j >= 150} if i >= 150 else set()
               for i in range(n)]]
    import torch
    p.q[...] = torch.abs(p.q) + 1.0
    p.k[...] = -torch.abs(p.k) - 2.0
    ref = p.reference()
    assert np.isfinite(ref[1][:, :, 150:]).all() and (ref[1][:, :, 150:] < -150).all()
    check(*run(p, cuda), p, ref)


@pytest.mark.parametrize("dtype,d", KINDS)
def test_nan_and_infinity_reach_their_rows_only(cuda, dtype, d):
    """NaN and infinities in V and K of drafts some rows see, of cache rows
    behind the drafts, and of blocks nobody holds; a NaN query row."""
    p = Problem(41, dtype, 2, 2, 1, 40, d, 16, [50, 70], "any")
    nan, inf = float("nan"), float("inf")

    def at(b, t):
        return int(p.tables[b, t // 16]), t % 16

    blk, row = at(0, 50 + 7)
    p.v[blk, 0, row, 3] = nan           # draft 7 of request 0
    blk, row = at(0, 50 + 20)
    p.v[blk, 0, row, 5] = inf
    blk, row = at(1, 70 + 11)
    p.k[blk, 0, row, 9] = nan           # every row that sees it is NaN
    p.q[1, 1, 30, 2] = nan
    for b, length in ((0, 50), (1, 70)):  # behind the last draft
        for t in range(length + 40, p.tables.shape[1] * 16):
            if p.tables[b, t // 16] >= 0:
                blk, row = at(b, t)
                p.k[blk, 0, row] = nan
                p.v[blk, 0, row] = nan
    ref = p.reference()
    assert np.isnan(ref[0]).any() and np.isfinite(ref[0]).any() and np.isinf(ref[0]).any()
    check(*run(p, cuda), p, ref)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("length", [90, 700])
def test_bad_pages_are_seen_by_nobody(cuda, dtype, d, length):
    p = Problem(43, dtype, 2, 2, 1, 3, d, 16, [length, length], "tree")
    blocks = p.k.shape[0]
    p.tables[0, 1] = -1
    p.tables[0, 3] = blocks
    p.tables[1, 0] = 2 ** 31 - 1
    p.tables[1, length // 32] = -(2 ** 31)
    p.tables[1, -1] = blocks + 5  # the drafts'
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
def test_no_page_is_good(cuda, dtype, d):
    import torch

    p = Problem(44, dtype, 1, 2, 1, 3, d, 16, [100], "tree")
    p.tables[:] = -1
    out, lse = run(p, cuda)
    assert bool((out == 0).all()) and bool(torch.isneginf(lse).all())


def test_lengths_past_the_table_are_clamped(cuda):
    """Every row of the table is a token then, and no draft has a key."""
    p = Problem(45, "float16", 2, 4, 2, 3, 64, 16, [61, 29], "tree")
    args = p.device(cuda)
    capacity = p.tables.shape[1] * 16
    args["lengths"][:] = args["lengths"].new_tensor([capacity + 1000, 2 ** 31 - 1])
    out = fl.forward_tree(**args)
    p.lengths = np.array([capacity, capacity])
    p.tables = np.where(p.tables < 0, -1, p.tables)
    check(out, None, p)
    args["lengths"][:] = -5
    p.lengths = np.array([0, 0])
    check(fl.forward_tree(**args), None, p)


def test_shared_mask_and_shared_blocks(cuda):
    """One mask for all requests; requests that share a prompt's blocks."""
    import torch

    p = Problem(46, "bfloat16", 3, 4, 2, 6, 128, 16, [64, 64, 64], "tree")
    p.seen = [p.seen[0]] * 3
    p.tables[1, :4] = p.tables[0, :4]
    p.tables[2, :4] = p.tables[0, :4]
    mask = torch.from_numpy(p.mask()[0]).to(cuda)
    check(*run(p, cuda, mask=mask), p)


def test_cache_of_one_block_a_request(cuda):
    """A cache that is not paged: blocks of all rows, strided."""
    import torch

    b, h, hk, n, d, most = 3, 4, 2, 2, 64, 301
    p = Problem(47, "float16", b, h, hk, n, d, most, [250, 0, 299], None)
    args = p.device(cuda)
    wide = torch.full((args["k_cache"].shape[0], hk, most, 2 * d), float("nan"), dtype=torch.float16,
                      device=cuda)
    wide[..., :d] = args["k_cache"]
    check(*run(p, cuda, k_cache=wide[..., :d]), p)


def test_same_as_causal_attention(cuda):
    """A chain over a cache is forward_flash2_ex's causal attention."""
    from flashlite_amd.workloads import make_qkv
    import torch

    q, k, v = (torch.from_numpy(x).to(cuda) for x in make_qkv(2, 4, 96, 64, seed=5))
    tables = torch.arange(2, dtype=torch.int32, device=cuda)[:, None]
    lengths = torch.full((2,), 64, dtype=torch.int32, device=cuda)
    got, lse = fl.forward_tree(q[:, :, 64:], k, v, tables, lengths, return_lse=True)
    want, want_lse = fl.forward_flash2_ex(q[:, :, 64:], k, v, is_causal=True, return_lse=True)
    assert float((got.float() - want.float()).abs().max()) <= 2e-3
    assert float((lse - want_lse).abs().max()) <= 2e-3


def test_new_outputs_and_empty_calls(cuda):
    import torch

    p = Problem(48, "float16", 3, 4, 2, 5, 64, 16, [20, 0, 33], "tree", ragged=True)
    p.counts = np.array([0, 5, 2])
    args = p.device(cuda)
    out, lse = fl.forward_tree(return_lse=True, **args)
    check(out, lse, p)
    assert bool((out[0] == 0).all()) and bool((out[2, :, 2:] == 0).all())
    assert bool((lse[0] == 0).all())
    for shape in ((0, 4, 5, 64), (3, 4, 0, 64), (3, 0, 5, 64)):
        q = torch.zeros(shape, dtype=torch.float16, device=cuda)
        out = fl.forward_tree(q, args["k_cache"], args["v_cache"], args["block_tables"][:shape[0]],
                              args["lengths"][:shape[0]])
        assert out.shape == q.shape


def test_far_cache_rows(cuda):
    """Keys and values past 32-bit byte offsets: a cache of 4.4 GB."""
    import torch

    d, block, blocks = 128, 16, 540000  # 4096 bytes a block: 2.2 GB each
    cache = torch.zeros((2, blocks, block, 1, d), dtype=torch.bfloat16, device=cuda)
    k, v = (c.transpose(1, 2) for c in cache)
    p = Problem(49, "bfloat16", 1, 3, 1, 2, d, block, [200], "tree")
    far = blocks - 1 - 37 * np.arange(p.tables.shape[1])
    args = p.device(cuda)
    own = args["block_tables"][0].long()
    where = torch.from_numpy(far.copy()).to(cuda)
    k[where] = args["k_cache"][own]
    v[where] = args["v_cache"][own]
    check(*run(p, cuda, k_cache=k, v_cache=v, block_tables=where.int()[None].contiguous()), p)


def test_other_stream_and_workspace(cuda):
    """The current stream is used; a workspace is enough where one is asked for."""
    import torch

    p = Problem(50, "bfloat16", 2, 8, 2, 4, 128, 16, [3000, 1200], "tree")
    args = p.device(cuda)
    want = fl.forward_tree(**args)
    need = fl.tree_workspace_bytes(args["q"], args["k_cache"])
    ws = torch.full((need // 4 + 4,), float("nan"), device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = torch.empty_like(args["q"])
        for _ in range(3):
            fl.forward_tree(out=out, workspace=ws, **args)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, want)
    check(out, None, p)


def test_refusals(cuda):
    import torch

    p = Problem(51, "float16", 2, 4, 2, 3, 64, 16, [20, 30], "tree")
    args = p.device(cuda)

    def refuse(text, **kw):
        with pytest.raises(RuntimeError, match=text):
            fl.forward_tree(**{**args, **kw})

    refuse("FP16", q=args["q"].float())
    refuse("dtype", k_cache=args["k_cache"].bfloat16())
    refuse("v_cache", v_cache=args["v_cache"][:1])
    refuse("block_tables", block_tables=args["block_tables"].long())
    refuse("block_tables", block_tables=args["block_tables"][:1])
    refuse("lengths", lengths=args["lengths"].long())
    refuse("lengths", lengths=args["lengths"][:1])
    refuse("counts", counts=args["lengths"].float())
    refuse("mask", mask=args["mask"].int())
    refuse("mask", mask=args["mask"][:, :2])
    refuse("multiple", q=args["q"][:, :3])
    refuse("out must", out=torch.empty_like(args["q"][:1]))
    refuse("lse= needs", lse=torch.empty((2, 4, 3), device=cuda))
    refuse("lse must", return_lse=True, lse=torch.empty((2, 4, 2), device=cuda))
    refuse("q must be 4D", q=args["q"][0])
    refuse("sm_scale", sm_scale=float("inf"))
