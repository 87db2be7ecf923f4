"""forward_tree's launches: units one work-group walks alone, and units whose
keys are dealt to many work-groups and joined.  Tables with room for far more
keys than the requests have call for the second; bounds in tree_util.py."""

import numpy as np
import pytest

import flashlite_amd as fl
from test_gpu_tree import KINDS, run
from tree_util import Problem, check

pytestmark = pytest.mark.gpu

ROOM = 4000  # blocks of 16 tokens: more steps than one work-group is given

# heads of one KV head and drafts: 12, 48, 120 and 150 rows
ROWS = [(4, 3), (4, 12), (4, 30), (1, 150)]


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("tree", [None, "tree", "any"])
def test_room_for_more(cuda, dtype, d, group, n, tree):
    """Short and empty requests in long tables."""
    p = Problem(60 + n, dtype, 3, 2 * group, 2, n, d, 16, [33, 0, 500], tree, ragged=True,
                table_pad=ROOM)
    p.counts[1] = n
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("room", [0, ROOM])
def test_many_requests(cuda, dtype, d, group, n, room):
    """More requests than lanes of a wave, whose shares begin and end anywhere."""
    rs = np.random.RandomState(n)
    b = 70
    lengths = rs.randint(0, 300, b) * (rs.rand(b) < 0.7)
    p = Problem(61 + n, dtype, b, group, 1, n, d, 16, lengths, "tree", ragged=True, table_pad=room)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n,hk", [(2, 4, 8), (4, 12, 8), (4, 30, 8), (1, 300, 4)])
@pytest.mark.parametrize("room", [0, ROOM])
def test_more_units_than_work_groups(cuda, dtype, d, group, n, hk, room):
    """Two units and more a CU."""
    b = 66
    lengths = np.random.RandomState(n).randint(0, 60, b)
    p = Problem(62 + n, dtype, b, group * hk, hk, n, d, 16, lengths, None, ragged=True,
                table_pad=room)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n,length", [(4, 1, 40000), (2, 24, 9000), (3, 40, 9000),
                                            (1, 140, 6000)])
def test_one_long_request(cuda, dtype, d, group, n, length):
    """As many parts as a unit is given."""
    p = Problem(63 + n, dtype, 1, group, 1, n, d, 16, [length], "any" if n > 1 else None)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
def test_sharp_rows_in_parts(cuda, dtype, d, group, n):
    """Parts whose largest scores lie far apart."""
    p = Problem(64 + n, dtype, 2, group, 1, n, d, 16, [3000, 700], "tree", q_scale=40.0,
                table_pad=ROOM)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
def test_nan_and_bad_pages_in_parts(cuda, dtype, d, group, n):
    """Blocks out of range and -1 entries, NaN keys and values that no row of
    some drafts sees, infinite values that some see, and a NaN query row: where
    they lie in one part only the rows of their own change."""
    p = Problem(65 + n, dtype, 2, group, 1, n, d, 16, [1500, 1400], "any", table_pad=ROOM)
    nan, inf = float("nan"), float("inf")

    def at(b, t):
        return int(p.tables[b, t // 16]), t % 16

    for b, length in enumerate((1500, 1400)):
        blk, row = at(b, length + n - 1)   # the last draft
        p.v[blk, 0, row, 3] = nan
        p.v[blk, 0, row, 5] = -inf
        blk, row = at(b, length + n // 2)
        if b == 1:
            p.k[blk, 0, row, 9] = nan
    p.q[0, group - 1, n - 1, 2] = nan
    p.tables[0, 1] = -1
    p.tables[0, 40] = p.k.shape[0]
    p.tables[1, 0] = 2 ** 31 - 1
    p.tables[1, 60:70] = -(2 ** 31)
    check(*run(p, cuda), p)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
def test_only_one_part_has_keys(cuda, dtype, d, group, n):
    """All pages but the last are bad: every part but one is empty."""
    p = Problem(66 + n, dtype, 1, group, 1, n, d, 16, [4000], None, table_pad=ROOM)
    p.tables[0, :249] = -1
    check(*run(p, cuda), p)
    p.tables[:] = -1
    p.seen = [[set()] * n]
    out, lse = run(p, cuda)
    assert bool((out == 0).all()) and bool((lse == -float("inf")).all())


@pytest.mark.parametrize("group,n", ROWS)
def test_workspace_is_not_read_before_it_is_written(cuda, group, n):
    """Calls of other sizes leave what they like in a workspace."""
    import torch

    kinds = [Problem(67, "float16", 3, 2 * group, 2, n, 64, 16, [900, 0, 40], "tree",
                     table_pad=ROOM),
             Problem(68, "float16", 2, 2 * group, 2, n, 64, 16, [10, 2000], None, table_pad=ROOM)]
    args = [p.device(cuda) for p in kinds]
    need = max(fl.tree_workspace_bytes(a["q"], a["k_cache"]) for a in args)
    ws = torch.empty(need // 4, device=cuda)
    first = None
    for fill in (float("nan"), -1.0, 3.0e38):
        ws.fill_(fill)
        got = [fl.forward_tree(workspace=ws, **a) for a in args for _ in range(2)]
        for i in (0, 2):
            assert torch.equal(got[i], got[i + 1])
        if first is None:
            first = got
            check(got[0], None, kinds[0])
            check(got[2], None, kinds[1])
        assert all(torch.equal(x, y) for x, y in zip(first, got))


def test_workspace_too_small_is_refused(cuda):
    import torch

    p = Problem(69, "float16", 1, 2, 1, 3, 64, 16, [900], "tree", table_pad=ROOM)
    args = p.device(cuda)
    need = fl.tree_workspace_bytes(args["q"], args["k_cache"])
    assert need > 0
    with pytest.raises(RuntimeError, match="workspace"):
        fl.forward_tree(workspace=torch.empty(need - 4, dtype=torch.uint8, device=cuda), **args)
    with pytest.raises(RuntimeError, match="workspace"):
        fl.forward_tree(workspace=torch.empty(need), **args)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("group,n", ROWS)
@pytest.mark.parametrize("room", [0, ROOM])
def test_infinite_scores(cuda, dtype, d, group, n, room):
    """Scores of -inf weigh nothing, a whole tile's or part's included; one of
    +inf makes its row NaN."""
    p = Problem(70 + n, dtype, 2, group, 1, n, d, 16, [900, 260], "tree", table_pad=room)
    for b, gone in ((0, 700), (1, 200)):  # the first tokens' scores: -inf or inf
        for t in range(gone):
            p.k[int(p.tables[b, t // 16]), 0, t % 16, 0] = float("inf")
    low = np.random.RandomState(n).rand(2, group, n) < 0.8
    import torch

    sign = torch.from_numpy(np.where(low, -1.0, 1.0))
    p.q[..., 0] = (p.q[..., 0].abs() + 0.1) * sign.to(p.q.dtype)
    ref = p.reference()
    assert np.isnan(ref[0]).any() and np.isfinite(ref[0]).any()
    check(*run(p, cuda), p, ref)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("b,h,hk,n,lengths,tree,room", [
    (1, 2, 2, 512, [40], "tree", 0),       # the widest mask plan_tree makes
    (2, 1, 1, 512, [0, 300], "any", ROOM),
    (1, 1, 1, 700, [33], None, 0),         # a prompt's chunk
    (1, 1, 1, 700, [0], None, ROOM),
])
def test_many_drafts(cuda, dtype, d, b, h, hk, n, lengths, tree, room):
    p = Problem(71 + n, dtype, b, h, hk, n, d, 16, lengths, tree, ragged=b > 1, table_pad=room)
    check(*run(p, cuda), p)


def test_outputs_that_overlap_are_refused(cuda):
    import torch

    p = Problem(72, "float16", 2, 2, 1, 3, 64, 16, [20, 5], "tree")
    args = p.device(cuda)
    one = torch.empty((1, 2, 3, 64), dtype=torch.float16, device=cuda).expand(2, 2, 3, 64)
    with pytest.raises(RuntimeError, match="overlap"):
        fl.forward_tree(out=one, **args)
    pos = torch.zeros((2, 3), dtype=torch.int32, device=cuda)
    freqs, _ = fl.rotary_frequencies(64, device=cuda)
    with pytest.raises(RuntimeError, match="overlap"):
        fl.forward_rotary(args["q"], None, pos, freqs, q_out=one)


@pytest.mark.parametrize("dtype,d", KINDS)
@pytest.mark.parametrize("b,h,hk,n,lengths,tree", [
    (2, 8, 8, 1, [3000, 0], None),
    (1, 16, 16, 1, [2500], None),
    (5, 8, 4, 3, [100, 0, 1700, 5, 64], "tree"),
    (3, 12, 12, 20, [7, 600, 0], "any"),
    (2, 32, 4, 4, [900, 2000], None),
])
@pytest.mark.parametrize("rows_first", [True, False])
def test_heads_side_by_side(cuda, dtype, d, b, h, hk, n, lengths, tree, rows_first):
    """Long tables of caches whose heads lie side by side, and of others; blocks
    nobody has and NaN rows among them."""
    p = Problem(73 + n, dtype, b, h, hk, n, d, 16, lengths, tree, ragged=n > 1, table_pad=ROOM,
                rows_first=rows_first)
    p.tables[0, 2] = -1
    p.k[int(p.tables[0, 3]), hk - 1, 5, 1] = float("nan")   # one head's rows
    p.v[int(p.tables[0, 4]), 0, 5, 1] = float("inf")
    check(*run(p, cuda), p)


@pytest.mark.parametrize("group,n", ROWS)
def test_less_workspace_runs_one_pass(cuda, group, n):
    """The C entry with no workspace, one byte too little, and enough; one
    that is not aligned is refused; the memory behind a workspace stays."""
    import ctypes

    import torch

    from flashlite_amd import capi

    p = Problem(74 + n, "bfloat16", 2, 4 * group, 4, n, 64, 16, [1800, 40], "tree", table_pad=ROOM)
    ref = p.reference()
    a = p.device(cuda)
    out = torch.zeros_like(a["q"])
    t3 = ctypes.c_int64 * 3
    f = capi.FlTreeParams(
        q=a["q"].data_ptr(), k_cache=a["k_cache"].data_ptr(), v_cache=a["v_cache"].data_ptr(),
        o=out.data_ptr(), lse=None, q_stride=t3(*a["q"].stride()[:3]),
        o_stride=t3(*out.stride()[:3]), k_stride=t3(*a["k_cache"].stride()[:3]),
        v_stride=t3(*a["v_cache"].stride()[:3]), block_tables=a["block_tables"].data_ptr(),
        table_stride=a["block_tables"].stride(0), lengths=a["lengths"].data_ptr(), counts=None,
        mask=a["mask"].data_ptr(), mask_stride=a["mask"].stride(0), batch=2, heads=4 * group,
        kv_heads=4, drafts=n, head_dim=64, num_blocks=a["k_cache"].shape[0], block_size=16,
        max_blocks=a["block_tables"].shape[1], sm_scale=0.0, dtype=capi.DTYPE_BF16)
    lib = capi.load()
    lib.fl_attn_tree_workspace_bytes.restype = ctypes.c_int64
    need = lib.fl_attn_tree_workspace_bytes(ctypes.byref(f))
    assert need > 0 and need == fl.tree_workspace_bytes(a["q"], a["k_cache"])
    ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device=cuda)
    st = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def call(at, size):
        out.zero_()
        rc = lib.fl_attn_tree_fwd(ctypes.byref(f), ctypes.c_void_p(at), ctypes.c_int64(size), st)
        torch.cuda.synchronize()
        return rc

    for at, size in ((None, 0), (None, need), (ws.data_ptr(), need - 1)):
        assert call(at, size) == capi.FL_OK
        check(out, None, p, ref)
        assert bool((ws == 77).all())
    assert call(ws.data_ptr() + 4, need) == capi.FL_ERR_MISALIGNED
    assert bool((out == 0).all())
    assert call(ws.data_ptr(), need) == capi.FL_OK
    check(out, None, p, ref)
    assert bool((ws[need:] == 77).all()) and not bool((ws[:need] == 77).all())
