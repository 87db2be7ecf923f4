"""Attention over packed sequences and its gradients against float64
(tests/packed_util.py has the bounds), one after the other as a training step
runs them."""

import numpy as np
import pytest

import flashlite_amd as fl
from packed_util import Problem, check, check_gradients

pytestmark = pytest.mark.gpu

BOTH = [("float16", 64), ("bfloat16", 64), ("float16", 128), ("bfloat16", 128)]


def run(p, dev, backward=True, ref=None):
    import torch

    a = p.device(dev)
    out = torch.full_like(a["q"], 7.0)
    lse = torch.full((1, p.h, p.rows), 7.0, device=dev)
    got, got_lse = fl.forward_packed(**a, out=out, return_lse=True, lse=lse)
    assert got is not None and got.data_ptr() == out.data_ptr()
    check(out, lse, p, ref)
    outside = torch.from_numpy(~p.inside()).to(dev)
    assert (out[:, :, outside] == 7.0).all() and (lse[:, :, outside] == 7.0).all()
    plain = fl.forward_packed(**a)  # (its own output: zeros where there is no sequence)
    assert torch.equal(torch.nan_to_num(plain[:, :, ~outside]),
                       torch.nan_to_num(out[:, :, ~outside]))
    assert (plain[:, :, outside] == 0).all()
    if not backward:
        return
    dout = p.view(p.dout, dev)
    grads = [torch.full_like(a[x], 7.0) for x in "qkv"]
    got = fl.backward_packed(dout, a["q"], a["k"], a["v"], out, lse, a["starts"], a["key_starts"],
                             a["sm_scale"], a["is_causal"], *grads)
    check_gradients(got, p, out, lse)
    key_outside = torch.from_numpy(~p.inside(True)).to(dev)
    for g, t, rows in zip(got, grads, (outside, key_outside, key_outside)):
        assert g.data_ptr() == t.data_ptr() and (t[:, :, rows] == 7.0).all()
    again = fl.backward_packed(dout, a["q"], a["k"], a["v"], out, lse, a["starts"],
                               a["key_starts"], a["sm_scale"], a["is_causal"])
    for g, t, rows in zip(again, grads, (outside, key_outside, key_outside)):
        assert (g[:, :, rows] == 0).all()
        assert torch.equal(g[:, :, ~rows].view(torch.int16), t[:, :, ~rows].view(torch.int16))


@pytest.mark.parametrize("dtype,d", BOTH)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,lengths,layout,gap", [
    (1, 1, [1], "rows", 0),
    (2, 2, [1, 0, 1], "heads", 3),
    (2, 1, [0, 0], "rows", 2),
    (3, 1, [17, 64, 3, 0, 129, 31, 32, 33], "rows", 0),
    (4, 2, [300, 5], "qkv", 1),
    (8, 1, [127, 128, 65], "heads", 0),
    (8, 8, [63, 200], "qkv", 70),
    (2, 2, [7] * 70, "rows", 0),
    (1, 1, [3, 0, 1, 2] * 160, "rows", 5),
])
def test_packed(cuda, dtype, d, causal, h, hk, lengths, layout, gap):
    run(Problem(len(lengths) + d, dtype, d, h, hk, lengths, None, causal, layout, gap), cuda)


@pytest.mark.parametrize("dtype,d", BOTH)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,lengths,keys", [
    (2, 1, [1, 1, 1, 1], [300, 1, 0, 65]),          # single tokens after cached ones
    (2, 2, [5, 0, 40, 130], [70, 33, 40, 129]),      # more, none, as many, fewer keys
    (4, 1, [200, 3], [20, 0]),                       # rows that see nothing
    (1, 1, [0, 0], [10, 200]),                       # keys that nobody sees
])
def test_packed_other_keys(cuda, dtype, d, causal, h, hk, lengths, keys):
    run(Problem(sum(keys) + d, dtype, d, h, hk, lengths, keys, causal, "rows", 1), cuda)


@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("lengths,keys", [
    ([0, 1, 130, 5, 0, 0, 257, 2] * 66, [3, 0, 200, 5, 1, 0, 20, 300] * 66),
    ([1, 0, 2] * 1500, None),
])
def test_packed_many_sequences(cuda, dtype, d, lengths, keys):
    """More than a wave or eight of them look at once."""
    run(Problem(6, dtype, d, 2, 1, lengths, keys, True, "rows", 3), cuda)


@pytest.mark.parametrize("dtype,d", BOTH)
@pytest.mark.parametrize("scale,q_scale", [(-0.3, 1.0), (1.0, 3.0), (0.02, 0.1)])
def test_packed_scales(cuda, dtype, d, scale, q_scale):
    """Negative, peaked (rows leave the first tile's range: the checked pass)
    and flat scores."""
    run(Problem(9, dtype, d, 2, 1, [150, 70], None, True, "rows", 0, scale, q_scale), cuda)


@pytest.mark.parametrize("dtype,d", BOTH)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_lowest_scores(cuda, dtype, d, causal):
    """Scores far apart and of the type's lowest values keep finite results."""
    import torch

    p = Problem(4, dtype, d, 2, 2, [90, 40], None, causal)
    p.q[0, 10:20] = 0.0
    p.k[0, 5:9] = -200.0
    p.q[1] = torch.abs(p.q[1]) * 8
    p.k[1, ::3] = -30.0
    run(p, cuda)


@pytest.mark.parametrize("dtype,d", BOTH)
def test_nan_and_infinities_stay_where_they_are_seen(cuda, dtype, d):
    """A NaN or infinity in a row of q, k, v or dout reaches the rows that see
    it, and neither earlier rows nor other sequences nor other heads."""
    for seed, plant in enumerate([("k", 40, np.nan), ("v", 40, np.nan), ("v", 41, np.inf),
                                  ("q", 70, np.nan), ("dout", 70, np.nan), ("k", 99, np.nan),
                                  ("v", 99, -np.inf), ("dout", 33, np.inf)]):
        name, row, value = plant
        p = Problem(seed, dtype, d, 2, 1, [33, 67, 50], None, True, "rows", 2)
        getattr(p, name)[0, 2 + row, 5] = value
        run(p, cuda)
        other = Problem(seed, dtype, d, 2, 1, [33, 67, 50], None, False, "heads", 2)
        getattr(other, name)[0, 2 + row, 5] = value
        run(other, cuda)


@pytest.mark.parametrize("dtype,d", BOTH)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h,hk,lengths", [
    (2, 1, [33, 67, 50] + [0] * 600),            # beyond what is ranked over all sequences
    (18, 1, [110, 129, 0, 40] + [0] * 58),       # key blocks in parts
])
def test_gradients_in_two_launches(cuda, dtype, d, causal, h, hk, lengths):
    """More work-groups than one launch takes for dq with dk and dv (empty
    sequences have work-groups too), with and without NaN and infinities."""
    for plant in (None, ("v", 40, np.nan)) if h > 2 else (None, ("dout", 70, np.inf),
                                                          ("k", 99, np.nan)):
        p = Problem(h + d, dtype, d, h, hk, lengths, None, causal, "rows", 2)
        if plant is not None:
            name, row, value = plant
            getattr(p, name)[0, 2 + row, 5] = value
        run(p, cuda)


def test_gradient_against_differences(cuda):
    """Directional differences of sum(dout out) in 64 bits of the oracle, which
    the kernel's gradients must follow: |g . e - slope| within the step's third
    order and the gradients' rounding."""
    from oracle import packed

    p = Problem(5, "float16", 64, 2, 1, [20, 13], [25, 13], True)
    a = p.device(cuda)
    out, lse = fl.forward_packed(**a, return_lse=True)
    dout = p.view(p.dout, cuda)
    grads = fl.backward_packed(dout, a["q"], a["k"], a["v"], out, lse, a["starts"],
                               a["key_starts"], is_causal=True)
    x = p.arrays()
    rs = np.random.RandomState(6)
    w = p.dout.double().numpy()

    def loss(y):
        return (w * packed.attention(*y, p.starts, p.key_starts, True, p.scale)[0]).sum()

    for i, g in enumerate(grads):
        e = rs.standard_normal(x[i].shape)
        e /= np.linalg.norm(e)
        step = 1e-4
        up, down = ([y + s * step * e if j == i else y for j, y in enumerate(x)] for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * step)
        g64 = g[0].double().cpu().numpy()
        # each gradient value is within 2^-9 of its own size and that of its
        # terms, which are at most some 8 times the root of the mean square
        bound = 8 * 2.0 ** -9 * np.linalg.norm(g64) + 1e-6
        assert abs((g64 * e).sum() - slope) <= bound


@pytest.mark.parametrize("seed", range(24))
def test_random_problems(cuda, seed):
    rs = np.random.RandomState(100 + seed)
    hk = int(rs.choice([1, 1, 2, 3]))
    h = hk * int(rs.choice([1, 2, 3, 7]))
    n = int(rs.choice([1, 2, 5, 20]))
    most = 500 // n + 1
    lengths = rs.randint(0, most, n).tolist()
    kind = rs.choice(["same", "same", "more", "apart"])
    keys = (None if kind == "same" else (rs.randint(0, most, n) + lengths).tolist()
            if kind == "more" else rs.randint(0, most, n).tolist())
    dtype, d = BOTH[seed % 4]
    layout = rs.choice(["rows", "heads"] + (["qkv"] if keys is None else []))
    run(Problem(seed, dtype, d, h, hk, lengths, keys, bool(rs.rand() < 0.6), str(layout),
                int(rs.choice([0, 9])), q_scale=float(rs.choice([0.3, 1.0, 2.0]))), cuda)


@pytest.mark.parametrize("dtype,d", BOTH)
def test_equals_the_dense_kernels_over_one_length(cuda, dtype, d):
    """Sequences of one length are a dense batch."""
    import torch

    b, h, n = 3, 2, 192
    q, k, v = (torch.randn((b, h, n, d), device=cuda).to(getattr(torch, dtype)) for _ in range(3))
    flat = [x.transpose(0, 1).reshape(1, h, b * n, d) for x in (q, k, v)]
    starts = torch.arange(0, (b + 1) * n, n, dtype=torch.int32, device=cuda)
    got, lse = fl.forward_packed(*flat, starts, is_causal=True, return_lse=True)
    want, want_lse = fl.forward_flash2_ex(q, k, v, is_causal=True, return_lse=True)
    got = got.view(h, b, n, d).transpose(0, 1)
    # two roundings of the same value, each as in packed_util
    step = 2.0 ** -8 if dtype == "bfloat16" else 2.0 ** -11
    assert (got.double() - want.double()).abs().max() <= 8 * step * want.double().abs().max()
    lse = lse.view(h, b, n).transpose(0, 1)
    assert (lse - want_lse).abs().max() <= 4 * step


def test_starts_out_of_range_are_not_followed(cuda):
    """Falling, negative and too large starts: memory outside is neither read
    nor written; sequences that are in order are as they should be."""
    import torch

    d, h, t = 64, 2, 100
    x = torch.full((3, 1, h, t + 200, d), float("nan"), dtype=torch.float16, device=cuda)
    q, k, v = (y[:, :, 100:100 + t] for y in x)
    for y in (q, k, v):
        y.copy_(torch.randn(y.shape, device=cuda))
    whole = torch.full((1, h, t + 200, d), 7.0, dtype=torch.float16, device=cuda)
    out = whole[:, :, 100:100 + t]
    lse = torch.zeros((1, h, t), device=cuda)
    starts = torch.tensor([-5, 40, 30, 90, 1 << 30], dtype=torch.int32, device=cuda)
    fl.forward_packed(q, k, v, starts, is_causal=True, out=out, return_lse=True, lse=lse)
    assert (whole[:, :, :100] == 7.0).all() and (whole[:, :, 100 + t:] == 7.0).all()
    one = fl.forward_packed(q[:, :, 90:], k[:, :, 90:], v[:, :, 90:],
                            torch.tensor([0, 10], dtype=torch.int32, device=cuda), is_causal=True)
    assert torch.equal(out[:, :, 90:], one)
    grads = fl.backward_packed(torch.ones_like(q), q, k, v, out, lse, starts, is_causal=True)
    assert all(torch.isfinite(g[:, :, 90:]).all() for g in grads)


@pytest.mark.parametrize("dtype,d", BOTH)
@pytest.mark.parametrize("h,hk,lengths,causal", [
    (7, 1, [400], True), (3, 3, [257, 31], False), (8, 2, [1500], True), (2, 1, [1, 700, 0], True)])
def test_key_blocks_in_parts(cuda, dtype, d, h, hk, lengths, causal):
    """Few key blocks: their queries are dealt to several work-groups."""
    run(Problem(sum(lengths), dtype, d, h, hk, lengths, None, causal, "heads", 3), cuda)
