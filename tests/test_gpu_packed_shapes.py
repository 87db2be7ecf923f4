"""Sequences long enough that each work-group shape of forward_packed is
launched (key ranges in halves, block pairs, 256 rows), against float64 on the
GPU within packed_util's bounds; one of them with a NaN in V."""

import numpy as np
import pytest

from packed_util import Problem, check
import flashlite_amd as fl

pytestmark = pytest.mark.gpu


def reference(p, dev):
    """packed.attention's results, one sequence and head at a time on the GPU."""
    import torch

    q, k, v = (x.to(dev).double() for x in (p.q, p.k, p.v))
    out, weight = torch.full_like(q, float("nan")), torch.zeros_like(q)
    lse, reach = torch.full(q.shape[:2], float("nan"), dtype=torch.float64, device=dev), None
    reach = torch.zeros_like(lse)
    for a, b, c, e in zip(p.starts, p.starts[1:], p.key_starts, p.key_starts[1:]):
        for h in range(p.h):
            kk, vv = (x[h // (p.h // p.hk), c:e] for x in (k, v))
            s = q[h, a:b] @ kk.t().contiguous() * p.scale
            hidden = torch.zeros((b - a, e - c), dtype=torch.bool, device=dev)
            if p.causal:
                hidden = (torch.arange(e - c, device=dev) - (e - c - (b - a))
                          > torch.arange(b - a, device=dev)[:, None])
            s = s.masked_fill(hidden, -float("inf"))
            lse[h, a:b] = torch.logsumexp(s, -1)
            w = torch.softmax(s, -1)
            odd = torch.isnan(vv)
            out[h, a:b] = w @ torch.where(odd, 0.0, vv)
            weight[h, a:b] = w @ torch.where(odd, 0.0, vv).abs()
            seen = (~hidden).double() @ odd.double()
            out[h, a:b] = torch.where(seen > 0, float("nan"), out[h, a:b])
            reach[h, a:b] = ((q[h, a:b].abs() @ kk.abs().t().contiguous())
                             .masked_fill(hidden, 0.0).amax(-1) * abs(p.scale))
    return tuple(x.cpu().numpy() for x in (out, lse, weight, reach))


@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 64), ("float16", 128),
                                     ("bfloat16", 128)])
@pytest.mark.parametrize("nan", [False, True])
@pytest.mark.parametrize("h,hk,lengths,causal", [
    (2, 1, [700], True),                      # 64 rows, key range in halves
    (2, 1, [700], False),
    (8, 2, [1450, 533, 1100, 900], True),     # 128 rows, in halves
    (8, 2, [4100], False),
    (8, 2, [4077], True),                     # pairs of 64-row blocks
    (8, 2, [4000, 4111], True),               # pairs of 128-row blocks
    (16, 16, [2301, 2050], False),            # 256 rows
    (16, 4, [4200], True),
])
def test_shapes(cuda, dtype, d, nan, h, hk, lengths, causal):
    p = Problem(sum(lengths) + h, dtype, d, h, hk, lengths, None, causal, "rows", 2)
    if nan:
        p.v[0, 2 + lengths[0] * 3 // 4, 7] = float("nan")
    out, lse = fl.forward_packed(**p.device(cuda), return_lse=True)
    check(out, lse, p, reference(p, cuda))


def test_more_keys_than_rows_over_long_sequences(cuda):
    """Chunks of a prompt after cached tokens, in each shape's key ranges."""
    for h, lengths, keys in ((2, [100, 1], [3000, 700]), (8, [900, 65], [2000, 3100]),
                             (8, [2000], [5000])):
        p = Problem(h, "bfloat16", 128, h, h // 2, lengths, keys, True, "heads", 1)
        out, lse = fl.forward_packed(**p.device(cuda), return_lse=True)
        check(out, lse, p, reference(p, cuda))


@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("nan", [False, True])
@pytest.mark.parametrize("h,hk,lengths,causal", [
    (4, 1, [130, 0, 61], True), (2, 1, [700], True), (8, 2, [1450, 533, 1100, 900], True),
    (8, 2, [4077], True), (8, 2, [4000, 4111], True), (16, 4, [4200], True),
    (16, 16, [2301, 2050], False)])
def test_out_over_q(cuda, dtype, d, nan, h, hk, lengths, causal):
    """The output in q's own place, in each shape."""
    import torch

    p = Problem(sum(lengths) + 1, dtype, d, h, hk, lengths, None, causal, "heads", 2)
    if nan:
        p.v[0, 2 + lengths[0] // 2, 7] = float("nan")
    a = p.device(cuda)
    want = fl.forward_packed(**a)
    a["q"] = a["q"].clone()
    got = fl.forward_packed(**a, out=a["q"])
    there = torch.from_numpy(p.inside()).to(cuda)
    assert got.data_ptr() == a["q"].data_ptr()
    assert torch.equal(torch.nan_to_num(got[:, :, there]), torch.nan_to_num(want[:, :, there]))
    assert torch.equal(got.isnan()[:, :, there], want.isnan()[:, :, there])


@pytest.mark.parametrize("dtype,d", [("float16", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("lengths", [[40, 0, 7], [300, 129]])
def test_gradient_of_a_broadcast(cuda, dtype, d, lengths):
    """dout of stride 0 along the heads, the rows, both: as one that is spelled
    out, bit for bit."""
    import torch

    p = Problem(sum(lengths), dtype, d, 4, 2, lengths, None, True, "rows", 1)
    a = p.device(cuda)
    out, lse = fl.forward_packed(**a, return_lse=True)
    dout = p.dout.nan_to_num().to(cuda)[None]
    how = (a["q"], a["k"], a["v"], out, lse, a["starts"], None, a["sm_scale"], True)
    for part in (dout[:, :1], dout[:, :, 3:4], dout[:, :1, 3:4]):
        wide = part.expand_as(a["q"])
        for x, y in zip(fl.backward_packed(wide, *how), fl.backward_packed(wide.contiguous(), *how)):
            assert torch.equal(x.nan_to_num(), y.nan_to_num())
