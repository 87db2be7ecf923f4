"""The rotary operators against float64, and the rows they store in a cache.

A rotated value is a cos - b sin with 32-bit sine and cosine of an angle that
was reduced in 64 bits: each is off by at most 2^-22 (the argument's rounding,
2^-24 of half a turn, and the function's last places), so the value by
2^-21 (|a| + |b|) scale, plus half a step of its own type.
"""

import numpy as np
import pytest

import flashlite_amd as fl
from oracle import paged

pytestmark = pytest.mark.gpu

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}


def draw(rs, shape, dtype, dev):
    """A contiguous tensor of `dtype` and its exact float64 values."""
    import torch

    t = torch.from_numpy(rs.standard_normal(shape).astype(np.float32)).to(getattr(torch, dtype))
    return t.to(dev), t.double().numpy()


def assert_rotated(got, x, want, dtype, pairs, inter, scale):
    bound = np.zeros_like(want)
    r = 2 * pairs
    if pairs:
        a, c = (x[..., 0:r:2], x[..., 1:r:2]) if inter else (x[..., :pairs], x[..., pairs:r])
        size = (np.abs(a) + np.abs(c)) * scale * 2.0 ** -21
        if inter:
            bound[..., 0:r:2] = bound[..., 1:r:2] = size
        else:
            bound[..., :pairs] = bound[..., pairs:r] = size
    bound[..., :r] += HALF_STEP[dtype] * np.abs(want[..., :r]) + 2.0 ** -25  # fp16's smallest step
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), f"{(err / np.maximum(bound, 1e-300)).max():.3g} of the bound"


def views(t, layout):
    """[B, H, N, D] tensors as the layout's view of the same values."""
    return t if layout == "bhnd" else t.transpose(1, 2).contiguous().transpose(1, 2)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,h,hk,n,d,pairs,layout,first,scale", [
    (1, 1, 1, 1, 64, 32, "bhnd", 0, 1.0),
    (2, 8, 2, 33, 64, 32, "bnhd", 100, 1.0),
    (1, 5, 5, 7, 128, 64, "bhnd", 131000, 1.2),
    (3, 7, 1, 65, 128, 32, "bnhd", 1 << 20, 0.5),
    (2, 3, 3, 17, 64, 10, "bnhd", 5, 1.0),
    (2, 3, 3, 17, 128, 5, "bhnd", 5, 1.0),
    (2, 3, 2, 19, 128, 4, "bhnd", 77, 1.0),
    (1, 2, 2, 9, 64, 1, "bnhd", 2000000000, 1.0),
    (2, 2, 2, 9, 64, 0, "bhnd", 3, 1.0),
    (1, 24, 8, 700, 128, 64, "bnhd", 0, 1.0),
])
def test_forward_and_backward(cuda, dtype, inter, b, h, hk, n, d, pairs, layout, first, scale):
    import torch

    rs = np.random.RandomState(n + d)
    q, q64 = draw(rs, (b, h, n, d), dtype, cuda)
    k, k64 = draw(rs, (b, hk, n, d), dtype, cuda)
    positions = first + rs.randint(0, 50, (b, 1)) + np.arange(n)
    freqs = 10000.0 ** (-np.arange(pairs) / max(pairs, 1))
    pos = torch.from_numpy(positions).to(cuda)
    pos = pos.int() if first < 2 ** 31 - 1000 and n % 2 else pos
    f = torch.from_numpy(freqs).to(cuda)
    for turn, transpose in ((fl.forward_rotary, False), (fl.backward_rotary, True)):
        qo, ko = turn(views(q, layout), views(k, layout), pos, f, inter, scale)
        assert qo.shape == q.shape and qo.dtype == q.dtype
        for got, x in ((qo, q64), (ko, k64)):
            assert_rotated(got, x, paged.rotary(x, positions, freqs, inter, scale, transpose),
                           dtype, pairs, inter, scale)
            assert torch.equal(got[..., 2 * pairs:].double().cpu(),
                               torch.from_numpy(x[..., 2 * pairs:].copy()))


@pytest.mark.parametrize("inter", [False, True])
def test_gradient_against_differences(cuda, inter):
    """d/dx of sum(w rotary(x)) by central differences of the forward pass
    (linear: the step 1 is exact up to rounding, 2^-22 of a value), and by
    torch's own derivative of the formula."""
    import torch

    rs = np.random.RandomState(3)
    n, d, pairs = 5, 64, 24
    x, x64 = draw(rs, (1, 2, n, d), "float32", cuda)
    w, w64 = draw(rs, (1, 2, n, d), "float32", cuda)
    pos = torch.arange(40, 40 + n, device=cuda)
    freqs = fl.rotary_frequencies(2 * pairs, device=cuda)[0]
    dx = fl.backward_rotary(w, None, pos, freqs, inter, 1.3)
    got = dx.double().cpu().numpy()
    for c in (0, 1, 23, 24, 47, 48, 63):
        e = torch.zeros_like(x)
        e[..., c] = 1.0
        up = fl.forward_rotary(x + e, None, pos, freqs, inter, 1.3)
        down = fl.forward_rotary(x - e, None, pos, freqs, inter, 1.3)
        slope = ((up.double() - down.double()) * w.double()).sum(-1).cpu().numpy() / 2
        # each of the two values that move is off by 2^-21 (|a| + |b|) 1.3 twice over
        size = 2.0 ** -19 * 1.3 * (np.abs(x64).max() + 1) * 2 * np.abs(w64).max()
        assert np.abs(slope - got[..., c]).max() <= size
    leaf = torch.from_numpy(x64).requires_grad_()
    angle = pos.double().cpu()[:, None] * freqs.cpu()
    cos, sin = angle.cos() * 1.3, angle.sin() * 1.3
    a, b = ((leaf[..., 0:2 * pairs:2], leaf[..., 1:2 * pairs:2]) if inter
            else (leaf[..., :pairs], leaf[..., pairs:2 * pairs]))
    wa, wb = ((w64[..., 0:2 * pairs:2], w64[..., 1:2 * pairs:2]) if inter
              else (w64[..., :pairs], w64[..., pairs:2 * pairs]))
    loss = ((a * cos - b * sin) * torch.from_numpy(wa.copy())).sum()
    loss = loss + ((a * sin + b * cos) * torch.from_numpy(wb.copy())).sum()
    loss = loss + (leaf[..., 2 * pairs:] * torch.from_numpy(w64[..., 2 * pairs:].copy())).sum()
    loss.backward()
    err = np.abs(got - leaf.grad.numpy())
    assert err.max() <= 2.0 ** -20 * 1.3 * 2 * np.abs(w64).max()


def test_shared_positions_in_place_and_no_k(cuda):
    import torch

    rs = np.random.RandomState(4)
    q, q64 = draw(rs, (3, 4, 21, 128), "bfloat16", cuda)
    f = fl.rotary_frequencies(128, device=cuda)[0]
    pos = torch.arange(21, device=cuda)
    want = fl.forward_rotary(q, None, pos[None].expand(3, 21), f)
    assert torch.equal(fl.forward_rotary(q, None, pos, f), want)
    assert torch.equal(fl.forward_rotary(q, None, pos.int(), f), want)
    k = q.clone()
    out = fl.forward_rotary(q, k, pos, f, q_out=q, k_out=k)
    assert out[0].data_ptr() == q.data_ptr() and out[1].data_ptr() == k.data_ptr()
    assert torch.equal(q, want) and torch.equal(k, want)


def test_slice_of_projections(cuda):
    """q and k as slices of one [B, N, (H + 2 H_k) D] projection; rows between
    stay as they were."""
    import torch

    rs = np.random.RandomState(5)
    b, n, h, hk, d = 2, 11, 6, 2, 64
    x, x64 = draw(rs, (b, n, (h + 2 * hk) * d), "float16", cuda)
    y = x.clone().view(b, n, h + 2 * hk, d).transpose(1, 2)
    f = fl.rotary_frequencies(d, device=cuda)[0]
    pos = torch.arange(n, device=cuda)
    q, k = y[:, :h], y[:, h:h + hk]
    fl.forward_rotary(q, k, pos, f, q_out=q, k_out=k)
    full = x64.reshape(b, n, h + 2 * hk, d).transpose(0, 2, 1, 3)
    want = paged.rotary(full, np.tile(np.arange(n), (b, 1)), f.cpu().numpy())
    assert_rotated(y[:, :h + hk], full[:, :h + hk], want[:, :h + hk], "float16", 32, False, 1.0)
    assert np.array_equal(y[:, h + hk:].double().cpu().numpy(), full[:, h + hk:])


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,h,hk,n,d,pairs,block,paged_rows", [
    (1, 1, 1, 1, 64, 32, 16, True), (32, 8, 2, 1, 128, 64, 16, True),
    (3, 6, 3, 40, 64, 32, 20, False), (2, 4, 4, 70, 128, 32, 257, False),
    (2, 3, 1, 9, 128, 10, 8, True), (4, 2, 2, 5, 64, 0, 1, False)])
def test_store(cuda, dtype, inter, b, h, hk, n, d, pairs, block, paged_rows):
    """Rotated k and v in their rows, everything else as it was; tokens
    without a slot, or with one past the cache, are passed over."""
    import torch

    rs = np.random.RandomState(n + b)
    blocks = (b * n + block - 1) // block + 3
    q, q64 = draw(rs, (b, h, n, d), dtype, cuda)
    k, k64 = draw(rs, (b, hk, n, d), dtype, cuda)
    v, v64 = draw(rs, (b, hk, n, d), dtype, cuda)
    shape = (blocks, block, hk, d) if paged_rows else (blocks, hk, block, d)
    caches = []
    for _ in range(2):
        c, c64 = draw(rs, shape, dtype, cuda)
        caches.append((c.transpose(1, 2), c64.transpose(0, 2, 1, 3)) if paged_rows else (c, c64))
    (kc, kc64), (vc, vc64) = caches
    slots = rs.permutation(blocks * block)[:b * n].reshape(b, n)
    slots[rs.rand(b, n) < 0.2] = -1
    if n > 4:
        slots[0, 1], slots[0, 2] = blocks * block, -(2 ** 40)
    positions = rs.randint(0, 9000, (b, n))
    freqs = 10000.0 ** (-np.arange(pairs) / max(pairs, 1))
    out = torch.full_like(q, 7.0)
    got = fl.rotary_to_cache(views(q, "bnhd"), views(k, "bnhd"), views(v, "bhnd"),
                             torch.from_numpy(positions).to(cuda), torch.from_numpy(slots).to(cuda),
                             torch.from_numpy(freqs).to(cuda), kc, vc, inter, 1.0, out)
    assert got.data_ptr() == out.data_ptr()
    there = (slots >= 0) & (slots < blocks * block)
    rows = np.broadcast_to(there[:, None], (b, h, n))
    qw = paged.rotary(q64, positions, freqs, inter)
    keep = torch.from_numpy(rows.copy())
    assert bool((out.cpu()[~keep] == 7.0).all())
    assert_rotated(out.cpu()[keep], q64[rows], qw[rows], dtype, pairs, inter, 1.0)
    kw = paged.rotary(k64, positions, freqs, inter)
    written = np.zeros((blocks, block), bool)
    kx = kc.double().cpu().numpy()
    vx = vc.double().cpu().numpy()
    for i, j in np.argwhere(there):
        blk, row = divmod(int(slots[i, j]), block)
        written[blk, row] = True
        assert_rotated(kc[blk, :, row], k64[i, :, j], kw[i, :, j], dtype, pairs, inter, 1.0)
        assert np.array_equal(vx[blk, :, row], v64[i, :, j])
    left = np.broadcast_to(~written[:, None], (blocks, hk, block))
    assert np.array_equal(kx[left], kc64[left]) and np.array_equal(vx[left], vc64[left])


def test_far_cache_rows(cuda):
    """Rows past 32-bit byte offsets of a cache of more than 4 GiB."""
    import torch

    blocks, block, d = 260, 65536, 64  # 2 x 2.2 GB: rows up to 2^31 bytes and beyond
    cache = torch.zeros((2, blocks, 1, block, d), dtype=torch.float16, device=cuda)
    kc, vc = cache[:, :, :, :, :].unbind(0)
    rs = np.random.RandomState(6)
    q, _ = draw(rs, (1, 1, 4, d), "float16", cuda)
    k, k64 = draw(rs, (1, 1, 4, d), "float16", cuda)
    slots = torch.tensor([[blocks * block - 1, 16777216, 16777215, 0]], device=cuda)
    f = torch.zeros((0,), dtype=torch.float64, device=cuda)
    fl.rotary_to_cache(q, k, k, torch.zeros((1, 4), dtype=torch.int32, device=cuda), slots, f, kc, vc)
    for c in (kc, vc):
        rows = c.reshape(blocks * block, d)[slots[0]]
        assert np.array_equal(rows.double().cpu().numpy(), k64[0, 0])
        assert int((c != 0).any(-1).sum()) == 4


def test_refusals(cuda):
    import torch

    x = torch.zeros((2, 3, 5, 64), dtype=torch.float16, device=cuda)
    f = torch.zeros((32,), dtype=torch.float64, device=cuda)
    pos = torch.zeros((2, 5), dtype=torch.int32, device=cuda)
    for args, text in (((x, x, pos, f.float()), "freqs"), ((x, x, pos.float(), f), "positions"),
                       ((x, x, pos[:, :4], f), "positions"), ((x, x.float(), pos, f), "dtype"),
                       ((x, x[:, :, :4], pos, f), "k must be"), ((x[0], x, pos, f), "4D"),
                       ((x.double(), None, pos, f), "FP16"),
                       ((x, x, pos, torch.zeros(33, dtype=torch.float64, device=cuda)), "pairs"),
                       ((x[..., :48], None, pos, f[:8]), "head_dim"),
                       ((x.transpose(2, 3).contiguous().transpose(2, 3), None, pos, f), "unit-stride")):
        with pytest.raises(RuntimeError, match=text):
            fl.forward_rotary(*args)
    with pytest.raises(RuntimeError, match="k_out"):
        fl.forward_rotary(x, None, pos, f, k_out=x)
    c = torch.zeros((4, 3, 16, 64), dtype=torch.float16, device=cuda)
    slots = torch.zeros((2, 5), dtype=torch.int64, device=cuda)
    for args, text in (((x, x, x, pos, slots.int(), f, c, c), "slots"),
                       ((x, x, x, pos, slots, f, c[:, :2], c[:, :2]), "caches"),
                       ((x, x, x[:, :2], pos, slots, f, c, c), "v must"),
                       ((x, x, x, pos, slots[0], f, c, c), "slots"),
                       ((x.float(), x.float(), x.float(), pos, slots, f, c.float(), c.float()),
                        "FP16")):
        with pytest.raises(RuntimeError, match=text):
            fl.rotary_to_cache(*args)
