"""Norms of q and k with rotary positions of one or several axes, their
gradients and the rows they store, against float64.

u is half a step of the element type.  A row's 1 / sqrt(mean + eps) is off by
half of the sum's (D + 8) 2^-24 and 2^-22 of the hardware's root: `root`,
relative; each product adds 2^-24.  Rotated values: 2^-21 (|a| + |b|) scale for
the sine and cosine (tests/test_gpu_rotary.py).  Gradients: g is such a rotated
value; dx's terms carry root three times and (D + 16) 2^-24 of their sums; dw's
root, a product and (rows + 64) 2^-24 of its terms' absolute sum.
"""

import numpy as np
import pytest

import flashlite_amd as fl
from oracle import packed

pytestmark = pytest.mark.gpu

HALF_STEP = {"float16": 2.0 ** -11, "bfloat16": 2.0 ** -8, "float32": 2.0 ** -24}
SMALL = 2.0 ** -25  # fp16's smallest step


def draw(rs, shape, dtype, dev, layout="bhnd"):
    import torch

    t = torch.from_numpy(rs.standard_normal(shape).astype(np.float32)).to(getattr(torch, dtype))
    x = t.double().numpy()
    t = t.to(dev)
    return (t if layout == "bhnd" else t.transpose(1, 2).contiguous().transpose(1, 2)), x


def root(d):
    return (d + 8) * 2.0 ** -25 + 2.0 ** -22 + 2.0 ** -22


def pair_size(x, pairs, inter):
    """|a| + |b| of each rotated column, 0 of the others."""
    out = np.zeros_like(x)
    cols = (np.arange(2 * pairs).reshape(-1, 2).T if inter
            else np.stack([np.arange(pairs), np.arange(pairs) + pairs]))
    a, b = cols
    size = np.abs(x[..., a]) + np.abs(x[..., b])
    out[..., a] = out[..., b] = size
    return out


def assert_within(got, want, bound, what):
    got = got.double().cpu().numpy()
    err = np.abs(got - want)
    assert np.isfinite(got).all(), what
    assert (err <= bound).all(), f"{what}: {(err / bound).max():.3g} of the bound"


def forward_bound(x, w, want, dtype, pairs, inter, scale, eps):
    y = x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    size = pair_size(y, pairs, inter) * scale
    size[..., 2 * pairs:] = np.abs(y[..., 2 * pairs:])
    rel = 0.0 if w is None else root(x.shape[-1])
    bound = size * (rel + 2.0 ** -22) + pair_size(y, pairs, inter) * scale * 2.0 ** -21
    return bound + HALF_STEP[dtype] * np.abs(want) + SMALL


CASES = [
    (1, 1, 1, 1, 64, 32, "bhnd", 0, 1.0, 0),
    (2, 8, 2, 33, 64, 32, "bnhd", 100, 1.0, 3),
    (1, 5, 5, 7, 128, 64, "bhnd", 131000, 1.2, 2),
    (3, 7, 1, 65, 128, 32, "bnhd", 1 << 20, 0.5, 0),
    (2, 3, 3, 17, 64, 10, "bnhd", 5, 1.0, 3),
    (2, 3, 3, 17, 128, 5, "bhnd", 5, 1.0, 2),
    (2, 3, 2, 19, 128, 4, "bhnd", 77, 1.0, 0),
    (1, 2, 2, 9, 64, 1, "bnhd", 2000000000, 1.0, 0),
    (2, 2, 2, 9, 64, 0, "bhnd", 3, 1.0, 0),
    (1, 24, 8, 700, 128, 64, "bnhd", 0, 1.0, 3),
]


def problem(rs, cuda, dtype, b, h, hk, n, d, pairs, layout, first, axes, weight):
    import torch

    q, q64 = draw(rs, (b, h, n, d), dtype, cuda, layout)
    k, k64 = draw(rs, (b, hk, n, d), dtype, cuda, layout)
    qw, qw64 = draw(rs, (d,), weight, cuda)
    kw, kw64 = draw(rs, (d,), weight, cuda)
    positions = first + rs.randint(0, 50, (max(axes, 1), b, 1)) + np.arange(n)
    which = rs.randint(0, axes, pairs) if axes else None
    freqs = 10000.0 ** (-np.arange(pairs) / max(pairs, 1))
    pos = torch.from_numpy(positions if axes else positions[0]).to(cuda)
    if first < 2 ** 31 - 1000 and n % 2:
        pos = pos.int()
    a = None if which is None else torch.tensor(which, dtype=torch.int32, device=cuda)
    return (q, q64, k, k64, qw, qw64, kw, kw64, pos, positions if axes else positions[0], a, which,
            torch.from_numpy(freqs).to(cuda), freqs)


# More rows than a work-group for each step of the heads: walks over whole tiles of
# tokens, all heads of a tile or shares of them.
MANY = [
    (1, 24, 8, 2501, 128, 64, "bnhd", 0, 1.0, 3),
    (2, 13, 3, 4099, 64, 32, "bnhd", 10, 1.1, 0),
    (3, 9, 2, 1801, 64, 10, "bhnd", 7, 1.0, 2),
    (1, 3, 0, 20000, 64, 32, "bhnd", 0, 1.0, 0),
    (1, 40, 40, 333, 64, 1, "bnhd", 0, 1.0, 2),
]


@pytest.mark.parametrize("dtype,inter", [("float16", True), ("bfloat16", False), ("float32", False),
                                         ("float32", True)])
@pytest.mark.parametrize("b,h,hk,n,d,pairs,layout,first,scale,axes", MANY)
def test_many_rows(cuda, dtype, inter, b, h, hk, n, d, pairs, layout, first, scale, axes):
    check_forward_and_backward(cuda, dtype, inter, b, h, hk, n, d, pairs, layout, first, scale, axes)


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("b,h,hk,n,d,pairs,layout,first,scale,axes", CASES)
def test_forward_and_backward(cuda, dtype, inter, b, h, hk, n, d, pairs, layout, first, scale, axes):
    check_forward_and_backward(cuda, dtype, inter, b, h, hk, n, d, pairs, layout, first, scale, axes)


def check_forward_and_backward(cuda, dtype, inter, b, h, hk, n, d, pairs, layout, first, scale, axes):
    rs = np.random.RandomState(n + d)
    weight = dtype if n % 3 else "float32"
    eps, offset = (1e-6, 0.0) if n % 2 else (1e-2, 1.0)
    (q, q64, k, k64, qw, qw64, kw, kw64, pos, positions, a, which, f, freqs) = problem(
        rs, cuda, dtype, b, h, hk, n, d, pairs, layout, first, axes, weight)
    how = dict(axes=a, eps=eps, weight_offset=offset, interleaved=inter, scale=scale)
    outs = fl.forward_norm_rotary(q, k, qw, kw, pos, f, **how)
    for got, x, w in zip(outs, (q64, k64), (qw64 + offset, kw64 + offset)):
        want = packed.norm_rotary(x, w, positions, freqs, which, eps, inter, scale)
        assert_within(got, want, forward_bound(x, w, want, dtype, pairs, inter, scale, eps), "y")
    dq, dq64 = draw(rs, (b, h, n, d), dtype, cuda, layout)
    dk, dk64 = draw(rs, (b, hk, n, d), dtype, cuda, layout)
    got = fl.backward_norm_rotary(dq, dk, q, k, qw, kw, pos, f, **how)
    again = fl.backward_norm_rotary(dq, dk, q, k, qw, kw, pos, f, **how)
    assert all((x == y).all() for x, y in zip(got, again))
    u = HALF_STEP[dtype]
    for i, (x, dy, w) in enumerate(((q64, dq64, qw64 + offset), (k64, dk64, kw64 + offset))):
        dx, dw, g, spread = packed.norm_rotary_gradients(x, dy, w, positions, freqs, which, eps,
                                                         inter, scale)
        r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
        eg = pair_size(dy, pairs, inter) * scale * 2.0 ** -21 + np.abs(g) * 2.0 ** -23
        through = r * (np.abs(w) * eg
                       + np.abs(x) * r * r * (np.abs(w * x) * eg).mean(-1, keepdims=True))
        bound = through + spread * (3 * root(d) + (d + 16) * 2.0 ** -24) + u * np.abs(dx) + SMALL
        assert_within(got[i], dx, bound, "dx")
        rows = x.shape[0] * x.shape[1] * x.shape[2]
        size = np.abs(g * x * r).sum((0, 1, 2))
        bound = ((np.abs(x) * r * eg).sum((0, 1, 2))
                 + size * (root(d) + (rows + 66) * 2.0 ** -24) + 2.0 ** -24 * np.abs(dw) + 1e-30)
        assert_within(got[2 + i], dw, bound, "dw")


def assert_as_rotary(got, want, x, dtype, pairs, scale):
    """Two rotations of x, each within 2^-21 (|a| + |b|) scale and half a step of
    the exact one (which is at most (|a| + |b|) scale): 2 (2^-21 + u) of that
    apart.  The columns that do not turn are equal."""
    x = x.double().cpu().numpy()
    size = pair_size(x, pairs, False) * scale
    err = (got.double() - want.double()).abs().cpu().numpy()
    assert (err <= 2 * (2.0 ** -21 + HALF_STEP[dtype]) * size + 2 * SMALL)[..., :2 * pairs].all()
    assert (err[..., 2 * pairs:] == 0).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16", "float32"])
def test_without_weights_it_is_the_rotation(cuda, dtype):
    """No weight: no norm; as forward_rotary and its gradient."""
    import torch

    rs = np.random.RandomState(7)
    q, _ = draw(rs, (2, 6, 41, 64), dtype, cuda, "bnhd")
    k, _ = draw(rs, (2, 2, 41, 64), dtype, cuda, "bnhd")
    pos = torch.arange(100, 141, device=cuda)
    f = fl.rotary_frequencies(48, device=cuda)[0]
    want = fl.forward_rotary(q, k, pos, f, scale=1.1)
    got = one = fl.forward_norm_rotary(q, k, None, None, pos, f, scale=1.1)
    for x, y, z in zip(got, want, (q, k)):
        assert_as_rotary(x, y, z, dtype, 24, 1.1)
    want = fl.backward_rotary(q, k, pos, f, scale=1.1)
    got = fl.backward_norm_rotary(q, k, q, k, None, None, pos, f, scale=1.1)
    for x, y, z in zip(got, want, (q, k)):
        assert_as_rotary(x, y, z, dtype, 24, 1.1)
    assert got[2] is None and got[3] is None
    # three equal axes are one
    three = fl.forward_norm_rotary(q, k, None, None, pos[None].expand(3, -1), f,
                                   axes=fl.rotary_axes([8, 8, 8], True, cuda), scale=1.1)
    assert all(torch.equal(x, y) for x, y in zip(three, one))


def test_one_tensor_only(cuda):
    """k left out, and a weight for one of the two."""
    import torch

    rs = np.random.RandomState(8)
    q, _ = draw(rs, (1, 3, 20, 128), "bfloat16", cuda)
    k, _ = draw(rs, (1, 2, 20, 128), "bfloat16", cuda)
    w, _ = draw(rs, (128,), "float32", cuda)
    pos = torch.arange(20, device=cuda)
    f = fl.rotary_frequencies(128, device=cuda)[0]
    both = fl.forward_norm_rotary(q, k, w, None, pos, f)
    alone = fl.forward_norm_rotary(q, None, w, None, pos, f)
    assert torch.equal(alone, both[0])
    assert_as_rotary(both[1], fl.forward_rotary(k, None, pos, f), k, "bfloat16", 64, 1.0)
    dq, dk, dqw, dkw = fl.backward_norm_rotary(q, k, q, k, None, w, pos, f)
    assert dqw is None and dkw is not None
    assert_as_rotary(dq, fl.backward_rotary(q, None, pos, f), q, "bfloat16", 64, 1.0)
    got = fl.backward_norm_rotary(q, None, q, None, w, None, pos, f)
    assert got[1] is None and got[3] is None
    assert torch.equal(got[2], fl.backward_norm_rotary(q, k, q, k, w, w, pos, f)[2])


def test_no_rows_and_no_heads(cuda):
    import torch

    w = torch.ones(64, device=cuda)
    f = fl.rotary_frequencies(64, device=cuda)[0]
    q = torch.zeros((2, 3, 0, 64), dtype=torch.float16, device=cuda)
    pos = torch.zeros((0,), dtype=torch.int64, device=cuda)
    got = fl.forward_norm_rotary(q, q, w, w, pos, f)
    assert got[0].shape == q.shape
    dirty = [torch.full((64,), 7.0, device=cuda) for _ in range(2)]
    fl.backward_norm_rotary(q, q, q, q, w, w, pos, f, dq_weight=dirty[0], dk_weight=dirty[1])
    assert all((x == 0).all() for x in dirty)
    k = torch.randn((2, 3, 5, 64), device=cuda).half()
    pos = torch.arange(5, device=cuda)
    got = fl.backward_norm_rotary(k[:, :0], k, k[:, :0], k, w, w, pos, f)
    assert (got[2] == 0).all()
    assert torch.equal(got[3], fl.backward_norm_rotary(k, k, k, k, w, w, pos, f)[3])


@pytest.mark.parametrize("layout", ["bhnd", "bnhd"])
def test_in_place(cuda, layout):
    import torch

    rs = np.random.RandomState(9)
    q, _ = draw(rs, (2, 5, 37, 64), "float16", cuda, layout)
    k, _ = draw(rs, (2, 5, 37, 64), "float16", cuda, layout)
    w, _ = draw(rs, (64,), "float16", cuda)
    pos = torch.arange(37, device=cuda)
    f = fl.rotary_frequencies(64, device=cuda)[0]
    want = fl.forward_norm_rotary(q, k, w, w, pos, f)
    a, b = q.clone(), k.clone()
    fl.forward_norm_rotary(a, b, w, w, pos, f, q_out=a, k_out=b)
    assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    want = fl.backward_norm_rotary(q, k, k, q, w, w, pos, f)
    a, b = q.clone(), k.clone()
    got = fl.backward_norm_rotary(a, b, k, q, w, w, pos, f, q_out=a, k_out=b)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_rows_of_zeros_and_far_values(cuda):
    """A row of zeros gives zeros and finite gradients; large and tiny rows are
    normed as the formula says."""
    import torch

    x64 = np.random.RandomState(10).standard_normal((1, 1, 4, 64))
    x64[0, 0, 0] = 0.0
    x64[0, 0, 1] *= 2.0 ** 40
    x64[0, 0, 2] *= 2.0 ** -40
    q = torch.from_numpy(x64).to(cuda).bfloat16()
    x64 = q.double().cpu().numpy()
    w = torch.ones(64, device=cuda)
    pos = torch.arange(4, device=cuda)
    f = fl.rotary_frequencies(64, device=cuda)[0]
    got = fl.forward_norm_rotary(q, None, w, None, pos, f)
    freqs = f.cpu().numpy()
    want = packed.norm_rotary(x64, 1.0, np.arange(4)[None], freqs)
    bound = forward_bound(x64, np.ones(64), want, "bfloat16", 32, False, 1.0, 1e-6)
    assert_within(got, want, bound, "y")
    assert (got[0, 0, 0] == 0).all()
    dx, _, dw, _ = fl.backward_norm_rotary(torch.ones_like(q), None, q, None, w, None, pos, f)
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("b,n,h,hk,d,pairs,block,axes,paged_rows", [
    (5, 1, 8, 2, 64, 32, 16, 0, True),
    (2, 37, 3, 3, 128, 64, 20, 3, True),
    (3, 9, 4, 1, 128, 10, 8, 2, False),
    (1, 300, 32, 8, 64, 16, 64, 0, True),
    (2, 2100, 12, 4, 128, 64, 64, 3, True),
    (1, 9001, 3, 2, 64, 10, 32, 0, False),
])
def test_rows_of_the_cache(cuda, dtype, b, n, h, hk, d, pairs, block, axes, paged_rows):
    """As forward_norm_rotary, in the rows of the slots; passed-over tokens and
    all other rows stay as they were."""
    import torch

    rs = np.random.RandomState(d + n)
    (q, _, k, _, qw, _, kw, _, pos, _, a, _, f, _) = problem(rs, cuda, dtype, b, h, hk, n, d, pairs,
                                                             "bnhd", 50, axes, "float32")
    v, _ = draw(rs, (b, hk, n, d), dtype, cuda, "bnhd")
    blocks = b * n // block + 3
    shape = (blocks, block, hk, d) if paged_rows else (blocks, hk, block, d)
    caches = [torch.full(shape, 5.0, dtype=q.dtype, device=cuda) for _ in range(2)]
    if paged_rows:
        caches = [c.transpose(1, 2) for c in caches]
    slots = torch.from_numpy(rs.permutation(blocks * block)[:b * n].reshape(b, n)).to(cuda)
    skip = torch.from_numpy(rs.rand(b, n) < 0.2).to(cuda)
    slots = torch.where(skip, torch.tensor([-1, 1 << 40, blocks * block], device=cuda)[
        torch.arange(b * n, device=cuda).view(b, n) % 3], slots)
    out = torch.full_like(q, 5.0)
    how = dict(axes=a, eps=1e-5, interleaved=pairs == 10, scale=1.1)
    fl.norm_rotary_to_cache(q, k, v, qw, kw, pos, slots, f, *caches, **how, out=out)
    yq, yk = fl.forward_norm_rotary(q, k, qw, kw, pos, f, **how)
    keep = (slots >= 0) & (slots < blocks * block)
    want = torch.where(keep[:, None, :, None], yq, torch.full_like(yq, 5.0))
    assert torch.equal(out, want)
    for cache, rows in zip(caches, (yk, v)):
        wanted = torch.full_like(cache, 5.0)
        s = slots[keep]
        wanted[s // block, :, s % block] = rows.transpose(1, 2)[keep]
        assert torch.equal(cache, wanted)


def test_axes_out_of_range_are_brought_into_it(cuda):
    import torch

    rs = np.random.RandomState(11)
    q, _ = draw(rs, (1, 2, 9, 64), "float16", cuda)
    pos = torch.stack([torch.arange(9), 100 + torch.arange(9)]).to(cuda)
    f = fl.rotary_frequencies(64, device=cuda)[0]
    axes = torch.tensor([0, 1] * 16, dtype=torch.int32, device=cuda)
    wild = torch.tensor([-7, 1 << 30] * 16, dtype=torch.int32, device=cuda)
    a, b = (fl.forward_norm_rotary(q, None, None, None, pos, f, axes=x) for x in (axes, wild))
    assert torch.equal(a, b)


def test_gradient_against_differences(cuda):
    """Differences of sum(w y) in the direction of each input, 32 bits: the
    kernel's own forward pass with a step of 2^-6, whose third order and
    rounding (2^-20 of a sum's terms over the step) bound the difference."""
    import torch

    rs = np.random.RandomState(12)
    n, d, pairs = 6, 64, 24
    x, _ = draw(rs, (1, 2, n, d), "float32", cuda)
    w, _ = draw(rs, (1, 2, n, d), "float32", cuda)
    weight, _ = draw(rs, (d,), "float32", cuda)
    pos = torch.arange(40, 40 + n, device=cuda)
    f = fl.rotary_frequencies(2 * pairs, device=cuda)[0]
    dx, _, dw, _ = fl.backward_norm_rotary(w, None, x, None, weight, None, pos, f)
    step = 2.0 ** -6

    def loss(a, b):
        return float((fl.forward_norm_rotary(a, None, b, None, pos, f).double() * w.double()).sum())

    for seed in range(4):
        e = torch.from_numpy(np.random.RandomState(seed).standard_normal(x.shape)).to(cuda).float()
        e /= e.double().norm().float()
        slope = (loss(x + step * e, weight) - loss(x - step * e, weight)) / (2 * step)
        size = float(dx.double().norm())
        assert abs(float((dx.double() * e.double()).sum()) - slope) <= 2.0 ** -8 * size
        e = torch.from_numpy(np.random.RandomState(seed).standard_normal(d)).to(cuda).float()
        slope = (loss(x, weight + step * e) - loss(x, weight - step * e)) / (2 * step)
        assert abs(float((dw.double() * e.double()).sum()) - slope) <= 2.0 ** -8 * float(
            dw.double().norm() * e.double().norm())


def test_binding_refusals(cuda):
    import torch

    q = torch.zeros((1, 2, 5, 64), dtype=torch.float16, device=cuda)
    w = torch.ones(64, device=cuda)
    pos, f = torch.arange(5, device=cuda), fl.rotary_frequencies(64, device=cuda)[0]
    axes = fl.rotary_axes([16, 16], device=cuda)
    bad = [
        (dict(q_weight=w.double()), "FP32 or of q's dtype"),
        (dict(q_weight=w.bfloat16()), "FP32 or of q's dtype"),
        (dict(q_weight=w[:32]), "contiguous \\[D\\]"),
        (dict(q_weight=torch.ones(128, device=cuda)[::2]), "contiguous \\[D\\]"),
        (dict(q_weight=w.cpu()), "same device"),
        (dict(q_weight=w, k_weight=w.half()), "same dtype"),
        (dict(axes=axes), "positions must be"),
        (dict(axes=axes[:5], positions=pos[None]), "an axis for each"),
        (dict(axes=axes.long(), positions=pos[None]), "int32"),
        (dict(eps=-1.0), "eps"),
        (dict(k=None, k_weight=w), "needs k"),
        (dict(k=None, k_out=q), "needs k"),
        (dict(q_out=q[:, :1]), "q's shape"),
    ]
    base = dict(q=q, k=q, q_weight=None, k_weight=None, positions=pos, freqs=f)
    for change, text in bad:
        with pytest.raises(RuntimeError, match=text):
            fl.forward_norm_rotary(**{**base, **change})
    grads = dict(base, dq=q, dk=q)
    for change, text in [(dict(k=None), "both"), (dict(q=q[:, :, :3]), "dq's shape"),
                         (dict(dq_weight=w), "needs q_weight"),
                         (dict(q_weight=w, dq_weight=w.half()), "dq_weight"),
                         (dict(q_weight=w, workspace=torch.zeros(8, device=cuda)), "bytes needed")]:
        with pytest.raises(RuntimeError, match=text):
            fl.backward_norm_rotary(**{**grads, **change})
