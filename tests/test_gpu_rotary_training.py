"""The rotary operators in a training step: autograd does not record them, a
Function around the two does."""

import numpy as np
import pytest

import flashlite_amd as fl
from oracle import paged

pytestmark = pytest.mark.gpu


def rotary_function():
    import torch

    class Rotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, positions, freqs, interleaved=False, scale=1.0):
            ctx.save_for_backward(positions, freqs)
            ctx.how = interleaved, scale
            return fl.forward_rotary(q, k, positions, freqs, interleaved, scale)

        @staticmethod
        def backward(ctx, dq, dk):
            dq, dk = (x if x.stride(-1) == 1 else x.contiguous() for x in (dq, dk))
            return *fl.backward_rotary(dq, dk, *ctx.saved_tensors, *ctx.how), None, None, None, None

    return Rotary


def test_results_are_not_recorded(cuda):
    import torch

    q = torch.randn((1, 2, 3, 64), device=cuda, requires_grad=True)
    freqs, _ = fl.rotary_frequencies(64, device=cuda)
    pos = torch.arange(3, device=cuda)
    out = fl.forward_rotary(q, None, pos, freqs)
    assert not out.requires_grad and out.grad_fn is None
    assert "autograd" in fl.forward_rotary.__doc__ and "autograd" in fl.backward_rotary.__doc__


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("summed", [False, True])
def test_gradients_of_a_step(cuda, inter, summed):
    """Of sum(w rotated): the transpose of the rotation of w, also where w is 1
    everywhere and autograd hands over an expanded gradient."""
    import torch

    b, h, hk, n, d, scale = 2, 3, 1, 50, 64, 1.2
    rs = np.random.RandomState(4)
    freqs, _ = fl.rotary_frequencies(d, device=cuda)
    pos = torch.arange(7, 7 + n, device=cuda)
    draw = lambda x: rs.standard_normal((b, x, n, d)).astype(np.float32)  # noqa: E731
    x = [torch.from_numpy(draw(i)).to(cuda).requires_grad_() for i in (h, hk)]
    w = [np.ones_like(draw(i)) if summed else draw(i) for i in (h, hk)]
    out = rotary_function().apply(*x, pos, freqs, inter, scale)
    if summed:
        loss = out[0].sum() + out[1].sum()
    else:
        loss = sum((o * torch.from_numpy(y).to(cuda)).sum() for o, y in zip(out, w))
    loss.backward()
    for t, y in zip(x, w):
        y = y.astype(np.float64)
        want = paged.rotary(y, np.broadcast_to(np.arange(7, 7 + n), (b, n)), freqs.cpu().numpy(),
                            inter, scale, transpose=True)
        # two products with factors of half a step each, and their sum
        bound = 2.0 ** -24 * 4 * scale * 2 * np.abs(y).max()
        assert (np.abs(t.grad.double().cpu().numpy() - want) <= bound).all()
