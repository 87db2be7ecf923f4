"""Views whose dimensions of one entry have strides of no meaning."""

import numpy as np
import pytest

import flashlite_amd as fl
from oracle import paged
from test_gpu_tree import run
from tree_util import Problem, check

pytestmark = pytest.mark.gpu


def odd(t, dim, stride):
    """`t` with another stride at a dimension of one entry."""
    st = list(t.stride())
    st[dim] = stride
    return t.as_strided(t.shape, st)


@pytest.mark.parametrize("stride", [1, 12, 1 << 40])
def test_one_request_of_one_token_in_blocks_of_one(cuda, stride):
    import torch

    p = Problem(91, "float16", 1, 4, 1, 1, 64, 1, [40], None)
    p.q = odd(odd(p.q, 0, stride), 2, stride)
    p.k, p.v = (odd(odd(x, 1, stride), 2, stride) for x in (p.k, p.v))
    args = p.device(cuda)
    for name in ("q", "k_cache", "v_cache"):
        x = args[name]
        for dim in range(3):
            x = odd(x, dim, stride) if x.shape[dim] == 1 else x
        args[name] = x
    out, lse = fl.forward_tree(return_lse=True, **args)
    check(out, lse, p)

    freqs, _ = fl.rotary_frequencies(64, device=cuda)
    pos = torch.tensor([[7]], dtype=torch.int32, device=cuda)
    turned = fl.forward_rotary(args["q"], None, pos, freqs)
    want = paged.rotary(p.q.double().numpy(), [[7]], freqs.cpu().numpy())
    err = np.abs(turned.double().cpu().numpy() - want)
    assert (err <= 2.0 ** -11 * np.abs(want) + 2.0 ** -20 * np.abs(want).max()).all()

    k = odd(args["q"][:, :1].clone(), 2, stride)
    slot = torch.tensor([[5]], device=cuda)
    fl.rotary_to_cache(args["q"], k, k, pos, slot, freqs, args["k_cache"], args["v_cache"])
    assert torch.equal(args["k_cache"][5, 0, 0], turned[0, 0, 0])
    assert torch.equal(args["v_cache"][5, 0, 0], k[0, 0, 0])
