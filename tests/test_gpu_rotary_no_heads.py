"""Rotary calls whose q or k has no heads."""

import pytest

import flashlite_amd as fl

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens_first", [False, True])
def test_only_k_and_v_are_stored(cuda, tokens_first):
    """q without heads: the cache gets what it gets with q."""
    import torch

    b, n, h, hk, d = 2, 9, 3, 2, 64
    g = torch.Generator(device=cuda)
    g.manual_seed(3)
    q, k, v = (torch.randn((b, x, n, d), generator=g, device=cuda).half() for x in (h, hk, hk))
    if tokens_first:
        q, k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    freqs, _ = fl.rotary_frequencies(d, device=cuda)
    pos = torch.arange(n, device=cuda).int()
    slots = torch.randperm(32, generator=g, device=cuda)[:b * n].view(b, n)
    caches = [torch.zeros((4, hk, 8, d), dtype=q.dtype, device=cuda) for _ in range(4)]
    fl.rotary_to_cache(q, k, v, pos, slots, freqs, *caches[:2])
    out = fl.rotary_to_cache(q[:, :0], k, v, pos, slots, freqs, *caches[2:])
    assert out.shape == (b, 0, n, d)
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    only = fl.forward_rotary(q[:, :0], k, pos, freqs)
    assert torch.equal(only[1], fl.forward_rotary(q, k, pos, freqs)[1])
    assert torch.equal(fl.forward_rotary(q, k[:, :0], pos, freqs)[0],
                       fl.forward_rotary(q, None, pos, freqs))
