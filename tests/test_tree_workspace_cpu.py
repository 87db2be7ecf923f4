"""Sizes of forward_tree's workspace: two partial results a work-group, each the
rows that a unit has in whole cache lines, and room for heads side by side only
where they lie so."""

import ctypes

import pytest

from flashlite_amd import capi

T3 = ctypes.c_int64 * 3
MOST_GROUPS = 2 * 256  # two work-groups a CU


def need(b, h, hk, n, d, heads_first, block=16):
    q = T3(h * n * d, d, h * d)
    kv = T3(hk * block * d, block * d, d) if heads_first else T3(hk * block * d, d, hk * d)
    p = capi.FlTreeParams(q_stride=q, o_stride=q, k_stride=kv, v_stride=kv, table_stride=20,
                          batch=b, heads=h, kv_heads=hk, drafts=n, head_dim=d, num_blocks=70,
                          block_size=block, max_blocks=20, dtype=capi.DTYPE_F16)
    return capi.load().fl_attn_tree_workspace_bytes(ctypes.byref(p))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,h,hk,n", [(2, 8, 8, 1), (1, 32, 8, 1), (2, 8, 4, 3), (4, 16, 4, 26),
                                      (1, 8, 1, 1), (2, 12, 3, 4), (1, 4, 2, 200)])
def test_a_part_has_the_rows_of_a_unit(b, h, hk, n, d):
    rows = min(h // hk * n, 256)
    for heads_first in (True, False):
        heads = 4 if not heads_first and hk % 4 == 0 and rows <= 32 else 1
        units = b * hk * -(-(h // hk * n) // 32)
        most = 2 * MOST_GROUPS * (heads * rows * (d + 4) * 4 + 128) + 8 * units
        got = need(b, h, hk, n, d, heads_first)
        assert 0 < got <= most


def test_many_units_of_a_cache_with_heads_first_need_none():
    assert need(64, 64, 8, 1, 128, heads_first=True) == 0
    assert need(64, 64, 8, 1, 128, heads_first=False) > 0


def test_one_token_of_a_small_batch():
    # 8 heads of 2 requests at head dim 64: K and V of 4096 tokens are 16.8 MB
    assert need(2, 8, 8, 1, 64, heads_first=False) < 1 << 20
