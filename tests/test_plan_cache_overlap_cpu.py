"""plan_cache's new held counts and ring state replace the old ones or lie
apart: work-groups read the old ones while others write the new."""

import ctypes

import pytest

from flashlite_amd import capi

A = 0x7F0000000000


def call(**kw):
    base = dict(lengths=A, counts=A, block_tables=A, held=A + 4096, held_out=A + 8192,
                free_blocks=A, free_state=A + 256, free_state_out=A + 512, positions=A,
                slots=A + 4, info=A, batch=40, width=3, block_size=16, max_blocks=10,
                table_stride=10, pool=40)
    base.update(kw)
    p = capi.FlCachePlanParams(**base)  # (slots that are not aligned are refused last)
    return capi.load().fl_attn_cache_plan(ctypes.byref(p), None)


@pytest.mark.parametrize("change,overlap", [
    (dict(held_out=A + 4096), False),            # in place
    (dict(held_out=A + 4096 + 160), False),      # right behind
    (dict(held_out=A + 4096 - 160), False),      # right before
    (dict(held_out=A + 4096 + 156), True),
    (dict(held_out=A + 4096 - 4), True),
    (dict(held_out=A + 4100), True),
    (dict(free_state_out=A + 256), False),
    (dict(free_state_out=A + 264), False),
    (dict(free_state_out=A + 260), True),
    (dict(free_state_out=A + 252), True),
])
def test_in_place_or_apart(change, overlap):
    rc = call(**change)
    if overlap:
        assert rc == capi.FL_ERR_INVALID_ARGUMENT
        assert "in place or apart" in capi.last_error()
    else:
        assert rc == capi.FL_ERR_MISALIGNED and "slots" in capi.last_error()
