"""The paged-cache operators on a machine without a GPU: refusals of the C ABI
and the binding, the rotary's frequencies, and the oracle's own pins."""

import ctypes
import math

import numpy as np
import pytest
import torch

import flashlite_amd as fl
from flashlite_amd import capi
from oracle import paged

A = 0x7F0000000000  # a fake aligned address: no call here reaches a launch


def refused(rc, code, text):
    assert rc == code, capi.last_error()
    assert text in capi.last_error()


# --- plan_cache ------------------------------------------------------------


def plan_params(**kw):
    base = dict(lengths=A, counts=A, block_tables=A, held=A, held_out=A, free_blocks=A,
                free_state=A, free_state_out=A, positions=A, slots=A, info=A, batch=4, width=3,
                block_size=16, max_blocks=10, table_stride=10, pool=40)
    base.update(kw)
    return capi.FlCachePlanParams(**base)


@pytest.mark.parametrize("change,code,text", [
    (dict(batch=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(width=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(block_size=0), capi.FL_ERR_INVALID_ARGUMENT, "block_size"),
    (dict(pool=0), capi.FL_ERR_INVALID_ARGUMENT, "pool"),
    (dict(batch=65536), capi.FL_ERR_UNSUPPORTED, "65535"),
    (dict(max_blocks=1 << 28, table_stride=1 << 28), capi.FL_ERR_UNSUPPORTED, "int32"),
    (dict(table_stride=9), capi.FL_ERR_INVALID_ARGUMENT, "table_stride"),
    (dict(free_state=0), capi.FL_ERR_INVALID_ARGUMENT, "free blocks"),
    (dict(slots=0), capi.FL_ERR_INVALID_ARGUMENT, "requests"),
    (dict(info=0), capi.FL_ERR_INVALID_ARGUMENT, "requests"),
    (dict(lengths=A + 2), capi.FL_ERR_MISALIGNED, "int32"),
    (dict(slots=A + 4), capi.FL_ERR_MISALIGNED, "slots"),
])
def test_plan_refusals(change, code, text):
    p = plan_params(**change)
    refused(capi.load().fl_attn_cache_plan(ctypes.byref(p), None), code, text)


# --- plan_tree -------------------------------------------------------------


@pytest.mark.parametrize("change,code,text", [
    (dict(batch=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(drafts=513, parent_stride=513), capi.FL_ERR_UNSUPPORTED, "512"),
    (dict(parent_stride=6), capi.FL_ERR_INVALID_ARGUMENT, "parent_stride"),
    (dict(mask=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(mask=A + 4), capi.FL_ERR_MISALIGNED, "aligned"),
])
def test_tree_plan_refusals(change, code, text):
    base = dict(parents=A, lengths=A, counts=0, mask=A, positions=A, batch=2, drafts=7,
                parent_stride=7)
    base.update(change)
    p = capi.FlTreePlanParams(**base)
    refused(capi.load().fl_attn_tree_plan(ctypes.byref(p), None), code, text)


def test_empty_tree_plan_is_a_noop():
    for batch, drafts in ((0, 5), (3, 0)):
        p = capi.FlTreePlanParams(batch=batch, drafts=drafts, parent_stride=drafts)
        assert capi.load().fl_attn_tree_plan(ctypes.byref(p), None) == capi.FL_OK


# --- rotary ----------------------------------------------------------------

T3 = ctypes.c_int64 * 3
T2 = ctypes.c_int64 * 2


def rotary_params(**kw):
    st = T3(8 * 100 * 64, 100 * 64, 64)
    base = dict(q=A, k=A, q_out=A, k_out=A, q_stride=st, k_stride=st, q_out_stride=st,
                k_out_stride=st, positions=A, position_stride=T2(100, 1), position_bits=32,
                dtype=capi.DTYPE_F16, freqs=A, pairs=32, batch=2, heads=8, kv_heads=8, rows=100,
                head_dim=64, scale=1.0)
    base.update(kw)
    return capi.FlRotaryParams(**base)


@pytest.mark.parametrize("change,code,text", [
    (dict(dtype=3), capi.FL_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(head_dim=96), capi.FL_ERR_UNSUPPORTED, "head_dim"),
    (dict(pairs=33), capi.FL_ERR_INVALID_ARGUMENT, "pairs"),
    (dict(rows=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(position_bits=16), capi.FL_ERR_INVALID_ARGUMENT, "position_bits"),
    (dict(scale=math.inf), capi.FL_ERR_INVALID_ARGUMENT, "finite"),
    (dict(scale=1e300), capi.FL_ERR_INVALID_ARGUMENT, "finite"),
    (dict(batch=1 << 20, rows=1 << 20), capi.FL_ERR_UNSUPPORTED, "2^26"),
    (dict(q_stride=T3(6400, 64, 12)), capi.FL_ERR_UNSUPPORTED, "q strides"),
    (dict(k_out_stride=T3(6400, 64, -64)), capi.FL_ERR_UNSUPPORTED, "k_out strides"),
    (dict(q_out_stride=T3(0, 6400, 64)), capi.FL_ERR_INVALID_ARGUMENT, "q_out is written"),
    (dict(k_out_stride=T3(51200, 0, 64)), capi.FL_ERR_INVALID_ARGUMENT, "k_out is written"),
    (dict(q=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(k_out=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(positions=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(q=A + 8), capi.FL_ERR_MISALIGNED, "16-byte"),
    (dict(position_bits=64, positions=A + 4), capi.FL_ERR_MISALIGNED, "positions"),
])
def test_rotary_refusals(change, code, text):
    p = rotary_params(**change)
    refused(capi.load().fl_attn_rotary(ctypes.byref(p), None), code, text)


def test_rotary_null_and_empty():
    lib = capi.load()
    refused(lib.fl_attn_rotary(None, None), capi.FL_ERR_INVALID_ARGUMENT, "NULL")
    p = rotary_params(rows=0, q=0, k=0)
    assert lib.fl_attn_rotary(ctypes.byref(p), None) == capi.FL_OK


@pytest.mark.parametrize("change,store,code,text", [
    (dict(dtype=capi.DTYPE_F32), {}, capi.FL_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(transpose=1), {}, capi.FL_ERR_INVALID_ARGUMENT, "transpose"),
    ({}, dict(num_blocks=0), capi.FL_ERR_INVALID_ARGUMENT, "blocks"),
    ({}, dict(block_size=1 << 31), capi.FL_ERR_UNSUPPORTED, "int32"),
    ({}, dict(v_cache_stride=T3(64, 64, 4)), capi.FL_ERR_UNSUPPORTED, "v_cache strides"),
    ({}, dict(k_cache_stride=T3(0, 1024, 64)), capi.FL_ERR_INVALID_ARGUMENT, "k_cache is written"),
    ({}, dict(v_cache_stride=T3(8192, 1024, 0)), capi.FL_ERR_INVALID_ARGUMENT, "v_cache is written"),
    ({}, dict(slots=0), capi.FL_ERR_INVALID_ARGUMENT, "slots"),
    (dict(k=0), {}, capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    ({}, dict(v=A + 4), capi.FL_ERR_MISALIGNED, "16-byte"),
    ({}, dict(slots=A + 4), capi.FL_ERR_MISALIGNED, "slots"),
])
def test_rotary_cache_refusals(change, store, code, text):
    p = rotary_params(**change)
    st = T3(8 * 16 * 64, 16 * 64, 64)
    base = dict(v=A, v_stride=st, k_cache=A, v_cache=A, k_cache_stride=st, v_cache_stride=st,
                num_blocks=30, block_size=16, slots=A, slot_stride=T2(100, 1))
    base.update(store)
    c = capi.FlCacheStore(**base)
    refused(capi.load().fl_attn_rotary_cache(ctypes.byref(p), ctypes.byref(c), None), code, text)


def test_rotary_cache_null_store():
    p = rotary_params()
    refused(capi.load().fl_attn_rotary_cache(ctypes.byref(p), None, None),
            capi.FL_ERR_INVALID_ARGUMENT, "cache is NULL")


# --- forward_tree ----------------------------------------------------------


def tree_params(**kw):
    st = T3(8 * 5 * 64, 5 * 64, 64)
    kv = T3(2 * 16 * 64, 16 * 64, 64)
    base = dict(q=A, k_cache=A, v_cache=A, o=A, lse=0, q_stride=st, o_stride=st, k_stride=kv,
                v_stride=kv, block_tables=A, table_stride=20, lengths=A, counts=0, mask=0,
                mask_stride=0, batch=3, heads=8, kv_heads=2, drafts=5, head_dim=64, num_blocks=70,
                block_size=16, max_blocks=20, sm_scale=0.0, dtype=capi.DTYPE_F16)
    base.update(kw)
    return capi.FlTreeParams(**base)


TREE_REFUSALS = [
    (dict(dtype=capi.DTYPE_F32), capi.FL_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(head_dim=96), capi.FL_ERR_UNSUPPORTED, "head_dim"),
    (dict(drafts=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(kv_heads=3), capi.FL_ERR_INVALID_ARGUMENT, "multiple"),
    (dict(kv_heads=0), capi.FL_ERR_INVALID_ARGUMENT, "multiple"),
    (dict(sm_scale=math.nan), capi.FL_ERR_INVALID_ARGUMENT, "sm_scale"),
    (dict(sm_scale=1e-60), capi.FL_ERR_INVALID_ARGUMENT, "sm_scale"),
    (dict(num_blocks=0), capi.FL_ERR_INVALID_ARGUMENT, "blocks"),
    (dict(max_blocks=0), capi.FL_ERR_INVALID_ARGUMENT, "tables"),
    (dict(max_blocks=1 << 27, table_stride=1 << 27), capi.FL_ERR_UNSUPPORTED, "2^31"),
    (dict(max_blocks=1, block_size=(1 << 31) - 65536), capi.FL_ERR_UNSUPPORTED, "2^31"),
    (dict(table_stride=19), capi.FL_ERR_INVALID_ARGUMENT, "table_stride"),
    (dict(mask_stride=-1), capi.FL_ERR_INVALID_ARGUMENT, "mask_stride"),
    (dict(k_stride=T3(2048, 1024, 60)), capi.FL_ERR_UNSUPPORTED, "k_cache strides"),
    (dict(o_stride=T3(-64, 64, 64)), capi.FL_ERR_UNSUPPORTED, "o strides"),
    (dict(batch=1 << 23), capi.FL_ERR_UNSUPPORTED, "work-groups"),
]


@pytest.mark.parametrize("change,code,text", TREE_REFUSALS)
def test_tree_refusals(change, code, text):
    p = tree_params(**change)
    lib = capi.load()
    refused(lib.fl_attn_tree_fwd(ctypes.byref(p), None, 0, None), code, text)
    assert lib.fl_attn_tree_workspace_bytes(ctypes.byref(p)) == -1
    assert text in capi.last_error()


@pytest.mark.parametrize("change,code,text", [
    (dict(lengths=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(o=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(o_stride=T3(2560, 320, 0)), capi.FL_ERR_INVALID_ARGUMENT, "o is written"),
    (dict(v_cache=A + 8), capi.FL_ERR_MISALIGNED, "16-byte"),
    (dict(mask=A + 4), capi.FL_ERR_MISALIGNED, "mask"),
    (dict(lse=A + 1), capi.FL_ERR_MISALIGNED, "lse"),
])
def test_tree_pointer_refusals(change, code, text):
    p = tree_params(**change)
    refused(capi.load().fl_attn_tree_fwd(ctypes.byref(p), None, 0, None), code, text)


def test_empty_tree_call_is_a_noop():
    lib = capi.load()
    for change in (dict(batch=0), dict(drafts=0), dict(heads=0)):
        p = tree_params(**change)
        assert lib.fl_attn_tree_fwd(ctypes.byref(p), None, 0, None) == capi.FL_OK
        assert lib.fl_attn_tree_workspace_bytes(ctypes.byref(p)) == 0


def test_cpu_tensors_are_refused():
    x = torch.zeros((1, 2, 8, 64), dtype=torch.float16)
    i = torch.zeros((1,), dtype=torch.int32)
    f = torch.zeros((32,), dtype=torch.float64)
    for call in (lambda: fl.forward_rotary(x, x, i, f), lambda: fl.backward_rotary(x, x, i, f),
                 lambda: fl.rotary_to_cache(x, x, x, i, i.long(), f, x, x),
                 lambda: fl.forward_tree(x, x, x, i[None], i),
                 lambda: fl.tree_workspace_bytes(x, x),
                 lambda: fl.plan_tree(i[None], i),
                 lambda: fl.plan_cache(i, i, i[None], i, i, i, 16, 1)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


# --- frequencies -----------------------------------------------------------


def test_frequencies():
    f, s = fl.rotary_frequencies(8)
    assert s == 1.0 and f.dtype == torch.float64
    assert f.tolist() == pytest.approx([1.0, 1e-1, 1e-2, 1e-3], rel=1e-15)
    lin, s = fl.rotary_frequencies(8, method="linear", factor=4.0)
    assert s == 1.0 and torch.equal(lin, f / 4.0)
    ntk, s = fl.rotary_frequencies(8, method="ntk", factor=4.0)
    assert ntk[0] == 1.0 and float(ntk[-1]) == pytest.approx(1e-3 / 4.0, rel=1e-12)
    assert fl.rotary_frequencies(0)[0].shape == (0,)


def test_yarn_frequencies():
    f, _ = fl.rotary_frequencies(128)
    y, s = fl.rotary_frequencies(128, method="yarn", factor=8.0, trained=4096)
    assert s == pytest.approx(0.1 * math.log(8.0) + 1.0)
    turns = f * 4096 / (2 * math.pi)
    # a pair's place on the ramp is within one pair of its exact one
    assert torch.equal(y[turns > 32 * 1.2], f[turns > 32 * 1.2])
    assert torch.allclose(y[turns < 1 / 1.2], f[turns < 1 / 1.2] / 8.0, rtol=1e-14)
    between = (turns < 32 / 1.2) & (turns > 1.2)
    assert bool(((y < f) & (y > f / 8.0))[between].all())
    assert bool((y[1:] < y[:-1]).all())


@pytest.mark.parametrize("kw", [dict(rot_dim=7), dict(rot_dim=-2), dict(rot_dim=8, base=1.0),
                                dict(rot_dim=8, method="other"),
                                dict(rot_dim=8, method="linear", factor=0.5),
                                dict(rot_dim=8, method="yarn", factor=2.0),
                                dict(rot_dim=8, method="yarn", factor=2.0, trained=4, fast=1.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        fl.rotary_frequencies(**kw)


# --- the oracle's pins -----------------------------------------------------


def test_oracle_tree_equals_causal_attention():
    """A chain over a cache is causal attention, bottom-right aligned."""
    from oracle import attention_fp64

    rs = np.random.RandomState(0)
    q = rs.standard_normal((1, 2, 3, 64))
    k, v = rs.standard_normal((2, 1, 2, 13, 64))
    tables = np.array([[2, 0, 1, 5]])
    caches = []
    for x in (k, v):
        c = np.full((3, 2, 5, 64), np.nan)
        for t in range(13):
            c[tables[0][t // 5], :, t % 5] = x[0, :, t]
        caches.append(c)
    out, lse, _, _ = paged.tree_attention(q, *caches, tables, [10])
    np.testing.assert_allclose(out, attention_fp64(q, k, v, 0.0, True), rtol=1e-6)
    seen = [[{0}, {0, 1}, {0, 1, 2}]]
    again = paged.tree_attention(q, *caches, tables, [10], seen)[0]
    np.testing.assert_array_equal(out, again)


def test_oracle_plan_by_hand():
    got = paged.plan_cache([3, 0, 7, 5], [2, 9, -1, 1], [[4, -1, -1], [-1] * 3, [7, 8, -1],
                                                          [2, 9, -1]],
                           [1, 0, 2, 2], [10, 11, 12, -1, -1], [1, 2], 4, 4)
    tables, held, ring, state, positions, slots, info = got
    # request 0 takes ring[1] = 11; request 1 (4 of its 9 tokens) takes ring[2] = 12
    assert tables[0] == [4, 11, -1] and tables[1] == [12, -1, -1]
    assert slots[0] == [4 * 4 + 3, 11 * 4, -1, -1] and slots[1] == [48, 49, 50, 51]
    # request 2 gives 7 and 8 back behind the ring's last
    assert ring == [10, 11, 12, 7, 8] and held == [2, 1, 0, 2] and state == [3, 2]
    assert slots[3] == [9 * 4 + 1, -1, -1, -1] and positions[3] == [5, -1, -1, -1]
    assert info == [[0, 1, 1, 1], [0, 0, 1, 2], [0, 2, -2, 3], [0, 2, 0, 3]]


def test_oracle_rotary_keeps_lengths_and_transposes():
    rs = np.random.RandomState(1)
    x = rs.standard_normal((2, 3, 5, 64))
    pos = rs.randint(0, 1000, (2, 5))
    f = np.exp(-rs.rand(20) * 5)
    for inter in (False, True):
        y = paged.rotary(x, pos, f, inter, 1.0)
        np.testing.assert_allclose((y ** 2).sum(-1), (x ** 2).sum(-1), rtol=1e-12)
        np.testing.assert_allclose(paged.rotary(y, pos, f, inter, 1.0, True), x, atol=1e-12)
        assert np.array_equal(y[..., 40:], x[..., 40:])
