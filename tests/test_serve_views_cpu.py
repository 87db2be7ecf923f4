"""Strides of the paged-cache operators' arguments at the C ABI: which written
views overlap.  No call here reaches a launch (fake addresses, and a refusal
that comes after the check of strides)."""

import ctypes

import pytest

from flashlite_amd import capi

A = 0x7F0000000000
T3, T2 = ctypes.c_int64 * 3, ctypes.c_int64 * 2
D = 64

# {batch, head, row} strides of 2 x 4 x 5 rows of 64 columns, and whether two rows meet
VIEWS = [
    ((1280, 320, 64), False),       # contiguous
    ((1280, 64, 256), False),       # a token's heads side by side
    ((64, 640, 128), False),        # batches innermost
    ((1 << 40, 1 << 20, 4096), False),
    ((1280, 320, 8), True),         # rows closer together than their columns
    ((1280, 320, 56), True),
    ((1280, 312, 64), True),        # a head begins in the last one's last row
    ((1272, 64, 256), True),
    ((1280, 8, 256), True),
    ((1280, 320, 320), True),       # two dimensions of one stride
    ((1280, 64, 192), True),        # a token's heads reach into the next one's
    ((1280, 320, 0), True),
]


def tree_call(o):
    q = T3(1280, 320, 64)
    kv = T3(2 * 16 * D, 16 * D, D)
    p = capi.FlTreeParams(
        q=A, k_cache=A, v_cache=A, o=A, lse=0, q_stride=q, o_stride=T3(*o), k_stride=kv,
        v_stride=kv, block_tables=A, table_stride=20, lengths=A, batch=2, heads=4, kv_heads=2,
        drafts=5, head_dim=D, num_blocks=70, block_size=16, max_blocks=20, dtype=capi.DTYPE_F16)
    # (a workspace that is not aligned is refused last)
    return capi.load().fl_attn_tree_fwd(ctypes.byref(p), A + 4, 1 << 40, None), "workspace"


def rotary_call(name, st):
    views = dict.fromkeys(("q_stride", "k_stride", "q_out_stride", "k_out_stride"),
                          T3(1280, 320, 64))
    views[name] = T3(*st)
    p = capi.FlRotaryParams(q=A, k=A, q_out=A, k_out=A, positions=A, position_stride=T2(5, 1),
                            position_bits=32, dtype=capi.DTYPE_F16, freqs=A + 4, pairs=32, batch=2,
                            heads=4, kv_heads=4, rows=5, head_dim=D, scale=1.0, **views)
    return capi.load().fl_attn_rotary(ctypes.byref(p), None), "freqs"


def cache_call(name, st):
    v = T3(1280, 320, 64)
    p = capi.FlRotaryParams(q=A, k=A, q_out=A, q_stride=v, k_stride=v, q_out_stride=v,
                            positions=A, position_stride=T2(5, 1), position_bits=32,
                            dtype=capi.DTYPE_F16, freqs=A, pairs=32, batch=2, heads=4, kv_heads=4,
                            rows=5, head_dim=D, scale=1.0)
    views = dict.fromkeys(("k_cache_stride", "v_cache_stride"), v)
    views[name] = T3(*st)
    c = capi.FlCacheStore(v=A, v_stride=v, k_cache=A, v_cache=A, num_blocks=2, block_size=5,
                          slots=A + 4, slot_stride=T2(5, 1), **views)
    return capi.load().fl_attn_rotary_cache(ctypes.byref(p), ctypes.byref(c), None), "slots"


CALLS = {
    "o": tree_call,
    "q_out": lambda st: rotary_call("q_out_stride", st),
    "k_out": lambda st: rotary_call("k_out_stride", st),
    "k_cache": lambda st: cache_call("k_cache_stride", st),
    "v_cache": lambda st: cache_call("v_cache_stride", st),
}


@pytest.mark.parametrize("what", CALLS)
@pytest.mark.parametrize("strides,overlap", VIEWS)
def test_written_rows_do_not_overlap(what, strides, overlap):
    rc, later = CALLS[what](strides)
    if overlap:
        assert rc == capi.FL_ERR_INVALID_ARGUMENT
        assert f"{what} is written, its rows must not overlap" in capi.last_error()
    else:
        assert rc == capi.FL_ERR_MISALIGNED and later in capi.last_error()


# --- dimensions of one entry -------------------------------------------------
# Their strides step nowhere, and torch leaves any number there.

ODD = (1, 12, -8, 1 << 40)


@pytest.mark.parametrize("stride", ODD)
@pytest.mark.parametrize("dim,sizes", [(0, (1, 4, 5)), (1, (2, 1, 5)), (2, (2, 4, 1))])
def test_strides_of_one_entry_are_not_looked_at(stride, dim, sizes):
    b, h, n = sizes
    st = [h * n * D, n * D, D]
    st[dim] = stride
    st = T3(*st)
    p = capi.FlRotaryParams(q=A, k=A, q_out=A, k_out=A, q_stride=st, k_stride=st, q_out_stride=st,
                            k_out_stride=st, positions=A, position_stride=T2(5, 1),
                            position_bits=32, dtype=capi.DTYPE_F16, freqs=A + 4, pairs=32, batch=b,
                            heads=h, kv_heads=h, rows=n, head_dim=D, scale=1.0)
    lib = capi.load()
    assert lib.fl_attn_rotary(ctypes.byref(p), None) == capi.FL_ERR_MISALIGNED
    assert "freqs" in capi.last_error()
    # a cache of b blocks of n rows
    c = capi.FlCacheStore(v=A, v_stride=st, k_cache=A, v_cache=A, k_cache_stride=st,
                          v_cache_stride=st, num_blocks=b, block_size=n, slots=A + 4,
                          slot_stride=T2(5, 1))
    p.freqs = A
    assert lib.fl_attn_rotary_cache(ctypes.byref(p), ctypes.byref(c), None) == \
        capi.FL_ERR_MISALIGNED
    assert "slots" in capi.last_error()
    t = capi.FlTreeParams(
        q=A, k_cache=A, v_cache=A, o=A, q_stride=st, o_stride=st, k_stride=st, v_stride=st,
        block_tables=A, table_stride=20, lengths=A, batch=b, heads=h, kv_heads=h, drafts=n,
        head_dim=D, num_blocks=b, block_size=n, max_blocks=20, dtype=capi.DTYPE_F16)
    assert lib.fl_attn_tree_workspace_bytes(ctypes.byref(t)) > 0
    assert lib.fl_attn_tree_fwd(ctypes.byref(t), A + 4, 1 << 40, None) == capi.FL_ERR_MISALIGNED
    assert "workspace" in capi.last_error()


def test_no_query_heads():
    """Without query heads only k and v are stored: q and out have no memory."""
    v = T3(1280, 320, 64)
    p = capi.FlRotaryParams(q=0, k=A, q_out=0, q_stride=v, k_stride=v, q_out_stride=v,
                            positions=A, position_stride=T2(5, 1), position_bits=32,
                            dtype=capi.DTYPE_F16, freqs=A, pairs=32, batch=2, heads=0, kv_heads=4,
                            rows=5, head_dim=D, scale=1.0)
    c = capi.FlCacheStore(v=A, v_stride=v, k_cache=A, v_cache=A, k_cache_stride=v,
                          v_cache_stride=v, num_blocks=2, block_size=5, slots=A + 4,
                          slot_stride=T2(5, 1))
    lib = capi.load()
    assert lib.fl_attn_rotary_cache(ctypes.byref(p), ctypes.byref(c), None) == \
        capi.FL_ERR_MISALIGNED
    p.k_out, p.k_out_stride, p.freqs = A, v, A + 4
    assert lib.fl_attn_rotary(ctypes.byref(p), None) == capi.FL_ERR_MISALIGNED
    # nor key heads
    p.q, p.q_out, p.k, p.k_out, p.heads, p.kv_heads = A, A, 0, 0, 4, 0
    assert lib.fl_attn_rotary(ctypes.byref(p), None) == capi.FL_ERR_MISALIGNED
    p.freqs = A
    assert lib.fl_attn_rotary_cache(ctypes.byref(p), ctypes.byref(c), None) == \
        capi.FL_ERR_MISALIGNED
    p.q = 0
    assert lib.fl_attn_rotary(ctypes.byref(p), None) == capi.FL_ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("sizes", [(0, 4, 5), (2, 0, 5), (2, 4, 0)])
def test_views_without_rows_do_not_overlap(sizes):
    """Nothing is written: no stride is too small, and the call does nothing."""
    b, h, n = sizes
    st = T3(8, 8, 8)
    p = capi.FlRotaryParams(q_stride=st, k_stride=st, q_out_stride=st, k_out_stride=st,
                            position_bits=32, dtype=capi.DTYPE_F16, pairs=32, batch=b, heads=h,
                            kv_heads=h, rows=n, head_dim=D, scale=1.0)
    assert capi.load().fl_attn_rotary(ctypes.byref(p), None) == capi.FL_OK
    kv = T3(2 * 16 * D, 16 * D, D)
    t = capi.FlTreeParams(q_stride=st, o_stride=st, k_stride=kv, v_stride=kv, table_stride=20,
                          batch=b, heads=h, kv_heads=2, drafts=n, head_dim=D, num_blocks=70,
                          block_size=16, max_blocks=20, dtype=capi.DTYPE_F16)
    assert capi.load().fl_attn_tree_fwd(ctypes.byref(t), None, 0, None) == capi.FL_OK
