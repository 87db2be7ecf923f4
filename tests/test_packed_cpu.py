"""Attention over packed sequences and the norms with rotary positions on a
machine without a GPU: refusals, and the oracle's own pins."""

import ctypes
import math

import numpy as np
import pytest
import torch

import flashlite_amd as fl
from flashlite_amd import capi
from oracle import attention_fp64, packed

A = 0x7F0000000000  # a fake aligned address: no call here reaches a launch
T2 = ctypes.c_int64 * 2
T3 = ctypes.c_int64 * 3


def refused(rc, code, text):
    assert rc == code, capi.last_error()
    assert text in capi.last_error()


def packed_params(**kw):
    q, k = T2(64, 512), T2(64, 128)
    base = dict(q=A, k=A, v=A, o=A, lse=A, q_stride=q, k_stride=k, v_stride=k, o_stride=q,
                starts=A, key_starts=A, sequences=3, rows=100, key_rows=120, heads=8, kv_heads=2,
                head_dim=64, sm_scale=0.0, causal=1, dtype=capi.DTYPE_F16)
    base.update(kw)
    return capi.FlPackedParams(**base)


def grads(**kw):
    q, k = T2(64, 512), T2(64, 128)
    base = dict(dout=A, dq=A, dk=A, dv=A, dout_stride=q, dq_stride=q, dk_stride=k, dv_stride=k)
    base.update(kw)
    return capi.FlPackedGrads(**base)


PACKED = [
    (dict(dtype=capi.DTYPE_F32), capi.FL_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(head_dim=96), capi.FL_ERR_UNSUPPORTED, "head_dim"),
    (dict(rows=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(sequences=-1), capi.FL_ERR_INVALID_ARGUMENT, "non-negative"),
    (dict(kv_heads=3), capi.FL_ERR_INVALID_ARGUMENT, "multiple"),
    (dict(kv_heads=0), capi.FL_ERR_INVALID_ARGUMENT, "multiple"),
    (dict(heads=0), capi.FL_ERR_INVALID_ARGUMENT, "multiple"),
    (dict(sm_scale=math.nan), capi.FL_ERR_INVALID_ARGUMENT, "sm_scale"),
    (dict(sm_scale=1e-60), capi.FL_ERR_INVALID_ARGUMENT, "sm_scale"),
    (dict(sm_scale=1e-31), capi.FL_ERR_UNSUPPORTED, "1e-30"),
    (dict(key_starts=0), capi.FL_ERR_INVALID_ARGUMENT, "key_starts"),
    (dict(rows=1 << 31), capi.FL_ERR_UNSUPPORTED, "2^30"),
    (dict(sequences=1 << 25), capi.FL_ERR_UNSUPPORTED, "2^24"),
    (dict(rows=1 << 29, heads=1024, kv_heads=1024), capi.FL_ERR_UNSUPPORTED, "work-groups"),
    (dict(q_stride=T2(64, 60)), capi.FL_ERR_UNSUPPORTED, "q strides"),
    (dict(k_stride=T2(64, 56)), capi.FL_ERR_UNSUPPORTED, "row stride of k"),
    (dict(v_stride=T2(64, 0)), capi.FL_ERR_UNSUPPORTED, "row stride of v"),
    (dict(q_stride=T2(64, 1 << 24)), capi.FL_ERR_UNSUPPORTED, "row stride of q"),
    (dict(key_rows=1 << 24), capi.FL_ERR_UNSUPPORTED, "2^31 bytes"),
    (dict(key_rows=65, v_stride=T2(64, (1 << 30) // 65 // 8 * 8)), capi.FL_ERR_UNSUPPORTED,
     "128 more"),
    (dict(k_stride=T2(-64, 128)), capi.FL_ERR_UNSUPPORTED, "k strides"),
]


@pytest.mark.parametrize("change,code,text", PACKED)
def test_packed_refusals(change, code, text):
    lib = capi.load()
    p = packed_params(**change)
    refused(lib.fl_attn_packed_fwd(ctypes.byref(p), None), code, text)
    assert lib.fl_attn_packed_bwd_workspace_bytes(ctypes.byref(p)) == -1
    assert text in capi.last_error()
    refused(lib.fl_attn_packed_bwd(ctypes.byref(p), ctypes.byref(grads()), A, 1 << 40, None), code,
            text)


@pytest.mark.parametrize("change,code,text", [
    (dict(q=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(v=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(starts=0), capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(k=A + 8), capi.FL_ERR_MISALIGNED, "16-byte"),
    (dict(starts=A + 2), capi.FL_ERR_MISALIGNED, "4-byte"),
    (dict(lse=A + 2), capi.FL_ERR_MISALIGNED, "4-byte"),
])
def test_packed_pointer_refusals(change, code, text):
    lib = capi.load()
    p = packed_params(**change)
    refused(lib.fl_attn_packed_fwd(ctypes.byref(p), None), code, text)
    refused(lib.fl_attn_packed_bwd(ctypes.byref(p), ctypes.byref(grads()), A, 1 << 40, None), code,
            text)


def test_packed_output_overlaps_are_refused():
    lib = capi.load()
    p = packed_params(o_stride=T2(0, 512))
    refused(lib.fl_attn_packed_fwd(ctypes.byref(p), None), capi.FL_ERR_INVALID_ARGUMENT,
            "o is written")
    for change, name in ((dict(dq_stride=T2(32, 512)), "dq"), (dict(dk_stride=T2(64, 0)), "dk"),
                         (dict(dv_stride=T2(0, 64)), "dv")):
        refused(lib.fl_attn_packed_bwd(ctypes.byref(packed_params()), ctypes.byref(grads(**change)),
                                       A, 1 << 40, None),
                capi.FL_ERR_INVALID_ARGUMENT, f"{name} is written")


@pytest.mark.parametrize("change,ws,code,text", [
    (dict(dout=0), A, capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(dk=0), A, capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(dv=A + 8), A, capi.FL_ERR_MISALIGNED, "16-byte"),
    ({}, 0, capi.FL_ERR_INVALID_ARGUMENT, "workspace"),
    ({}, A + 4, capi.FL_ERR_MISALIGNED, "workspace"),
])
def test_packed_gradient_refusals(change, ws, code, text):
    lib = capi.load()
    p = packed_params()
    refused(lib.fl_attn_packed_bwd(ctypes.byref(p), ctypes.byref(grads(**change)), ws or None,
                                   1 << 40, None), code, text)


def test_packed_null_empty_and_small_workspace():
    lib = capi.load()
    refused(lib.fl_attn_packed_fwd(None, None), capi.FL_ERR_INVALID_ARGUMENT, "NULL")
    refused(lib.fl_attn_packed_bwd(ctypes.byref(packed_params()), None, A, 1 << 40, None),
            capi.FL_ERR_INVALID_ARGUMENT, "NULL")
    need = lib.fl_attn_packed_bwd_workspace_bytes(ctypes.byref(packed_params()))
    assert need >= 8 * 100 * 8
    refused(lib.fl_attn_packed_bwd(ctypes.byref(packed_params()), ctypes.byref(grads()), A,
                                   need - 1, None), capi.FL_ERR_INVALID_ARGUMENT, "workspace")
    for change in (dict(sequences=0), dict(heads=0, kv_heads=0), dict(rows=0)):
        p = packed_params(**change)
        assert lib.fl_attn_packed_fwd(ctypes.byref(p), None) == capi.FL_OK
    for change in (dict(sequences=0), dict(heads=0, kv_heads=0)):
        p = packed_params(**change)
        assert lib.fl_attn_packed_bwd_workspace_bytes(ctypes.byref(p)) == 0
        assert lib.fl_attn_packed_bwd(ctypes.byref(p), ctypes.byref(grads()), None, 0,
                                      None) == capi.FL_OK


# --- norms -------------------------------------------------------------------


def rotary_params(**kw):
    st = T3(8 * 100 * 64, 100 * 64, 64)
    base = dict(q=A, k=A, q_out=A, k_out=A, q_stride=st, k_stride=st, q_out_stride=st,
                k_out_stride=st, positions=A, position_stride=T2(100, 1), position_bits=32,
                dtype=capi.DTYPE_F16, freqs=A, pairs=32, batch=2, heads=8, kv_heads=8, rows=100,
                head_dim=64, scale=1.0)
    base.update(kw)
    return capi.FlRotaryParams(**base)


def norm_params(**kw):
    base = dict(q_weight=A, k_weight=A, weight_dtype=capi.DTYPE_F32, eps=1e-6, weight_offset=0.0,
                axes=A, num_axes=3, axis_stride=200)
    base.update(kw)
    return capi.FlNormParams(**base)


def norm_grads(**kw):
    st = T3(8 * 100 * 64, 100 * 64, 64)
    base = dict(q=A, k=A, q_stride=st, k_stride=st, dq_weight=A, dk_weight=A)
    base.update(kw)
    return capi.FlNormGrads(**base)


def store():
    st = T3(8 * 16 * 64, 16 * 64, 64)
    return capi.FlCacheStore(v=A, v_stride=st, k_cache=A, v_cache=A, k_cache_stride=st,
                             v_cache_stride=st, num_blocks=30, block_size=16, slots=A,
                             slot_stride=T2(100, 1))


@pytest.mark.parametrize("change,norm,code,text", [
    (dict(dtype=3), {}, capi.FL_ERR_INVALID_ARGUMENT, "dtype"),
    (dict(head_dim=96), {}, capi.FL_ERR_UNSUPPORTED, "head_dim"),
    (dict(q_out_stride=T3(0, 6400, 64)), {}, capi.FL_ERR_INVALID_ARGUMENT, "q_out is written"),
    (dict(q=A + 8), {}, capi.FL_ERR_MISALIGNED, "16-byte"),
    ({}, dict(weight_dtype=capi.DTYPE_BF16), capi.FL_ERR_INVALID_ARGUMENT, "weights"),
    ({}, dict(eps=-1e-6), capi.FL_ERR_INVALID_ARGUMENT, "eps"),
    ({}, dict(eps=math.nan), capi.FL_ERR_INVALID_ARGUMENT, "eps"),
    ({}, dict(eps=1e300), capi.FL_ERR_INVALID_ARGUMENT, "eps"),
    ({}, dict(weight_offset=math.inf), capi.FL_ERR_INVALID_ARGUMENT, "weight_offset"),
    ({}, dict(q_weight=A + 2), capi.FL_ERR_MISALIGNED, "weights"),
    ({}, dict(axes=A + 2), capi.FL_ERR_MISALIGNED, "axes"),
    ({}, dict(num_axes=0), capi.FL_ERR_INVALID_ARGUMENT, "axis"),
])
def test_norm_refusals(change, norm, code, text):
    lib = capi.load()
    p, n = rotary_params(**change), norm_params(**norm)
    refused(lib.fl_attn_norm_rotary(ctypes.byref(p), ctypes.byref(n), None), code, text)
    refused(lib.fl_attn_norm_rotary_bwd(ctypes.byref(p), ctypes.byref(n),
                                        ctypes.byref(norm_grads()), A, 1 << 30, None), code, text)
    refused(lib.fl_attn_norm_rotary_cache(ctypes.byref(p), ctypes.byref(n), ctypes.byref(store()),
                                          None), code, text)


@pytest.mark.parametrize("change,ws,code,text", [
    (dict(q=0), A, capi.FL_ERR_INVALID_ARGUMENT, "non-NULL"),
    (dict(k=A + 8), A, capi.FL_ERR_MISALIGNED, "16-byte"),
    (dict(dq_weight=A + 2), A, capi.FL_ERR_MISALIGNED, "dq_weight"),
    (dict(q_stride=T3(1, 1, 1)), A, capi.FL_ERR_UNSUPPORTED, "q strides"),
    ({}, 0, capi.FL_ERR_INVALID_ARGUMENT, "workspace"),
    ({}, A + 8, capi.FL_ERR_MISALIGNED, "workspace"),
])
def test_norm_gradient_refusals(change, ws, code, text):
    lib = capi.load()
    refused(lib.fl_attn_norm_rotary_bwd(ctypes.byref(rotary_params()), ctypes.byref(norm_params()),
                                        ctypes.byref(norm_grads(**change)), ws or None, 1 << 30,
                                        None), code, text)


def test_norm_null_and_empty():
    lib = capi.load()
    p, n = rotary_params(), norm_params()
    refused(lib.fl_attn_norm_rotary(None, ctypes.byref(n), None), capi.FL_ERR_INVALID_ARGUMENT,
            "NULL")
    refused(lib.fl_attn_norm_rotary(ctypes.byref(p), None, None), capi.FL_ERR_INVALID_ARGUMENT,
            "NULL")
    refused(lib.fl_attn_norm_rotary_cache(ctypes.byref(p), ctypes.byref(n), None, None),
            capi.FL_ERR_INVALID_ARGUMENT, "cache is NULL")
    empty = rotary_params(rows=0, q=0, k=0)
    assert lib.fl_attn_norm_rotary(ctypes.byref(empty), ctypes.byref(n), None) == capi.FL_OK
    none = norm_grads(dq_weight=0, dk_weight=0)
    assert lib.fl_attn_norm_rotary_bwd(ctypes.byref(empty), ctypes.byref(n), ctypes.byref(none),
                                       None, 0, None) == capi.FL_OK
    assert lib.fl_attn_norm_rotary_workspace_bytes(None) == -1
    assert lib.fl_attn_norm_rotary_workspace_bytes(ctypes.byref(rotary_params(head_dim=32))) == -1


def test_cpu_tensors_are_refused():
    x = torch.zeros((1, 2, 8, 64), dtype=torch.float16)
    i = torch.zeros((2,), dtype=torch.int32)
    f = torch.zeros((32,), dtype=torch.float64)
    l = torch.zeros((1, 2, 8))
    for call in (lambda: fl.forward_packed(x, x, x, i), lambda: fl.packed_workspace_bytes(x, x, i),
                 lambda: fl.backward_packed(x, x, x, x, x, l, i),
                 lambda: fl.forward_norm_rotary(x, x, None, None, i, f),
                 lambda: fl.backward_norm_rotary(x, x, x, x, None, None, i, f),
                 lambda: fl.norm_rotary_to_cache(x, x, x, None, None, i, i.long(), f, x, x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


# --- axes and the oracle -----------------------------------------------------


def test_axes():
    assert fl.rotary_axes([2, 1, 3]).tolist() == [0, 0, 1, 2, 2, 2]
    assert fl.rotary_axes([2, 1, 3], interleaved=True).tolist() == [0, 1, 2, 0, 2, 2]
    assert fl.rotary_axes([0, 2]).tolist() == [1, 1]
    assert fl.rotary_axes([4]).dtype == torch.int32
    for bad in ([], [3, -1]):
        with pytest.raises(ValueError):
            fl.rotary_axes(bad)


def test_oracle_equals_causal_attention():
    rs = np.random.RandomState(0)
    q, k, v = rs.standard_normal((3, 2, 11, 64))
    starts, out = [0, 4, 4, 11], np.zeros((2, 11, 64))
    for a, b in ((0, 4), (4, 11)):
        out[:, a:b] = attention_fp64(*(x[None, :, a:b] for x in (q, k, v)), 0.0, True)[0]
    got, lse, _, _ = packed.attention(q, k, v, starts, starts, True, 0.125)
    np.testing.assert_allclose(got, out, rtol=1e-6, atol=1e-9)
    assert np.isfinite(lse).all()


@pytest.mark.parametrize("causal", [True, False])
def test_oracle_gradients_are_torchs(causal):
    rs = np.random.RandomState(1)
    q, do = rs.standard_normal((2, 4, 9, 8))
    k, v = rs.standard_normal((2, 2, 12, 8))
    starts, key_starts = [0, 5, 9], [0, 3, 12]
    out, lse, _, _ = packed.attention(q, k, v, starts, key_starts, causal, 0.3)
    g = packed.gradients(q, k, v, out, lse, do, starts, key_starts, causal, 0.3)
    leaves = [torch.from_numpy(x).requires_grad_() for x in (q, k, v)]
    loss = 0.0
    for a, b, c, e in zip(starts, starts[1:], key_starts, key_starts[1:]):
        for h in range(4):
            s = leaves[0][h, a:b] @ leaves[1][h // 2, c:e].T * 0.3
            if causal:
                hidden = torch.arange(e - c) - (e - c - (b - a)) > torch.arange(b - a)[:, None]
                s = s.masked_fill(hidden, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1)) if not causal else torch.exp(
                s - torch.from_numpy(np.where(np.isfinite(lse[h, a:b]), lse[h, a:b], 0.0))[:, None])
            if causal:  # (a softmax of given log-sum-exps: its own derivative)
                total = p.sum(-1, keepdim=True)
                p = p / torch.where(total > 0, total, torch.ones_like(total))
            loss = loss + (p @ leaves[2][h // 2, c:e] * torch.from_numpy(do[h, a:b])).sum()
    loss.backward()
    for name, leaf in zip(("dq", "dk", "dv"), leaves):
        np.testing.assert_allclose(g[name]["value"], leaf.grad.numpy(), atol=1e-12)


@pytest.mark.parametrize("axes", [None, [0, 2, 1, 1, 0]])
@pytest.mark.parametrize("inter", [False, True])
def test_oracle_norm_gradients_are_torchs(axes, inter):
    rs = np.random.RandomState(2)
    x, dy = rs.standard_normal((2, 2, 3, 4, 16))
    w = rs.standard_normal(16)
    pos = rs.randint(0, 50, (2, 4) if axes is None else (3, 2, 4))
    freqs = np.exp(-rs.rand(5))
    dx, dw, _, _ = packed.norm_rotary_gradients(x, dy, w, pos, freqs, axes, 1e-3, inter, 1.3)
    xl, wl = torch.from_numpy(x).requires_grad_(), torch.from_numpy(w).requires_grad_()
    y = xl / torch.sqrt((xl * xl).mean(-1, keepdim=True) + 1e-3) * wl
    p = pos[..., None] if axes is None else np.moveaxis(pos[np.array(axes)], 0, -1)
    angle = torch.from_numpy((p * freqs)[:, None])
    a, b = (y[..., 0:10:2], y[..., 1:10:2]) if inter else (y[..., :5], y[..., 5:10])
    u = (a * angle.cos() - b * angle.sin()) * 1.3
    v = (a * angle.sin() + b * angle.cos()) * 1.3
    turned = torch.stack([u, v], -1).flatten(-2) if inter else torch.cat([u, v], -1)
    out = torch.cat([turned, y[..., 10:]], -1)
    np.testing.assert_allclose(packed.norm_rotary(x, w, pos, freqs, axes, 1e-3, inter, 1.3),
                               out.detach().numpy(), atol=1e-12)
    (out * torch.from_numpy(dy)).sum().backward()
    np.testing.assert_allclose(dx, xl.grad.numpy(), atol=1e-12)
    np.testing.assert_allclose(dw, wl.grad.numpy(), atol=1e-12)


def test_norm_gradient_workspace_follows_the_sums():
    """Sums over no heads of q pass through the workspace too."""
    lib = capi.load()
    p = rotary_params(heads=0)
    n = norm_params(k_weight=0)
    refused(lib.fl_attn_norm_rotary_bwd(ctypes.byref(p), ctypes.byref(n),
                                        ctypes.byref(norm_grads(dk_weight=0)), None, 0, None),
            capi.FL_ERR_INVALID_ARGUMENT, "workspace")
