"""The packed and normed operators as a program uses them: a training step
through autograd, streams, captured graphs, far rows, a prompt that goes into
the cache and on to single tokens."""

import numpy as np
import pytest

import flashlite_amd as fl
from packed_util import Problem, check, check_gradients

pytestmark = pytest.mark.gpu


def functions():
    import torch

    class NormRotary(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, q_weight, k_weight, positions, freqs, axes=None):
            ctx.save_for_backward(q, k, q_weight, k_weight, positions, freqs, axes)
            return fl.forward_norm_rotary(q, k, q_weight, k_weight, positions, freqs, axes)

        @staticmethod
        def backward(ctx, dq, dk):
            dq, dk = (x if x.stride(-1) == 1 else x.contiguous() for x in (dq, dk))
            q, k, q_weight, k_weight, *how = ctx.saved_tensors
            dq, dk, dqw, dkw = fl.backward_norm_rotary(dq, dk, q, k, q_weight, k_weight, *how)
            return dq, dk, dqw.to(q_weight.dtype), dkw.to(k_weight.dtype), None, None, None

    class Packed(torch.autograd.Function):
        @staticmethod
        def forward(ctx, q, k, v, starts, is_causal=True):
            out, lse = fl.forward_packed(q, k, v, starts, is_causal=is_causal, return_lse=True)
            ctx.save_for_backward(q, k, v, out, lse, starts)
            ctx.is_causal = is_causal
            return out

        @staticmethod
        def backward(ctx, dout):
            dout = dout if dout.stride(-1) == 1 else dout.contiguous()
            return *fl.backward_packed(dout, *ctx.saved_tensors, is_causal=ctx.is_causal), None, None

    return NormRotary, Packed


def plain_step(x, qw, kw, positions, freqs, axes, starts, h, hk):
    """The same step by elementary operations, in 64 bits."""
    import torch

    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    pos = positions.double()[axes.long()].movedim(0, -1)
    angle = (pos * freqs)[:, None]
    half = freqs.numel()

    def turn(y, w):
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + 1e-6) * w
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(),
                          y[..., 2 * half:]], -1)

    q, k = turn(q, qw), turn(k, kw)
    outs = []
    for a, b in zip(starts, starts[1:]):
        s = torch.matmul(q[0, :, a:b], k[0, :, a:b].repeat_interleave(h // hk, 0).transpose(
            1, 2).contiguous()) / np.sqrt(q.shape[-1])
        s = s.masked_fill(torch.ones(b - a, b - a, dtype=torch.bool).triu(1), -np.inf)
        outs.append(torch.matmul(torch.softmax(s, -1),
                                 v[0, :, a:b].repeat_interleave(h // hk, 0)))
    return torch.cat(outs, 1)[None]


@pytest.mark.parametrize("d", [64, 128])
def test_a_training_step(cuda, d):
    """Projection -> norms and rotation with three axes -> packed attention, and
    back: every gradient against torch's own in 64 bits.  Roundings of 16 bits
    in a chain of four operators: q, k, out, dout, the gradients of q and k and
    what the products round; each is within half a step of values whose sizes
    follow the root mean square, so 16 half steps of it bound a value by far."""
    import torch

    NormRotary, Packed = functions()
    rs = np.random.RandomState(d)
    h, hk, starts = 4, 2, [0, 37, 37, 120, 150]
    t = starts[-1]
    x = torch.from_numpy(rs.standard_normal((1, h + 2 * hk, t, d)).astype(np.float32)).to(
        torch.bfloat16)
    qw, kw = (torch.from_numpy(1 + 0.1 * rs.standard_normal(d)).float() for _ in range(2))
    positions = torch.stack([torch.arange(t) // 9, torch.arange(t) % 9, torch.arange(t) % 3])[:, None]
    freqs, _ = fl.rotary_frequencies(d)
    axes = fl.rotary_axes([d // 4, d // 8, d // 8])
    w = torch.from_numpy(rs.standard_normal((1, h, t, d)).astype(np.float32)).to(torch.bfloat16)

    leaf, qwl, kwl = (y.double().requires_grad_() for y in (x, qw, kw))
    want = plain_step(leaf, qwl, kwl, positions, freqs, axes, starts, h, hk)
    (want * w.double()).sum().backward()

    gx = x.to(cuda).transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    gq, gk = qw.to(cuda).requires_grad_(), kw.to(cuda).requires_grad_()
    q, k = NormRotary.apply(gx[:, :h], gx[:, h:h + hk], gq, gk, positions.to(cuda),
                            freqs.to(cuda), axes.to(cuda))
    assert q.requires_grad
    out = Packed.apply(q, k, gx[:, h + hk:],
                       torch.tensor(starts, dtype=torch.int32, device=cuda))
    (out * w.to(cuda)).sum().backward()
    for got, ref, share in ((out, want, 16), (gx.grad, leaf.grad, 16), (gq.grad, qwl.grad, 16),
                            (gk.grad, kwl.grad, 16)):
        got, ref = got.detach().double().cpu(), ref.detach()
        rms = ref.pow(2).mean().sqrt()
        assert ((got - ref).abs() <= share * 2.0 ** -8 * (rms + ref.abs())).all()


def test_results_are_not_recorded(cuda):
    import torch

    p = Problem(0, "float16", 64, 2, 2, [5])
    a = p.device(cuda)
    a["q"] = a["q"].detach().requires_grad_()
    assert not fl.forward_packed(**a).requires_grad
    for f in (fl.forward_packed, fl.backward_packed, fl.forward_norm_rotary,
              fl.backward_norm_rotary):
        assert "autograd" in f.__doc__


def test_on_another_stream(cuda):
    """A call runs on the current stream, behind what that stream still does."""
    import torch

    p = Problem(1, "bfloat16", 128, 4, 2, [100, 30])
    a = p.device(cuda)
    dout = p.view(p.dout, cuda)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        big = torch.randn((4096, 4096), device=cuda)
        q = a["q"] * 0
        for _ in range(4):
            big = big @ big * 1e-3
        q = q + a["q"] + (big[0, 0] * 0).to(q.dtype)
        out, lse = fl.forward_packed(**{**a, "q": q}, return_lse=True)
        g = fl.backward_packed(dout, q, a["k"], a["v"], out, lse, a["starts"], is_causal=True)
    torch.cuda.current_stream().wait_stream(stream)
    check(out, lse, p)
    check_gradients(g, p, out, lse)


def test_captured_and_replayed(cuda):
    """A step captured into a graph, replayed with new inputs in the same
    memory and with the program's own work between: each replay as the eager
    step.  Two captured steps have workspaces of their own."""
    import torch

    h, hk, d = 4, 2, 64
    lengths = [70, 1, 129]
    p = Problem(2, "float16", d, h, hk, lengths)
    a = p.device(cuda)
    w = torch.rand(d, device=cuda) + 0.5
    pos = torch.arange(p.rows, device=cuda)
    freqs = fl.rotary_frequencies(d, device=cuda)[0]
    dout = p.view(p.dout, cuda)
    k_in, q_in = a["k"].clone(), a["q"].clone()
    steps = []

    def make():
        ws = torch.empty(fl.packed_workspace_bytes(q_in, k_in, a["starts"]) // 4 + 1, device=cuda)
        nws = torch.empty(fl.norm_rotary_workspace_bytes(q_in, k_in) // 4 + 1, device=cuda)

        def step():
            q, k = fl.forward_norm_rotary(q_in, k_in, w, w, pos, freqs)
            out, lse = fl.forward_packed(q, k, a["v"], a["starts"], is_causal=True,
                                         return_lse=True)
            g = fl.backward_packed(dout, q, k, a["v"], out, lse, a["starts"], is_causal=True,
                                   workspace=ws)
            return (out, lse, *g, *fl.backward_norm_rotary(g[0], g[1], q_in, k_in, w, w, pos,
                                                           freqs, workspace=nws))

        return step

    for _ in range(2):
        step = make()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        steps.append((graph, res, step))
    for i in range(4):
        q_in.copy_(torch.randn(q_in.shape, device=cuda) * (i + 1))
        k_in.copy_(torch.randn(k_in.shape, device=cuda))
        torch.cuda.synchronize()
        for graph, _, _ in steps:
            graph.replay()
        torch.cuda.synchronize()
        want = steps[0][2]()
        for _, res, _ in steps:
            for x, y in zip(res, want):
                assert torch.equal(x, y)


def test_calls_with_their_outputs_allocate_nothing(cuda):
    import torch

    p = Problem(3, "bfloat16", 128, 4, 1, [100, 90])
    a = p.device(cuda)
    dout = p.view(p.dout, cuda)
    out, lse = torch.empty_like(a["q"]), torch.empty((1, p.h, p.rows), device=cuda)
    g = [torch.empty_like(a[x]) for x in "qkv"]
    ws = torch.empty(fl.packed_workspace_bytes(a["q"], a["k"], a["starts"]) // 4 + 1, device=cuda)
    w, dw = torch.ones(128, device=cuda), torch.empty((2, 128), device=cuda)
    nws = torch.empty(fl.norm_rotary_workspace_bytes(a["q"], a["k"]) // 4 + 1, device=cuda)
    pos, f = torch.arange(p.rows, device=cuda), fl.rotary_frequencies(128, device=cuda)[0]
    before = torch.cuda.memory_stats()["allocation.all.allocated"]
    fl.forward_packed(**a, out=out, return_lse=True, lse=lse)
    fl.backward_packed(dout, a["q"], a["k"], a["v"], out, lse, a["starts"], None, 0.0, True, *g, ws)
    fl.forward_norm_rotary(a["q"], a["k"], w, w, pos, f, q_out=g[0], k_out=g[1])
    fl.backward_norm_rotary(a["q"], a["k"], a["q"], a["k"], w, w, pos, f, q_out=g[0], k_out=g[1],
                            dq_weight=dw[0], dk_weight=dw[1], workspace=nws)
    assert torch.cuda.memory_stats()["allocation.all.allocated"] == before


def test_far_rows(cuda):
    """Query rows 2^21 elements apart: offsets past 32 bits in q, out, dout and dq."""
    import torch

    p = Problem(4, "float16", 64, 1, 1, [700, 400], gap=1)
    a = p.device(cuda)
    far = []
    for _ in range(4):
        far.append(torch.empty(((p.rows - 1) << 21) + 64, dtype=torch.float16, device=cuda)
                   .as_strided((1, 1, p.rows, 64), (0, 0, 1 << 21, 1)))
    q, out, dout, dq = far
    q.copy_(a["q"])
    dout.copy_(p.view(p.dout, cuda))
    lse = torch.zeros((1, 1, p.rows), device=cuda)
    fl.forward_packed(**{**a, "q": q}, out=out, return_lse=True, lse=lse)
    near, near_lse = fl.forward_packed(**a, return_lse=True)
    there = torch.from_numpy(p.inside()).to(cuda)
    assert torch.equal(out[:, :, there], near[:, :, there])
    want = fl.backward_packed(p.view(p.dout, cuda), a["q"], a["k"], a["v"], near, near_lse,
                              a["starts"], is_causal=True)
    got = fl.backward_packed(dout, q, a["k"], a["v"], out, lse, a["starts"], is_causal=True, dq=dq)
    assert torch.equal(got[0][:, :, there], want[0][:, :, there])
    assert torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


def test_a_prompt_goes_on_in_the_cache(cuda):
    """Prompts through forward_packed with their normed keys stored, then single
    tokens by forward_tree: as one attention over the whole sequences."""
    import torch

    h, hk, d, block = 4, 2, 64, 16
    lengths = [37, 5, 80]
    rs = np.random.RandomState(13)
    total = [n + 1 for n in lengths]
    freqs = fl.rotary_frequencies(d, device=cuda)[0]
    w = (torch.rand(d, device=cuda) + 0.5).half()
    x = torch.from_numpy(rs.standard_normal((1, h + 2 * hk, sum(total), d)).astype(np.float32))
    x = x.half().to(cuda)
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    starts = np.concatenate([[0], np.cumsum(total)])
    i32 = lambda y: torch.tensor(y, dtype=torch.int32, device=cuda)  # noqa: E731
    positions = i32(np.concatenate([np.arange(n) for n in total]))[None]
    qn, kn = fl.forward_norm_rotary(q, k, w, w, positions, freqs)
    want = fl.forward_packed(qn, kn, v, i32(starts), is_causal=True)

    tables = i32(np.arange(18).reshape(3, 6))
    k_cache, v_cache = (torch.zeros((18, hk, block, d), dtype=torch.float16, device=cuda)
                        for _ in range(2))
    token = np.concatenate([np.arange(n) for n in total])
    owner = np.repeat(np.arange(3), total)
    slots = torch.from_numpy((owner * 6 + token // block) * block + token % block).to(cuda)
    last = starts[1:] - 1
    prompt = slots.clone()
    prompt[last] = -1  # the single tokens come in a step of their own
    qp = fl.norm_rotary_to_cache(q, k, v, w, w, positions, prompt[None], freqs, k_cache, v_cache)
    keep = prompt >= 0
    assert torch.equal(qp[:, :, keep], qn[:, :, keep])
    step = lambda y: y[0][:, last].transpose(0, 1)[:, :, None].contiguous()  # noqa: E731
    q1 = fl.norm_rotary_to_cache(step(q), step(k), step(v), w, w, positions[0, last][:, None],
                                 slots[last][:, None], freqs, k_cache, v_cache)
    got = fl.forward_tree(q1, k_cache, v_cache, tables, i32(lengths))
    want = want[0][:, last].transpose(0, 1)[:, :, None]
    # two kernels' roundings of the same value (packed_util, tree_util): 2 u of p
    # and u of the output each, of values of at most max |v|
    assert (got.double() - want.double()).abs().max() <= 6 * 2.0 ** -11 * v.abs().max().double()


def test_binding_refusals(cuda):
    import torch

    p = Problem(5, "float16", 64, 4, 2, [5, 6])
    a = p.device(cuda)
    q, k, v, s = a["q"], a["k"], a["v"], a["starts"]
    lse = torch.zeros((1, 4, 11), device=cuda)
    for change, text in [
            (dict(q=q.float(), k=k.float(), v=v.float()), "FP16"),
            (dict(k=k.bfloat16()), "dtype"),
            (dict(q=q[0]), "4D"),
            (dict(q=q.expand(2, -1, -1, -1)), "one batch"),
            (dict(v=v[:, :1]), "k and v must be"),
            (dict(k=k[:, :, :5], v=v[:, :, :5]), "without key_starts"),
            (dict(starts=s.long()), "int32"),
            (dict(starts=s[:0]), "starts must be"),
            (dict(starts=s.cpu()), "same device"),
            (dict(key_starts=s[:2]), "as many entries"),
            (dict(out=q[:, :, :5]), "q's shape"),
            (dict(lse=lse), "return_lse"),
            (dict(lse=lse.half(), return_lse=True), "lse"),
            (dict(lse=lse[0], return_lse=True), "lse"),
            (dict(q=q[:, :3]), "multiple"),
            (dict(sm_scale=float("inf")), "sm_scale"),
            (dict(out=q[:, :1].expand(1, 4, -1, -1)), "o is written")]:
        with pytest.raises(RuntimeError, match=text):
            fl.forward_packed(**{**a, **change})
    base = dict(dout=q, q=q, k=k, v=v, out=q, lse=lse, starts=s)
    for change, text in [
            (dict(dout=q[:, :2]), "q's shape"), (dict(out=q[:, :2]), "q's shape"),
            (dict(lse=lse[..., :5]), "lse"), (dict(dk=q), "input's shape"),
            (dict(dq=q.bfloat16()), "dtype"),
            (dict(dv=v[:, :1].expand(1, 2, -1, -1)), "dv is written"),
            (dict(workspace=torch.zeros(4, device=cuda)), "bytes needed"),
            (dict(workspace=torch.zeros(4)), "workspace must be")]:
        with pytest.raises(RuntimeError, match=text):
            fl.backward_packed(**{**base, **change})
