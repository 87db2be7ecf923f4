"""More operators whose speed counts, and their plain forms: attention over
packed sequences with its gradient, and the norms of queries and keys for each
head with the position rotation in the same pass.

``forward_packed`` and ``backward_packed``: sequences of different lengths lie
one behind the other in a batch of one, [1, H, T, D], and attend to their own
keys only; query heads share key heads.  ``forward_norm_rotary``,
``backward_norm_rotary`` and ``norm_rotary_to_cache``: y = R(x r w) with r =
1 / sqrt(mean(x x) + eps) of each head's row, w the head's weight and R the
rotation of its position, which may have several axes (time, height, width).

A case is a dict of plain values; ``op`` names the operator:
  attend  seqs sequences of lo to hi tokens, h, hk, dim, dtype, causal, keys
          ("same": the queries' own tokens; "more": some cached ones before
          them; "apart": lengths of their own), layout ("qkv": views of one
          projection, "rows": [T, H, D], "heads": [H, T, D]), tail (rows
          behind the last sequence), lse
  grad    the same, the gradients of q, k and v from out and lse
  norm    b, h, hk, n, dim, rot (rotated part), style ("half", "inter"),
          axes (0: one position a token), dtype, layout ("bhnd", "bnhd"),
          weight ("f32" or the rows' type)
  normgrad  the same, the gradients of q, k and the weights
  store   b, n, h, hk, dim, rot, style, axes, dtype, block, weight
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}
_EPS = 1e-6


def _packed(name, op, seqs, lo, hi, h, hk, dim, dtype, causal=True, keys="same", layout="rows",
            tail=0, lse=True):
    return dict(name=name, op=op, seqs=seqs, lo=lo, hi=hi, h=h, hk=hk, dim=dim, dtype=dtype,
                causal=causal, keys=keys, layout=layout, tail=tail, lse=lse)


def _norm(name, op, b, h, hk, n, dim, rot, style, axes, dtype, layout, weight):
    return dict(name=name, op=op, b=b, h=h, hk=hk, n=n, dim=dim, rot=rot, style=style, axes=axes,
                dtype=dtype, layout=layout, weight=weight)


def _store(name, b, n, h, hk, dim, rot, style, axes, dtype, block, weight):
    return dict(name=name, op="store", b=b, n=n, h=h, hk=hk, dim=dim, rot=rot, style=style,
                axes=axes, dtype=dtype, block=block, weight=weight)


def listed():
    return [
        # A few short prompts admitted together; latency.
        _packed("packed-prompts", "attend", 5, 17, 300, 8, 8, 64, "f16", lse=False),
        # The forward pass of a training batch: documents of all lengths packed
        # to about 16k tokens, views of one projection, some padding.
        _packed("packed-train", "attend", 16, 64, 2000, 32, 8, 128, "bf16", layout="qkv", tail=100),
        # Pictures' patches through an encoder: everything sees everything.
        _packed("packed-patches", "attend", 12, 196, 1999, 12, 12, 64, "f16", causal=False,
                layout="qkv", lse=False),
        # A small batch's training step; latency.
        _packed("grad-short", "grad", 4, 33, 257, 8, 2, 64, "bf16"),
        # The backward pass of packed-train.
        _packed("grad-train", "grad", 16, 64, 2000, 32, 8, 128, "bf16", layout="qkv", tail=100),
        # Two long documents, one key head for eight query heads.
        _packed("grad-long", "grad", 2, 7000, 8192, 16, 2, 128, "f16", layout="heads"),
        # A short text's queries and keys on their way into attention.
        _norm("norm-short", "norm", 1, 8, 2, 333, 64, 64, "half", 0, "bf16", "bnhd", "bf16"),
        # A training batch of text and pictures: positions of three axes.
        _norm("norm-train", "norm", 2, 32, 8, 4096, 128, 128, "half", 3, "bf16", "bnhd", "f32"),
        # The gradients' way back through a short one in 32 bits.
        _norm("normgrad-short", "normgrad", 2, 8, 8, 257, 64, 32, "inter", 0, "f32", "bhnd", "f32"),
        # The backward pass of norm-train.
        _norm("normgrad-train", "normgrad", 2, 32, 8, 4096, 128, 128, "half", 3, "bf16", "bnhd",
              "f32"),
        # One token a request: normed, rotated, and stored in its cache row.
        _store("normstore-decode", 32, 1, 32, 8, 128, 128, "half", 0, "bf16", 16, "bf16"),
        # A prompt's rows, with pictures in it.
        _store("normstore-prompt", 4, 4096, 32, 8, 128, 128, "half", 3, "f16", 64, "f32"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_FLOPS = 6.0e11
_MOST_BYTES = 5.0e8


def draw(rng):
    while True:
        op = rng.choice(["attend", "attend", "grad", "grad", "norm", "normgrad", "store"])
        dim = rng.choice([64, 128])
        hk = rng.choice([1, 2, 4, 8, 16])
        h = hk * rng.choice([1, 1, 2, 3, 4, 7, 8])
        dtype = rng.choice(["f16", "bf16"])
        style = rng.choice(["half", "inter"])
        rot = rng.choice([dim, dim, dim // 2, dim // 4, 20])
        axes = rng.choice([0, 0, 2, 3])
        weight = rng.choice(["f32", dtype])
        if op in ("attend", "grad"):
            hi = _log_int(rng, 1, 8192)
            lo = rng.choice([hi, max(1, hi // 2), max(1, hi // 16), 0])
            seqs = _log_int(rng, 1, max(1, min(256, 32768 // hi)))
            c = _packed(None, op, seqs, lo, hi, h, hk, dim, dtype, rng.random() < 0.7,
                        rng.choice(["same", "same", "more", "apart"]),
                        rng.choice(["qkv", "rows", "heads"]), rng.choice([0, 0, 77]),
                        op == "grad" or rng.random() < 0.5)
            if c["keys"] != "same" and c["layout"] == "qkv":
                continue
            w = work(c)
            # the plain form's scores of one sequence
            if h * hi * hi * (4 if c["keys"] == "more" else 1) > 1 << 31:
                continue
        elif op in ("norm", "normgrad"):
            c = _norm(None, op, rng.choice([1, 2, 3, 8]), h, hk, _log_int(rng, 1, 16384), dim, rot,
                      style, axes, rng.choice([dtype, dtype, "f32"]),
                      rng.choice(["bhnd", "bnhd"]), weight)
            if weight != "f32" and c["dtype"] != weight:
                continue
            w = work(c)
        else:
            n = rng.choice([1, 1, 7, _log_int(rng, 2, 8192)])
            b = _log_int(rng, 1, max(1, min(256, 16384 // n)))
            c = _store(None, b, n, h, hk, dim, rot, style, axes, dtype,
                       rng.choice([8, 16, 16, 32, 64, 128, 20, 257]), weight)
            w = work(c)
        del c["name"]
        if w["flops"] <= _MOST_FLOPS and w["bytes"] <= _MOST_BYTES:
            return c


# ---------------------------------------------------------------------------
# Inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 31)
    return g


def _randint(g, lo, hi, shape):
    """Whole numbers in [lo, hi]."""
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda")


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * std).to(dtype)


def _freqs(rot):
    """Radians a position, 64 bits: base 10000."""
    j = torch.arange(rot // 2, dtype=torch.float64, device="cuda")
    return torch.pow(10000.0, -2.0 * j / rot)


def _axes(rot, axes):
    """The axis of each pair: sections of pairs, the first axis' the largest."""
    if axes == 0:
        return None
    pairs = rot // 2
    other = pairs * 3 // (4 * axes)
    each = [pairs - other * (axes - 1)] + [other] * (axes - 1)
    return torch.repeat_interleave(torch.arange(axes, device="cuda"),
                                   torch.tensor(each, device="cuda")).int()


def _positions(g, b, n, axes):
    first = _randint(g, 0, 4096, (b, 1))
    if axes == 0:
        return (first + torch.arange(n, device="cuda")).int()
    # pictures of 24 columns among text: time stands still in one, height and
    # width run
    i = torch.arange(n, device="cuda")
    time, place = i // 240, i % 240
    grid = [time, place // 24, place % 24][:axes]
    return torch.stack([first + x for x in grid]).int()


def _heads(g, b, h, n, dim, dtype, layout="bnhd"):
    """[b, h, n, dim]: the view of a projection's [b, n, h, dim], or contiguous."""
    if layout == "bhnd":
        return _randn(g, (b, h, n, dim), dtype)
    return _randn(g, (b, n, h, dim), dtype).transpose(1, 2)


def _weight(g, c):
    return (1.0 + 0.2 * torch.randn(c["dim"], generator=g, device="cuda")).to(_DT[c["weight"]])


def prepare(case, seed):
    return dict(_PREPARE[case["op"]](case, _gen(seed)), case=case)


def _lengths(g, lo, hi, count):
    """Whole numbers in [lo, hi], of a sum that is a case's own: in pairs
    around the middle, in random order."""
    half = _randint(g, lo, hi, (count // 2,))
    middle = torch.full((count % 2,), (lo + hi) // 2, device="cuda")
    return torch.cat([half, lo + hi - half, middle])[
        torch.randperm(count, generator=g, device="cuda")]


def _starts(lengths):
    return torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"),
                      torch.cumsum(lengths, 0)]).int()


def _prepare_attend(c, g):
    dt, d, h, hk = _DT[c["dtype"]], c["dim"], c["h"], c["hk"]
    lengths = _lengths(g, c["lo"], c["hi"], c["seqs"])
    starts = _starts(lengths)
    key_starts = None
    if c["keys"] == "more":
        key_starts = _starts(lengths + _lengths(g, 0, c["hi"], c["seqs"]))
    elif c["keys"] == "apart":
        key_starts = _starts(_lengths(g, c["lo"], c["hi"], c["seqs"]))
    ends = starts.tolist(), (starts if key_starts is None else key_starts).tolist()
    t, tk = ends[0][-1] + c["tail"], ends[1][-1] + c["tail"]
    if c["layout"] == "qkv":
        x = _randn(g, (t, h + 2 * hk, d), dt).transpose(0, 1)[None]
        q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    else:
        layout = "bhnd" if c["layout"] == "heads" else "bnhd"
        q = _heads(g, 1, h, t, d, dt, layout)
        k, v = (_heads(g, 1, hk, tk, d, dt, layout) for _ in range(2))
    s = dict(q=q, k=k, v=v, starts=starts, key_starts=key_starts, ends=ends,
             out=torch.zeros_like(q), lse=torch.zeros((1, h, t), device="cuda"))
    return s


def _prepare_grad(c, g):
    s = dict(_prepare_attend(c, g), case=c)
    _plain_attend(s)
    s["dout"] = _randn(g, (1, s["q"].shape[2], c["h"], c["dim"]), s["q"].dtype).transpose(1, 2)
    for x in ("q", "k", "v"):
        s["d" + x] = torch.zeros_like(s[x])
    return s


def _prepare_norm(c, g):
    dt = _DT[c["dtype"]]
    s = dict(positions=_positions(g, c["b"], c["n"], c["axes"]), freqs=_freqs(c["rot"]),
             axes=_axes(c["rot"], c["axes"]), q_weight=_weight(g, c), k_weight=_weight(g, c))
    for x, heads in (("q", c["h"]), ("k", c["hk"])):
        s[x] = _heads(g, c["b"], heads, c["n"], c["dim"], dt, c["layout"])
        s[x + "_out"] = torch.empty_like(s[x])
        if c["op"] == "normgrad":
            s["d" + x] = _heads(g, c["b"], heads, c["n"], c["dim"], dt, c["layout"])
            s["d%s_weight" % x] = torch.empty(c["dim"], device="cuda")
    return s


def _prepare_store(c, g):
    b, n, block, dt = c["b"], c["n"], c["block"], _DT[c["dtype"]]
    q = _heads(g, b, c["h"], n, c["dim"], dt)
    k, v = (_heads(g, b, c["hk"], n, c["dim"], dt) for _ in range(2))
    blocks = (b * n + block - 1) // block + 8
    # the new tokens' rows: runs of a block each, the blocks in random order
    order = torch.randperm(blocks, generator=g, device="cuda")
    if n == 1:
        slots = torch.randperm(blocks * block, generator=g, device="cuda")[:b]
    else:
        i = torch.arange(b * n, device="cuda")
        slots = order[i // block] * block + i % block
    counts = _randint(g, max(1, n - n // 8), n, (b, 1))
    slots = torch.where(torch.arange(n, device="cuda") < counts, slots.view(b, n), -1)
    caches = [_randn(g, (blocks, block, c["hk"], c["dim"]), dt).transpose(1, 2) for _ in range(2)]
    return dict(q=q, k=k, v=v, slots=slots, positions=_positions(g, b, n, c["axes"]),
                freqs=_freqs(c["rot"]), axes=_axes(c["rot"], c["axes"]), q_weight=_weight(g, c),
                k_weight=_weight(g, c), k_cache=caches[0], v_cache=caches[1],
                out=torch.zeros_like(q))


_PREPARE = {"attend": _prepare_attend, "grad": _prepare_grad, "norm": _prepare_norm,
            "normgrad": _prepare_norm, "store": _prepare_store}


# ---------------------------------------------------------------------------
# One pass


def run(state):
    if own:
        return _CALL[state["case"]["op"]](state)
    return _PLAIN[state["case"]["op"]](state)


def _call_attend(s):
    import flashlite_amd as fl

    c = s["case"]
    return fl.forward_packed(s["q"], s["k"], s["v"], s["starts"], s["key_starts"],
                             is_causal=c["causal"], out=s["out"], return_lse=c["lse"],
                             lse=s["lse"] if c["lse"] else None)


def _call_grad(s):
    import flashlite_amd as fl

    if "ws" not in s:  # a training loop makes its workspace with its first step
        need = fl.packed_workspace_bytes(s["q"], s["k"], s["starts"])
        s["ws"] = torch.empty(need // 4 + 1, dtype=torch.float32, device=s["q"].device)
    return fl.backward_packed(s["dout"], s["q"], s["k"], s["v"], s["out"], s["lse"], s["starts"],
                              s["key_starts"], is_causal=s["case"]["causal"], dq=s["dq"],
                              dk=s["dk"], dv=s["dv"], workspace=s["ws"])


def _call_norm(s):
    import flashlite_amd as fl

    return fl.forward_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"],
                                  s["freqs"], axes=s["axes"], eps=_EPS,
                                  interleaved=s["case"]["style"] == "inter", q_out=s["q_out"],
                                  k_out=s["k_out"])


def _call_normgrad(s):
    import flashlite_amd as fl

    if "ws" not in s:
        need = fl.norm_rotary_workspace_bytes(s["q"], s["k"])
        s["ws"] = torch.empty(need // 4 + 1, dtype=torch.float32, device=s["q"].device)
    return fl.backward_norm_rotary(s["dq"], s["dk"], s["q"], s["k"], s["q_weight"], s["k_weight"],
                                   s["positions"], s["freqs"], axes=s["axes"], eps=_EPS,
                                   interleaved=s["case"]["style"] == "inter", q_out=s["q_out"],
                                   k_out=s["k_out"], dq_weight=s["dq_weight"],
                                   dk_weight=s["dk_weight"], workspace=s["ws"])


def _call_store(s):
    import flashlite_amd as fl

    fl.norm_rotary_to_cache(s["q"], s["k"], s["v"], s["q_weight"], s["k_weight"], s["positions"],
                            s["slots"], s["freqs"], s["k_cache"], s["v_cache"], axes=s["axes"],
                            eps=_EPS, interleaved=s["case"]["style"] == "inter", out=s["out"])
    return s["out"], s["k_cache"], s["v_cache"]


_CALL = {"attend": _call_attend, "grad": _call_grad, "norm": _call_norm,
         "normgrad": _call_normgrad, "store": _call_store}


def _sequences(s):
    """(first query, end, first key, end) of the sequences that have queries or keys."""
    a, b = s["ends"]
    return [x for x in zip(a, a[1:], b, b[1:]) if x[0] < x[1] or x[2] < x[3]]


def _hidden(nq, nk, dev):
    """[nq, nk]: keys behind a query, the last query seeing all keys."""
    return (torch.arange(nk, device=dev) - (nk - nq)) > torch.arange(nq, device=dev)[:, None]


def _scores(s, q0, q1, k0, k1):
    """The sequence's scaled scores [hk, group, nq, nk] in 32 bits, hidden ones
    -inf, and its q [hk, group nq, d] and k [hk, nk, d]."""
    c = s["case"]
    hk, group, nq, nk = c["hk"], c["h"] // c["hk"], q1 - q0, k1 - k0
    q = s["q"][0, :, q0:q1].float().reshape(hk, group * nq, c["dim"])
    k = s["k"][0, :, k0:k1].float().contiguous()
    x = torch.matmul(q, k.transpose(1, 2).contiguous()) * (1.0 / math.sqrt(c["dim"]))
    x = x.view(hk, group, nq, nk)
    if c["causal"]:
        x = x.masked_fill(_hidden(nq, nk, q.device), -math.inf)
    return x, q, k


def _plain_attend(s):
    c = s["case"]
    hk, h, d = c["hk"], c["h"], c["dim"]
    for q0, q1, k0, k1 in _sequences(s):
        if q0 == q1:
            continue
        if k0 == k1:
            s["out"][0, :, q0:q1] = 0
            s["lse"][0, :, q0:q1] = -math.inf
            continue
        x = _scores(s, q0, q1, k0, k1)[0]
        top = x.amax(-1, keepdim=True).clamp(min=-1e30)
        x = (x - top).exp()
        total = x.sum(-1, keepdim=True)
        v = s["v"][0, :, k0:k1].float().contiguous()
        o = torch.matmul(x.view(hk, -1, k1 - k0), v).view(hk, h // hk, q1 - q0, d)
        o = o / total.clamp(min=1e-37)
        s["out"][0, :, q0:q1] = o.view(h, q1 - q0, d).to(s["out"].dtype)
        s["lse"][0, :, q0:q1] = (top + total.log()).view(h, q1 - q0)
    return (s["out"], s["lse"]) if c["lse"] else s["out"]


def _plain_grad(s):
    c = s["case"]
    hk, h, d = c["hk"], c["h"], c["dim"]
    scale = 1.0 / math.sqrt(d)
    for q0, q1, k0, k1 in _sequences(s):
        nq, nk = q1 - q0, k1 - k0
        if nq == 0 or nk == 0:
            s["dq"][0, :, q0:q1] = 0
            s["dk"][0, :, k0:k1] = 0
            s["dv"][0, :, k0:k1] = 0
            continue
        x, q, k = _scores(s, q0, q1, k0, k1)
        lse = s["lse"][0, :, q0:q1].reshape(hk, h // hk, nq, 1)
        p = (x - lse.clamp(min=-1e30)).exp().view(hk, -1, nk)
        do = s["dout"][0, :, q0:q1].float().reshape(hk, -1, d)
        delta = (do * s["out"][0, :, q0:q1].float().reshape(hk, -1, d)).sum(-1, keepdim=True)
        v = s["v"][0, :, k0:k1].float().transpose(1, 2).contiguous()
        s["dv"][0, :, k0:k1] = torch.matmul(p.transpose(1, 2).contiguous(), do).to(s["dv"].dtype)
        ds = p * (torch.matmul(do, v) - delta) * scale
        s["dk"][0, :, k0:k1] = torch.matmul(ds.transpose(1, 2).contiguous(), q).to(s["dk"].dtype)
        s["dq"][0, :, q0:q1] = torch.matmul(ds, k).view(h, nq, d).to(s["dq"].dtype)
    return s["dq"], s["dk"], s["dv"]


def _turns(s, dtype):
    """Cosine and sine [b, 1, n, pairs] of the tokens' angles, taken in 64 bits."""
    positions = s["positions"].double()
    if s["axes"] is None:
        positions = positions[..., None]
    else:
        positions = positions[s["axes"].long()].movedim(0, -1)
    angle = (positions * s["freqs"])[:, None]
    return angle.cos().to(dtype), angle.sin().to(dtype)


def _parts(x, pairs, inter):
    part = x[..., :2 * pairs]
    return (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :pairs], part[..., pairs:])


def _turned(x, cos, sin, inter):
    """The pairs of x's first columns rotated by the angles."""
    pairs = cos.shape[-1]
    a, b = _parts(x, pairs, inter)
    a, b = a * cos - b * sin, a * sin + b * cos
    part = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([part, x[..., 2 * pairs:]], -1)


def _normed(x, weight):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * weight.float()


def _plain_norm(s):
    cos, sin = _turns(s, torch.float32)
    for x in ("q", "k"):
        y = _turned(_normed(s[x], s[x + "_weight"]), cos, sin, s["case"]["style"] == "inter")
        s[x + "_out"].copy_(y)
    return s["q_out"], s["k_out"]


def _plain_normgrad(s):
    cos, sin = _turns(s, torch.float32)
    for x in ("q", "k"):
        g = _turned(s["d" + x].float(), cos, -sin, s["case"]["style"] == "inter")
        rows = s[x].float()
        r = torch.rsqrt((rows * rows).mean(-1, keepdim=True) + _EPS)
        rows = rows * r
        s["d%s_weight" % x].copy_((g * rows).sum((0, 1, 2), dtype=torch.float64))
        g = g * s[x + "_weight"].float()
        s[x + "_out"].copy_(r * (g - rows * (g * rows).mean(-1, keepdim=True)))
    return s["q_out"], s["k_out"], s["dq_weight"], s["dk_weight"]


def _plain_store(s):
    inter, block = s["case"]["style"] == "inter", s["case"]["block"]
    cos, sin = _turns(s, torch.float32)
    keep = s["slots"] >= 0
    q = _turned(_normed(s["q"], s["q_weight"]), cos, sin, inter).to(s["q"].dtype)
    k = _turned(_normed(s["k"], s["k_weight"]), cos, sin, inter).to(s["q"].dtype)
    s["out"].copy_(torch.where(keep[:, None, :, None], q, s["out"]))
    rows = s["slots"][keep]
    s["k_cache"][rows // block, :, rows % block] = k.transpose(1, 2)[keep]
    s["v_cache"][rows // block, :, rows % block] = s["v"].transpose(1, 2)[keep]
    return s["out"], s["k_cache"], s["v_cache"]


_PLAIN = {"attend": _plain_attend, "grad": _plain_grad, "norm": _plain_norm,
          "normgrad": _plain_normgrad, "store": _plain_store}


# ---------------------------------------------------------------------------
# Work and exact values


def work(case):
    c = case
    size = _SIZE[c["dtype"]]
    if c["op"] in ("attend", "grad"):
        lo, hi, seqs = c["lo"], c["hi"], c["seqs"]
        mean, square = (lo + hi) / 2, (lo * lo + lo * hi + hi * hi) / 3
        keys = mean + (hi / 2 if c["keys"] == "more" else 0)
        pairs = seqs * {"same": square, "more": square + mean * hi / 2,
                        "apart": mean * mean}[c["keys"]]
        if c["causal"]:  # the triangle in front of each sequence's end is hidden
            pairs -= seqs * (square - mean) / 2
        pairs = max(pairs, 0.0)
        rows = seqs * mean * c["h"] * c["dim"] * size      # q, or what has its shape
        cols = seqs * keys * c["hk"] * c["dim"] * size     # k or v
        lse = 4 * seqs * mean * c["h"] if c["lse"] else 0
        if c["op"] == "attend":
            return {"bytes": 2 * rows + 2 * cols + lse + 8 * seqs,
                    "flops": 4 * c["h"] * c["dim"] * pairs}
        return {"bytes": 4 * rows + 4 * cols + lse + 8 * seqs,
                "flops": 10 * c["h"] * c["dim"] * pairs}
    heads, b, n = c["h"] + c["hk"], c["b"], c["n"]
    rest = 4 * b * n * max(1, c["axes"]) + 4 * c["rot"] + 2 * c["dim"] * _SIZE[c["weight"]]
    rows = b * n * heads * c["dim"]
    if c["op"] == "norm":
        return {"bytes": 2 * rows * size + rest, "flops": 6 * rows}
    if c["op"] == "normgrad":
        return {"bytes": 3 * rows * size + rest + 8 * c["dim"], "flops": 14 * rows}
    v = b * n * c["hk"] * c["dim"]
    return {"bytes": 2 * (rows + v) * size + rest + 8 * b * n, "flops": 6 * rows}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "grad": _exact_grad, "norm": _exact_norm,
            "normgrad": _exact_normgrad, "store": _exact_store}[case["op"]](s)


def _head_scores(s, i, q0, q1, k0, k1):
    """One query head's scaled scores [nq, nk], 64 bits, hidden ones -inf."""
    c = s["case"]
    q = s["q"][0, i, q0:q1].double()
    k = s["k"][0, i * c["hk"] // c["h"], k0:k1].double()
    x = torch.matmul(q, k.t().contiguous()) / math.sqrt(c["dim"])
    if c["causal"]:
        x = x.masked_fill(_hidden(q1 - q0, k1 - k0, x.device), -math.inf)
    return x


def _exact_attend(s):
    """64 bits, one sequence and query head at a time."""
    c = s["case"]
    out = s["out"].double()
    lse = s["lse"].double()
    for q0, q1, k0, k1 in _sequences(s):
        for i in range(c["h"]):
            if q0 == q1:
                continue
            if k0 == k1:
                lse[0, i, q0:q1] = -math.inf
                continue
            x = _head_scores(s, i, q0, q1, k0, k1)
            norm = torch.logsumexp(x, -1)
            lse[0, i, q0:q1] = norm
            seen = norm > -math.inf
            p = torch.exp(x - torch.where(seen, norm, 0.0)[:, None])
            v = s["v"][0, i * c["hk"] // c["h"], k0:k1].double()
            out[0, i, q0:q1] = torch.matmul(p, v)
    return (out, lse) if c["lse"] else out


def _exact_grad(s):
    """64 bits from out and lse as they are given, one sequence and query head
    at a time: p = exp(s - lse), dv = p' dout, ds = p (dout v' - dout . out),
    dq = ds k, dk = ds' q, the last two times the scale."""
    c = s["case"]
    scale = 1.0 / math.sqrt(c["dim"])
    dq, dk, dv = (s["d" + x].double() * 0 for x in ("q", "k", "v"))
    for q0, q1, k0, k1 in _sequences(s):
        if q0 == q1 or k0 == k1:
            continue
        for i in range(c["h"]):
            j = i * c["hk"] // c["h"]
            lse = s["lse"][0, i, q0:q1].double()
            p = torch.exp(_head_scores(s, i, q0, q1, k0, k1)
                          - torch.where(lse > -math.inf, lse, 0.0)[:, None])
            do, o = s["dout"][0, i, q0:q1].double(), s["out"][0, i, q0:q1].double()
            dv[0, j, k0:k1] += torch.matmul(p.t().contiguous(), do)
            v = s["v"][0, j, k0:k1].double()
            ds = p * (torch.matmul(do, v.t().contiguous()) - (do * o).sum(-1)[:, None])
            dq[0, i, q0:q1] = scale * torch.matmul(ds, s["k"][0, j, k0:k1].double())
            dk[0, j, k0:k1] += scale * torch.matmul(ds.t().contiguous(),
                                                    s["q"][0, i, q0:q1].double())
    return dq, dk, dv


def _exact_turn(x, s, b, sign):
    """Request b's x [h, n, dim] in 64 bits, its pairs as complex numbers times e^(i sign a)."""
    pos = s["positions"].double()
    pos = pos[b][:, None] if s["axes"] is None else pos[:, b].t()[:, s["axes"].long()]
    angle = pos * s["freqs"]
    half = s["freqs"].numel()
    turn = torch.polar(torch.ones_like(angle), sign * angle)
    x = x.clone()
    if s["case"]["style"] == "inter":
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
    return x


def _exact_rows(s, x, b):
    rows = s[x][b].double()
    r = 1.0 / torch.sqrt(torch.sum(rows ** 2, -1, keepdim=True) / rows.shape[-1] + _EPS)
    return _exact_turn(rows * r * s[x + "_weight"].double(), s, b, 1.0)


def _exact_norm(s):
    return tuple(torch.stack([_exact_rows(s, x, b) for b in range(s["case"]["b"])])
                 for x in ("q", "k"))


def _exact_normgrad(s):
    """The chain rule: through the rotation (its transpose), the weight, and
    x / sqrt(mean(x x) + eps), whose derivative is (g - x (g . x) / (n rms^2)) / rms."""
    out = {}
    for x in ("q", "k"):
        dx, dw = [], torch.zeros(s["case"]["dim"], dtype=torch.float64, device="cuda")
        for b in range(s["case"]["b"]):
            g = _exact_turn(s["d" + x][b].double(), s, b, -1.0)
            rows = s[x][b].double()
            square = torch.sum(rows ** 2, -1, keepdim=True) / rows.shape[-1] + _EPS
            rms = torch.sqrt(square)
            dw += torch.sum(g * rows / rms, (0, 1))
            g = g * s[x + "_weight"].double()
            along = torch.sum(g * rows, -1, keepdim=True) / rows.shape[-1]
            dx.append((g - rows * along / square) / rms)
        out[x] = torch.stack(dx), dw
    return out["q"][0], out["k"][0], out["q"][1], out["k"][1]


def _exact_store(s):
    block = s["case"]["block"]
    out = s["out"].double()
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    for b in range(s["case"]["b"]):
        q, k = _exact_rows(s, "q", b), _exact_rows(s, "k", b)
        rows = torch.nonzero(s["slots"][b] >= 0)[:, 0]
        slot = s["slots"][b][rows]
        out[b][:, rows] = q[:, rows]
        for cache, x in zip(caches, (k, s["v"][b].double())):
            cache[slot // block, :, slot % block] = x[:, rows].transpose(0, 1)
    return out, caches[0], caches[1]
