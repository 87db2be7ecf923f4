"""The serving operators whose speed counts, and their plain forms.

One step of decoding over a paged cache, with or without drafted tokens:
``plan_cache`` (blocks, slots and positions of the new tokens), ``plan_tree``
(the drafts' ancestors and positions), ``rotary_to_cache`` (rotated q out,
rotated k and v into the cache) and ``forward_tree`` (attention over it); and
the rotary of a training step, ``forward_rotary`` and ``backward_rotary``.

A case is a dict of plain values; ``op`` names the operator:
  plan    b requests, width n of the maps, block size, table width m, ended
          (share of requests that end), short (whether the pool runs out)
  tree    b trees of up to n drafts, branch (mean number of children)
  rotary  b, h, hk, n, dim, rot (rotated part of the head), style
          ("half", "inter"), dtype, layout ("bhnd", "bnhd"), far (largest
          position), back (the backward pass), scale
  store   b, n, h, hk, dim, rot, style, dtype, block, far
  attend  b, n, h, hk, dim, dtype, block, lo and hi (lengths of the
          requests), tree (a mask of ancestors; a chain without), ragged
          (requests with fewer than n drafts), lse, paged ("rows": a block is
          [block, heads, dim], "heads": [heads, block, dim])
"""

from __future__ import annotations

import math

import torch

own = False

_DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def _plan(name, b, n, block, m, ended=0.0, short=False):
    return dict(name=name, op="plan", b=b, n=n, block=block, m=m, ended=ended, short=short)


def _tree(name, b, n, branch):
    return dict(name=name, op="tree", b=b, n=n, branch=branch)


def _rotary(name, b, h, hk, n, dim, rot, style, dtype, layout, far, back, scale):
    return dict(name=name, op="rotary", b=b, h=h, hk=hk, n=n, dim=dim, rot=rot, style=style,
                dtype=dtype, layout=layout, far=far, back=back, scale=scale)


def _store(name, b, n, h, hk, dim, rot, style, dtype, block, far):
    return dict(name=name, op="store", b=b, n=n, h=h, hk=hk, dim=dim, rot=rot, style=style,
                dtype=dtype, block=block, far=far)


def _attend(name, b, n, h, hk, dim, dtype, block, lo, hi, tree, ragged=False, lse=False,
            paged="rows"):
    return dict(name=name, op="attend", b=b, n=n, h=h, hk=hk, dim=dim, dtype=dtype, block=block,
                lo=lo, hi=hi, tree=tree, ragged=ragged, lse=lse, paged=paged)


def listed():
    return [
        # A decode step of a batch: one token a request, a few take a block.
        _plan("plan-decode", 32, 1, 16, 256, ended=0.1),
        # Prompts admitted together: every block and every slot of them.
        _plan("plan-prompts", 64, 4096, 64, 80),
        # Small drafts of a small batch; latency.
        _tree("tree-small", 8, 16, 2.0),
        # Wide drafts of a large batch.
        _tree("tree-wide", 128, 192, 3.0),
        # The rotary of a training step over projection outputs, ragged length.
        _rotary("rotary-train", 2, 8, 8, 1999, 64, 64, "half", "bf16", "bnhd", 1999, False, 1.0),
        # The gradients' way back through it on a very long sequence, the
        # positions scaled for long contexts.
        _rotary("rotary-back-long", 1, 16, 16, 16384, 128, 128, "inter", "f16", "bhnd", 16384,
                True, 1.2),
        # One token a request: rotated, and stored in its cache row.
        _store("store-decode", 32, 1, 32, 8, 128, 128, "half", "f16", 16, 4096),
        # A prompt's rows, part of the head rotated.
        _store("store-prompt", 4, 4096, 32, 8, 128, 64, "half", "bf16", 64, 16384),
        # The smallest decode step: 16 heads of 4096 keys.
        _attend("decode-step", 2, 1, 8, 8, 64, "f16", 64, 4096, 4096, False),
        # A tree of drafts checked over caches of about 5000 keys.
        _attend("verify-tree", 4, 26, 16, 4, 128, "bf16", 16, 4500, 5500, True, ragged=True,
                lse=True),
        # A large decode batch of very different lengths.
        _attend("decode-ragged", 32, 1, 32, 8, 128, "bf16", 16, 256, 8192, False),
        # Many drafts over long caches: as much product as traffic.
        _attend("verify-long", 8, 64, 32, 8, 128, "f16", 64, 15000, 16384, True, paged="heads"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_MOST_FLOPS = 1.3e11
_MOST_BYTES = 5.0e8


def draw(rng):
    while True:
        op = rng.choice(["plan", "tree", "rotary", "store", "attend", "attend", "attend"])
        dim = rng.choice([64, 128])
        hk = rng.choice([1, 2, 4, 8, 16])
        h = hk * rng.choice([1, 1, 2, 3, 4, 7, 8])
        block = rng.choice([8, 16, 16, 32, 64, 128, 20, 257])
        dtype = rng.choice(["f16", "bf16"])
        style = rng.choice(["half", "inter"])
        rot = rng.choice([dim, dim, dim // 2, dim // 4, 20])
        if op == "plan":
            n = rng.choice([1, 1, 5, _log_int(rng, 2, 8192)])
            b = _log_int(rng, 1, max(1, min(1024, (1 << 20) // n)))
            m = n // block + rng.choice([40, 300])
            if b * m > 1 << 20:
                continue
            c = _plan(None, b, n, block, m, rng.choice([0.0, 0.0, 0.1, 0.5]), rng.random() < 0.2)
        elif op == "tree":
            n = _log_int(rng, 1, 512)
            c = _tree(None, _log_int(rng, 1, max(1, min(512, (1 << 16) // n))), n,
                      rng.choice([1.0, 2.0, 4.0, 16.0]))
        elif op == "rotary":
            c = _rotary(None, rng.choice([1, 2, 3, 8]), h, hk, _log_int(rng, 1, 16384), dim, rot,
                        style, rng.choice(["f16", "bf16", "f32"]), rng.choice(["bhnd", "bnhd"]),
                        rng.choice([0, 4096, 131072, 1 << 20]), rng.random() < 0.5,
                        rng.choice([1.0, 1.0, 1.2]))
        elif op == "store":
            n = rng.choice([1, 1, 7, _log_int(rng, 2, 8192)])
            b = _log_int(rng, 1, max(1, min(256, 16384 // n)))
            c = _store(None, b, n, h, hk, dim, rot, style, dtype, block,
                       rng.choice([4096, 131072, 1 << 20]))
        else:
            kind = rng.choice(["decode", "decode", "verify", "verify", "chunk"])
            n = (1 if kind == "decode" else _log_int(rng, 2, 96) if kind == "verify"
                 else _log_int(rng, 97, 700))
            hi = _log_int(rng, 1, 32768)
            lo = rng.choice([hi, hi, max(1, hi // 2), max(1, hi // 32)])
            c = _attend(None, rng.choice([1, 2, 3, 5, 8, 16, 40]), n, h, hk, dim, dtype, block,
                        lo, hi, kind == "verify" and rng.random() < 0.8, rng.random() < 0.3,
                        rng.random() < 0.3, rng.choice(["rows", "heads"]))
        del c["name"]
        w = work(c)
        if w["flops"] > _MOST_FLOPS or w["bytes"] > _MOST_BYTES:
            continue
        if c["op"] == "attend":  # the plain form's scores and gathered keys
            if c["b"] * (c["hi"] + c["n"]) * (c["h"] * c["n"] + 2 * c["hk"] * c["dim"]) > 1 << 30:
                continue
        return c


# ---------------------------------------------------------------------------
# Inputs


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * int(seed) + 29)
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


def _heads(g, b, h, n, dim, dtype, layout="bnhd"):
    """[b, h, n, dim]: the view of a projection's [b, n, h, dim], or contiguous."""
    if layout == "bhnd":
        return _randn(g, (b, h, n, dim), dtype)
    return _randn(g, (b, n, h, dim), dtype).transpose(1, 2)


def _pages(g, lengths, block, spare=0):
    """Tables of distinct blocks in random order for `lengths` tokens a
    request, -1 behind them, and the number of blocks."""
    need = (lengths + block - 1) // block
    total, m = int(need.sum()) + spare, max(1, int(need.max()))
    ids = torch.randperm(max(1, total), generator=g, device="cuda")
    at = (torch.cumsum(need, 0) - need)[:, None] + torch.arange(m, device="cuda")
    tables = torch.where(torch.arange(m, device="cuda") < need[:, None],
                         ids[at.clamp(max=max(0, total - 1))], -1)
    return tables.to(torch.int32), max(1, total)


def _parents(g, b, n, branch):
    """Each draft's parent among the earlier ones (-1: the prompt), about
    `branch` children each, as sorted drafts of a beam come."""
    i = torch.arange(n, device="cuda").expand(b, n)
    mean = torch.floor(i / branch) - 1
    jitter = torch.floor(torch.rand((b, n), generator=g, device="cuda") * 2 * branch)
    return torch.minimum((mean + jitter - branch // 2).long().clamp(min=-1), i - 1).to(torch.int32)


def _cache(g, c, blocks):
    shape = ((blocks, c["block"], c["hk"], c["dim"]) if c.get("paged", "rows") == "rows"
             else (blocks, c["hk"], c["block"], c["dim"]))
    k, v = (_randn(g, shape, _DT[c["dtype"]]) for _ in range(2))
    return (k.transpose(1, 2), v.transpose(1, 2)) if c.get("paged", "rows") == "rows" else (k, v)


def prepare(case, seed):
    g = _gen(seed)
    return dict(_PREPARE[case["op"]](case, g), case=case)


def _prepare_plan(c, g):
    b, n, block, m = c["b"], c["n"], c["block"], c["m"]
    lengths = _randint(g, 0, m * block - n, (b,))
    if n > 64:
        lengths = lengths // 8  # prompts come with a short shared prefix
    counts = torch.full((b,), n, device="cuda") if n == 1 else _randint(g, max(1, n // 2), n, (b,))
    ended = torch.rand((b,), generator=g, device="cuda") < c["ended"]
    counts = torch.where(ended, -1, counts)
    tables, used = _pages(g, lengths, block)
    held = (lengths + block - 1) // block
    full = torch.full((b, m), -1, dtype=torch.int32, device="cuda")
    full[:, :tables.shape[1]] = tables
    # the pool behind the blocks in use: a ring that starts somewhere
    need = int(((lengths + counts.clamp(min=0) + block - 1) // block - held).clamp(min=0).sum())
    size = b * m
    free = min(size - used, need // 2 if c["short"] else need + 64)
    head = int(_randint(g, 0, size - 1, (1,)))
    ring = torch.full((size,), -1, dtype=torch.int32, device="cuda")
    at = (head + torch.arange(free, device="cuda")) % size
    ring[at] = (used + torch.randperm(free, generator=g, device="cuda")).to(torch.int32)
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(lengths=lengths.int(), counts=counts.int(), tables=full, held=held.int(),
                free=ring, state=torch.tensor([head, free], **i32),
                held_out=torch.zeros(b, **i32), state_out=torch.zeros(2, **i32),
                positions=torch.empty((b, n), **i32),
                slots=torch.empty((b, n), dtype=torch.int64, device="cuda"),
                info=torch.empty((b, 4), **i32))


def _prepare_tree(c, g):
    b, n = c["b"], c["n"]
    words = (n + 63) // 64
    return dict(parents=_parents(g, b, n, c["branch"]), lengths=_randint(g, 0, 8192, (b,)).int(),
                counts=_randint(g, max(1, n // 2), n, (b,)).int(),
                mask=torch.empty((b, n, words), dtype=torch.int64, device="cuda"),
                positions=torch.empty((b, n), dtype=torch.int32, device="cuda"))


def _prepare_rotary(c, g):
    b, n = c["b"], c["n"]
    q = _heads(g, b, c["h"], n, c["dim"], _DT[c["dtype"]], c["layout"])
    k = _heads(g, b, c["hk"], n, c["dim"], _DT[c["dtype"]], c["layout"])
    first = _randint(g, 0, max(0, c["far"] - n), (b, 1))
    positions = (first + torch.arange(n, device="cuda")).int()
    return dict(q=q, k=k, positions=positions, freqs=_freqs(c["rot"]), q_out=torch.empty_like(q),
                k_out=torch.empty_like(k))


def _prepare_store(c, g):
    b, n, block = c["b"], c["n"], c["block"]
    dt = _DT[c["dtype"]]
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
    k_cache, v_cache = _cache(g, c, blocks)
    first = _randint(g, 0, max(0, c["far"] - n), (b, 1))
    return dict(q=q, k=k, v=v, slots=slots, positions=(first + torch.arange(n, device="cuda")).int(),
                freqs=_freqs(c["rot"]), k_cache=k_cache, v_cache=v_cache, out=torch.zeros_like(q))


def _bits(seen):
    """[..., n] of truth values -> the int64 words of their bits."""
    n = seen.shape[-1]
    words = (n + 63) // 64
    wide = torch.zeros(seen.shape[:-1] + (64 * words,), dtype=torch.int64, device=seen.device)
    wide[..., :n] = seen
    return (wide.view(seen.shape[:-1] + (words, 64)) << torch.arange(64, device=seen.device)).sum(-1)


def _ancestors(parents):
    """[b, n, n]: whether draft j is i or above it."""
    b, n = parents.shape
    index = torch.arange(n, device=parents.device)
    up = torch.where((parents >= 0) & (parents < index), parents.long(), n)
    up = torch.cat([up, torch.full((b, 1), n, device=parents.device)], 1)
    seen = torch.eye(n + 1, dtype=torch.bool, device=parents.device)[:, :n].expand(b, n + 1, n)
    for _ in range(max(1, (n - 1).bit_length())):  # the way up doubles each time
        seen = seen | seen.gather(1, up[:, :, None].expand(b, n + 1, n))
        up = up.gather(1, up)
    return seen[:, :n]


def _prepare_attend(c, g):
    b, n, dt = c["b"], c["n"], _DT[c["dtype"]]
    lengths = _randint(g, c["lo"], c["hi"], (b,))
    if c["lo"] < c["hi"]:
        lengths[0] = c["hi"]
    tables, blocks = _pages(g, lengths + n, c["block"], spare=4)
    counts = _randint(g, max(1, n // 2), n, (b,)) if c["ragged"] else None
    mask = _bits(_ancestors(_parents(g, b, n, 2.0))) if c["tree"] else None
    q = _heads(g, b, c["h"], n, c["dim"], dt)
    k_cache, v_cache = _cache(g, c, blocks)
    lse = torch.zeros((b, c["h"], n), device="cuda") if c["lse"] else None
    return dict(q=q, k_cache=k_cache, v_cache=v_cache, tables=tables, lengths=lengths.int(),
                counts=None if counts is None else counts.int(), mask=mask,
                out=torch.zeros_like(q), lse=lse)


_PREPARE = {"plan": _prepare_plan, "tree": _prepare_tree, "rotary": _prepare_rotary,
            "store": _prepare_store, "attend": _prepare_attend}


# ---------------------------------------------------------------------------
# One pass


def run(state):
    if own:
        return _call(state)
    return _PLAIN[state["case"]["op"]](state)


def _call(s):
    import flashlite_amd as fl

    c = s["case"]
    if c["op"] == "plan":
        fl.plan_cache(s["lengths"], s["counts"], s["tables"], s["held"], s["free"], s["state"],
                      c["block"], c["n"], held_out=s["held_out"], state_out=s["state_out"],
                      positions=s["positions"], slots=s["slots"], info=s["info"])
        return {k: s[k] for k in _PLANNED}
    if c["op"] == "tree":
        return fl.plan_tree(s["parents"], s["lengths"], s["counts"], mask=s["mask"],
                            positions=s["positions"])
    if c["op"] == "rotary":
        turn = fl.backward_rotary if c["back"] else fl.forward_rotary
        return turn(s["q"], s["k"], s["positions"], s["freqs"], c["style"] == "inter", c["scale"],
                    s["q_out"], s["k_out"])
    if c["op"] == "store":
        fl.rotary_to_cache(s["q"], s["k"], s["v"], s["positions"], s["slots"], s["freqs"],
                           s["k_cache"], s["v_cache"], c["style"] == "inter", 1.0, s["out"])
        return s["out"], s["k_cache"], s["v_cache"]
    if "ws" not in s:  # a serving loop makes its workspace with its first step
        need = fl.tree_workspace_bytes(s["q"], s["k_cache"])
        s["ws"] = torch.empty(need // 4 + 1, dtype=torch.float32, device=s["q"].device)
    return fl.forward_tree(s["q"], s["k_cache"], s["v_cache"], s["tables"], s["lengths"],
                           s["mask"], s["counts"], 0.0, s["out"], c["lse"], s["lse"], s["ws"])


_PLANNED = ("positions", "slots", "info", "held_out", "state_out", "tables", "free")


def _plain_plan(s):
    c = s["case"]
    n, block, m, size = c["n"], c["block"], c["m"], s["free"].numel()
    lengths, counts = s["lengths"].long().clamp(min=0), s["counts"].long()
    ended, new = counts < 0, counts.clamp(0, n)
    held = s["held"].long().clamp(0, m)
    head, count = s["state"].long().unbind()
    want = (lengths + new + block - 1) // block
    wide = (new > 0) & (want > m)
    need = torch.where((new > 0) & ~wide, (want - held).clamp(min=0), 0)
    before = torch.cumsum(need, 0) - need
    served = ~wide & ((need == 0) | (before + need <= count))
    taken = torch.where(served, need, 0)
    cols = torch.arange(m, device=held.device)
    from_ring = s["free"][(head + before[:, None] + cols - held[:, None]) % size]
    filled = (cols >= held[:, None]) & (cols < (held + taken)[:, None])
    # blocks of ended requests go behind the ring's last
    back = torch.where(ended, held, 0)
    behind = (torch.cumsum(back, 0) - back)[:, None] + cols
    given = torch.minimum(back, (size - count - behind[:, 0]).clamp(min=0))
    put = cols < given[:, None]
    ring = torch.cat([s["free"], s["free"][:1]])
    ring.scatter_(0, torch.where(put, (head + count + behind) % size, size).view(-1),
                  s["tables"].view(-1))
    s["free"].copy_(ring[:size])
    s["tables"].copy_(torch.where(filled, from_ring, s["tables"]))
    s["held_out"].copy_(torch.where(ended, 0, held + taken))
    total = taken.sum()
    s["state_out"].copy_(torch.stack([(head + total) % size,
                                      count - total + given.sum()]))
    s["info"].copy_(torch.stack([torch.where(wide, 2, torch.where(served, 0, 1)), held,
                                 taken - given,
                                 (head + torch.where(ended, count + behind[:, 0], before)) % size],
                                1))
    i = torch.arange(n, device=held.device)
    at = lengths[:, None] + i
    ids = s["tables"].long().gather(1, (at // block).clamp(max=m - 1))
    there = (i < new[:, None]) & served[:, None] & (ids >= 0)
    s["slots"].copy_(torch.where(there, ids * block + at % block, -1))
    s["positions"].copy_(torch.where(there, at, -1))
    return {k: s[k] for k in _PLANNED}


def _plain_tree(s):
    n = s["case"]["n"]
    index = torch.arange(n, device=s["parents"].device)
    there = index < s["counts"][:, None]
    seen = _ancestors(s["parents"]) & there[:, :, None]
    s["mask"].copy_(_bits(seen))
    depth = seen.sum(-1) - 1
    s["positions"].copy_(torch.where(there, s["lengths"][:, None] + depth, -1))
    return s["mask"], s["positions"]


def _turned(x, positions, freqs, inter, scale, back):
    """x [b, h, n, dim] with its first 2 len(freqs) columns rotated, 32 bits."""
    half = freqs.numel()
    angle = positions.double()[:, None, :, None] * freqs
    cos, sin = (angle.cos() * scale).float(), (angle.sin() * (-scale if back else scale)).float()
    x = x.float()
    part = x[..., :2 * half]
    a, b = (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :half], part[..., half:])
    a, b = a * cos - b * sin, a * sin + b * cos
    part = torch.stack([a, b], -1).flatten(-2) if inter else torch.cat([a, b], -1)
    return torch.cat([part, x[..., 2 * half:]], -1)


def _plain_rotary(s):
    c = s["case"]
    inter = c["style"] == "inter"
    s["q_out"].copy_(_turned(s["q"], s["positions"], s["freqs"], inter, c["scale"], c["back"]))
    s["k_out"].copy_(_turned(s["k"], s["positions"], s["freqs"], inter, c["scale"], c["back"]))
    return s["q_out"], s["k_out"]


def _plain_store(s):
    c = s["case"]
    inter, block = c["style"] == "inter", c["block"]
    keep = s["slots"] >= 0
    q = _turned(s["q"], s["positions"], s["freqs"], inter, 1.0, False).to(s["q"].dtype)
    k = _turned(s["k"], s["positions"], s["freqs"], inter, 1.0, False).to(s["q"].dtype)
    s["out"].copy_(torch.where(keep[:, None, :, None], q, s["out"]))
    rows = s["slots"][keep]
    s["k_cache"][rows // block, :, rows % block] = k.transpose(1, 2)[keep]
    s["v_cache"][rows // block, :, rows % block] = s["v"].transpose(1, 2)[keep]
    return s["out"], s["k_cache"], s["v_cache"]


def _seen_drafts(s):
    """[b, n, n]: whether draft i sees draft j."""
    c, dev = s["case"], s["q"].device
    n, b = c["n"], c["b"]
    index = torch.arange(n, device=dev)
    if s["mask"] is None:
        seen = (index <= index[:, None]).expand(b, n, n)
    else:
        seen = ((s["mask"][:, :, index // 64] >> (index % 64)) & 1).bool()
    return seen if s["counts"] is None else seen & (index < s["counts"][:, None, None])


def _plain_attend(s):
    c, q = s["case"], s["q"]
    b, h, n, d = q.shape
    hk, block, dev = c["hk"], c["block"], q.device
    most = c["hi"] + n
    key = torch.arange(most, device=dev)
    at = s["tables"].long()[:, (key // block).clamp(max=s["tables"].shape[1] - 1)].clamp(min=0)
    k = s["k_cache"][at, :, key % block].float().permute(0, 2, 3, 1).contiguous()
    v = s["v_cache"][at, :, key % block].float().permute(0, 2, 1, 3).contiguous()
    draft = key - s["lengths"].long()[:, None]
    seen = (draft < 0)[:, None] | (((draft >= 0) & (draft < n))[:, None] & _seen_drafts(s).gather(
        2, draft.clamp(0, n - 1)[:, None].expand(b, n, most)))
    v = v * seen.any(1)[:, None, :, None]
    x = q.float().reshape(b, hk, (h // hk) * n, d).contiguous()
    x = torch.matmul(x, k).view(b, hk, h // hk, n, most) * (1.0 / math.sqrt(d))
    x = x.masked_fill(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True).clamp(min=-1e30)
    x = (x - top).exp()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, hk, -1, most), v).view(b, hk, h // hk, n, d) / total.clamp(min=1e-37)
    there = (torch.arange(n, device=dev) < (n if s["counts"] is None else s["counts"][:, None]))
    there = there.expand(b, n)[:, None, :]
    s["out"].copy_(torch.where(there[..., None], o.reshape(b, h, n, d).to(q.dtype), s["out"]))
    if not c["lse"]:
        return s["out"]
    lse = (top + total.log()).reshape(b, h, n)
    s["lse"].copy_(torch.where(there, lse, s["lse"]))
    return s["out"], s["lse"]


_PLAIN = {"plan": _plain_plan, "tree": _plain_tree, "rotary": _plain_rotary,
          "store": _plain_store, "attend": _plain_attend}


# ---------------------------------------------------------------------------
# Work and exact values


def work(case):
    c = case
    op, b, n = c["op"], c["b"], c["n"]
    if op == "plan":
        blocks = b * (n // c["block"] + 1)
        # lengths, counts, held in and out, info; a table entry a block touched,
        # read or taken and written; position and slot of each new token
        return {"bytes": 32 * b + 8 * blocks + 12 * b * n, "flops": 4 * b * n}
    if op == "tree":
        words = (n + 63) // 64
        return {"bytes": 8 * b + b * n * (4 + 8 * words + 4), "flops": b * n * words}
    size = _SIZE[c["dtype"]]
    if op == "rotary":
        heads = c["h"] + c["hk"]
        return {"bytes": 2 * b * n * heads * c["dim"] * size + 4 * b * n + 4 * c["rot"],
                "flops": 3 * b * n * heads * c["rot"]}
    if op == "store":
        heads = c["h"] + c["hk"]
        return {"bytes": 2 * b * n * (heads + c["hk"]) * c["dim"] * size + 12 * b * n + 4 * c["rot"],
                "flops": 3 * b * n * heads * c["rot"]}
    mean = (c["lo"] + c["hi"]) / 2
    kv = b * c["hk"] * (mean + n) * 2 * c["dim"] * size
    qo = 2 * b * c["h"] * n * c["dim"] * size
    rest = b * (4 + 4 * mean / c["block"]) + (4 * b * c["h"] * n if c["lse"] else 0)
    return {"bytes": kv + qo + rest,
            "flops": 4 * b * c["h"] * n * c["dim"] * (mean + (n + 1) / 2)}


def exact(case, seed):
    """64 bits, one request (and for attention one key head) at a time."""
    if case["op"] in ("plan", "tree"):
        return None  # whole numbers
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "store": _exact_store, "attend": _exact_attend}[case["op"]](s)


def _exact_turn(x, positions, freqs, inter, scale, sign):
    """One request's x [h, n, dim] as complex numbers times scale e^(i sign a)."""
    half = freqs.numel()
    x = x.double()
    turn = torch.polar(torch.full((positions.numel(), half), float(scale), dtype=torch.float64,
                                  device=x.device), sign * torch.outer(positions.double(), freqs))
    if inter:
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2]) * turn
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = z.real, z.imag
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half]) * turn
        x[..., :half], x[..., half:2 * half] = z.real, z.imag
    return x


def _exact_rotary(s):
    c = s["case"]
    args = (s["freqs"], c["style"] == "inter", c["scale"], -1.0 if c["back"] else 1.0)
    return tuple(torch.stack([_exact_turn(x[i], s["positions"][i], *args)
                              for i in range(c["b"])]) for x in (s["q"], s["k"]))


def _exact_store(s):
    c, block = s["case"], s["case"]["block"]
    out = s["out"].double()
    caches = [s["k_cache"].double(), s["v_cache"].double()]
    for i in range(c["b"]):
        args = (s["positions"][i], s["freqs"], c["style"] == "inter", 1.0, 1.0)
        q, k = _exact_turn(s["q"][i], *args), _exact_turn(s["k"][i], *args)
        rows = torch.nonzero(s["slots"][i] >= 0)[:, 0]
        slot = s["slots"][i][rows]
        out[i][:, rows] = q[:, rows]
        for cache, x in zip(caches, (k, s["v"][i].double())):
            cache[slot // block, :, slot % block] = x[:, rows].transpose(0, 1)
    return out, caches[0], caches[1]


def _exact_attend(s):
    c, q = s["case"], s["q"]
    b, h, n, d = q.shape
    hk, block, dev = c["hk"], c["block"], q.device
    group = h // hk
    out = s["out"].double()
    lse = torch.zeros((b, h, n), dtype=torch.float64, device=dev)
    for i in range(b):
        length = int(s["lengths"][i])
        count = n if s["counts"] is None else int(s["counts"][i])
        key = torch.arange(length + count, device=dev)
        page = s["tables"][i].long()[key // block]
        hidden = torch.zeros((count, length + count), dtype=torch.bool, device=dev)
        j = torch.arange(count, device=dev)
        if s["mask"] is None:
            hidden[:, length:] = j[None, :] > j[:, None]
        else:
            hidden[:, length:] = (s["mask"][i][:count][:, j // 64] >> (j % 64)) % 2 == 0
        for kh in range(hk):
            k = s["k_cache"][page, kh, key % block].double()
            v = s["v_cache"][page, kh, key % block].double()
            for r in range(kh * group, (kh + 1) * group):
                x = torch.matmul(q[i, r, :count].double(), k.t().contiguous()) / math.sqrt(d)
                x = x.masked_fill(hidden, -math.inf)
                lse[i, r, :count] = torch.logsumexp(x, -1)
                out[i, r, :count] = torch.matmul(torch.softmax(x, -1), v)
    return (out, lse) if c["lse"] else out
