"""plan_cache and plan_tree against the oracle: whole numbers, equal."""

import numpy as np
import pytest

import flashlite_amd as fl
from oracle import paged

pytestmark = pytest.mark.gpu


def i32(x, dev):
    import torch

    return torch.tensor(x, dtype=torch.int32, device=dev)


def make(seed, b, width, block, m, ended=0.2, free=None, idle=0.1):
    """Requests whose blocks are distinct, and a ring that starts anywhere."""
    rs = np.random.RandomState(seed)
    lengths = rs.randint(0, max(1, m * block - width + 1), b)
    counts = rs.randint(0 if idle else 1, width + 1, b)
    counts[rs.rand(b) < ended] = -1
    held = -(-lengths // block)
    ids = rs.permutation(b * m + 5)
    tables = np.full((b, m), -1)
    at = 0
    for i in range(b):
        tables[i, :held[i]] = ids[at:at + held[i]]
        at += held[i]
    pool = b * m + 5
    need = int(np.maximum(-(-(lengths + np.maximum(counts, 0)) // block) - held, 0).sum())
    count = min(pool - at, need + 3 if free is None else free)
    head = rs.randint(0, pool)
    ring = np.full(pool, -7)
    ring[(head + np.arange(count)) % pool] = ids[at:at + count]
    return [x.tolist() for x in (lengths, counts, tables, held, ring)] + [[head, count]]


def call(args, block, width, dev, in_place=True, table_pad=0):
    import torch

    lengths, counts, tables, held, ring, state = args
    t = i32(tables, dev)
    if table_pad:
        wide = torch.full((t.shape[0], t.shape[1] + table_pad), 12345, dtype=torch.int32, device=dev)
        wide[:, :t.shape[1]] = t
        t = wide[:, :t.shape[1]]
    h, r, s = i32(held, dev), i32(ring, dev), i32(state, dev)
    kw = {}
    if not in_place:
        kw = dict(held_out=torch.full_like(h, 99), state_out=torch.full_like(s, 99))
    positions, slots, info = fl.plan_cache(i32(lengths, dev), i32(counts, dev), t, h, r, s, block,
                                           width, **kw)
    if not in_place:
        assert h.tolist() == held and s.tolist() == state
        h, s = kw["held_out"], kw["state_out"]
    if table_pad:
        assert bool((wide[:, t.shape[1]:] == 12345).all())
    return [x.tolist() for x in (t, h, r, s, positions, slots, info)]


NAMES = ("tables", "held", "ring", "state", "positions", "slots", "info")


def check(args, block, width, dev, **kw):
    want = paged.plan_cache(*args, block, width)
    got = call(args, block, width, dev, **kw)
    for name, a, b in zip(NAMES, got, want):
        assert a == b, name


@pytest.mark.parametrize("b,width,block,m", [
    (1, 1, 16, 4), (3, 1, 1, 9), (32, 1, 16, 40), (7, 5, 16, 3), (5, 300, 16, 40), (2, 1000, 64, 20),
    (70, 7, 20, 6), (33, 257, 257, 3), (1000, 1, 8, 5), (1500, 2, 16, 3), (2100, 1, 16, 2)])
@pytest.mark.parametrize("in_place", [True, False])
def test_plan(cuda, b, width, block, m, in_place):
    check(make(b + width, b, width, block, m), block, width, cuda, in_place=in_place,
          table_pad=0 if in_place else 3)


@pytest.mark.parametrize("free", [0, 1, 7, 60])
def test_pool_runs_out(cuda, free):
    """Requests are served in order; one that needs nothing always is."""
    args = make(5, 90, 40, 16, 8, ended=0.1, free=free)
    info = np.array(paged.plan_cache(*args, 16, 40)[6])
    assert (info[:, 0] == 1).any() and (info[:, 0] == 0).any()
    check(args, 16, 40, cuda)


def test_row_too_short_and_values_out_of_range(cuda):
    args = make(6, 20, 10, 4, 6, ended=0.0)
    lengths, counts, tables, held, ring, state = args
    lengths[3] = 6 * 4 - 2          # needs a seventh block
    counts[3] = 9
    counts[4], held[4] = 50, 9      # more than the width; more than the row
    lengths[5] = 2 ** 31 - 3        # far past the row
    counts[5] = 10
    lengths[6], held[6] = -5, -2
    tables[7][0] = -1               # an entry that is no block: no slots there
    lengths[7], held[7], counts[7] = 0, 1, 3
    status = [r[0] for r in paged.plan_cache(*args, 4, 10)[6]]
    assert status[3] == 2 and status[5] == 2
    check(args, 4, 10, cuda)


def test_everything_ends_and_a_full_ring_drops(cuda):
    args = make(8, 12, 3, 16, 5, ended=1.0)
    check(args, 16, 3, cuda)
    # a ring without room for the blocks (more given back than it lacks)
    lengths, counts, tables, held, ring, state = args
    small = ring[:6]
    check([lengths, counts, tables, held, small, [4, 3]], 16, 3, cuda)


def test_no_requests_and_no_width(cuda):
    import torch

    t = torch.zeros((0, 4), dtype=torch.int32, device=cuda)
    e = torch.zeros((0,), dtype=torch.int32, device=cuda)
    s = i32([1, 2], cuda)
    out = fl.plan_cache(e, e, t, e, i32([3, 4, 5], cuda), s, 16, 5)
    assert [tuple(x.shape) for x in out] == [(0, 5), (0, 5), (0, 4)] and s.tolist() == [1, 2]
    args = make(9, 6, 1, 16, 4)
    lengths, counts = args[0], [min(c, 0) for c in args[1]]
    check([lengths, counts] + args[2:], 16, 0, cuda)


def test_steps_in_a_row(cuda):
    """A pool over many steps: every block has one owner, and slots never meet."""
    import torch

    b, width, block, m, pool = 9, 4, 4, 12, 60
    rs = np.random.RandomState(11)
    lengths, held = np.zeros(b, int), i32([0] * b, cuda)
    tables = torch.full((b, m), -1, dtype=torch.int32, device=cuda)
    ring, state = i32(list(range(pool)), cuda), i32([0, pool], cuda)
    for step in range(30):
        counts = rs.randint(0, width + 1, b)
        counts[(lengths > 30) | (rs.rand(b) < 0.05)] = -1
        positions, slots, info = fl.plan_cache(i32(lengths, cuda), i32(counts, cuda), tables, held,
                                               ring, state, block, width)
        s = slots.cpu().numpy()
        live = s[s >= 0]
        assert len(set(live.tolist())) == len(live)
        served = info.cpu().numpy()[:, 0] == 0
        lengths = np.where(counts < 0, 0, lengths + np.where(served, np.maximum(counts, 0), 0))
        own = [set(tables[i, :int(held[i])].tolist()) for i in range(b)]
        head, count = state.tolist()
        free = [ring[(head + k) % pool].item() for k in range(count)]
        everything = [x for o in own for x in o] + free
        assert sorted(everything) == list(range(pool)), f"step {step}"
        for i in range(b):
            assert len(own[i]) * block >= lengths[i]


@pytest.mark.parametrize("b,n", [(1, 1), (3, 2), (8, 16), (5, 63), (4, 64), (3, 65), (2, 200), (2, 512)])
@pytest.mark.parametrize("kind", ["random", "chain", "wide", "bad"])
@pytest.mark.parametrize("ragged", [False, True])
def test_tree(cuda, b, n, kind, ragged):
    rs = np.random.RandomState(n)
    if kind == "chain":
        parents = np.tile(np.arange(n) - 1, (b, 1))
    elif kind == "wide":
        parents = np.maximum(np.tile(np.arange(n), (b, 1)) // 3 - 1, -1)
    else:
        parents = np.floor(rs.rand(b, n) * (np.arange(n) + 1)).astype(int) - 1
    if kind == "bad":  # not earlier drafts: they follow the prompt
        bad = rs.rand(b, n) < 0.3
        parents = np.where(bad, rs.choice([-7, n, n - 1, 2 ** 30], (b, n)), parents)
    lengths = rs.randint(0, 5000, b)
    counts = rs.randint(0, n + 1, b) if ragged else None
    seen, positions = paged.plan_tree(parents.tolist(), lengths, counts)
    mask, pos = fl.plan_tree(i32(parents, cuda), i32(lengths, cuda),
                             None if counts is None else i32(counts, cuda))
    assert pos.tolist() == positions
    want = np.stack([paged.words(s, n) for s in seen])
    assert np.array_equal(mask.cpu().numpy(), want)


def test_tree_shared_parents(cuda):
    """One tree for all requests: an expanded tensor."""
    p = i32([[-1, 0, 0, 1]], cuda)
    lengths = i32([5, 0, 70], cuda)
    mask, pos = fl.plan_tree(p.expand(3, 4), lengths)
    again = fl.plan_tree(p.expand(3, 4).contiguous(), lengths)
    assert mask.equal(again[0]) and pos.equal(again[1])
    assert pos.tolist() == [[5, 6, 6, 7], [0, 1, 1, 2], [70, 71, 71, 72]]


def test_refusals(cuda):
    import torch

    e = i32([1, 2], cuda)
    t = torch.zeros((2, 4), dtype=torch.int32, device=cuda)
    with pytest.raises(RuntimeError, match="counts must have one entry"):
        fl.plan_cache(e, e[:1], t, e, e, e, 16, 1)
    with pytest.raises(RuntimeError, match="held must be int32"):
        fl.plan_cache(e, e, t, e.long(), e, e, 16, 1)
    with pytest.raises(RuntimeError, match="block_size"):
        fl.plan_cache(e, e, t, e, e, e, 0, 1)
    with pytest.raises(RuntimeError, match="slots"):
        fl.plan_cache(e, e, t, e, e, e, 16, 1, slots=torch.zeros((2, 1), device=cuda))
    with pytest.raises(RuntimeError, match="512"):
        fl.plan_tree(torch.zeros((1, 513), dtype=torch.int32, device=cuda), e[:1])
    with pytest.raises(RuntimeError, match="lengths"):
        fl.plan_tree(t, e[:1])
