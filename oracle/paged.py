"""CPU oracle of the paged-cache operators (test infrastructure only): plain
Python and float64 numpy, one request, head and row at a time.

No counterpart in the reference; the definitions are the comments of
``include/flashlite_attn.h``.
"""

from __future__ import annotations

import numpy as np


def plan_cache(lengths, counts, tables, held, ring, state, block, width):
    """(tables, held, ring, state, positions, slots, info) after the call;
    the arguments are lists and are not changed."""
    tables, ring = [list(t) for t in tables], list(ring)
    head, count = state
    pool, rows = len(ring), len(lengths)
    out_held, info = list(held), [[0] * 4 for _ in range(rows)]
    wanted = 0  # blocks asked for by the requests before, served or not
    back = 0    # blocks given back by the requests before
    taken_all = given_all = 0
    old_ring = list(ring)
    for b in range(rows):
        limit = len(tables[b])
        own = min(max(held[b], 0), limit)
        length = max(lengths[b], 0)
        new = min(max(counts[b], 0), width)
        info[b][1] = own
        if counts[b] < 0:
            info[b][3] = (head + count + back) % pool
            given = min(own, max(pool - count - back, 0))
            for k in range(given):
                ring[(head + count + back + k) % pool] = tables[b][k]
            info[b][2] = -given
            back += own
            given_all += given
            out_held[b] = 0
            continue
        need = 0
        if new > 0:
            blocks = -(-(length + new) // block)
            if blocks > limit:
                info[b][0] = 2
            else:
                need = max(blocks - own, 0)
        info[b][3] = (head + wanted) % pool
        if info[b][0] == 0 and need > 0 and wanted + need > count:
            info[b][0] = 1
        if info[b][0] == 0:
            for k in range(need):
                tables[b][own + k] = old_ring[(head + wanted + k) % pool]
            info[b][2] = need
            taken_all += need
            out_held[b] = own + need
        else:
            out_held[b] = own
        wanted += need
    positions = [[-1] * width for _ in range(rows)]
    slots = [[-1] * width for _ in range(rows)]
    for b in range(rows):
        if counts[b] <= 0 or info[b][0] != 0:
            continue
        for i in range(min(counts[b], width)):
            at = max(lengths[b], 0) + i
            block_id = tables[b][at // block]
            if block_id >= 0:
                positions[b][i] = at
                slots[b][i] = block_id * block + at % block
    new_state = [(head + taken_all) % pool, count - taken_all + given_all]
    return tables, out_held, ring, new_state, positions, slots, info


def plan_tree(parents, lengths, counts):
    """(seen, positions): seen[b][i] is the set of drafts that i sees."""
    seen, positions = [], []
    for b, row in enumerate(parents):
        n = len(row)
        there = n if counts is None else min(max(counts[b], 0), n)
        s, p = [], []
        for i in range(n):
            if i >= there:
                s.append(set())
                p.append(-1)
                continue
            up = row[i]
            mine = {i} | (s[up] if 0 <= up < i else set())
            s.append(mine)
            p.append(max(lengths[b], 0) + len(mine) - 1)
        seen.append(s)
        positions.append(p)
    return seen, positions


def words(seen, n):
    """Sets of drafts as int64 words [len(seen), ceil(n / 64)]."""
    out = np.zeros((len(seen), (n + 63) // 64), dtype=np.uint64)
    for i, s in enumerate(seen):
        for j in s:
            out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def rotary(x, positions, freqs, interleaved=False, scale=1.0, transpose=False):
    """x [B, H, N, D] float64 with the pairs of its first columns rotated."""
    out = np.array(x, dtype=np.float64)
    pairs = len(freqs)
    for j in range(pairs):
        a, c = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
        angle = np.asarray(positions, dtype=np.float64) * float(freqs[j])
        if transpose:
            angle = -angle
        cos, sin = np.cos(angle)[:, None, :] * scale, np.sin(angle)[:, None, :] * scale
        out[..., a] = x[..., a] * cos - x[..., c] * sin
        out[..., c] = x[..., a] * sin + x[..., c] * cos
    return out


def tree_attention(q, k_cache, v_cache, tables, lengths, seen=None, counts=None, sm_scale=0.0):
    """(out, lse, weight, reach) in float64 over q [B, H, n, D] and caches
    [blocks, H_k, block, D]: `weight` is sum_j p_j |v_j| / sum_j p_j per output
    value and `reach` the largest sum_i |q_i k_i| |scale| per row, the sizes
    that rounding errors follow.  Rows of drafts that are not there are NaN.
    seen[b][i]: the drafts that draft i sees (None: a chain)."""
    bsz, heads, n, d = q.shape
    blocks, kv_heads, block, _ = k_cache.shape
    scale = sm_scale if sm_scale != 0.0 else 1.0 / np.sqrt(d)
    capacity = tables.shape[1] * block
    out = np.full((bsz, heads, n, d), np.nan)
    weight = np.zeros((bsz, heads, n, d))
    lse = np.full((bsz, heads, n), np.nan)
    reach = np.zeros((bsz, heads, n))
    for b in range(bsz):
        length = min(max(int(lengths[b]), 0), capacity)
        there = n if counts is None else min(max(int(counts[b]), 0), n)
        drafts = min(there, capacity - length)
        at = np.arange(length + drafts)
        ids = tables[b][at // block]
        good = (ids >= 0) & (ids < blocks)
        safe = np.where(good, ids, 0)
        for h in range(heads):
            hk = h // (heads // kv_heads)
            k = k_cache[safe, hk, at % block].astype(np.float64)
            v = v_cache[safe, hk, at % block].astype(np.float64)
            for i in range(there):
                vis = good.copy()
                for j in range(drafts):
                    vis[length + j] &= (j <= i) if seen is None else (j in seen[b][i])
                if not vis.any():
                    out[b, h, i] = 0.0
                    lse[b, h, i] = -np.inf
                    continue
                x = q[b, h, i].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = k[vis] @ x * scale
                    reach[b, h, i] = (np.abs(k[vis]) @ np.abs(x)).max() * abs(scale)
                    top = s.max()
                    p = np.exp(s - top)
                    out[b, h, i] = p @ v[vis] / p.sum()
                    weight[b, h, i] = p @ np.abs(v[vis]) / p.sum()
                    lse[b, h, i] = top + np.log(p.sum())
    return out, lse, weight, reach
