"""Decoding goes on from an accepted path of a tree: its drafts lie anywhere in the
cache's draft rows, and are stored again behind the request's tokens."""

import numpy as np
import pytest

import flashlite_amd as fl

pytestmark = pytest.mark.gpu


def paths(rs, parents):
    """A root-to-leaf path of each request's tree, that is not its first drafts
    where the tree has another."""
    out = []
    for row in parents:
        up = {int(p) for p in row}
        leaves = [i for i in range(len(row)) if i not in up]
        i, path = int(rs.choice(leaves[-2:])), []
        while i >= 0:
            path.append(i)
            i = int(row[i])
        out.append(path[::-1])
    return out


@pytest.mark.parametrize("dtype,d,h,hk,block", [("float16", 64, 4, 2, 16),
                                                ("bfloat16", 128, 6, 2, 20)])
def test_an_accepted_path_equals_its_tokens_in_order(cuda, dtype, d, h, hk, block):
    import torch

    rs, b, n, pool = np.random.RandomState(8), 4, 13, 80
    t = getattr(torch, dtype)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=cuda)  # noqa: E731
    freqs, scale = fl.rotary_frequencies(d, device=cuda)

    def state():
        shape = (pool, block, hk, d)
        k, v = (torch.full(shape, float("nan"), dtype=t, device=cuda).transpose(1, 2)
                for _ in range(2))
        return dict(tables=torch.full((b, 20), -1, dtype=torch.int32, device=cuda),
                    held=i32([0] * b), ring=i32(np.random.RandomState(9).permutation(pool)),
                    state=i32([5, pool]), lengths=i32([0] * b), k=k, v=v)

    def rows(m):
        return [torch.from_numpy(rs.standard_normal((b, x, m, d)).astype(np.float32)).to(cuda).to(t)
                for x in (h, hk, hk)]

    def step(s, qkv, counts, parents=None):
        q, k, v = qkv
        m = q.shape[2]
        positions, slots, info = fl.plan_cache(s["lengths"], counts, s["tables"], s["held"],
                                               s["ring"], s["state"], block, m)
        assert bool((info[:, 0] == 0).all())
        mask = None
        if parents is not None:
            mask, positions = fl.plan_tree(parents, s["lengths"], counts)
        turned = fl.rotary_to_cache(q, k, v, positions, slots, freqs, s["k"], s["v"], scale=scale)
        return slots, fl.forward_tree(turned, s["k"], s["v"], s["tables"], s["lengths"], mask,
                                      counts)

    tree, line = state(), state()
    prompt, lengths = rows(40), i32([40, 17, 1, 33])
    most = float(prompt[2].abs().max())
    for s in (tree, line):
        step(s, prompt, lengths)
        s["lengths"] += lengths
    moved = 0
    for _ in range(3):
        parents = np.floor(rs.rand(b, n) * (np.arange(n) + 1)).astype(int) - 1
        drafts = rows(n)
        most = max(most, float(drafts[2].abs().max()))
        slots, out = step(tree, drafts, i32([n] * b), i32(parents))
        accepted = paths(rs, parents)
        count, m = [len(x) for x in accepted], max(len(x) for x in accepted)
        moved += sum(x != list(range(len(x))) for x in accepted)
        path = torch.tensor([x + [0] * (m - len(x)) for x in accepted], device=cuda)

        def of_path(x):
            return x.gather(2, path[:, None, :, None].expand(b, x.shape[1], m, d))

        q, k, v = (of_path(x) for x in drafts)
        at = torch.arange(m, device=cuda)
        positions = (tree["lengths"][:, None] + at).int()
        stay = torch.where(at < i32(count)[:, None], slots[:, :m], -1)
        fl.rotary_to_cache(q[:, :0], k, v, positions, stay, freqs, tree["k"], tree["v"],
                           scale=scale)
        # the same tokens in order, as a chain
        _, want = step(line, (q, k, v), i32(count))
        for r in range(b):
            for j, draft in enumerate(accepted[r]):
                # The rows are the same, what is summed lies in other tiles: each
                # is off by half a step of itself and of the p, so by eps
                # max |v| at most, and by less than a tenth of that in its sums.
                err = (out[r, :, draft].float() - want[r, :, j].float()).abs()
                assert float(err.max()) <= 2.1 * torch.finfo(t).eps * most
        for s in (tree, line):
            s["lengths"] += i32(count)
        token = rows(1)
        most = max(most, float(token[2].abs().max()))
        got, want = (step(s, token, i32([1] * b))[1] for s in (tree, line))
        assert torch.equal(got, want)
        for s in (tree, line):
            s["lengths"] += 1
    assert moved >= 3
