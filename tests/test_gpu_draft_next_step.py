"""The step after a step with drafted tokens: what follows the verification and the compaction
against the kept tokens run one at a time on the cache as it was before the drafts."""
import pytest
import torch

import hxm.ops as ops
from test_gpu_draft_step import V, Model, i32, prompt, slot

pytestmark = pytest.mark.gpu

# Two ways through three layers of f16, as in the step before (test_gpu_draft_step.py).
NEAR = dict(rtol=5e-2, atol=1e-2)


def test_the_next_step_is_the_kept_tokens_one_at_a_time(dev):
    g = torch.Generator().manual_seed(17)
    ctx, T, B = [5, 14, 9], 9, 3
    rows = [[-1, 0, 0, 0, 3, 2, 4, 4, 7], [-1, 0, 1, 0, 3, 4, 4, 6, 6],
            [-1, 0, 0, 1, 2, 4, -2, -2, -2]]
    kept = [[0, 3, 4, 7, 8], [0, 3, 4, 6], [0, 2, 4, 5]]       # none of them where it has to go
    order = torch.randperm(12, generator=g).int()
    table = torch.stack([order[:4], order[4:8], order[8:12]])
    model = Model(dev, 16, seed=3)
    prompt(model, table, ctx, dev, g)
    before = model.k.clone(), model.v.clone()
    depth = [[0] * T for _ in rows]
    for b, row in enumerate(rows):
        for i in range(1, T):
            depth[b][i] = depth[b][row[i]] + 1 if row[i] >= 0 else 0
    tokens = torch.randperm(V, generator=g)[:B * T].view(B, T).int()
    at = lambda b, t: slot(table, b, t)                                          # noqa: E731
    p = model.run(tokens.to(dev),
                  i32([[ctx[b] + depth[b][i] for i in range(T)] for b in range(B)], dev),
                  i32([[at(b, ctx[b] + i) if rows[b][i] > -2 else -1 for i in range(T)]
                       for b in range(B)], dev),
                  table.to(dev), i32([n + T for n in ctx], dev), i32(rows, dev))
    # A target that is certain of the branch, and its own at the branch's end.
    sure = torch.zeros_like(p)
    for b, path in enumerate(kept):
        for i, j in zip(path, path[1:]):
            sure[b, i, tokens[b, j]] = 1
        sure[b, path[-1]] = p[b, path[-1]]
    u = torch.rand(B, T, generator=g).to(dev)
    path, counts, following = ops.verify_draft(tokens.to(dev), sure, u, i32(rows, dev))
    assert path.tolist() == [k + [-1] * (T - len(k)) for k in kept]
    lens = i32([n + T for n in ctx], dev)
    drafted = model.k.clone(), model.v.clone()
    new = ops.compact_cache(model.k, model.v, table.to(dev), lens, path, counts)
    assert new.tolist() == [n + len(k) for n, k in zip(ctx, kept)]
    moved = model.k.clone(), model.v.clone()

    # The next step: the token that follows, and a tree of five behind it.
    rows2 = [[-1, 0, 0, 1, 3, 2]] * B
    depth2 = [0, 1, 1, 2, 3, 2]
    tokens2 = torch.cat((following[:, None].cpu(),
                         torch.randint(0, V, (B, 5), generator=g).int()), 1)

    def one_more():
        return model.run(following[:, None].contiguous(), new[:, None].contiguous(),
                         i32([[at(b, int(new[b]))] for b in range(B)], dev), table.to(dev), new + 1)

    def tree_more():
        return model.run(tokens2.to(dev),
                         i32([[int(new[b]) + d for d in depth2] for b in range(B)], dev),
                         i32([[at(b, int(new[b]) + i) for i in range(6)] for b in range(B)], dev),
                         table.to(dev), new + 6, i32(rows2, dev))

    one = one_more()
    model.k.copy_(moved[0]), model.v.copy_(moved[1])
    tree = tree_more()
    model.k.copy_(drafted[0]), model.v.copy_(drafted[1])
    astray = one_more()                                        # the drafts left where they were
    for b in range(B):
        model.k.copy_(before[0]), model.v.copy_(before[1])

        def step(word, t):
            return model.run(i32([[int(word)]], dev), i32([[t]], dev), i32([[at(b, t)]], dev),
                             table[b:b + 1].to(dev), i32([t + 1], dev))[0, 0]
        for n, i in enumerate(kept[b]):
            end = step(tokens[b, i], ctx[b] + n)
        assert torch.allclose(end, p[b, kept[b][-1]], **NEAR)
        first = step(following[b], int(new[b]))
        assert torch.allclose(first, one[b, 0], **NEAR), b
        assert torch.allclose(first, tree[b, 0], **NEAR), b
        assert not torch.allclose(first, astray[b, 0], **NEAR), b
        here = model.k.clone(), model.v.clone()
        for branch in ((1, 3, 4), (2, 5)):
            model.k.copy_(here[0]), model.v.copy_(here[1])
            for n, i in enumerate(branch):
                got = step(tokens2[b, i], int(new[b]) + 1 + n)
                assert torch.allclose(got, tree[b, i], **NEAR), (b, i)
