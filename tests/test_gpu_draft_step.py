"""A step with drafted tokens through all of its operators, as a serving program runs it:
head norms, rotation and append of a tree, its attention, the head's probabilities, the
verification, the compaction, and the next token's attention over what is left; sequences
that fork.  Each is checked against the same tokens run one at a time."""
import pytest
import torch

import hxm.ops as ops

pytestmark = pytest.mark.gpu

HQ, HKV, D, PAGE, V, LAYERS = 8, 2, 64, 16, 512, 3


class Model:
    """A decoder of attention layers alone, its cache for `pages` pages."""

    def __init__(self, dev, pages, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g)).half().to(dev)  # noqa: E731
        H = HQ * D
        self.embed = r(V, H)
        self.qkv = [r((HQ + 2 * HKV) * D, H, scale=H ** -0.5) for _ in range(LAYERS)]
        self.o = [r(H, H, scale=H ** -0.5) for _ in range(LAYERS)]
        self.norms = [(r(D), r(D)) for _ in range(LAYERS)]
        self.head = r(V, H, scale=3.0 * H ** -0.5)
        self.k = r(LAYERS, pages, HKV, PAGE, D)
        self.v = r(LAYERS, pages, HKV, PAGE, D)
        ang = torch.arange(512)[:, None] * 10000.0 ** (-torch.arange(D // 2) / (D // 2))
        self.cos_sin = torch.cat((ang.cos(), ang.sin()), 1).to(dev)

    def run(self, tokens, positions, slots, table, lens, parents=None):
        """Probabilities [B, T, V] of tokens [B, T], their keys and values stored."""
        B, T = tokens.shape
        x = self.embed[tokens.flatten().long()]
        for n in range(LAYERS):
            _, z = ops.residual_norm(torch.zeros_like(x), x)
            qkv = ops.matmul(z, self.qkv[n], b_layout="nk").view(B * T, HQ + 2 * HKV, D)
            q, k, v = qkv.split((HQ, HKV, HKV), 1)
            q = ops.norm_rope_append(q, k, v, self.k[n], self.v[n], slots.flatten(),
                                     positions.flatten(), self.cos_sin, q_weight=self.norms[n][0],
                                     k_weight=self.norms[n][1])
            if T == 1:
                a = ops.paged_attention(q, self.k[n], self.v[n], table, lens)
            else:
                a = ops.tree_attention(q.view(B, T, HQ, D), self.k[n], self.v[n], table, lens,
                                       parents)
            x = x + ops.matmul(a.reshape(B * T, -1), self.o[n], b_layout="nk")
        _, z = ops.residual_norm(torch.zeros_like(x), x)
        logits = ops.matmul(z, self.head, b_layout="nk", out_dtype=torch.float32)
        return ops.softmax(logits).view(B, T, V)


def i32(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def slot(table, b, at):
    return int(table[b, at // PAGE]) * PAGE + at % PAGE


def prompt(model, table, ctx, dev, g):
    """The prompts token by token; returns them."""
    text = [torch.randint(0, V, (n,), generator=g).tolist() for n in ctx]
    for b, words in enumerate(text):
        for t, w in enumerate(words):
            model.run(i32([[w]], dev), i32([[t]], dev), i32([[slot(table, b, t)]], dev),
                      table[b:b + 1].to(dev), i32([t + 1], dev))
    return text


def test_a_tree_step_is_its_branches_token_by_token(dev):
    g = torch.Generator().manual_seed(7)
    ctx, T = [20, 33, 5], 10
    rows = [[-1, 0, 0, 1, 1, 2, 3, 3, 5, 6], [-1, 0, 1, 2, 3, 4, 5, 6, 7, 8],
            [-1, 0, 0, 0, 2, 4, -2, -2, -2, -2]]
    order = torch.randperm(12, generator=g).int()
    table = torch.stack([order[:4], order[4:8], order[8:12]])
    model = Model(dev, 16)
    prompt(model, table, ctx, dev, g)
    depth = [[0] * T for _ in rows]
    for b, row in enumerate(rows):
        for i in range(1, T):
            depth[b][i] = depth[b][row[i]] + 1 if row[i] >= 0 else 0
    tokens = torch.randint(0, V, (3, T), generator=g).int()
    pos = [[ctx[b] + depth[b][i] for i in range(T)] for b in range(3)]
    slots = [[slot(table, b, ctx[b] + i) if rows[b][i] > -2 else -1 for i in range(T)]
             for b in range(3)]
    before = model.k.clone(), model.v.clone()
    lens = i32([n + T for n in ctx], dev)
    p = model.run(tokens.to(dev), i32(pos, dev), i32(slots, dev), table.to(dev), lens,
                  i32(rows, dev))
    after = model.k.clone(), model.v.clone()
    u = torch.rand(3, T, generator=g)
    path, counts, following = ops.verify_draft(tokens.to(dev), p, u.to(dev), i32(rows, dev))
    # Every branch to its leaf, one token at a time on the cache as it was.
    for b in range(3):
        for leaf in range(T):
            if rows[b][leaf] < -1 or leaf in rows[b]:
                continue
            branch = [leaf]
            while rows[b][branch[0]] >= 0:
                branch.insert(0, rows[b][branch[0]])
            model.k.copy_(before[0]), model.v.copy_(before[1])
            for n, i in enumerate(branch):
                at = ctx[b] + n
                one = model.run(i32([[int(tokens[b, i])]], dev), i32([[at]], dev),
                                i32([[slot(table, b, at)]], dev), table[b:b + 1].to(dev),
                                i32([at + 1], dev))
                # Two ways through three layers of f16 (11 bits): 1e-2 is some twenty
                # roundings of the largest probability.
                assert torch.allclose(one[0, 0], p[b, i], rtol=5e-2, atol=1e-2), (b, i)
    # The kept rows move behind the context, in every layer.
    model.k.copy_(after[0]), model.v.copy_(after[1])
    new = ops.compact_cache(model.k, model.v, table.to(dev), lens, path, counts)
    for b in range(3):
        kept = path[b, :counts[b]].tolist()
        assert new[b].item() == ctx[b] + len(kept)
        for x, old in ((model.k, after[0]), (model.v, after[1])):
            for n, i in enumerate(kept):
                a, z = ctx[b] + i, ctx[b] + n
                assert torch.equal(x[:, table[b, z // PAGE], :, z % PAGE],
                                   old[:, table[b, a // PAGE], :, a % PAGE])
    # And the next step goes on from there.
    nxt = model.run(following[:, None].contiguous(), new[:, None].contiguous(),
                    i32([[slot(table, b, int(new[b]))] for b in range(3)], dev), table.to(dev),
                    new + 1)
    assert nxt.isfinite().all() and (nxt.sum(-1) - 1).abs().max() < 1e-3


def test_certain_drafts_are_kept_whole(dev):
    """A chain of the target's own best tokens, the target made certain: all of it is kept."""
    g = torch.Generator().manual_seed(9)
    T, ctx = 5, [17]
    table = torch.arange(3, dtype=torch.int32)[None]
    model = Model(dev, 4)
    text = prompt(model, table, ctx, dev, g)[0]
    keep = model.k.clone(), model.v.clone()
    tokens = [text[0]]
    for t in range(T):
        at = ctx[0] + t
        p = model.run(i32([[tokens[-1]]], dev), i32([[at]], dev), i32([[slot(table, 0, at)]], dev),
                      table.to(dev), i32([at + 1], dev))
        tokens.append(int(p[0, 0].argmax()))
    model.k.copy_(keep[0]), model.v.copy_(keep[1])
    at = [[ctx[0] + t for t in range(T)]]
    p = model.run(i32([tokens[:T]], dev), i32(at, dev), i32([[slot(table, 0, a) for a in at[0]]], dev),
                  table.to(dev), i32([ctx[0] + T], dev))
    sure = torch.nn.functional.one_hot(p.argmax(-1), V).float()
    path, counts, following = ops.verify_draft(i32([tokens[:T]], dev), sure,
                                               torch.rand(1, T, generator=g).to(dev))
    assert counts.tolist() == [T] and path.tolist() == [list(range(T))]
    assert following.tolist() == [tokens[T]]


def test_a_fork_goes_its_own_way(dev):
    """A sequence forks: its full pages shared, the last one copied; both go on and give
    what each gives alone."""
    g = torch.Generator().manual_seed(8)
    ctx = 21
    table = torch.tensor([[5, 2]], dtype=torch.int32)
    model = Model(dev, 8)
    prompt(model, table, [ctx], dev, g)
    ops.copy_pages(model.k, model.v, i32([2], dev), i32([6], dev), i32([ctx - PAGE], dev))
    both = torch.tensor([[5, 2], [5, 6]], dtype=torch.int32)
    words = torch.randint(0, V, (2, 3), generator=g).int()
    keep = model.k.clone(), model.v.clone()
    pos = i32([[ctx + t for t in range(3)]] * 2, dev)
    slots = i32([[slot(both, b, ctx + t) for t in range(3)] for b in range(2)], dev)
    p = model.run(words.to(dev), pos, slots, both.to(dev), i32([ctx + 3] * 2, dev))
    for b in range(2):
        model.k.copy_(keep[0]), model.v.copy_(keep[1])
        alone = model.run(words[b:b + 1].to(dev), pos[:1], i32([[slot(table, 0, ctx + t)
                                                                 for t in range(3)]], dev),
                          table.to(dev), i32([ctx + 3], dev))
        assert torch.allclose(alone[0], p[b], rtol=5e-2, atol=1e-2)
