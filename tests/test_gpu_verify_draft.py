"""hxm_verify_draft against the rule walked node by node in 64 bits (numpy): paths, counts
and tokens equal."""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def walk(parents, tokens, p, q, u):
    """(path, the following token) of one sequence: parents, tokens [T]; p, q [T, V] fp64."""
    T, V = p.shape
    if parents[0] != -1:
        return [], -1
    clean = lambda x: np.where(x > 0, x, 0.0)                                    # noqa: E731
    path = [0]
    while True:
        node = path[-1]
        row, w, left, kept = clean(p[node]), clean(p[node]), 1.0, None
        children = [i for i in range(node + 1, T) if parents[i] == node and 0 <= tokens[i] < V]
        had = set()
        for i in children[:1] if q is not None else children:
            x = tokens[i]
            if x in had:
                continue
            had.add(x)
            qx = 1.0 if q is None else clean(q[node])[x]
            if u[i] * qx * left < row[x]:
                kept = i
                break
            if q is None:
                left -= row[x]
                w = w.copy()
                w[x] = 0
            else:
                w = np.maximum(row - clean(q[node]), 0)
        if kept is not None:
            path.append(kept)
            continue
        if not w.sum() > 0:
            w = row
        total = w.sum()
        if not 0 < total < np.inf:
            return path, -1
        past = np.nonzero((np.cumsum(w) > u[0] * total) & (w > 0))[0]
        return path, int(past[0] if len(past) else np.nonzero(w > 0)[0][-1])


def expect(parents, tokens, p, q, u):
    B, T = tokens.shape
    got = [walk(parents[b], tokens[b], p[b], None if q is None else q[b], u[b]) for b in range(B)]
    path = np.full((B, T), -1)
    for b, (x, _) in enumerate(got):
        path[b, :len(x)] = x
    return path, np.array([len(x) for x, _ in got]), np.array([t for _, t in got])


def run(dev, parents, tokens, p, q, u, null_parents=False):
    f = lambda t: None if t is None else t.double().numpy()                     # noqa: E731
    want = expect(parents.numpy(), tokens.numpy(), f(p), f(q), f(u))
    got = ops.verify_draft(tokens.to(dev), p.to(dev), u.to(dev),
                           None if null_parents else parents.to(dev),
                           None if q is None else q.to(dev))
    for g, w, what in zip(got, want, ("path", "counts", "next")):
        assert g.dtype == torch.int32
        bad = np.argwhere(g.cpu().numpy() != w)
        assert not len(bad), (what, bad[:4].tolist(), g.cpu().numpy()[tuple(bad[0])],
                              w[tuple(bad[0])])
    return want


def case(g, B, T, V, kind, dtype, with_draft, pad=0, sharp=8.0):
    """Random probabilities with a few likely tokens, drafted tokens that meet them often."""
    likely = torch.randint(0, V, (B, T, 4), generator=g)
    logits = torch.randn(B, T, V, generator=g)
    logits.scatter_(2, likely, sharp + torch.randn(B, T, 4, generator=g))
    p = logits.softmax(-1).to(dtype)
    q = (logits + torch.randn(B, T, V, generator=g)).softmax(-1).to(dtype) if with_draft else None
    parents = torch.full((B, T), -2, dtype=torch.int32)
    for b in range(B - pad):
        n = T if kind != "ragged" else int(torch.randint(1, T + 1, (1,), generator=g))
        parents[b, 0] = -1
        for i in range(1, n):
            parents[b, i] = i - 1 if kind == "chain" else max(
                0, i - 1 - int(torch.randint(0, 5, (1,), generator=g)))
    at = parents.clamp(min=0).long()
    pick = torch.randint(0, 4, (B, T), generator=g)
    tokens = likely.gather(1, at[..., None].expand(B, T, 4)).gather(2, pick[..., None])[..., 0]
    wild = torch.rand(B, T, generator=g) < 0.1
    tokens = torch.where(wild, torch.randint(0, V, (B, T), generator=g), tokens).int()
    return parents, tokens, p, q, torch.rand(B, T, generator=g)


@pytest.mark.parametrize("V", [1, 2, 7, 63, 257, 1000, 4096, 4097, 33001])
@pytest.mark.parametrize("name", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("with_draft", [False, True])
def test_vocabularies(dev, V, name, with_draft):
    g = torch.Generator().manual_seed(V)
    for kind in ("chain", "tree", "ragged"):
        run(dev, *case(g, 9, 6, V, kind, TDT[name], with_draft, pad=2))


@pytest.mark.parametrize("T", [1, 2, 3, 16, 17, 33, 63, 64])
@pytest.mark.parametrize("with_draft", [False, True])
def test_nodes(dev, T, with_draft):
    g = torch.Generator().manual_seed(T)
    deepest = 0
    for kind in ("chain", "tree", "ragged"):
        for sharp in (3.0, 14.0):
            want = run(dev, *case(g, 40, T, 501, kind, torch.float32, with_draft, sharp=sharp))
            deepest = max(deepest, want[1].max())
    assert deepest > 1 or T == 1


@pytest.mark.parametrize("B,V", [(1, 128000), (3, 50000), (200, 3001), (1100, 300), (2, 300001)])
def test_batches(dev, B, V):
    g = torch.Generator().manual_seed(B)
    run(dev, *case(g, B, 4, V, "chain", torch.float32, True))
    run(dev, *case(g, B, 4, V, "tree", torch.bfloat16, False))


def test_chains_without_parents(dev):
    g = torch.Generator().manual_seed(1)
    parents, tokens, p, q, u = case(g, 20, 5, 900, "chain", torch.float32, True)
    run(dev, parents, tokens, p, q, u, null_parents=True)
    run(dev, parents, tokens, p, None, u, null_parents=True)


def test_random_numbers_at_their_ends(dev):
    g = torch.Generator().manual_seed(2)
    for kind, with_draft in (("chain", True), ("tree", False)):
        parents, tokens, p, q, u = case(g, 6, 5, 5000, kind, torch.float32, with_draft)
        p[..., :3] = 0                             # the first token drawn at 0 is not one of them
        run(dev, parents, tokens, p, q, torch.zeros_like(u))
        run(dev, parents, tokens, p, q, torch.full_like(u, 1 - 2.0 ** -24))


def test_certain_targets(dev):
    """One-hot probabilities: a token is kept where it is the target's, and the one that
    follows is the target's, whatever the random numbers."""
    B, T, V = 8, 6, 1000
    g = torch.Generator().manual_seed(3)
    best = torch.randint(0, V, (B, T), generator=g)
    p = torch.nn.functional.one_hot(best, V).float()
    parents = torch.arange(-1, T - 1, dtype=torch.int32).expand(B, T).contiguous()
    tokens = torch.cat((torch.zeros(B, 1, dtype=torch.long), best[:, :-1]), 1)
    for b in range(B):
        if b + 1 < T:
            tokens[b, b + 1] = (tokens[b, b + 1] + 1) % V
    u = torch.rand(B, T, generator=g)
    path, counts, following = run(dev, parents, tokens.int(), p, None, u)
    assert counts.tolist() == [min(b + 1, T) for b in range(B)]
    assert following.tolist() == [int(best[b, counts[b] - 1]) for b in range(B)]


def test_what_is_no_probability_token_or_parent(dev):
    g = torch.Generator().manual_seed(4)
    parents, tokens, p, q, u = case(g, 10, 6, 700, "tree", torch.float32, False)
    tokens[0, 1:] = torch.tensor([-1, 700, 2 ** 31 - 1, -2 ** 31, 3], dtype=torch.int32)
    p[1, :, ::3] = float("nan")
    p[2, :, ::2] = -0.5
    p[3] = 0                                       # nothing to draw from
    p[4] = float("nan")
    p[5, 0, 10] = float("inf")
    tokens[5, 1:] = 20
    parents[6] = torch.tensor([-1, 1, 5, 2, 9, 2 ** 31 - 1], dtype=torch.int32)
    parents[7, 0] = 0
    parents[8, 0] = -2
    parents[9] = torch.tensor([-1, -1, 0, -2, 2, 4], dtype=torch.int32)
    want = run(dev, parents, tokens, p, None, u)
    assert want[2][3] == want[2][4] == want[2][5] == want[2][7] == want[2][8] == -1


def test_children_of_one_token(dev):
    """The second child of a token is not tried again, nor does its probability count twice."""
    p = torch.zeros(1, 5, 8)
    p[0, :, 2], p[0, :, 3], p[0, :, 4] = 0.25, 0.25, 0.5
    parents = torch.tensor([[-1, 0, 0, 0, 0]], dtype=torch.int32)
    tokens = torch.tensor([[1, 2, 2, 3, 4]], dtype=torch.int32)
    for u3, kept in ((0.33, [0, 3]), (0.34, [0, 4])):      # 0.25 of the 0.75 that are left
        u = torch.tensor([[0.5, 0.9, 0.0, u3, 0.99]])
        path, _, _ = run(dev, parents, tokens, p, None, u)
        assert path[0, :2].tolist() == kept


def test_target_below_the_draft_everywhere(dev):
    """Nothing is left where a token is not kept: the target's own row."""
    p = torch.full((2, 2, 4), 0.2)
    q = torch.full((2, 2, 4), 0.25)
    parents = torch.tensor([[-1, 0]] * 2, dtype=torch.int32)
    tokens = torch.tensor([[0, 1]] * 2, dtype=torch.int32)
    _, counts, following = run(dev, parents, tokens, p, q, torch.tensor([[0.6, 0.9], [0.1, 0.9]]))
    assert counts.tolist() == [1, 1] and following.tolist() == [2, 0]


def test_strided_probabilities_and_a_stream(dev):
    g = torch.Generator().manual_seed(5)
    parents, tokens, p, q, u = case(g, 4, 5, 1003, "chain", torch.bfloat16, True)
    want = ops.verify_draft(tokens.to(dev), p.to(dev), u.to(dev), parents.to(dev), q.to(dev))
    wide = [torch.full((4, 5, 1100), 9.0, dtype=torch.bfloat16, device=dev) for _ in range(2)]
    wide[0][..., 1:1004], wide[1][..., 7:1010] = p.to(dev), q.to(dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.verify_draft(tokens.to(dev), wide[0][..., 1:1004], u.to(dev), parents.to(dev),
                               wide[1][..., 7:1010])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured(dev):
    g = torch.Generator().manual_seed(6)
    parents, tokens, p, q, u = (t.to(dev) for t in case(g, 6, 5, 20000, "chain", torch.float32,
                                                        True))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        ops.verify_draft(tokens, p, u, parents, q)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = ops.verify_draft(tokens, p, u, parents, q)
    for r in range(4):
        u.copy_(torch.rand(u.shape, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b)
                   for a, b in zip(got, ops.verify_draft(tokens, p, u, parents, q))), r


def test_wrong_arguments_are_refused(dev):
    z = lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, device=dev)       # noqa: E731
    i = torch.int32
    ok = (z(2, 4, dt=i), z(2, 4, 50), z(2, 4), z(2, 4, dt=i), z(2, 4, 50))
    ops.verify_draft(*ok)
    for n, bad in ((0, z(2, 3, dt=i)), (0, z(2, 4)), (1, z(4, 50)), (1, z(2, 4, 50, dt=i)),
                   (1, z(2, 4, 50).cpu()), (1, z(4, 2, 50).transpose(0, 1)),
                   (1, z(2, 4, 100)[..., ::2]), (2, z(2, 4).double()), (2, z(4, 2).t()),
                   (3, z(2, 5, dt=i)), (4, z(2, 4, 49)), (4, z(2, 4, 50).half())):
        args = list(ok)
        args[n] = bad
        with pytest.raises((ValueError, TypeError)):
            ops.verify_draft(*args)
    with pytest.raises(hxm.HxmError, match="tile-alignment"):
        ops.verify_draft(z(1, 65, dt=i), z(1, 65, 8), z(1, 65))
    with pytest.raises(hxm.HxmError, match="invalid-argument"):
        ops.verify_draft(z(1, 4, dt=i), z(1, 4, 0), z(1, 4))
    none = ops.verify_draft(z(0, 4, dt=i), z(0, 4, 8), z(0, 4))
    assert [tuple(t.shape) for t in none] == [(0, 4), (0,), (0,)]


def test_offsets_past_32_bits(dev):
    """Rows of the tables beyond 2^31 elements."""
    B, T, V = 3, 4, 200_000_000
    p = torch.zeros(B, T, V, dtype=torch.float16, device=dev)
    assert p.numel() > 2 ** 31
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)                 # noqa: E731
    far = [V - 3, 150_000_001, 7]
    for b in range(B):
        p[b, :, far[b]], p[b, :, 5] = 0.75, 0.25
    tokens = i([[1] + [f] * 3 for f in far])
    u = torch.full((B, T), 0.5, device=dev)
    u[:, 3] = 0.9                                  # 0.9 of 1 is not below 0.75
    path, counts, following = ops.verify_draft(tokens, p, u)
    assert counts.tolist() == [3] * B and path.tolist() == [[0, 1, 2, -1]] * B
    assert following.tolist() == [5] * B           # what is left of the third row
    u[:, 3] = 0.1
    path, counts, following = ops.verify_draft(tokens, p, u)
    assert counts.tolist() == [4] * B
    assert following.tolist() == far


def test_streams_at_once(dev):
    """Calls on two streams beside each other: each has its own sums and counters."""
    g = torch.Generator().manual_seed(8)
    jobs = [tuple(t.to(dev) for t in case(g, B, 5, V, "chain", torch.float32, True))
            for B, V in ((20, 30000), (7, 120000))]
    call = lambda j, s=None: ops.verify_draft(j[1], j[2], j[4], j[0], j[3], stream=s)  # noqa: E731
    want = [call(j) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = [call(j, s) for j, s in zip(jobs, streams)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
