"""hxm_compact_cache and hxm_copy_pages against plain indexing, bit by bit."""
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu


def caches(g, layers, pages, heads, page, dim, layout, dev, dtype=torch.float16):
    """(k, v) [layers, pages, heads, page, dim] of random bits in several memory orders."""
    bits = lambda *s: torch.randint(-2 ** 15, 2 ** 15, s, generator=g).short().to(dev)  # noqa: E731
    if layout == "hnd":
        k, v = bits(layers, pages, heads, page, dim), bits(layers, pages, heads, page, dim)
    elif layout == "nhd":
        k, v = (bits(layers, pages, page, heads, dim).transpose(2, 3) for _ in "kv")
    elif layout == "kv_in_layer":
        k, v = bits(layers, 2, pages, heads, page, dim).unbind(1)
    elif layout == "kv_in_page":
        k, v = bits(layers, pages, 2, heads, page, dim).unbind(2)
    elif layout == "kv_in_row":
        k, v = bits(layers, pages, page, heads, 2, dim).transpose(2, 3).unbind(4)
    else:                                    # layers inside the pages, wider rows
        k, v = (bits(pages, layers, heads, page, dim + 8)[..., 3:3 + dim].transpose(0, 1)
                for _ in "kv")
    return k.view(dtype), v.view(dtype)


def bits(t):
    return t.view(torch.int16).cpu()


LAYOUTS = ["hnd", "nhd", "kv_in_layer", "kv_in_page", "kv_in_row", "layers_in_page"]


def make_table(g, lens, page, width=None):
    need = [-(-max(n, 0) // page) for n in lens]
    order = torch.randperm(sum(need) + 2, generator=g)
    table = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    return table, sum(need) + 2


def compacted(x, table, lens, T, paths, page):
    old, x = x.clone(), x.clone()
    for b, path in enumerate(paths):
        for i, node in enumerate(path or []):
            a, z = lens[b] - T + node, lens[b] - T + i
            x[:, table[b, z // page], :, z % page] = old[:, table[b, a // page], :, a % page]
    return x


def run_compact(dev, layout, lens, T, paths, page, layers=3, heads=2, dim=64,
                dtype=torch.float16):
    g = torch.Generator().manual_seed(T + page)
    table, pages = make_table(g, lens, page)
    k, v = caches(g, layers, pages, heads, page, dim, layout, dev, dtype)
    want = [compacted(bits(x), table, lens, T, paths, page) for x in (k, v)]
    path = torch.full((len(lens), T), -1, dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    counts = torch.tensor([len(p) for p in paths], dtype=torch.int32)
    out = ops.compact_cache(k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                            path.to(dev), counts.to(dev))
    assert torch.equal(bits(k), want[0]) and torch.equal(bits(v), want[1])
    assert out.tolist() == [n - T + len(p) for n, p in zip(lens, paths)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page", [1, 3, 8, 16, 100])
def test_compact(dev, layout, page):
    T = 12
    paths = [[0], [0, 1, 2, 3], [0, 4, 7, 11], [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11], [0, 2, 3, 4],
             list(range(12)), [], [11]]
    run_compact(dev, layout, [12, 13, 25, 44, 90, 31, 60, 17], T, paths, page)
    run_compact(dev, layout, [40, 40], T, [[0, 5], [0, 2, 3]], page, layers=1, heads=5, dim=40,
                dtype=torch.bfloat16)


@pytest.mark.parametrize("T", [1, 2, 9, 33, 64])
@pytest.mark.parametrize("layers,heads,dim", [(1, 1, 8), (5, 3, 256), (33, 8, 128)])
def test_compact_sizes(dev, T, layers, heads, dim):
    g = torch.Generator().manual_seed(T)
    lens = torch.randint(T, T + 100, (6,), generator=g).tolist()
    paths = [sorted(torch.randperm(T, generator=g)[:int(torch.randint(0, T + 1, (1,),
                                                                      generator=g))].tolist())
             for _ in lens]
    run_compact(dev, "nhd", lens, T, paths, 16, layers, heads, dim)


def test_compact_one_layer_without_its_dimension(dev):
    g = torch.Generator().manual_seed(0)
    table, pages = make_table(g, [30], 8)
    k, v = caches(g, 1, pages, 2, 8, 64, "hnd", dev)
    want = compacted(bits(k), table, [30], 6, [[0, 3, 5]], 8)
    out = ops.compact_cache(k[0], v[0], table.to(dev), torch.tensor([30], dtype=torch.int32,
                                                                    device=dev),
                            torch.tensor([[0, 3, 5, -1, -1, -1]], dtype=torch.int32, device=dev),
                            torch.tensor([3], dtype=torch.int32, device=dev))
    assert torch.equal(bits(k), want) and out.tolist() == [27]


def test_compact_leaves_what_is_wrong_as_it_is(dev):
    g = torch.Generator().manual_seed(1)
    T, page, lens = 4, 4, [20] * 9
    table, pages = make_table(g, lens, page)
    k, v = caches(g, 2, pages, 2, page, 64, "hnd", dev)
    path = torch.tensor([[0, 2, 1, -1], [1, 1, 3, -1], [0, 4, -1, -1], [0, -1, 3, -1], [0, 3, -1, -1],
                         [0, 3, -1, -1], [0, 3, -1, -1], [0, 3, -1, -1], [-5, 3, -1, -1]],
                        dtype=torch.int32)
    counts = torch.tensor([3, 3, 2, 3, 5, -1, 2, 2, 2], dtype=torch.int32)
    ln = torch.tensor([20, 20, 20, 20, 20, 20, 3, 21, 20], dtype=torch.int32)
    before = bits(k).clone(), bits(v).clone()
    out = ops.compact_cache(k, v, table.to(dev), ln.to(dev), path.to(dev), counts.to(dev))
    assert torch.equal(bits(k), before[0]) and torch.equal(bits(v), before[1])
    assert out.tolist() == ln.tolist()
    # No tokens at all, and a page that is none: that row stays, the others move.
    lens = [0, 22]
    table, pages = make_table(g, lens, page)
    k, v = caches(g, 2, pages, 2, page, 64, "hnd", dev)
    want = compacted(bits(k), table, [4, 22], T, [[], [0, 1, 3]], page)
    keep = table[1, 19 // page].item(), 19 % page
    want[:, keep[0], :, keep[1]] = bits(k)[:, keep[0], :, keep[1]]
    broken = table.clone()
    broken[1, 20 // page] = pages                      # offsets 20 .. 23: rows 2 and 3 of the four
    rows = torch.tensor([[-1] * 4, [1, 2, -1, -1]], dtype=torch.int32)
    cnt = torch.tensor([0, 2], dtype=torch.int32)
    now = compacted(bits(k), table, [4, 22], T, [[], [1]], page)
    out = ops.compact_cache(k, v, broken.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev),
                            rows.to(dev), cnt.to(dev))
    assert torch.equal(bits(k), now) and out.tolist() == [0, 20]


def test_offsets_past_32_bits(dev):
    pages, page, heads, dim = 35000, 16, 8, 256
    kv = torch.zeros(2, pages, heads, page, dim, dtype=torch.bfloat16, device=dev)
    vv = torch.zeros_like(kv)
    assert kv[0].numel() > 2 ** 30 and kv.numel() > 2 ** 31
    kv[1, pages - 1] = 3
    vv[1, pages - 1] = 5
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)                # noqa: E731
    ops.copy_pages(kv, vv, i(pages - 1), i(pages - 3))
    assert (kv[1, pages - 3] == 3).all() and (vv[1, pages - 3] == 5).all()
    assert (kv[0, pages - 3] == 0).all() and (kv[1, pages - 2] == 0).all()
    kv[1, pages - 1, :, 9] = 7
    ops.compact_cache(kv, vv, i(pages - 2, pages - 1).view(1, 2), i(26), i(0, 9, -1, -1, -1, -1, -1,
                                                                           -1, -1, -1).view(1, 10),
                      i(2))
    assert (kv[1, pages - 1, :, 1] == 7).all() and (kv[1, pages - 1, :, 0] == 3).all()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page,heads,dim", [(1, 1, 8), (16, 8, 128), (24, 3, 80), (100, 2, 256)])
@pytest.mark.parametrize("part", [False, True])
def test_copy(dev, layout, page, heads, dim, part):
    g = torch.Generator().manual_seed(page)
    pages, layers = 23, 3
    k, v = caches(g, layers, pages, heads, page, dim, layout, dev, torch.bfloat16)
    order = torch.randperm(pages, generator=g).tolist()
    src = [order[0], order[0], order[1], -1, order[2], pages, 3, order[3]]
    dst = [order[10], order[11], order[12], order[13], -1, order[14], 2 ** 31 - 1, order[15]]
    rows = torch.randint(-1, page + 2, (8,), generator=g).tolist()
    want = [bits(x).clone() for x in (k, v)]
    for w in want:
        old = w.clone()
        for a, z, n in zip(src, dst, rows):
            if 0 <= a < pages and 0 <= z < pages:
                n = min(max(n, 0), page) if part else page
                w[:, z, :, :n] = old[:, a, :, :n]
    i = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)                 # noqa: E731
    ops.copy_pages(k, v, i(src), i(dst), i(rows) if part else None)
    assert torch.equal(bits(k), want[0]) and torch.equal(bits(v), want[1])
    ops.copy_pages(k, v, i([]), i([]))
    ops.copy_pages(k[1], v[1], i([order[10]]), i([order[20]]))
    for x, w in zip((k, v), want):
        w[1, order[20]] = w[1, order[10]]
        assert torch.equal(bits(x), w)


def test_captured_on_another_stream(dev):
    g = torch.Generator().manual_seed(3)
    lens, T, page = [40, 33], 8, 16
    table, pages = make_table(g, lens, page)
    k, v = caches(g, 4, pages + 4, 2, page, 64, "nhd", dev)
    k0, v0 = k.clone(), v.clone()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)                # noqa: E731
    args = table.to(dev), i(*lens)
    path, counts, src, dst = i(0, 2, 4, *[-1] * 5, 0, 1, 7, *[-1] * 5).view(2, 8), i(3, 3), i(0), \
        i(pages)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.copy_pages(k, v, src, dst)
        out = ops.compact_cache(k, v, *args, path, counts)
    for r in range(3):
        k.copy_(k0), v.copy_(v0)
        src.fill_(r), dst.fill_(pages + r)
        counts.fill_(r)
        graph.replay()
        ke, ve = k0.clone(), v0.clone()
        ops.copy_pages(ke, ve, src, dst)
        want = ops.compact_cache(ke, ve, *args, path, counts)
        torch.cuda.synchronize()
        assert torch.equal(bits(k), bits(ke)) and torch.equal(bits(v), bits(ve)), r
        assert torch.equal(out, want)


def test_wrong_arguments_are_refused(dev):
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)       # noqa: E731
    i = torch.int32
    k, v = z(3, 4, 2, 16, 64), z(3, 4, 2, 16, 64)
    ok = (k, v, z(2, 2, dt=i), z(2, dt=i), z(2, 5, dt=i), z(2, dt=i))
    ops.compact_cache(*ok)
    for n, bad in ((0, z(4, 2, 16, 64)), (0, z(3, 4, 2, 16, 64).float()), (1, z(2, 4, 2, 16, 64)),
                   (0, z(0, 4, 2, 16, 64)), (0, k.cpu()), (2, z(3, 2, dt=i)), (3, z(3, dt=i)),
                   (4, z(10, dt=i)), (4, z(5, 2, dt=i).t()), (5, z(2)), (5, z(3, dt=i))):
        args = list(ok)
        args[n] = bad
        with pytest.raises((ValueError, TypeError)):
            ops.compact_cache(*args)
    with pytest.raises(hxm.HxmError, match="share elements"):
        ops.compact_cache(k, k, *ok[2:])
    with pytest.raises(hxm.HxmError, match="share elements"):
        ops.compact_cache(k[:1].expand(3, 4, 2, 16, 64), v, *ok[2:])
    with pytest.raises(hxm.HxmError, match="tile-alignment"):
        ops.compact_cache(k, v, *ok[2:4], z(2, 65, dt=i), ok[5])
    for src, dst, rows in ((z(2, dt=i), z(3, dt=i), None), (z(2), z(2, dt=i), None),
                           (z(2, dt=i), z(2, dt=i), z(3, dt=i)), (z(2, dt=i).cpu(), z(2, dt=i), None)):
        with pytest.raises((ValueError, TypeError)):
            ops.copy_pages(k, v, src, dst, rows)
    flat = z(2 * 3 * 4 * 2 * 16 * 64)
    with pytest.raises(hxm.HxmError, match="share elements"):
        ops.copy_pages(flat[:k.numel()].view(k.shape), flat[64:64 + k.numel()].view(k.shape),
                       z(1, dt=i), z(1, dt=i))
