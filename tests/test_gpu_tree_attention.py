"""hxm_tree_attention against softmax(scale q K^T) V over what each node sees, in 64 bits.

Every cache row outside a sequence's tokens and those of padded nodes hold NaN, every
table entry past its pages an invalid number.  Tolerances, from arithmetic alone, with A
the mean of |v| under the exact probabilities and u = eps / 2 of the dtype:
* out is rounded once: u |o|;
* each probability enters the product with V as two halves of the dtype, the second
  the rounded rest of the first: 2 u^2 A at most (the sum that normalises adds the
  unrounded ones), and in f16 a subnormal second half is off by half of 2^-24, at
  least 2^7 below the scaled maximum: n 2^-32 max|v|;
* scores: fp32 sums of dim products, (dim + 8) 2^-24 of scale sum|q k|, move a
  probability by that much relatively, and the mean of v by twice that of A;
* the exponential, the rescalings and the chains of the fp32 sums, n / 2 terms
  long at most (a lane adds the probabilities of every other four tokens):
  (n / 2 + 64) 2^-24 A.
"""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16}
NAN = float("nan")


def trees(g, lens, T, kind):
    """Parents [B][T]: -1 the context, -2 padding."""
    rows = []
    for n in lens:
        if kind == "chain":
            row = list(range(-1, T - 1))
        else:
            live = T if kind == "full" else int(torch.randint(1, T + 1, (1,), generator=g))
            row = [-1] + [int(torch.randint(-1, i, (1,), generator=g)) for i in range(1, live)]
            row += [-2] * (T - live)
            if kind == "holes":                  # padding among the nodes, not only behind them
                order = torch.randperm(T, generator=g).sort().values.tolist()
                row = row[:live] + [-2] * (T - live)
                for i in range(1, T, 3):
                    row[i] = -2
                row = [p if p < 0 or row[p] >= -1 else -1 for p in row]
                assert order == list(range(T))
        rows.append(row if n > 0 else [-2] * T)
    return rows


def above(row, i):
    out = []
    while i >= 0:
        out.append(i)
        i = row[i]
    return out


def visible(row, n, T, window):
    """Bool [T, n]: the tokens each node sees."""
    see = np.zeros((T, max(n, 0)), dtype=bool)
    for i in range(T if n > 0 else 0):
        if row[i] < -1:
            continue
        up = above(row, i)
        depth = len(up) - 1
        first = max(0, n - T + depth - window + 1) if window else 0
        see[i, first:n - T] = True
        for j in up:
            if not window or len(above(row, j)) - 1 > depth - window:
                see[i, n - T + j] = True
    return see


def build(g, name, lens, T, rows, hkv, group, dim, page, layout, dev, spread=1.0, spare=2):
    dt = TDT[name]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    width = max(need) + 1
    table = torch.tensor([-7, 2 ** 31 - 1])[torch.arange(len(lens) * width) % 2].view(
        len(lens), width).int()
    kc = torch.full((pages, hkv, page, dim), NAN, dtype=dt)
    vc = kc.clone()
    seqs, at = [], 0
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = torch.tensor(ids, dtype=torch.int32)
        k = (spread * torch.randn(n, hkv, dim, generator=g)).to(dt)
        v = torch.randn(n, hkv, dim, generator=g).to(dt)
        for i, p in enumerate(rows[b]):
            if p < -1 and n:
                k[n - T + i] = NAN
                v[n - T + i] = NAN
        for t in range(need[b]):
            part = slice(t * page, min(n, (t + 1) * page))
            kc[ids[t], :, :part.stop - part.start] = k[part].transpose(0, 1)
            vc[ids[t], :, :part.stop - part.start] = v[part].transpose(0, 1)
        seqs.append((k.double().numpy(), v.double().numpy()))
    q = torch.randn(len(lens), T, hkv * group, dim, generator=g).to(dt)
    if layout == "nhd":
        kc, vc = (c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for c in (kc, vc))
    else:
        kc, vc = kc.to(dev), vc.to(dev)
    return q, kc, vc, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), seqs


def check(out, lse, q, seqs, rows, group, scale, window, name):
    u, dt = torch.finfo(TDT[name]).eps / 2, TDT[name]
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    T = q.shape[1]
    for b, (k, v) in enumerate(seqs):
        n = len(k)
        see = visible(rows[b], n, T, window)
        for h in range(q.shape[2]):
            got, gl = out[b, :, h].double().numpy(), lse[b, :, h].double().numpy()
            dead = ~see.any(1) if n else np.ones(T, dtype=bool)
            assert (got[dead] == 0).all() and (gl[dead] == -np.inf).all(), (b, h)
            if dead.all():
                continue
            qh, kh, vh = q[b, :, h].double().numpy(), k[:, h // group], v[:, h // group]
            ok = np.isfinite(kh).all(1) & np.isfinite(vh).all(1)
            assert not (see & ~ok).any()
            kh, vh = np.where(ok[:, None], kh, 0), np.where(ok[:, None], vh, 0)
            s = np.where(see, scale * (qh @ kh.T), -np.inf)[~dead]
            mag = abs(scale) * np.where(see, np.abs(qh) @ np.abs(kh).T, 0).max(1)[~dead]
            top = s.max(1, keepdims=True)
            p = np.exp(s - top)
            L = top[:, 0] + np.log(p.sum(1))
            p /= p.sum(1, keepdims=True)
            want, A = p @ vh, p @ np.abs(vh)
            d = 2.0 ** -24 * ((q.shape[3] + 8) * mag + n / 2 + 64)
            tol = u * np.abs(want) + (2 * u * u + 2 * d[:, None]) * A + tiny
            if name == "f16":
                tol = tol + n * 2.0 ** -32 * np.abs(vh).max()
            bad = ~(np.abs(got[~dead] - want) <= tol)
            assert not bad.any(), (b, h, n, np.argwhere(bad)[:4].tolist(), got[~dead][bad][:4],
                                   want[bad][:4])
            assert (np.abs(gl[~dead] - L) <= d + 2.0 ** -22 * np.abs(L)).all(), (b, h, n)


def run_case(dev, name, lens, T, hkv, group, dim, page, layout, kind="full", window=0, scale=None,
             spread=1.0, seed=0):
    print(f"{name} lens={lens[:8]} T={T} heads={hkv}x{group} dim={dim} page={page} {layout} "
          f"{kind} window={window}", flush=True)
    g = torch.Generator().manual_seed(seed + dim + page + group + T)
    rows = trees(g, lens, T, kind)
    q, kc, vc, table, ld, seqs = build(g, name, lens, T, rows, hkv, group, dim, page, layout, dev,
                                       spread)
    parents = None if kind == "chain" and min(lens) > 0 else torch.tensor(
        rows, dtype=torch.int32, device=dev)
    out, lse = ops.tree_attention(q.to(dev), kc, vc, table, ld, parents, window=window,
                                  scale=scale, return_lse=True)
    check(out.cpu(), lse.cpu(), q, seqs, rows, group, dim ** -0.5 if scale is None else scale,
          window, name)
    return out, lse


@pytest.mark.parametrize("T", [1, 2, 5, 8, 9, 16, 17, 31, 32, 33, 63, 64])
@pytest.mark.parametrize("kind", ["chain", "full", "ragged", "holes"])
def test_nodes(dev, T, kind):
    lens = [T, T + 1, 0, T + 31, T + 32, 64 + T, 200 + T, 300]
    run_case(dev, "f16", lens, T, 2, 2, 64, 16, "hnd", kind)
    run_case(dev, "bf16", lens[:3] + [333], T, 1, 4, 128, 24, "nhd", kind)


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_dims(dev, name, dim):
    for T, group in ((3, 4), (11, 4), (20, 5)):       # one, two and four waves over the rows
        run_case(dev, name, [T, 100, 0, 257], T, 2, group, dim, 16, "hnd", "ragged")
        run_case(dev, name, [63, 64, 90], T, 1, group, dim, 24, "nhd", "full")


@pytest.mark.parametrize("page", [1, 3, 8, 12, 16, 24, 33, 64, 100, 4096])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages(dev, page, layout):
    run_case(dev, "f16", [12, 13, 31, 33, 150, 0, 300], 12, 2, 3, 64, page, layout)
    run_case(dev, "bf16", [700, 0, 41], 9, 1, 8, 128, page, layout, window=100)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 8, 15, 16, 17, 32, 40])
def test_shared_heads(dev, group):
    run_case(dev, "f16", [257, 0, 64, 7], 7, 2, group, 128, 16, "hnd", "ragged")
    run_case(dev, "bf16", [100, 31], 25, 1, group, 64, 32, "nhd")


@pytest.mark.parametrize("window", [1, 2, 7, 31, 32, 33, 100, 299, 300, 2 ** 31 - 1, 2 ** 40])
@pytest.mark.parametrize("T", [1, 10, 40])
def test_windows(dev, window, T):
    lens = [T, T + 1, T + 33, 129 + T, 300 + T, 0]
    run_case(dev, "f16", lens, T, 2, 2, 64, 16, "hnd", "ragged", window=window)
    run_case(dev, "bf16", lens[:-1], T, 1, 4, 128, 5, "nhd", "chain", window=window)


@pytest.mark.parametrize("lens", [[5000], [4097, 6, 0, 2500], [20011, 30], [1000] * 40])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_long(dev, name, lens):
    run_case(dev, name, lens, 6, 2, 4, 128, 16, "nhd", "ragged")
    run_case(dev, name, lens, 5, 1, 9, 256, 40, "hnd", "chain" if 0 not in lens else "full")
    run_case(dev, name, lens[:4], 5, 1, 30, 64, 128, "hnd", window=1500)


@pytest.mark.parametrize("batch", [63, 64, 65, 200, 256, 257, 400])
def test_many_sequences(dev, batch):
    r = np.random.default_rng(batch)
    lens = r.integers(4, 70, batch).tolist()
    lens[batch // 2] = 2600
    run_case(dev, "f16", lens, 4, 2, 2, 64, 16, "hnd", "ragged")
    run_case(dev, "bf16", [640 if b < batch - 9 else 0 for b in range(batch)], 3, 1, 2, 64, 32,
             "nhd", "full")


@pytest.mark.parametrize("hkv,group", [(32, 1), (8, 8), (2, 33), (300, 1)])
def test_many_heads(dev, hkv, group):
    run_case(dev, "bf16", [1000, 0, 1085, 5], 5, hkv, group, 64, 16, "nhd", "ragged")
    run_case(dev, "f16", [700], 3, hkv, group, 32, 16, "hnd", window=530)


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_peaked_and_flat_scores(dev, name):
    for T, group in ((4, 4), (16, 8)):
        run_case(dev, name, [3000, 77], T, 1, group, 128, 16, "hnd", spread=20.0)
        run_case(dev, name, [3000, 77], T, 1, group, 128, 16, "hnd", scale=0.0)
        run_case(dev, name, [3000, 77], T, 1, group, 64, 16, "hnd", scale=-0.7)


def test_one_node_is_paged_attention(dev):
    """Within both operators' rounding of the output (eps / 2 each) of the same sums."""
    g = torch.Generator().manual_seed(3)
    lens = [1, 33, 700, 0, 2000]
    rows = [[-1] if n else [-2] for n in lens]
    q, kc, vc, table, ld, _ = build(g, "f16", lens, 1, rows, 2, 4, 128, 16, "hnd", dev)
    a, la = ops.tree_attention(q.to(dev), kc, vc, table, ld, return_lse=True)
    b, lb = ops.paged_attention(q[:, 0].to(dev), kc, vc, table, ld, return_lse=True)
    assert torch.allclose(a[:, 0].float(), b.float(), rtol=2.0 ** -10, atol=2.0 ** -12)
    assert torch.allclose(la[:, 0], lb, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("T,group", [(6, 2), (12, 4), (40, 4)])
@pytest.mark.parametrize("what", ["nan", "inf"])
def test_what_a_node_does_not_see_never_reaches_it(dev, T, group, what):
    """Keys and values of one drafted token (and one of the context, behind the window of some)
    that are no numbers: those that do not see them stay as they were."""
    g = torch.Generator().manual_seed(T)
    n, dim, bad = 150 + T, 64, T // 2
    rows = [[-1] + [int(torch.randint(-1, i, (1,), generator=g)) for i in range(1, T)]]
    q, kc, vc, table, ld, _ = build(g, "f16", [n], T, rows, 1, group, dim, 16, "hnd", dev)
    parents = torch.tensor(rows, dtype=torch.int32, device=dev)
    window = 60
    ref = ops.tree_attention(q.to(dev), kc, vc, table, ld, parents, window=window)
    see = visible(rows[0], n, T, window)
    for tok in (n - T + bad, n - T - window + 1):
        assert not see[:, tok].all()
        k2, v2 = kc.clone(), vc.clone()
        k2[table[0, tok // 16].item(), :, tok % 16, 5] = NAN if what == "nan" else 0.0
        v2[table[0, tok // 16].item(), :, tok % 16, 7] = NAN if what == "nan" else float("inf")
        got = ops.tree_attention(q.to(dev), k2, v2, table, ld, parents, window=window)
        blind = torch.tensor(~see[:, tok])
        if what == "nan":
            assert torch.equal(got.cpu()[0, blind], ref.cpu()[0, blind])
            assert got.cpu()[0, ~blind].isnan().all()
        else:  # an infinite value is one of its dim, a zero in the key of finite numbers no harm
            assert not got.cpu()[0, blind].isnan().any()
            assert got.cpu()[0, blind].isfinite().all()
            assert not got.cpu()[0, ~blind][..., 7].isfinite().any()
            keep = [d for d in range(dim) if d != 7]
            assert got.cpu()[0][..., keep].isfinite().all()


def test_bad_parents_pages_and_lengths(dev):
    g = torch.Generator().manual_seed(0)
    T, lens = 5, [40, 40, 40, 40, 3, 1000, 40]
    rows = [[-1, 0, 1, 2, 3] for _ in lens]
    q, kc, vc, table, ld, _ = build(g, "f16", [40] * 7, T, rows, 2, 2, 64, 16, "hnd", dev)
    ld = torch.tensor(lens, dtype=torch.int32, device=dev)
    rows[0] = [-1, 0, 2, 1, 2]        # its own parent, and its child
    rows[1] = [-1, 4, 0, 1, 0]        # a later node, and its child
    rows[2] = [-1, -2, 1, 0, 2]       # below padding, and its child
    table[3, 1] = kc.shape[0]         # a page that is none
    parents = torch.tensor(rows, dtype=torch.int32, device=dev)
    out, lse = (t.cpu() for t in ops.tree_attention(q.to(dev), kc, vc, table, ld, parents,
                                                    return_lse=True))
    nan = [[0, 0, 1, 0, 1], [0, 1, 0, 1, 0], [0, 0, 1, 0, 1], [1] * 5, [1] * 5, [1] * 5, [0] * 5]
    nan = torch.tensor(nan).bool()
    assert torch.equal(out.isnan().all(-1).all(-1), nan)
    assert torch.equal(out.isnan().any(-1).any(-1), nan)
    assert torch.equal(lse.isnan().all(-1), nan)
    assert (out[2, 1] == 0).all() and (lse[2, 1] == -np.inf).all()
    chain = ops.tree_attention(q.to(dev), kc, vc, table, ld).cpu()
    assert torch.equal(chain[6], out[6]) and chain[3:6].isnan().all()


def test_strided_views_outputs_and_streams(dev):
    """q as heads of a fused projection, an output of other strides, another stream."""
    g = torch.Generator().manual_seed(1)
    lens, T = [50, 700], 7
    rows = trees(g, lens, T, "full")
    q, kc, vc, table, ld, _ = build(g, "bf16", lens, T, rows, 2, 3, 64, 16, "nhd", dev)
    parents = torch.tensor(rows, dtype=torch.int32, device=dev)
    ref, rl = ops.tree_attention(q.to(dev), kc, vc, table, ld, parents, return_lse=True)
    fused = torch.zeros(2, T, 10, 64, dtype=torch.bfloat16, device=dev)
    fused[:, :, 2:8] = q.to(dev)
    big = torch.full((2, T, 9, 72), 7.0, dtype=torch.bfloat16, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got, gl = ops.tree_attention(fused[:, :, 2:8], kc, vc, table, ld, parents,
                                 out=big[:, :, 1:7, :64], return_lse=True, stream=s)
    s.synchronize()
    assert torch.equal(got, ref) and torch.equal(gl, rl)
    assert (big[:, :, 0] == 7).all() and (big[:, :, 7:] == 7).all() and (big[..., 64:] == 7).all()
    wide = torch.zeros(2, 12, dtype=torch.int32, device=dev).fill_(-1)
    wide = torch.cat((table, wide), 1)[:, :table.shape[1]]
    assert torch.equal(ops.tree_attention(q.to(dev), kc, vc, wide, ld, parents), ref)


def test_captured_graph(dev):
    """Replayed with the program's own calls in between, against the eager result each time."""
    g = torch.Generator().manual_seed(2)
    lens, T = [2000, 40, 900], 8
    rows = trees(g, lens, T, "ragged")
    q, kc, vc, table, ld, _ = build(g, "f16", lens, T, rows, 2, 4, 128, 16, "hnd", dev)
    q, parents = q.to(dev), torch.tensor(rows, dtype=torch.int32, device=dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out = torch.empty_like(q)
    with torch.cuda.stream(s):
        ops.tree_attention(q, kc, vc, table, ld, parents, out=out)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.tree_attention(q, kc, vc, table, ld, parents, out=out)
    for turn in range(4):
        q.copy_(torch.randn(q.shape, generator=g).half())
        ld.copy_(torch.tensor([2000 - 300 * turn, 40, 900 + turn], dtype=torch.int32)
                 .clamp(max=2000))
        ld[2] = 900 - turn
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.tree_attention(q, kc, vc, table, ld, parents)), turn


def test_no_sequences(dev):
    kc = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device=dev)
    q = torch.zeros(0, 4, 2, 64, dtype=torch.float16, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    out, lse = ops.tree_attention(q, kc, kc.clone(), none.view(0, 1), none, return_lse=True)
    assert out.shape == q.shape and lse.shape == (0, 4, 2)


def test_wrong_arguments_are_refused(dev):
    z = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)     # noqa: E731
    kc, vc = z(4, 2, 16, 64), z(4, 2, 16, 64)
    table, lens = z(3, 2, dt=torch.int32), z(3, dt=torch.int32)
    q, parents = z(3, 5, 4, 64), z(3, 5, dt=torch.int32)
    ok = (q, kc, vc, table, lens, parents)
    ops.tree_attention(*ok)

    def refused(error, *args, **kw):
        with pytest.raises(error):
            ops.tree_attention(*args, **kw)
    for i, bad in [(0, z(3, 4, 64)), (0, z(3, 5, 4, 64, dt=torch.bfloat16)), (0, q.cpu()),
                   (0, z(5, 3, 4, 64).transpose(0, 1)), (0, z(3, 5, 4, 128)[..., ::2]),
                   (3, z(2, 2, dt=torch.int32)), (3, z(3, 2, dt=torch.int64)),
                   (4, z(2, dt=torch.int32)), (5, z(3, 4, dt=torch.int32)),
                   (5, z(5, 3, dt=torch.int32).t()), (5, parents.long())]:
        args = list(ok)
        args[i] = bad
        refused((ValueError, TypeError), *args)
    refused(hxm.HxmError, z(3, 5, 3, 64), *ok[1:])               # 3 heads over 2
    refused(hxm.HxmError, z(3, 65, 4, 64), *ok[1:5])             # 65 nodes
    refused(hxm.HxmError, z(3, 0, 4, 64), *ok[1:5])
    refused(hxm.HxmError, *ok, window=-1)
    refused(hxm.HxmError, *ok, scale=NAN)
    refused(hxm.HxmError, *ok, out=q)
    refused(ValueError, *ok, out=z(3, 5, 4, 32))


def test_offsets_past_32_bits(dev):
    """A cache of more than 2^31 elements, its last pages in use; and rows too far apart for
    32-bit offsets within a page."""
    pages, page, heads, dim, T = 70000, 16, 8, 256, 3
    kc = torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    assert kc.numel() > 2 ** 31
    g = torch.Generator().manual_seed(5)
    ids = [pages - 1, 3, pages - 2]
    small = [torch.randn(4, heads, page, dim, generator=g).bfloat16().to(dev) for _ in range(2)]
    for i, p in enumerate(ids):
        kc[p], vc[p] = small[0][i], small[1][i]
    q = torch.randn(1, T, 16, dim, generator=g).bfloat16().to(dev)
    lens = torch.tensor([45], dtype=torch.int32, device=dev)
    near = ops.tree_attention(q, *small, torch.tensor([[0, 1, 2]], dtype=torch.int32, device=dev),
                              lens)
    far = ops.tree_attention(q, kc, vc, torch.tensor([ids], dtype=torch.int32, device=dev), lens)
    assert torch.equal(near, far)
    del kc, vc
    apart = 2 ** 26 + 8
    wide = [torch.zeros(16 * apart, dtype=torch.bfloat16, device=dev).as_strided(
        (1, 1, 16, 64), (16 * apart, 16 * apart, apart, 1)) for _ in range(2)]
    packed = [torch.randn(1, 1, 16, 64, generator=g).bfloat16().to(dev) for _ in range(2)]
    for w, p in zip(wide, packed):
        w.copy_(p)
    q = torch.randn(1, T, 2, 64, generator=g).bfloat16().to(dev)
    table = torch.zeros(1, 1, dtype=torch.int32, device=dev)
    lens = torch.tensor([14], dtype=torch.int32, device=dev)
    assert torch.equal(ops.tree_attention(q, *packed, table, lens),
                       ops.tree_attention(q, *wide, table, lens))


def test_same_results_every_time_and_on_streams_at_once(dev):
    """Results repeat bit for bit, also beside another stream's calls, whose workspace is its own."""
    g = torch.Generator().manual_seed(6)
    jobs = []
    for lens, T, group in (([3000, 40, 700], 6, 4), ([900, 2000], 20, 5)):
        rows = trees(g, lens, T, "ragged")
        q, kc, vc, table, ld, _ = build(g, "f16", lens, T, rows, 2, group, 128, 16, "nhd", dev)
        jobs.append((q.to(dev), kc, vc, table, ld, torch.tensor(rows, dtype=torch.int32, device=dev)))
    want = [ops.tree_attention(*j, return_lse=True) for j in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(10):
        got = [ops.tree_attention(*j, return_lse=True, stream=s) for j, s in zip(jobs, streams)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_call_of_its_own_beside_other_sequences(dev):
    """A sequence that is not cut gives the same alone and in a batch."""
    g = torch.Generator().manual_seed(7)
    lens, T = [100, 333, 500, 64], 5
    rows = trees(g, lens, T, "full")
    q, kc, vc, table, ld, _ = build(g, "bf16", lens, T, rows, 2, 4, 64, 16, "hnd", dev)
    parents = torch.tensor(rows, dtype=torch.int32, device=dev)
    q = q.to(dev)
    all_of_them = ops.tree_attention(q, kc, vc, table, ld, parents)
    for b in range(len(lens)):
        one = ops.tree_attention(q[b:b + 1], kc, vc, table[b:b + 1].contiguous(), ld[b:b + 1],
                                 parents[b:b + 1])
        assert torch.equal(one[0], all_of_them[b]), b
