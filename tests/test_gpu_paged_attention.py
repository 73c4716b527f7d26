"""hxm_paged_attention against softmax(scale q K^T) V in 64 bits.

Every cache row outside a sequence's tokens holds NaN, every table entry past
its pages an invalid number.  Tolerances, from arithmetic alone, with A the
mean of |v| under the exact probabilities and u = eps / 2 of the dtype:
* out is rounded once: u |o|;
* each probability enters the product with V as two halves of the dtype, the second
  the rounded rest of the first: 2 u^2 A at most (the sum that normalises adds the
  unrounded ones), and in f16 a subnormal second half is off by half of 2^-24, at
  least 2^7 below the scaled maximum: n 2^-32 max|v|;
* scores: fp32 sums of dim products, (dim + 8) 2^-24 of scale sum|q k|, move a
  probability by that much relatively, and the mean of v by twice that of A;
* the exponential, the rescalings and the chains of the fp32 sums, n / 16 terms
  long at most: (n / 16 + 64) 2^-24 A.
"""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16}


def build(g, name, lens, hkv, group, dim, page, layout, dev, spread=1.0, spare=2):
    """(q, k_cache, v_cache, table, lens) on dev and each sequence's K, V in 64 bits."""
    dt = TDT[name]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=g).tolist()
    width = max(need) + 1
    table = torch.tensor([-7, 2 ** 31 - 1])[torch.arange(len(lens) * width) % 2].view(
        len(lens), width).int()
    kc = torch.full((pages, hkv, page, dim), float("nan"), dtype=dt)
    vc = kc.clone()
    seqs, at = [], 0
    for b, n in enumerate(lens):
        ids = order[at:at + need[b]]
        at += need[b]
        table[b, :need[b]] = torch.tensor(ids, dtype=torch.int32)
        k = (spread * torch.randn(n, hkv, dim, generator=g)).to(dt)
        v = torch.randn(n, hkv, dim, generator=g).to(dt)
        for t in range(need[b]):
            part = slice(t * page, min(n, (t + 1) * page))
            kc[ids[t], :, :part.stop - part.start] = k[part].transpose(0, 1)
            vc[ids[t], :, :part.stop - part.start] = v[part].transpose(0, 1)
        seqs.append((k.double().numpy(), v.double().numpy()))
    q = torch.randn(len(lens), hkv * group, dim, generator=g).to(dt)
    if layout == "nhd":
        kc, vc = (c.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for c in (kc, vc))
    else:
        kc, vc = kc.to(dev), vc.to(dev)
    return q, kc, vc, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), seqs


def check(out, lse, q, seqs, group, scale, window, name):
    u, dt = torch.finfo(TDT[name]).eps / 2, TDT[name]
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    for b, (k, v) in enumerate(seqs):
        lo = max(0, len(k) - window) if window else 0
        k, v, n = k[lo:], v[lo:], len(k) - lo
        if n <= 0:
            assert (out[b] == 0).all() and (lse[b] == -np.inf).all(), b
            continue
        dim = k.shape[2]
        for h in range(q.shape[1]):
            qh, kh, vh = q[b, h].double().numpy(), k[:, h // group], v[:, h // group]
            s = scale * (kh @ qh)
            mag = abs(scale) * (np.abs(kh) @ np.abs(qh)).max()
            p = np.exp(s - s.max())
            L = s.max() + np.log(p.sum())
            p /= p.sum()
            want, A = p @ vh, p @ np.abs(vh)
            d = 2.0 ** -24 * ((dim + 8) * mag + n / 16 + 64)
            tol = u * np.abs(want) + (2 * u * u + 2 * d) * A + tiny
            if name == "f16":
                tol = tol + n * 2.0 ** -32 * np.abs(vh).max()
            got = out[b, h].double().numpy()
            bad = ~(np.abs(got - want) <= tol)
            assert not bad.any(), (b, h, n, np.argwhere(bad)[:4].tolist(), got[bad][:4],
                                   want[bad][:4])
            assert abs(lse[b, h].item() - L) <= d + 2.0 ** -22 * abs(L), (b, h, n, lse[b, h], L)


def run_case(dev, name, lens, hkv, group, dim, page, layout, window=0, scale=None, spread=1.0,
             seed=0):
    print(f"{name} lens={lens[:8]} heads={hkv}x{group} dim={dim} page={page} {layout} "
          f"window={window}", flush=True)
    g = torch.Generator().manual_seed(seed + dim + page + group)
    q, kc, vc, table, ld, seqs = build(g, name, lens, hkv, group, dim, page, layout, dev, spread)
    out, lse = ops.paged_attention(q.to(dev), kc, vc, table, ld, window=window, scale=scale,
                                   return_lse=True)
    check(out.cpu(), lse.cpu(), q, seqs, group, dim ** -0.5 if scale is None else scale, window,
          name)
    return out, lse


LENS = [0, 1, 2, 7, 8, 9, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300, 0]


@pytest.mark.parametrize("dim", [8, 40, 64, 72, 80, 96, 128, 136, 192, 256])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_dims_and_lengths(dev, name, dim):
    run_case(dev, name, LENS, 2, 4, dim, 16, "hnd")
    run_case(dev, name, LENS, 3, 1, dim, 24, "nhd")


@pytest.mark.parametrize("page", [1, 3, 5, 8, 12, 16, 24, 32, 33, 64, 100, 256, 4096])
@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_pages(dev, page, layout):
    run_case(dev, "f16", LENS, 2, 3, 64, page, layout)
    run_case(dev, "bf16", [700, 0, 41], 1, 8, 128, page, layout, window=100)


@pytest.mark.parametrize("group", [1, 2, 3, 5, 7, 8, 12, 15, 16, 17, 32, 40])
def test_shared_heads(dev, group):
    run_case(dev, "f16", [257, 0, 64, 1], 2, group, 128, 16, "hnd")
    run_case(dev, "bf16", [100, 31], 1, group, 64, 32, "nhd")


@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 299, 300, 301, 2 ** 31 - 1, 2 ** 40])
def test_windows(dev, window):
    run_case(dev, "f16", LENS, 2, 2, 64, 16, "hnd", window=window)
    run_case(dev, "bf16", LENS, 1, 4, 128, 5, "nhd", window=window)


@pytest.mark.parametrize("lens", [[5000], [4097, 1, 0, 2500], [20011, 3], [1000] * 40])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_long(dev, name, lens):
    run_case(dev, name, lens, 2, 4, 128, 16, "nhd")
    run_case(dev, name, lens, 1, 1, 256, 40, "hnd")
    run_case(dev, name, lens, 4, 2, 64, 128, "hnd", window=1500)


@pytest.mark.parametrize("batch", [63, 64, 65, 128, 200, 255, 256, 257, 513])
def test_many_sequences(dev, batch):
    """Batches in and past one wave's lanes, of one long sequence among short ones, all
    alike, and with rows of padding (no tokens) at the end."""
    r = np.random.default_rng(batch)
    lens = r.integers(0, 70, batch).tolist()
    lens[batch // 2] = 2600
    run_case(dev, "f16", lens, 2, 4, 64, 16, "hnd")
    run_case(dev, "bf16", [640 if b < batch - 9 else 0 for b in range(batch)], 1, 2, 64, 32, "nhd")


@pytest.mark.parametrize("hkv,group", [(32, 1), (8, 8), (64, 2), (2, 33), (300, 1)])
def test_many_heads(dev, hkv, group):
    run_case(dev, "bf16", [1000, 0, 2085, 1], hkv, group, 64, 16, "nhd")
    run_case(dev, "f16", [700], hkv, group, 32, 16, "hnd", window=530)


def test_calls_of_changing_sizes(dev):
    """One stream, one workspace: larger calls after smaller ones and back, the same
    results as before."""
    cases = [([3000], 2, 4, 128), ([700] * 70, 4, 2, 64), ([2000, 0, 900], 8, 20, 64),
             ([30] * 300, 2, 1, 64), ([9000, 5], 1, 16, 256)]
    first = []
    for turn in range(3):
        for i, (lens, hkv, group, dim) in enumerate(cases[::-1] if turn == 1 else cases):
            got = run_case(dev, "f16", lens, hkv, group, dim, 16, "hnd") if turn == 0 else None
            if turn == 0:
                first.append(got)
                continue
            i = len(cases) - 1 - i if turn == 1 else i
            g = torch.Generator().manual_seed(dim + 16 + group)
            q, kc, vc, table, ld, _ = build(g, "f16", lens, hkv, group, dim, 16, "hnd", dev)
            out, lse = ops.paged_attention(q.to(dev), kc, vc, table, ld, return_lse=True)
            assert torch.equal(out, first[i][0]) and torch.equal(lse, first[i][1])


@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_peaked_and_flat_scores(dev, name):
    """Scores spread over hundreds (the running maximum moves often), all equal,
    and of another sign."""
    run_case(dev, name, [3000, 77], 2, 4, 128, 16, "hnd", spread=20.0)
    run_case(dev, name, [3000, 77], 2, 4, 128, 16, "hnd", scale=0.0)
    run_case(dev, name, [3000, 77], 2, 4, 64, 16, "hnd", scale=-0.7)


def test_growing_scores(dev):
    """Each token scores above all before it: every step moves the maximum."""
    n, dim = 2000, 64
    k = (torch.arange(n)[:, None, None] / 64).expand(n, 1, dim).half()
    kc = torch.zeros(n // 16, 1, 16, dim, dtype=torch.float16)
    kc[:] = k.reshape(n // 16, 16, 1, dim).transpose(1, 2)
    vc = torch.randn(kc.shape).half()
    q = torch.ones(1, 1, dim).half()
    table = torch.arange(n // 16, dtype=torch.int32)[None]
    out, lse = ops.paged_attention(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                   torch.tensor([n], dtype=torch.int32, device=dev),
                                   return_lse=True)
    v64 = vc.transpose(1, 2).reshape(n, 1, dim).double().numpy()
    check(out.cpu(), lse.cpu(), q, [(k.double().numpy(), v64)], 1, dim ** -0.5, 0, "f16")


def test_values_far_apart(dev):
    """Keys and values near the f16 limit; an infinite key gives what softmax does."""
    q, kc, vc, table, lens, seqs = build(torch.Generator().manual_seed(1), "f16", [64, 64, 64], 1,
                                         2, 64, 16, "hnd", dev)
    vc.clamp_(-1, 1).mul_(60000)
    seqs = [(k, np.clip(v, -1, 1) * 60000) for k, v in seqs]
    seqs = [(k, torch.from_numpy(v).half().double().numpy()) for k, v in seqs]
    q[1] = 0
    q[1, :, 0] = 1
    row = kc[table[1, 1], 0, 3]
    row[:] = 0
    row[0] = -float("inf")                       # token 19 of sequence 1 counts for nothing
    seqs[1][0][19] = 0
    out, lse = ops.paged_attention(q.to(dev), kc, vc, table, lens, return_lse=True)
    keep = np.arange(64) != 19
    check(out.cpu(), lse.cpu(), q, [seqs[0], (seqs[1][0][keep], seqs[1][1][keep]), seqs[2]], 2,
          64 ** -0.5, 0, "f16")
    row[0] = float("inf")
    out = ops.paged_attention(q.to(dev), kc, vc, table, lens)
    assert out[1].isnan().all() and out[0].isfinite().all() and out[2].isfinite().all()


def test_bad_pages_and_lengths(dev):
    """A page number out of range, or a length past the table, makes that sequence
    NaN and leaves the others as they are."""
    g = torch.Generator().manual_seed(3)
    q, kc, vc, table, lens, seqs = build(g, "f16", [100, 90, 80, 70, 0], 2, 2, 64, 16, "hnd", dev)
    good, glse = ops.paged_attention(q.to(dev), kc, vc, table, lens, return_lse=True)
    for page in (-1, kc.shape[0], 2 ** 31 - 1, -2 ** 31):
        t = table.clone()
        t[1, 3] = page
        ln = lens.clone()
        ln[2] = table.shape[1] * 16 + 1
        ln[4] = -5
        out, lse = ops.paged_attention(q.to(dev), kc, vc, t, ln, return_lse=True)
        assert out[1:3].isnan().all() and lse[1:3].isnan().all()
        for b in (0, 3, 4):
            assert torch.equal(out[b], good[b]) and torch.equal(lse[b], glse[b])
        # A window that does not reach the bad page does not see it.
        out = ops.paged_attention(q.to(dev), kc, vc, t, ln, window=20)
        assert out[1].isfinite().all() and out[2].isnan().all()


def test_strided_views_and_in_place(dev):
    g = torch.Generator().manual_seed(5)
    q, kc, vc, table, lens, seqs = build(g, "bf16", [130, 40, 0], 2, 4, 96, 16, "nhd", dev)
    want, wl = ops.paged_attention(q.to(dev), kc, vc, table, lens, return_lse=True)
    wide = torch.full((3, 8 * 2 + 1, 101), 3.0, dtype=torch.bfloat16, device=dev)
    qs = wide[:, 1:17:2, 5:101]                  # strided heads, off the 16-byte boundary
    qs.copy_(q)
    rest = wide.clone()
    out = torch.full((3, 8, 100), 7.0, dtype=torch.bfloat16, device=dev)
    got, gl = ops.paged_attention(qs, kc, vc, table, lens, out=out[..., 3:99], return_lse=True)
    assert torch.equal(got, want) and torch.equal(gl, wl)
    assert (out[..., :3] == 7).all() and (out[..., 99:] == 7).all()
    wt = torch.full((3, table.shape[1] + 5), -1, dtype=torch.int32, device=dev)
    wt[:, 2:2 + table.shape[1]] = table
    ops.paged_attention(qs, kc, vc, wt[:, 2:2 + table.shape[1]], lens, out=qs)
    assert torch.equal(qs, want)
    rest[:, 1:17:2, 5:101] = qs
    assert torch.equal(rest, wide), "wrote outside the heads"


def test_offsets_past_32_bits(dev):
    pages, page, heads, dim = 70000, 16, 8, 256
    kc = torch.zeros(pages, heads, page, dim, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    assert kc.numel() > 2 ** 31
    g = torch.Generator().manual_seed(6)
    ids = [pages - 1, 66001, 3]
    k, v = (torch.randn(48, heads, dim, generator=g).bfloat16() for _ in range(2))
    for i, p in enumerate(ids):
        kc[p] = k[16 * i:16 * i + 16].transpose(0, 1)
        vc[p] = v[16 * i:16 * i + 16].transpose(0, 1)
    q = torch.randn(1, heads, dim, generator=g).bfloat16()
    out, lse = ops.paged_attention(q.to(dev), kc, vc,
                                   torch.tensor([ids], dtype=torch.int32, device=dev),
                                   torch.tensor([45], dtype=torch.int32, device=dev),
                                   return_lse=True)
    check(out.cpu(), lse.cpu(), q, [(k[:45].double().numpy(), v[:45].double().numpy())], 1,
          dim ** -0.5, 0, "bf16")


def test_same_results_every_time_and_beside_other_sequences(dev):
    """Bit-identical over calls, and on two streams at once."""
    g = torch.Generator().manual_seed(7)
    q, kc, vc, table, lens, _ = build(g, "f16", [3000, 500, 20], 2, 4, 128, 16, "hnd", dev)
    q = q.to(dev)
    want = ops.paged_attention(q, kc, vc, table, lens)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.paged_attention(q, kc, vc, table, lens))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_captured(dev):
    """A captured step replayed while the lengths, the table and the cache move."""
    g = torch.Generator().manual_seed(8)
    q, kc, vc, table, lens, _ = build(g, "f16", [3000, 500, 20, 0], 2, 4, 128, 16, "hnd", dev)
    kc.nan_to_num_(0), vc.nan_to_num_(0)
    q = q.to(dev)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        ops.paged_attention(q, kc, vc, table, lens, out=out)
        with torch.cuda.graph(graph, stream=s):
            ops.paged_attention(q, kc, vc, table, lens, out=out)
    torch.cuda.synchronize()
    for ln in ([3000, 500, 20, 0], [1, 499, 0, 0], [2999, 0, 19, 0], [0, 0, 0, 0], [3000] * 4):
        table[1:] = table[0] if ln[3] else table[1:]
        lens.copy_(torch.tensor(ln, dtype=torch.int32))
        q.normal_()
        want = ops.paged_attention(q, kc, vc, table, lens)
        torch.cuda.synchronize()
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), ln


def test_refusals(dev):
    B, hkv, D = 3, 2, 64
    mk = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)      # noqa: E731
    ok = dict(q=mk(B, 4, D), k_cache=mk(5, hkv, 16, D), v_cache=mk(5, hkv, 16, D),
              block_table=mk(B, 2, dt=torch.int32), seq_lens=mk(B, dt=torch.int32))
    ops.paged_attention(**ok)
    for kw in (dict(q=mk(B, 4, D + 8)), dict(q=mk(B, 4, D, dt=torch.bfloat16)), dict(q=mk(B, D)),
               dict(v_cache=mk(5, hkv, 8, D)), dict(k_cache=mk(5, 16, D)),
               dict(k_cache=mk(5, hkv, 16, D).cpu()), dict(block_table=mk(B + 1, 2, dt=torch.int32)),
               dict(seq_lens=mk(B + 1, dt=torch.int32)), dict(out=mk(B, 4, D + 8)),
               dict(out=mk(B, 4, D, dt=torch.float32)),
               dict(block_table=mk(2, B, dt=torch.int32).t())):
        with pytest.raises(ValueError):
            ops.paged_attention(**{**ok, **kw})
    for kw in (dict(block_table=mk(B, 2, dt=torch.int64)), dict(seq_lens=mk(B, dt=torch.int64)),
               dict(k_cache=mk(5, hkv, 16, D, dt=torch.float32))):
        with pytest.raises(TypeError):
            ops.paged_attention(**{**ok, **kw})
    big = mk(B + 1, 4, D)
    for kw, word in ((dict(q=mk(B, 3, D)), "query heads"), (dict(window=-1), "window"),
                     (dict(scale=float("nan")), "scale"),
                     (dict(q=big[:B], out=big[1:]), "overlaps"),
                     (dict(out=mk(1, 4, D).expand(B, 4, D)), "share elements"),
                     (dict(k_cache=mk(0, hkv, 16, D), v_cache=mk(0, hkv, 16, D)), "cache")):
        with pytest.raises(hxm.HxmError, match=word):
            ops.paged_attention(**{**ok, **kw})
    for d in (12, 264):
        with pytest.raises(hxm.HxmError, match="tile-alignment"):
            ops.paged_attention(mk(B, 4, d), mk(5, hkv, 16, d), mk(5, hkv, 16, d),
                                ok["block_table"], ok["seq_lens"])
    out, lse = ops.paged_attention(mk(0, 4, D), ok["k_cache"], ok["v_cache"],
                                   mk(0, 2, dt=torch.int32), mk(0, dt=torch.int32),
                                   return_lse=True)
    assert out.shape == (0, 4, D) and lse.shape == (0, 4)
    out = ops.paged_attention(**{**ok, "block_table": mk(B, 0, dt=torch.int32)})
    assert (out == 0).all()


@pytest.mark.parametrize("lens", [[40, 70], [3000, 70]])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_infinite_and_nan_values_keep_to_their_dims(dev, name, lens):
    """An infinite or NaN value of a live token: its sequence, key head and dim are not finite,
    all else is as without it."""
    g = torch.Generator().manual_seed(11)
    q, kc, vc, table, ln, _ = build(g, name, lens, 2, 3, 64, 16, "hnd", dev)
    q = q.to(dev)
    want, wl = ops.paged_attention(q, kc, vc, table, ln, return_lse=True)
    t = lens[0] - 3
    row = vc[table[0, t // 16], 1, t % 16]
    row[5], row[9], row[40] = float("inf"), -float("inf"), float("nan")
    out, lse = ops.paged_attention(q, kc, vc, table, ln, return_lse=True)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, 3:, [5, 9, 40]] = True
    assert not out[hit].isfinite().any() and out[0, 3:, 40].isnan().all()
    assert torch.equal(out[~hit], want[~hit]) and torch.equal(lse, wl)
