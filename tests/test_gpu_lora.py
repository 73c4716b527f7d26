"""hxm_lora_add against y + scale (x A^T) B^T in 64 bits.

Tolerances, from arithmetic alone: out is rounded once (eps / 2 of |out|, or half
the smallest subnormal).  With Tm = |x| |A|^T, t's fp32 sum is off by at most
(K + 16) 2^-24 Tm (K terms in any order); as two 16-bit halves of a scaled row
it is off by 2^-21 (f16) or 2^-15 (bf16) of the row's largest |t|, h below; the
second product's sums over 2 R terms and its epilogue add (2 R + 16) 2^-24.  So
  scale (((K + 2 R + 32) 2^-24 Tm + h max|t|) |B|^T) + 2^-23 |y|."""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16}
HALVES = {"f16": 2.0 ** -21, "bf16": 2.0 ** -15}


def run_case(dev, name, M, N, K, R, index, L, scaled=True, inplace=False, pad=3, seed=0):
    print(f"{name} M={M} N={N} K={K} R={R} adapters={L} in place={inplace}", flush=True)
    g = torch.Generator().manual_seed(seed + M + N + K + R)
    dt = TDT[name]
    x = torch.randn(M, K, generator=g).to(dt)
    y = torch.randn(M, N, generator=g).to(dt)
    A = (torch.randn(L, R, K, generator=g) / K ** 0.5).to(dt)
    B = (torch.randn(L, N, R, generator=g) / R ** 0.5).to(dt)
    sc = torch.rand(L, generator=g) * 2 - 0.5 if scaled else None
    index = torch.as_tensor(index, dtype=torch.int32)
    # Rows off the 16-byte boundary inside padding that must keep its fill.
    xb, yb, ob = (torch.full((M * (w + pad) + 1,), 7.0, dtype=dt, device=dev) for w in (K, N, N))
    xd, yd, od = (t[1:].view(M, w + pad)[:, :w] for t, w in ((xb, K), (yb, N), (ob, N)))
    xd.copy_(x), yd.copy_(y)
    out = ops.lora_add(yd, xd, A.to(dev), B.to(dev), index.to(dev),
                       None if sc is None else sc.to(dev), out=yd if inplace else od)
    assert out is (yd if inplace else od)
    got = out.double().cpu().numpy()
    t = torch.finfo(dt)
    x64, y64 = x.double().numpy(), y.double().numpy()
    for m, a in enumerate(index.tolist()):
        if a < 0:
            assert torch.equal(out[m].cpu(), y[m]), m
            continue
        if a >= L:
            assert out[m].isnan().all(), m
            continue
        A64, B64 = A[a].double().numpy(), B[a].double().numpy()
        s = 1.0 if sc is None else float(sc[a])
        tt, tm = A64 @ x64[m], np.abs(A64) @ np.abs(x64[m])
        want = y64[m] + s * (B64 @ tt)
        e = (K + 2 * R + 32) * 2.0 ** -24 * tm + HALVES[name] * np.abs(tt).max()
        tol = (t.eps / 2 * np.abs(want) + t.smallest_normal * t.eps / 2
               + abs(s) * (np.abs(B64) @ e) + 2.0 ** -23 * np.abs(y64[m]))
        bad = ~(np.abs(got[m] - want) <= tol)
        assert not bad.any(), (m, a, np.argwhere(bad)[:4].tolist(), got[m][bad][:4], want[bad][:4])
    for buf, w in ((xb, K), (yb, N), (ob, N)):
        assert (buf[1:].view(M, w + pad)[:, w:] == 7).all() and buf[0] == 7, "wrote past a row"


def mixed(M, L, seed=0, none=0.2, run=1):
    r = np.random.default_rng(seed)
    out = []
    while len(out) < M:
        out += [-1 if r.random() < none else int(r.integers(L))] * run
    return out[:M]


@pytest.mark.parametrize("R", [8, 16, 24, 32, 40, 64, 72, 128, 136, 256])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_ranks(dev, name, R):
    run_case(dev, name, 21, 300, 264, R, mixed(21, 5), 5)
    run_case(dev, name, 40, 129, 1032, R, mixed(40, 3, run=7), 3, inplace=True)


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 48, 100, 515])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_rows(dev, name, M):
    run_case(dev, name, M, 512, 512, 16, mixed(M, 20), 20)
    run_case(dev, name, M, 200, 4096, 16, mixed(M, 2, run=30, none=0.0), 2, scaled=False)


@pytest.mark.parametrize("N,K", [(1, 8), (7, 16), (8, 40), (31, 64), (33, 128), (128, 136),
                                 (1000, 520), (5003, 1024)])
def test_odd_sizes(dev, N, K):
    for name in ("f16", "bf16"):
        run_case(dev, name, 19, N, K, 8, mixed(19, 4), 4)
        run_case(dev, name, 33, N, K, 32, mixed(33, 4), 4, inplace=True)


def test_many_rows(dev):
    run_case(dev, "bf16", 3001, 96, 256, 64, mixed(3001, 6, run=113), 6)
    run_case(dev, "f16", 2048, 128, 512, 16, mixed(2048, 6), 6)


@pytest.mark.parametrize("R", [8, 16, 24, 32, 40, 64, 72, 128, 136, 200, 256])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_ranks_of_many_rows(dev, name, R):
    """Tiles of 64 rows with one adapter, several, and none; K that ends inside a step of 256,
    columns that end inside a block."""
    run_case(dev, name, 300, 173, 520, R, mixed(300, 5, run=40), 5)
    run_case(dev, name, 257, 264, 264, R, mixed(257, 9), 9, inplace=True)


@pytest.mark.parametrize("M", [255, 256, 257, 320, 700])
@pytest.mark.parametrize("N,K", [(1, 8), (31, 256), (129, 248), (136, 264), (1000, 2056)])
def test_odd_sizes_of_many_rows(dev, M, N, K):
    run_case(dev, "f16", M, N, K, 16, mixed(M, 30), 30)
    run_case(dev, "bf16", M, N, K, 48, mixed(M, 2, run=90), 2, inplace=True, scaled=False)


def test_bad_indexes_and_sick_weights_of_many_rows(dev):
    run_case(dev, "f16", 260, 70, 64, 16, [-5, 3, 0, 2 ** 31 - 1, -2 ** 31] * 52, 3)
    run_case(dev, "bf16", 320, 70, 64, 16, [-1] * 130 + [2] * 60 + [-1] * 130, 3, inplace=True)
    g = torch.Generator().manual_seed(7)
    M, N, K, R, L = 400, 160, 512, 16, 6
    x, y = (torch.randn(M, w, generator=g).half().to(dev) for w in (K, N))
    A, B = (torch.randn(L, a, b, generator=g).half().to(dev) * 0.1 for a, b in ((R, K), (N, R)))
    index = torch.tensor(mixed(M, L, none=0.1), dtype=torch.int32, device=dev)
    want = ops.lora_add(y, x, A, B, index)
    A[2], B[4, 3] = float("nan"), float("inf")
    sick = int((index == 0).nonzero()[0])
    x[sick] = float("nan")
    out = ops.lora_add(y, x, A, B, index)
    for m, a in enumerate(index.tolist()):
        if a == 2 or m == sick:
            assert out[m].isnan().all(), m
        elif a == 4:
            assert not out[m, 3].isfinite() and torch.equal(out[m, 4:], want[m, 4:]), m
        else:
            assert torch.equal(out[m], want[m]), m


def test_rows_beyond_one_set_of_launches(dev):
    """65536 rows of rank 256 fill one set's planes: the next set starts at row 65536, and takes
    the form for few rows where 100 are left."""
    R, K, N, L = 256, 16, 24, 3
    for M in (65536 + 100, 65536 + 300):
        g = torch.Generator().manual_seed(M)
        x, y = (torch.randn(M, w, generator=g).half().to(dev) for w in (K, N))
        A, B = (torch.randn(L, a, b, generator=g).half().to(dev) / 16 for a, b in ((R, K), (N, R)))
        index = (torch.arange(M, device=dev) // 1000 % (L + 1) - 1).int()
        out = ops.lora_add(y, x, A, B, index)
        for a in range(-1, L):
            rows = index == a
            want = y[rows].double()
            err = torch.zeros_like(want)
            if a >= 0:
                t = x[rows].double() @ A[a].double().t()
                tm = x[rows].double().abs() @ A[a].double().abs().t()
                want = want + t @ B[a].double().t()
                e = (K + 2 * R + 32) * 2.0 ** -24 * tm + HALVES["f16"] * t.abs().amax(1, True)
                err = e @ B[a].double().abs().t() + 2.0 ** -23 * y[rows].double().abs()
            tol = 2.0 ** -11 * (want.abs() + err) + 2.0 ** -25 + err
            assert ((out[rows].double() - want).abs() <= (tol if a >= 0 else 0)).all(), (M, a)


def test_many_rows_captured_after_other_sizes(dev):
    """One stream's workspace under calls of changing sizes, then a captured one."""
    g = torch.Generator().manual_seed(8)
    L, R, K, N = 4, 64, 1024, 640
    A, B = (torch.randn(L, a, b, generator=g).bfloat16().to(dev) * 0.1
            for a, b in ((R, K), (N, R)))
    x, y = (torch.randn(600, w, generator=g).bfloat16().to(dev) for w in (K, N))
    index = torch.tensor(mixed(600, L, run=50), dtype=torch.int32, device=dev)
    s, graph, out = torch.cuda.Stream(), torch.cuda.CUDAGraph(), torch.empty_like(y)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        want = ops.lora_add(y, x, A, B, index)
        for m in (1, 300, 600, 17, 256):
            part = ops.lora_add(y[:m], x[:m], A, B, index[:m])
            if m >= 256:
                assert torch.equal(part[:192], want[:192])
    with torch.cuda.graph(graph, stream=s):
        ops.lora_add(y, x, A, B, index, out=out)
    for k in range(3):
        x.normal_()
        index.copy_(torch.tensor(mixed(600, L, seed=k, run=70), dtype=torch.int32))
        want = ops.lora_add(y, x, A, B, index)
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), k


def test_no_adapters_and_bad_indexes(dev):
    run_case(dev, "f16", 20, 100, 64, 16, [-1] * 20, 3)
    run_case(dev, "f16", 20, 100, 64, 16, [-5, 3, 0, 2 ** 31 - 1, -2 ** 31] * 4, 3)
    run_case(dev, "bf16", 20, 100, 64, 16, [-1] * 20, 3, inplace=True)
    y = torch.randn(4, 32).half().to(dev)
    x = torch.randn(4, 64).half().to(dev)
    none = torch.tensor([-1, 0, -1, 5], dtype=torch.int32, device=dev)
    out = ops.lora_add(y, x, x.new_empty(0, 16, 64), x.new_empty(0, 32, 16), none)
    assert torch.equal(out[::2], y[::2]) and out[1::2].isnan().all()


def test_other_rows_and_adapters_do_not_reach_a_row(dev):
    """NaN and infinities in one adapter's weights and in one row of x stay with
    the rows that use them, in any tile."""
    g = torch.Generator().manual_seed(4)
    M, N, K, R, L = 48, 160, 256, 16, 6
    x, y = (torch.randn(M, w, generator=g).half().to(dev) for w in (K, N))
    A, B = (torch.randn(L, a, b, generator=g).half().to(dev) * 0.1 for a, b in ((R, K), (N, R)))
    index = torch.tensor(mixed(M, L, none=0.1), dtype=torch.int32, device=dev)
    want = ops.lora_add(y, x, A, B, index)
    A[2], B[4, 3] = float("nan"), float("inf")
    sick = int((index == 0).nonzero()[0])
    x[sick] = float("nan")
    out = ops.lora_add(y, x, A, B, index)
    for m, a in enumerate(index.tolist()):
        if a == 2 or m == sick:
            assert out[m].isnan().all(), m
        elif a == 4:
            assert not out[m, 3].isfinite() and torch.equal(out[m, 4:], want[m, 4:]), m
        else:
            assert torch.equal(out[m], want[m]), m


def test_large_and_small_t(dev):
    """x A^T beyond the f16 range, and far below its smallest number, with B
    bringing the product back."""
    for big in (2.0 ** 9, 2.0 ** -13):
        x = torch.full((3, 512), big).half()
        A = torch.full((1, 16, 512), big).half()      # t = 512 big^2 = 2^27 or 2^-17
        B = torch.full((1, 40, 16), 2.0 ** -12 if big > 1 else 2.0 ** 12).half()
        y = torch.ones(3, 40).half()
        sc = torch.tensor([2.0 ** -17 if big > 1 else 2.0])
        out = ops.lora_add(y.to(dev), x.to(dev), A.to(dev), B.to(dev),
                           torch.tensor([0, -1, 0], dtype=torch.int32, device=dev), sc.to(dev))
        t = 512.0 * big * big
        want = 1 + float(sc) * t * 16 * float(B[0, 0, 0])
        assert (out[0] == torch.tensor(want).half().to(dev)).all() and (out[1] == 1).all()
        assert torch.equal(out[0], out[2])


def test_captured_and_on_two_streams(dev):
    g = torch.Generator().manual_seed(5)
    x, y = (torch.randn(50, w, generator=g).half().to(dev) for w in (2048, 512))
    A, B = (torch.randn(4, a, b, generator=g).half().to(dev) * 0.1
            for a, b in ((16, 2048), (512, 16)))
    index = torch.tensor(mixed(50, 4), dtype=torch.int32, device=dev)
    want = ops.lora_add(y, x, A, B, index)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.lora_add(y, x, A, B, index))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    out = torch.empty_like(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        ops.lora_add(y, x, A, B, index, out=out)
    for k in range(3):
        x.normal_()
        index.copy_(torch.tensor(mixed(50, 4, seed=k + 9), dtype=torch.int32))
        want = ops.lora_add(y, x, A, B, index)
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), k


def test_refusals(dev):
    mk = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)      # noqa: E731
    ok = dict(y=mk(4, 48), x=mk(4, 64), A=mk(2, 16, 64), B=mk(2, 48, 16),
              index=mk(4, dt=torch.int32), scale=mk(2, dt=torch.float32))
    ops.lora_add(**ok)
    for kw in (dict(x=mk(5, 64)), dict(x=mk(4, 64, dt=torch.bfloat16)), dict(A=mk(2, 16, 72)),
               dict(A=mk(2, 64, 16).transpose(1, 2)), dict(B=mk(2, 48, 8)), dict(B=mk(3, 48, 16)),
               dict(index=mk(5, dt=torch.int32)), dict(scale=mk(3, dt=torch.float32)),
               dict(scale=mk(2)), dict(out=mk(4, 40)), dict(y=mk(4, 48).cpu()),
               dict(y=mk(48, 4).t())):
        with pytest.raises(ValueError):
            ops.lora_add(**{**ok, **kw})
    for kw in (dict(index=mk(4, dt=torch.int64)), dict(y=mk(4, 48, dt=torch.float32)),
               dict(out=mk(4, 48, dt=torch.float32))):
        with pytest.raises(TypeError):
            ops.lora_add(**{**ok, **kw})
    for r in (4, 12, 264):
        with pytest.raises(hxm.HxmError, match="tile-alignment"):
            ops.lora_add(**{**ok, "A": mk(2, r, 64), "B": mk(2, 48, r)})
    with pytest.raises(hxm.HxmError, match="tile-alignment"):
        ops.lora_add(**{**ok, "x": mk(4, 60), "A": mk(2, 16, 60)})
    big = mk(5, 64)
    with pytest.raises(hxm.HxmError, match="overlaps"):
        ops.lora_add(**{**ok, "y": big[:4, :48], "out": big[1:, :48]})
    with pytest.raises(hxm.HxmError, match="overlaps"):
        ops.lora_add(**{**ok, "x": big[:4], "out": big[:4, :48]})
    assert ops.lora_add(mk(0, 48), mk(0, 64), ok["A"], ok["B"], ok["index"][:0]).shape == (0, 48)


# What a rank is off by as two halves of a row scaled to [2^14, 2^15): two roundings of the
# dtype, and in f16 half of the smallest subnormal, 2^-25, at least 2^14 below the largest.
SPLIT = {"f16": (2.0 ** -21, 2.0 ** -39), "bf16": (2.0 ** -15, 0.0)}


@pytest.mark.parametrize("M", [5, 300])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_ranks_far_apart(dev, name, M):
    """t falls by 2^20 from a row's first rank to its last while B grows by as much, so that
    every rank adds about the same to the output: each keeps its own precision."""
    R, N, L = 16, 200, 2
    K = 8 * R
    g = torch.Generator().manual_seed(M)
    dt, t = TDT[name], torch.finfo(TDT[name])
    e = 20.0 * torch.arange(R) / (R - 1)
    x = (torch.randn(M, R, 8, generator=g) * 2.0 ** (-e / 2)[:, None]).reshape(M, K).to(dt)
    A = torch.zeros(L, R, R, 8)                       # rank r reads its own eight columns
    A[:, range(R), range(R)] = torch.randn(L, R, 8, generator=g) * 2.0 ** (-e / 2)[:, None]
    A = A.view(L, R, K).to(dt)
    B = (torch.randn(L, N, R, generator=g) * 2.0 ** (e - 10)).to(dt)
    index = torch.arange(M, dtype=torch.int32) % L
    out = ops.lora_add(torch.zeros(M, N, dtype=dt, device=dev), x.to(dev), A.to(dev), B.to(dev),
                       index.to(dev)).double().cpu().numpy()
    half, floor = SPLIT[name]
    for m, a in enumerate(index.tolist()):
        A64, B64, x64 = (v.double().numpy() for v in (A[a], B[a], x[m]))
        tt, tm = A64 @ x64, np.abs(A64) @ np.abs(x64)
        want = B64 @ tt
        err = (K + 2 * R + 32) * 2.0 ** -24 * tm + half * np.abs(tt) + floor * np.abs(tt).max()
        tol = t.eps / 2 * np.abs(want) + t.smallest_normal * t.eps / 2 + np.abs(B64) @ err
        bad = ~(np.abs(out[m] - want) <= tol)
        assert not bad.any(), (m, np.argwhere(bad)[:4].tolist(), out[m][bad][:4], want[bad][:4])
