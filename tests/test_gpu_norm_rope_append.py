"""hxm_norm_rope_append against the norm and the rotation of each head in 64 bits.

Tolerances, from arithmetic alone, with u = eps / 2 of the dtype, r the norm's factor and
M_j = r (|x_j| + mean|x|) |gamma_j| + |beta_j| (mean|x| for LayerNorm's subtraction):
one rounding of the result, u |y|; the fp32 sums of dim terms, the factor, the products
and the rotation move it by (dim + 32) 2^-24 of M_j |cos| + M_i |sin| at most.  Values are
stored as they are."""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16}


def table(far, rot):
    half = rot // 2
    ang = torch.arange(far, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, dtype=torch.float64) / max(half, 1))
    return torch.cat((ang.cos(), ang.sin()), 1).float()


def want(x, kind, w, b, eps, pos, cs, rot, pairs):
    """(y, the bound's magnitude) in 64 bits of x [T, H, D]."""
    x = x.double()
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    c = x - mean
    r = 1 / (c.square().mean(-1, keepdim=True) + eps).sqrt() if kind != "none" else 1.0
    w = torch.ones(x.shape[-1]).double() if w is None else w.double()
    b = torch.zeros(x.shape[-1]).double() if b is None else b.double()
    y = c * r * w + b
    M = (x.abs() + (x.abs().mean(-1, keepdim=True) if kind == "layer" else 0)) * r * w.abs() + b.abs()
    half = rot // 2
    i = torch.arange(half)
    i, j = (2 * i, 2 * i + 1) if pairs else (i, i + half)
    cos, sin = (t[:, None] for t in cs.double()[pos.long()].split((half, half), 1))
    out, mag = y.clone(), M.clone()
    out[..., i] = y[..., i] * cos - y[..., j] * sin
    out[..., j] = y[..., j] * cos + y[..., i] * sin
    mag[..., i] = M[..., i] * cos.abs() + M[..., j] * sin.abs()
    mag[..., j] = M[..., j] * cos.abs() + M[..., i] * sin.abs()
    return out, mag


def close(got, y, mag, name, dim):
    dt = TDT[name]
    tiny = torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2
    tol = torch.finfo(dt).eps / 2 * y.abs() + (dim + 32) * 2.0 ** -24 * mag + tiny
    bad = ~((got.double() - y).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), got[bad][:4], y[bad][:4])


def run_case(dev, name, T, hq, hkv, dim, rot, pairs, page, layout, norm="rms", each=False,
             bias=False, weight=True, pad=0, inplace=False, with_q=True, shift=0.0):
    print(f"{name} T={T} heads={hq}+{hkv} dim={dim} rot={rot} pairs={pairs} page={page} {layout} "
          f"{norm} each={each} bias={bias}", flush=True)
    g = torch.Generator().manual_seed(T + dim + rot)
    dt = TDT[name]
    qkv = (torch.randn(T, hq + 2 * hkv, dim, generator=g) * 2 + shift).to(dt)
    q, k, v = qkv.to(dev).split((hq, hkv, hkv), 1)
    par = {}
    for n, h in (("q", hq), ("k", hkv)):
        shape = (h, dim) if each else (dim,)
        par[n + "_weight"] = (1 + 0.3 * torch.randn(shape, generator=g)).to(dt) if weight else None
        par[n + "_bias"] = torch.randn(shape, generator=g).to(dt) if bias else None
    pages = T // page + 3
    order = (0, 1, 2, 3) if layout == "hnd" else (0, 2, 1, 3)
    mk = lambda: torch.full([(pages, hkv, page, dim)[i] for i in order], 7.0, dtype=dt,  # noqa: E731
                            device=dev).permute(*order)
    kc, vc = mk(), mk()
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    slots[T - pad:] = -1
    pos = torch.randint(0, 500, (T,), generator=g).int()
    cs = table(500, rot)
    out = ops.norm_rope_append(
        q if with_q else None, k, v, kc, vc, slots.to(dev), pos.to(dev) if rot else None,
        cs.to(dev) if rot else None, norm=norm, eps=1e-5, interleaved=pairs,
        q_out=q if inplace and with_q else None,
        **{n: None if t is None or (not with_q and n[0] == "q") else t.to(dev)
           for n, t in par.items()})
    if with_q:
        y, mag = want(qkv[:, :hq], norm, par["q_weight"], par["q_bias"], 1e-5, pos, cs, rot, pairs)
        close(out.cpu(), y, mag, name, dim)
        assert (out.data_ptr() == q.data_ptr()) == inplace
    else:
        assert out is None
    y, mag = want(qkv[:, hq:hq + hkv], norm, par["k_weight"], par["k_bias"], 1e-5, pos, cs, rot,
                  pairs)
    live = slots >= 0
    at = slots[live].long()
    rows = kc.cpu().transpose(1, 2).reshape(pages * page, hkv, dim)
    close(rows[at], y[live], mag[live], name, dim)
    vrows = vc.cpu().transpose(1, 2).reshape(pages * page, hkv, dim)
    assert torch.equal(vrows[at], qkv[live, hq + hkv:])
    rest = torch.ones(pages * page, dtype=torch.bool)
    rest[at] = False
    assert (rows[rest] == 7).all() and (vrows[rest] == 7).all()


@pytest.mark.parametrize("dim,rot", [(8, 8), (8, 2), (64, 64), (80, 40), (80, 80), (96, 48),
                                     (120, 90), (128, 128), (128, 0), (256, 256), (256, 2),
                                     (200, 34), (256, 250), (72, 72)])
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_dims(dev, name, pairs, dim, rot):
    run_case(dev, name, 37, 5, 2, dim, rot, pairs, 16, "nhd", pad=3)
    run_case(dev, name, 5, 3, 3, dim, rot, pairs, 7, "hnd", norm="layer", bias=True, each=True)


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
@pytest.mark.parametrize("T,hq,hkv,page", [(1, 32, 8, 16), (2, 1, 1, 1), (64, 32, 8, 16),
                                           (333, 28, 4, 24), (2051, 16, 2, 64), (17, 96, 96, 3)])
def test_sizes(dev, T, hq, hkv, page, layout):
    run_case(dev, "f16", T, hq, hkv, 128, 128, False, page, layout, pad=min(4, T // 3))
    run_case(dev, "bf16", T, hq, hkv, 64, 32, True, page, layout, norm="layer", bias=True,
             inplace=True)


@pytest.mark.parametrize("norm", ["none", "rms", "layer"])
def test_norms(dev, norm):
    run_case(dev, "f16", 33, 4, 2, 96, 96, False, 16, "hnd", norm=norm, weight=False)
    run_case(dev, "bf16", 33, 4, 2, 96, 96, False, 16, "hnd", norm=norm, with_q=False,
             weight=norm != "none")
    if norm != "none":
        run_case(dev, "f16", 33, 4, 2, 128, 64, False, 16, "hnd", norm=norm, weight=False, bias=True)
        run_case(dev, "f16", 33, 4, 2, 128, 64, False, 16, "hnd", norm=norm, each=True, shift=30.0)


def test_one_norm_without_the_other(dev):
    """The norms of q and k are apart in the C entry: without either it is hxm_rope_append."""
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.randn(6, h, 64, generator=g).half().to(dev) for h in (4, 2, 2))
    slots = torch.arange(6, dtype=torch.int32, device=dev)
    pos, cs = slots * 7, table(64, 64).to(dev)
    a, b = (torch.zeros(2, 2, 2, 8, 64, dtype=torch.float16, device=dev) for _ in range(2))
    x = ops.rope_append(q, k, v, a[0], a[1], slots, pos, cs)
    y = ops.norm_rope_append(q, k, v, b[0], b[1], slots, pos, cs, norm="none")
    assert torch.equal(x, y) and torch.equal(a, b)


def test_zero_rows_and_values_that_are_no_numbers(dev):
    """A head of zeros stays zeros (eps), one with a NaN or an infinite element is NaN, and
    its neighbours are untouched."""
    T, D = 4, 128
    q = torch.randn(T, 4, D).half()
    q[1, 2] = 0
    q[2, 1, 5] = float("nan")
    q[3, 0, 9] = float("inf")
    k, v = torch.randn(T, 2, D).half().to(dev), torch.randn(T, 2, D).half().to(dev)
    kc, vc = (torch.zeros(1, 2, 16, D, dtype=torch.float16, device=dev) for _ in range(2))
    out = ops.norm_rope_append(q.to(dev), k, v, kc, vc,
                               torch.arange(T, dtype=torch.int32, device=dev)).cpu()
    assert (out[1, 2] == 0).all() and out[2, 1].isnan().all()
    fine = torch.ones(T, 4, dtype=torch.bool)
    fine[2, 1] = fine[3, 0] = False
    assert out[fine].isfinite().all()


def test_positions_outside_the_table(dev):
    T, rot = 5, 32
    q, k, v = (torch.randn(T, 2, 64).half().to(dev) for _ in range(3))
    kc, vc = (torch.zeros(2, 2, 8, 64, dtype=torch.float16, device=dev) for _ in range(2))
    pos = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    out = ops.norm_rope_append(q, k, v, kc, vc, slots, pos, table(10, rot).to(dev))
    for t, good in enumerate((True, False, True, False, False)):
        for x in (out[t], kc[0, :, t]):
            assert x[:, :rot].isnan().all() != good and not x[:, rot:].isnan().any()
    assert torch.equal(vc[0, :, :T].transpose(0, 1), v)


def test_captured_on_another_stream(dev):
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(9, h, 128, generator=g).half().to(dev) for h in (8, 2, 2))
    w = torch.randn(128, generator=g).half().to(dev)
    kc, vc = (torch.zeros(3, 2, 16, 128, dtype=torch.float16, device=dev) for _ in range(2))
    slots = torch.arange(9, dtype=torch.int32, device=dev)
    pos, cs, out = slots.clone(), table(64, 128).to(dev), torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.norm_rope_append(q, k, v, kc, vc, slots, pos, cs, q_weight=w, k_weight=w, q_out=out)
    for r in range(3):
        pos.add_(3)
        slots.copy_(torch.randperm(48, generator=g)[:9].int())
        kc.fill_(0), vc.fill_(0), out.fill_(0)
        graph.replay()
        ke, ve = torch.zeros_like(kc), torch.zeros_like(vc)
        ref = ops.norm_rope_append(q, k, v, ke, ve, slots, pos, cs, q_weight=w, k_weight=w)
        torch.cuda.synchronize()
        assert torch.equal(out, ref) and torch.equal(kc, ke) and torch.equal(vc, ve), r


def test_wrong_arguments_are_refused(dev):
    T, hq, hkv, D = 4, 4, 2, 64
    mk = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)      # noqa: E731
    ok = dict(q=mk(T, hq, D), k=mk(T, hkv, D), v=mk(T, hkv, D), k_cache=mk(2, hkv, 16, D),
              v_cache=mk(2, hkv, 16, D), slots=torch.arange(T, dtype=torch.int32, device=dev),
              positions=mk(T, dt=torch.int32), cos_sin=mk(8, D, dt=torch.float32),
              q_weight=mk(D), k_weight=mk(hkv, D), k_bias=mk(hkv, D))
    ops.norm_rope_append(**ok)
    for kw in (dict(q_weight=mk(D - 8)), dict(q_weight=mk(D).float()), dict(q_weight=mk(D).cpu()),
               dict(q_weight=mk(hkv, D)), dict(k_weight=mk(D)), dict(k_bias=mk(D)),
               dict(norm="l2"), dict(q=None, q_out=mk(T, hq, D)), dict(k=mk(T, hkv, D - 8))):
        with pytest.raises(ValueError):
            ops.norm_rope_append(**{**ok, **kw})
    for kw in (dict(eps=-1.0), dict(eps=float("nan")), dict(norm="none"),
               dict(cos_sin=mk(8, D + 8, dt=torch.float32))):
        with pytest.raises(hxm.HxmError):
            ops.norm_rope_append(**{**ok, **kw})
