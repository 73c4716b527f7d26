"""hxm_residual_norm_rows against its formulas in 64 bits.

Tolerances, from arithmetic alone.  y and z are each rounded once (half a step
of the dtype, eps / 2 relative, or half the smallest subnormal).  Before that
everything is fp32: C = 64 units of 2^-24 covers a row sum (at most 32 terms in
a chain per lane, then 12 pairwise levels) and the dozen operations around
it, relative to the size of the terms added:
  Ym = |rs x| + |bs g| (|gamma| rstd (|h| + mean|h|) + |beta|)
for y; for z, whose input carries y's error and whose rstd that of the row,
  |gamma| rstd (Ym + mean Ym) + |beta| + |z - beta| rstd rms(Ym).
"""
import numpy as np
import pytest
import torch

import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
C = 64 * 2.0 ** -24
EPS = 1e-5


def norm64(v, mag, kind, w, b, eps):
    """(norm of v, size of its terms, the rows' rstd) for v of term sizes mag."""
    if kind == "none":
        return v, mag, None
    mean = v.mean(1, keepdims=True) if kind == "layer" else 0.0
    rstd = 1 / np.sqrt(((v - mean) ** 2).mean(1, keepdims=True) + eps)
    n = (v - mean) * rstd * w
    m = np.abs(w) * rstd * (mag + (mag.mean(1, keepdims=True) if kind == "layer" else 0.0))
    m += np.abs(n) * rstd * np.sqrt((mag ** 2).mean(1, keepdims=True)) + np.abs(b)
    return n + b, m, rstd


def check(got, want, mag, name, what):
    t = torch.finfo(TDT[name])
    tol = t.eps / 2 * np.abs(want) + t.smallest_normal * t.eps / 2 + C * mag
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


def params(g, kind, cols, name, dev, bias):
    if kind == "none":
        return None, None, 1.0, 0.0
    w = (1 + 0.2 * torch.randn(cols, generator=g)).to(TDT[name])
    b = (0.2 * torch.randn(cols, generator=g)).to(TDT[name]) if bias else None
    return (w.to(dev), None if b is None else b.to(dev), w.double().numpy(),
            b.double().numpy() if bias else 0.0)


def run_case(dev, name, rows, cols, post, pre, gates, bias=True, pad=3, alias=None, seed=0):
    print(f"{name} {rows}x{cols} {post}/{pre} gates={gates} alias={alias}", flush=True)
    g = torch.Generator().manual_seed(rows * 131 + cols + seed)
    dt = TDT[name]
    h = (0.8 * torch.randn(rows, cols, generator=g) + 0.3).to(dt)
    x = (2 * torch.randn(rows, cols, generator=g) - 0.5).to(dt)
    gate = torch.randn(gates, cols, generator=g).to(dt) if gates else None
    # Rows off the 16-byte boundary, leading dimensions that are no multiple of
    # a vector, outputs inside padding that must keep its fill.
    hb, xb, yb, zb = (torch.full((rows * (cols + pad + i) + 1,), 7.0, dtype=dt, device=dev)
                      for i in range(4))
    view = lambda t, i: t[1:].view(rows, cols + pad + i)                    # noqa: E731
    hd, xd, yd, zd = (view(t, i)[:, :cols] for i, t in enumerate((hb, xb, yb, zb)))
    hd.copy_(h), xd.copy_(x)
    pw, pb, pw64, pb64 = params(g, post, cols, name, dev, bias)
    nw, nb, nw64, nb64 = params(g, pre, cols, name, dev, bias)
    if alias == "y=x":
        yd = xd
    elif alias == "y=h z=x":
        yd, zd = hd, xd
    elif alias == "z=h":
        zd = hd
    y, z = ops.residual_norm(hd, xd, post=post, post_weight=pw, post_bias=pb, post_eps=EPS,
                             pre=pre, pre_weight=nw, pre_bias=nb, pre_eps=EPS,
                             gate=None if gate is None else gate.to(dev), block_scale=1.25,
                             residual_scale=0.5, out=yd,
                             normed_out=zd if pre != "none" else None)
    assert y is yd and (z is zd if pre != "none" else z is None)
    h64, x64 = h.double().numpy(), x.double().numpy()
    p, pm, _ = norm64(h64, np.abs(h64), post, pw64, pb64, EPS)
    g64 = 1.25 * (np.repeat(gate.double().numpy(), rows // gates, 0) if gates else 1.0)
    want, mag = 0.5 * x64 + g64 * p, 0.5 * np.abs(x64) + np.abs(g64) * pm
    check(y, want, mag, name, "y")
    if pre != "none":
        want, mag, _ = norm64(want, mag, pre, nw64, nb64, EPS)
        check(z, want, mag, name, "z")
    for i, t in enumerate((hb, xb, yb, zb)):
        assert (view(t, i)[:, cols:] == 7).all() and t[0] == 7, "wrote outside the rows"


WIDTHS = (1, 7, 64, 512, 1024, 1536, 2048, 4096, 6144, 8192, 12288, 16384, 24576, 32768)


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_widths(dev, name, cols):
    """One element either side of each width where the launch changes (f32 rows
    take half of each), the streamed rows past the last."""
    cols = max(1, cols // 2) if name == "f32" else cols
    for c in sorted({max(1, cols - 1), cols, cols + 1}):
        run_case(dev, name, 3, c, "rms", "layer", 0)
        run_case(dev, name, 3, c, "layer", "rms", 3)


@pytest.mark.parametrize("pre", ["none", "rms", "layer"])
@pytest.mark.parametrize("post", ["none", "rms", "layer"])
@pytest.mark.parametrize("rows,cols,gates", [(1, 4096, 1), (6, 1000, 3), (37, 300, 37),
                                             (5, 40000, 5), (130, 64, 0), (257, 515, 1)])
def test_kinds_and_gates(dev, post, pre, rows, cols, gates):
    for name in ("f16", "bf16", "f32"):
        run_case(dev, name, rows, cols, post, pre, gates, bias=cols != 515)


@pytest.mark.parametrize("alias", ["y=x", "y=h z=x", "z=h"])
@pytest.mark.parametrize("cols", [37, 4096, 33000])
def test_in_place(dev, alias, cols):
    for name in ("f16", "f32"):
        run_case(dev, name, 9, cols, "layer", "rms", 1, alias=alias)


def test_dense_views_and_returned_shapes(dev):
    g = torch.Generator().manual_seed(4)
    h = torch.randn(2, 5, 96, generator=g).half().to(dev)
    x = torch.randn(2, 5, 96, generator=g).half().to(dev)
    y, z = ops.residual_norm(h, x, pre_eps=EPS)
    assert y.shape == z.shape == h.shape and y.dtype == z.dtype == torch.float16
    yf = x.float() + h.float()
    torch.testing.assert_close(y, yf.half(), rtol=0, atol=0)
    want = yf * torch.rsqrt(yf.square().mean(-1, keepdim=True) + EPS)
    torch.testing.assert_close(z.float(), want, rtol=2.0 ** -10, atol=1e-6)
    e = torch.empty(0, 96, dtype=torch.float16, device=dev)
    y, z = ops.residual_norm(e, e)
    assert y.shape == z.shape == (0, 96)


def test_z_is_the_norm_of_the_unrounded_y(dev):
    """x = 1 and h far below half a step of 1: y rounds to 1 everywhere, but the
    LayerNorm of the exact sum is that of h."""
    h = torch.where(torch.arange(256) % 2 == 0, 2.0 ** -16, -2.0 ** -16).half().to(dev)[None]
    x = torch.ones(1, 256, dtype=torch.float16, device=dev)
    y, z = ops.residual_norm(h, x, pre="layer", pre_eps=0.0)
    assert (y == 1).all()
    torch.testing.assert_close(z.float(), torch.sign(h.float()), rtol=1e-2, atol=0)


@pytest.mark.parametrize("cols", [500, 4096, 40000])
def test_rows_keep_to_themselves(dev, cols):
    """A row of zeros, a constant row, rows with a NaN or an infinity: only
    those rows are touched by them."""
    g = torch.Generator().manual_seed(cols)
    h = torch.randn(6, cols, generator=g).to(dev)
    x = torch.randn(6, cols, generator=g).to(dev)
    kw = dict(post="layer", pre="layer", post_eps=EPS, pre_eps=EPS)
    y0, z0 = ops.residual_norm(h, x, **kw)
    h[1], x[1] = 0, 0
    h[2] = 3.0
    h[3, cols // 2], x[4, cols - 1] = float("nan"), float("inf")
    y, z = ops.residual_norm(h, x, **kw)
    assert (y[1] == 0).all() and (z[1] == 0).all()
    assert torch.equal(y[2], x[2])                       # a constant block adds nothing
    assert y[3].isnan().all() and z[3].isnan().all() and z[4].isnan().all()
    for r in (0, 5):
        assert torch.equal(y[r], y0[r]) and torch.equal(z[r], z0[r])


def test_a_stream_of_its_own_and_a_graph(dev):
    g = torch.Generator().manual_seed(9)
    h, x = (torch.randn(33, 4096, generator=g).half().to(dev) for _ in range(2))
    w = torch.randn(4096, generator=g).half().to(dev)
    y, z = torch.empty_like(h), torch.empty_like(h)
    call = lambda: ops.residual_norm(h, x, post="rms", post_weight=w, pre_weight=w,  # noqa: E731
                                     out=y, normed_out=z)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        call()
        with torch.cuda.graph(graph, stream=s):
            call()
    torch.cuda.synchronize()
    for k in range(3):
        h.copy_(torch.randn(33, 4096, generator=g).half())
        ye, ze = ops.residual_norm(h, x, post="rms", post_weight=w, pre_weight=w)
        y.fill_(9), z.fill_(9)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ye) and torch.equal(z, ze), k


def test_refusals(dev):
    h = torch.zeros(6, 32, dtype=torch.float16, device=dev)
    x = torch.zeros_like(h)
    for kw in (dict(x=x[:5]), dict(x=x.float()), dict(x=x.cpu()), dict(post="batch"),
               dict(pre="none", normed_out=x), dict(gate=torch.zeros(4, 32).half().to(dev)),
               dict(gate=torch.zeros(31).half().to(dev)), dict(gate=torch.zeros(32, device=dev)),
               dict(pre_weight=torch.zeros(31).half().to(dev)), dict(out=x[:, :16]),
               dict(out=torch.zeros(32, 6).half().to(dev).t()),
               dict(normed_out=torch.zeros(6, 32, device=dev))):
        with pytest.raises(ValueError):
            ops.residual_norm(**{"h": h, "x": x, **kw})
    with pytest.raises(TypeError):
        ops.residual_norm(h.int(), x.int())
    for kw in (dict(pre_eps=-1.0), dict(post_eps=float("nan"), post="rms"),
               dict(post="none", post_weight=torch.ones(32).half().to(dev)),
               dict(out=h, normed_out=h)):
        with pytest.raises(ops.HxmError, match="invalid-argument"):
            ops.residual_norm(h, x, **kw)
    buf = torch.zeros(8, 32, dtype=torch.float16, device=dev)
    with pytest.raises(ops.HxmError, match="overlaps"):   # the rows of x, one further down
        ops.residual_norm(h, buf[:6], out=buf[1:7])
    wide = torch.zeros(6, 64, dtype=torch.float16, device=dev)
    y, z = ops.residual_norm(h, wide[:, :32], out=wide[:, 32:])      # other columns: disjoint
    assert y.data_ptr() == wide.data_ptr() + 64


@pytest.mark.parametrize("cols,rows", [(300, 1028), (1000, 1028), (1536, 1028), (2043, 1028),
                                       (4096, 260), (6100, 260), (8192, 260), (12000, 260),
                                       (16384, 260)])
@pytest.mark.parametrize("name", ["f16", "bf16", "f32"])
def test_more_than_a_workgroup_a_cu(dev, name, cols, rows):
    """Past 256 workgroups parameters are loaded where they are used: every width that takes
    a row in registers of 1, 4 or 8 waves, at the last row count before the change and past it."""
    cols = max(1, cols // 2) if name == "f32" else cols
    run_case(dev, name, rows, cols, "rms", "layer", 4)
    run_case(dev, name, rows, cols, "layer", "rms", 1, alias="y=x")
    run_case(dev, name, rows - 4, cols, "none", "rms", rows - 4, bias=False, alias="y=h z=x")
    run_case(dev, name, rows - 3, cols, "layer", "none", 0)


def test_permuted_rows(dev):
    """Sequences first or tokens first: rows of a permuted tensor, new outputs."""
    import torch.nn.functional as F

    g = torch.Generator().manual_seed(12)
    h, x = (torch.randn(7, 5, 96, generator=g).half().to(dev).transpose(0, 1) for _ in range(2))
    for a, b in zip(ops.residual_norm(h, x, post="rms", pre_eps=EPS),
                    ops.residual_norm(h.contiguous(), x.contiguous(), post="rms", pre_eps=EPS)):
        assert a.shape == h.shape and torch.equal(a, b)
    assert torch.equal(ops.softmax(h), ops.softmax(h.contiguous()))
    assert torch.equal(ops.rms_norm(h, (96,)), ops.rms_norm(h.contiguous(), (96,)))
    torch.testing.assert_close(ops.layer_norm(h, (96,)).float(), F.layer_norm(h.float(), (96,)),
                               rtol=1e-2, atol=2e-3)
