"""hxm_rope_append against its formulas in 64 bits.

A rotated element is a cos - b sin in fp32, three roundings at 2^-24 of the two
terms' size at most, then one to the dtype (half a step: eps / 2 relative, half
the smallest subnormal below).  Everything that is not rotated is equal, and so
is every cache row that no slot names."""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops

pytestmark = pytest.mark.gpu

TDT = {"f16": torch.float16, "bf16": torch.bfloat16}


def table(max_pos, rot):
    inv = 10000.0 ** (-np.arange(rot // 2) / max(1, rot // 2))
    ang = np.arange(max_pos)[:, None] * inv
    return torch.from_numpy(np.concatenate((np.cos(ang), np.sin(ang)), 1)).float()


def rotate64(x, cs, rot, interleaved):
    """(rotated x, size of its terms) for x [T, H, D], cs [T, rot]."""
    x = x.double().numpy()
    y, mag = x.copy(), np.zeros_like(x)
    half = rot // 2
    i = 2 * np.arange(half) if interleaved else np.arange(half)
    j = i + 1 if interleaved else i + half
    c, s = (cs[:, None, :half].double().numpy(), cs[:, None, half:].double().numpy())
    y[..., i] = x[..., i] * c - x[..., j] * s
    y[..., j] = x[..., j] * c + x[..., i] * s
    mag[..., i] = np.abs(x[..., i] * c) + np.abs(x[..., j] * s)
    mag[..., j] = np.abs(x[..., j] * c) + np.abs(x[..., i] * s)
    return y, mag


def close(got, want, mag, name):
    t = torch.finfo(TDT[name])
    tol = t.eps / 2 * np.abs(want) + t.smallest_normal * t.eps / 2 + 3 * 2.0 ** -24 * mag
    tol[mag == 0] = 0
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


def make_cache(pages, heads, page, dim, layout, dt, dev):
    shape = (pages, heads, page, dim) if layout == "hnd" else (pages, page, heads, dim)
    both = torch.full((2,) + shape, 5.0, dtype=dt, device=dev)
    if layout == "interleaved":                    # keys and values of a page side by side
        both = torch.full((pages, 2, page, heads, dim), 5.0, dtype=dt, device=dev).transpose(0, 1)
    k, v = both[0], both[1]
    return (k, v) if layout == "hnd" else (k.transpose(1, 2), v.transpose(1, 2))


def run_case(dev, name, T, hq, hkv, dim, rot, interleaved, page, layout, pad=0, inplace=False,
             with_q=True):
    print(f"{name} T={T} {hq}/{hkv}x{dim} rot={rot} pairs={interleaved} page={page} {layout}",
          flush=True)
    g = torch.Generator().manual_seed(T * 7 + dim + rot)
    dt = TDT[name]
    qkv = torch.randn(T, hq + 2 * hkv, dim, generator=g).to(dt)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    buf = torch.full((T * (hq + 2 * hkv) * dim + 3,), 9.0, dtype=dt, device=dev)
    qkvd = buf[3:].view(T, hq + 2 * hkv, dim)      # off every 16-byte boundary
    qkvd.copy_(qkv)
    qd, kd, vd = qkvd.split((hq, hkv, hkv), 1)
    pages = T // page + 2
    kc, vc = make_cache(pages, hkv, page, dim, layout, dt, dev)
    slots = torch.randperm(pages * page, generator=g)[:T].int()
    if pad:
        slots[T - pad:] = torch.tensor([-1, -2 ** 31, pages * page, 2 ** 31 - 1])[
            torch.arange(pad) % 4].int()
    max_pos = 4099
    positions = torch.randint(0, max_pos, (T,), generator=g).int()
    positions[0] = max_pos - 1
    cs = table(max_pos, rot)
    got = ops.rope_append(qd if with_q else None, kd, vd, kc, vc, slots.to(dev), positions.to(dev),
                          cs.to(dev) if rot else None, interleaved=interleaved,
                          q_out=qd if inplace else None)
    c = cs[positions.long()]
    if with_q:
        assert (got is qd) == inplace
        close(got, *rotate64(q, c, rot, interleaved), name)
    else:
        assert got is None
    wantk, magk = rotate64(k, c, rot, interleaved)
    live = [(t, s) for t, s in enumerate(slots.tolist()) if 0 <= s < pages * page]
    assert len(live) == T - pad
    ts, ss = np.array([t for t, _ in live], int), np.array([s for _, s in live], int)
    close(kc.transpose(1, 2)[ss // page, ss % page], wantk[ts], magk[ts], name)
    assert torch.equal(vc.transpose(1, 2)[ss // page, ss % page].cpu(), v[ts])
    kc.transpose(1, 2)[ss // page, ss % page] = 5.0
    vc.transpose(1, 2)[ss // page, ss % page] = 5.0
    assert (kc == 5).all() and (vc == 5).all(), "wrote a row no slot names"
    assert torch.equal(kd.cpu(), k) and torch.equal(vd.cpu(), v) and (buf[:3] == 9).all()


@pytest.mark.parametrize("dim,rot", [(8, 8), (8, 2), (64, 64), (80, 40), (80, 80), (96, 48),
                                     (120, 90), (128, 128), (128, 0), (256, 256), (256, 2),
                                     (200, 34)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("name", ["f16", "bf16"])
def test_dims(dev, name, interleaved, dim, rot):
    run_case(dev, name, 37, 5, 2, dim, rot, interleaved, 16, "nhd", pad=3)
    run_case(dev, name, 5, 3, 3, dim, rot, interleaved, 7, "hnd")


@pytest.mark.parametrize("layout", ["hnd", "nhd", "interleaved"])
@pytest.mark.parametrize("T,hq,hkv,page", [(1, 32, 8, 16), (2, 1, 1, 1), (64, 32, 8, 16),
                                           (333, 28, 4, 24), (2051, 16, 2, 64), (17, 96, 96, 3)])
def test_sizes(dev, T, hq, hkv, page, layout):
    run_case(dev, "f16", T, hq, hkv, 128, 128, False, page, layout, pad=min(4, T // 3))
    run_case(dev, "bf16", T, hq, hkv, 64, 32, True, page, layout, inplace=True)


def test_keys_without_queries_and_no_rotation(dev):
    run_case(dev, "f16", 33, 2, 4, 96, 96, False, 16, "hnd", with_q=False)
    run_case(dev, "bf16", 33, 2, 4, 96, 0, False, 16, "hnd", inplace=True)


def test_positions_outside_the_table(dev):
    """The rotated dims of such a token are NaN, its other dims and its values are stored."""
    T, rot = 5, 32
    q, k, v = (torch.randn(T, 2, 64).half().to(dev) for _ in range(3))
    kc, vc = make_cache(2, 2, 8, 64, "hnd", torch.float16, dev)
    pos = torch.tensor([0, -1, 9, 10, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    slots = torch.arange(T, dtype=torch.int32, device=dev)
    out = ops.rope_append(q, k, v, kc, vc, slots, pos, table(10, rot).to(dev))
    for t, good in enumerate((True, False, True, False, False)):
        for x in (out[t], kc[0, :, t]):
            assert x[:, :rot].isnan().all() != good and not x[:, rot:].isnan().any()
    assert torch.equal(vc[0, :, :T].transpose(0, 1), v) and torch.equal(out[..., rot:], q[..., rot:])


def test_far_positions_and_long_caches(dev):
    """Slots whose element offset passes 2^31."""
    pages, page, heads, dim = 70000, 16, 8, 256
    kc = torch.empty(pages, heads, page, dim, dtype=torch.bfloat16, device=dev)
    vc = torch.empty_like(kc)
    assert kc.numel() > 2 ** 31
    k, v = (torch.randn(3, heads, dim).bfloat16().to(dev) for _ in range(2))
    slots = torch.tensor([pages * page - 1, 1, 66001 * 16 + 5], dtype=torch.int32, device=dev)
    ops.rope_append(None, k, v, kc, vc, slots)
    for t, s in enumerate(slots.tolist()):
        assert torch.equal(kc[s // page, :, s % page], k[t])
        assert torch.equal(vc[s // page, :, s % page], v[t])


def test_captured(dev):
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(9, h, 128, generator=g).half().to(dev) for h in (8, 2, 2))
    kc, vc = make_cache(3, 2, 16, 128, "nhd", torch.float16, dev)
    slots = torch.randperm(48, generator=g)[:9].int().to(dev)
    pos = torch.arange(9, dtype=torch.int32, device=dev)
    cs = table(64, 128).to(dev)
    out = torch.empty_like(q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        ops.rope_append(q, k, v, kc, vc, slots, pos, cs, q_out=out)
    for r in range(3):
        pos.add_(3)
        slots.copy_(torch.randperm(48, generator=g)[:9].int())
        kc.fill_(0), vc.fill_(0), out.fill_(0)
        graph.replay()
        ke, ve = make_cache(3, 2, 16, 128, "nhd", torch.float16, dev)
        ke.fill_(0), ve.fill_(0)
        want = ops.rope_append(q, k, v, ke, ve, slots, pos, cs)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kc, ke) and torch.equal(vc, ve), r


def test_refusals(dev):
    T, hq, hkv, D = 4, 4, 2, 64
    mk = lambda *s, dt=torch.float16: torch.zeros(*s, dtype=dt, device=dev)      # noqa: E731
    ok = dict(q=mk(T, hq, D), k=mk(T, hkv, D), v=mk(T, hkv, D), k_cache=mk(2, hkv, 16, D),
              v_cache=mk(2, hkv, 16, D), slots=torch.arange(T, dtype=torch.int32, device=dev),
              positions=mk(T, dt=torch.int32), cos_sin=mk(8, D, dt=torch.float32))
    ops.rope_append(**ok)
    for kw in (dict(k=mk(T, hkv, D - 8)), dict(v=mk(T + 1, hkv, D)), dict(q=mk(T, D)),
               dict(k=mk(T, hkv, D, dt=torch.bfloat16)), dict(v_cache=mk(3, hkv, 16, D)),
               dict(k_cache=mk(2, hkv, 16, D).cpu()), dict(slots=ok["slots"][:3]),
               dict(positions=None), dict(cos_sin=mk(8, D)), dict(q=None, q_out=mk(T, hq, D)),
               dict(q=mk(T, hq, 2 * D)[..., ::2]), dict(q_out=mk(T, hq, D).float())):
        with pytest.raises(ValueError):
            ops.rope_append(**{**ok, **kw})
    for kw in (dict(slots=ok["slots"].long()), dict(positions=ok["positions"].long()),
               dict(k_cache=mk(2, hkv, 16, D, dt=torch.float32))):
        with pytest.raises(TypeError):
            ops.rope_append(**{**ok, **kw})
    flat = mk(2, hkv, 16, D)
    for kw, word in (
            (dict(cos_sin=mk(8, D + 8, dt=torch.float32)), "rot_dim"),
            (dict(cos_sin=mk(8, 31, dt=torch.float32)), "rot_dim"),
            (dict(cos_sin=mk(0, D, dt=torch.float32)), "max_pos"),
            (dict(k_cache=flat[:1].expand(2, hkv, 16, D)), "share elements"),
            (dict(q_out=mk(1, hq, D).expand(T, hq, D)), "share elements"),
            (dict(q=mk(T + 1, hq, D)[1:], q_out=None), None),
            (dict(v_cache=flat.as_strided((2, hkv, 16, D), (hkv * 16 * D, 16 * D, D - 8, 1))),
             "share elements")):
        if word is None:
            ops.rope_append(**{**ok, **kw})
            continue
        with pytest.raises(hxm.HxmError, match=word):
            ops.rope_append(**{**ok, **kw})
    big = mk(T + 1, hq, D)
    with pytest.raises(hxm.HxmError, match="overlaps"):
        ops.rope_append(**{**ok, "q": big[:T], "q_out": big[1:]})
    with pytest.raises(hxm.HxmError, match="tile-alignment"):
        ops.rope_append(None, mk(T, hkv, 12), mk(T, hkv, 12), mk(2, hkv, 16, 12),
                        mk(2, hkv, 16, 12), ok["slots"])
    e = mk(0, hkv, D)
    assert ops.rope_append(mk(0, hq, D), e, e, ok["k_cache"], ok["v_cache"], ok["slots"][:0],
                           ok["positions"][:0], ok["cos_sin"]).shape == (0, hq, D)


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_between_the_heads_of_k_and_v(dev, T, interleaved):
    """A fused projection whose heads hold q, k and v side by side, q turned in place."""
    H, D, page = 6, 64, 16
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(T, H, 3, D, generator=g).half()
    fused = qkv.to(dev)
    q, k, v = fused.unbind(2)
    kc, vc = make_cache(T // page + 1, H, page, D, "nhd", torch.float16, dev)
    slots = torch.randperm((T // page + 1) * page, generator=g)[:T].int()
    pos = torch.randint(0, 512, (T,), generator=g).int()
    cs = table(512, D)
    out = ops.rope_append(q, k, v, kc, vc, slots.to(dev), pos.to(dev), cs.to(dev),
                          interleaved=interleaved, q_out=q)
    assert out is q
    c, s = cs[pos.long()], slots.long()
    close(fused[:, :, 0], *rotate64(qkv[:, :, 0], c, D, interleaved), "f16")
    assert torch.equal(fused[:, :, 1:].cpu(), qkv[:, :, 1:])
    close(kc.transpose(1, 2)[s // page, s % page], *rotate64(qkv[:, :, 1], c, D, interleaved), "f16")
    assert torch.equal(vc.transpose(1, 2)[s // page, s % page].cpu(), qkv[:, :, 2])
