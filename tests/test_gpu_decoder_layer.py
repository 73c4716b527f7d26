"""The decoder-layer operators together, as a serving loop runs them beside the
W8A16 GEMMs: residual_norm -> qkv GEMM + lora_add -> rope_append ->
paged_attention -> output GEMM + lora_add -> residual_norm -> gate/up GEMM ->
down GEMM, through two layers.

Each operator's output is compared with its formula in 64 bits on the inputs it
had in the run; what the loop as a whole must give is compared exactly: a prompt
appended in one call, in pieces or token by token, a captured step replayed,
and a batch padded to a larger one (the operators' part)."""
import numpy as np
import pytest
import torch

import hxm
import hxm.ops as ops
from test_gpu_paged_attention import check as check_attention
from test_gpu_rope_append import close, rotate64, table as rope_table

pytestmark = pytest.mark.gpu

H, HQ, HKV, D, I, R, ADAPTERS, PAGE, EPS = 512, 8, 2, 64, 704, 16, 3, 16, 1e-5
WIDE = (HQ + 2 * HKV) * D
U = 2.0 ** -11


def f64(t):
    return t.double().cpu().numpy()


def near(got, want, err, what):
    """got: want rounded once to f16 after an error of up to err."""
    tol = U * (np.abs(want) + err) + 2.0 ** -25 + err
    got = f64(got)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:4].tolist(), got[bad][:4], want[bad][:4])


class Layer:
    def __init__(self, g, dev):
        w8 = lambda n, k: (torch.randint(-127, 128, (n, k), generator=g,             # noqa: E731
                                         dtype=torch.int8).to(dev),
                           ((torch.rand(n, generator=g) + 0.5) / (74 * k ** 0.5)).to(dev))
        lo = lambda n, k: ((torch.randn(ADAPTERS, R, k, generator=g) / k ** 0.5)     # noqa: E731
                           .half().to(dev),
                           (torch.randn(ADAPTERS, n, R, generator=g) / 4).half().to(dev))
        self.qkv, self.o, self.down = w8(WIDE, H), w8(H, HQ * D), w8(H, I)
        (wg, sg), (wu, su) = w8(I, H), w8(I, H)
        self.gate_up = ops.swiglu_pack(wg, wu, sg, su)
        self.lora_qkv, self.lora_o = lo(WIDE, H), lo(H, HQ * D)
        self.norm1, self.norm2 = ((1 + 0.1 * torch.randn(H, generator=g)).half().to(dev)
                                  for _ in range(2))


class Model:
    def __init__(self, dev, pages=40, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.layers = [Layer(g, dev) for _ in range(2)]
        self.cos_sin = rope_table(512, D).to(dev)
        self.alpha = (torch.rand(ADAPTERS, generator=g) + 0.5).to(dev)
        shape = (2, 2, pages, PAGE, HKV, D)          # layer, k or v
        self.cache = torch.full(shape, float("nan"), dtype=torch.float16, device=dev)

    def kv(self, i):
        return self.cache[i, 0].transpose(1, 2), self.cache[i, 1].transpose(1, 2)

    def step(self, x, index, positions, slots, block_table, lens, record=None):
        """One new token of every sequence; x [B, H] the embeddings."""
        rec = record.append if record is not None else lambda r: None
        h = torch.zeros_like(x)
        B = x.shape[0]
        for i, l in enumerate(self.layers):
            kc, vc = self.kv(i)
            y, z = ops.residual_norm(h, x, pre="rms", pre_weight=l.norm1, pre_eps=EPS)
            rec(("norm", h, x, l.norm1, y, z))
            x = y
            p = ops.gemm_w8a16(z, *l.qkv)
            qkv = ops.lora_add(p, z, *l.lora_qkv, index, self.alpha)
            rec(("lora", p, z, *l.lora_qkv, index, self.alpha, qkv.clone()))  # q turns in place
            q, k, v = qkv.view(B, -1, D).split((HQ, HKV, HKV), 1)
            q0 = q.clone() if record is not None else q
            q = ops.rope_append(q, k, v, kc, vc, slots, positions, self.cos_sin, q_out=q)
            rec(("rope", q0, k, v, kc, vc, slots, positions, self.cos_sin, q.clone()))
            a, lse = ops.paged_attention(q, kc, vc, block_table, lens, return_lse=True)
            rec(("attention", q, kc, vc, block_table, lens, a, lse))
            a = a.view(B, HQ * D)
            p = ops.gemm_w8a16(a, *l.o)
            h = ops.lora_add(p, a, *l.lora_o, index, self.alpha)
            rec(("lora", p, a, *l.lora_o, index, self.alpha, h))
            y, z = ops.residual_norm(h, x, pre="rms", pre_weight=l.norm2, pre_eps=EPS)
            rec(("norm", h, x, l.norm2, y, z))
            x = y
            h = ops.gemm_w8a16(ops.gemm_w8a16_swiglu(z, *l.gate_up, I), *l.down)
        return ops.residual_norm(h, x, pre="none")[0]


def check_norm(h, x, w, y, z):
    """fp32 sums and a dozen operations: 64 2^-24 of the terms."""
    h, x, w = f64(h), f64(x), f64(w)
    mag, c = np.abs(h) + np.abs(x), 64 * 2.0 ** -24
    near(y, h + x, c * mag, "y")
    s = h + x
    r = 1 / np.sqrt((s * s).mean(1, keepdims=True) + EPS)
    rms = np.sqrt((mag ** 2).mean(1, keepdims=True))
    err = c * (np.abs(w) * r * mag + np.abs(s * r * w) * r * rms)
    near(z, s * r * w, err, "z")


def check_lora(y, x, A, B, index, alpha, out):
    """The x A^T sum in fp32, its two halves (2^-21 of the row's largest), the second
    product's sums and epilogue."""
    y64, x64, K = f64(y), f64(x), x.shape[1]
    for m, a in enumerate(index.tolist()):
        if a < 0:
            assert torch.equal(out[m], y[m])
            continue
        A64, B64, s = f64(A[a]), f64(B[a]), float(alpha[a])
        t, tm = A64 @ x64[m], np.abs(A64) @ np.abs(x64[m])
        err = ((K + 2 * R + 32) * 2.0 ** -24 * tm + 2.0 ** -21 * np.abs(t).max())
        near(out[m], y64[m] + s * (B64 @ t),
             s * (np.abs(B64) @ err) + 2.0 ** -23 * np.abs(y64[m]), m)


def check_rope(q0, k, v, kc, vc, slots, positions, cos_sin, q):
    cs = cos_sin.cpu()[positions.long().cpu()]
    close(q, *rotate64(q0.cpu(), cs, D, False), "f16")
    live = slots.cpu() >= 0
    s = slots.cpu()[live].long()
    wk, mk = rotate64(k.cpu(), cs, D, False)
    close(kc.transpose(1, 2)[s // PAGE, s % PAGE], wk[live], mk[live], "f16")
    assert torch.equal(vc.transpose(1, 2)[s // PAGE, s % PAGE], v[live.to(v.device)])


def check_att(q, kc, vc, table, lens, out, lse):
    seqs = []
    for b, n in enumerate(lens.tolist()):
        t = torch.arange(n)
        at = table[b].cpu()[t // PAGE].long(), t % PAGE
        seqs.append(tuple(f64(c.transpose(1, 2)[at[0], at[1]]) for c in (kc, vc)))
    check_attention(out.cpu(), lse.cpu(), q.cpu(), seqs, HQ // HKV, D ** -0.5, 0, "f16")


CHECKS = {"norm": check_norm, "lora": check_lora, "rope": check_rope, "attention": check_att}


class Batch:
    """Sequences of given lengths on pages of their own, in a random order."""

    def __init__(self, dev, lens, pages=40, steps=8, pad=0, seed=1):
        g = torch.Generator().manual_seed(seed)
        need = [-(-(n + steps) // PAGE) for n in lens]
        order = torch.randperm(pages, generator=g).int()
        self.table = torch.full((len(lens) + pad, max(need) + 1), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        assert at <= pages
        self.live, self.pad, self.dev = len(lens), pad, dev
        self.lens = torch.tensor(list(lens) + [0] * pad, dtype=torch.int32)
        self.index = torch.tensor([b % (ADAPTERS + 1) - 1 for b in range(len(lens))] + [-1] * pad,
                                  dtype=torch.int32, device=dev)
        self.table_d = self.table.to(dev)

    def slot(self, b, t):
        return self.table[b, t // PAGE] * PAGE + t % PAGE

    def advance(self):
        """(positions, slots, table, lens) of the next token of every live sequence."""
        pos = self.lens.clone()
        slots = torch.full_like(pos, -1)
        for b in range(self.live):
            slots[b] = self.slot(b, int(pos[b]))
        self.lens[:self.live] += 1
        return [t.to(self.dev) for t in (pos, slots)] + [self.table_d, self.lens.to(self.dev)]


def prefill(model, batch, lens, pieces, seed=2):
    """Keys and values of the prompts, each appended in `pieces` calls."""
    g = torch.Generator().manual_seed(seed)
    for i in range(2):
        kc, vc = model.kv(i)
        for b, n in enumerate(lens):
            k, v = (torch.randn(n, HKV, D, generator=g).half().to(kc.device) for _ in range(2))
            pos = torch.arange(n, dtype=torch.int32)
            slots = torch.stack([batch.slot(b, t) for t in range(n)]).int() if n else pos
            edges = np.linspace(0, n, pieces + 1).astype(int) if pieces else np.arange(n + 1)
            for lo, hi in zip(edges[:-1], edges[1:]):
                ops.rope_append(None, k[lo:hi], v[lo:hi], kc, vc, slots[lo:hi].to(kc.device),
                                pos[lo:hi].to(kc.device), model.cos_sin)


LENS = [200, 0, 37, 16, 15, 1, 90]


def test_every_stage_of_a_decode_loop(dev):
    model, batch = Model(dev), Batch(dev, LENS)
    prefill(model, batch, LENS, 1)
    g = torch.Generator().manual_seed(3)
    for step in range(3):
        record = []
        x = torch.randn(len(LENS), H, generator=g).half().to(dev)
        out = model.step(x, batch.index, *batch.advance(), record=record)
        assert out.isfinite().all()
        print("step", step, len(record), "operators", flush=True)
        for name, *args in record:
            CHECKS[name](*args)


def test_prompts_in_pieces(dev):
    """One call, three, and one a token leave the same cache and the same step."""
    outs = []
    for pieces in (1, 3, 0):
        model, batch = Model(dev), Batch(dev, LENS)
        prefill(model, batch, LENS, pieces)
        x = torch.randn(len(LENS), H, generator=torch.Generator().manual_seed(4)).half().to(dev)
        outs.append((model.step(x, batch.index, *batch.advance()), model.cache.clone()))
    for out, cache in outs[1:]:
        assert torch.equal(out, outs[0][0])
        assert torch.equal(cache.view(torch.int16), outs[0][1].view(torch.int16))


def test_captured_step(dev):
    """The step captured once and replayed over eight tokens, eager steps of a second
    model between the replays."""
    a, b = Model(dev), Model(dev)
    ba, bb = Batch(dev, LENS), Batch(dev, LENS)
    prefill(a, ba, LENS, 1), prefill(b, bb, LENS, 1)
    x = torch.zeros(len(LENS), H, dtype=torch.float16, device=dev)
    static = [t.clone() for t in Batch(dev, LENS).advance()]
    start = a.cache.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        a.step(x, ba.index, *static)
        with torch.cuda.graph(graph, stream=s):
            out = a.step(x, ba.index, *static)
    torch.cuda.synchronize()
    a.cache.copy_(start)
    g = torch.Generator().manual_seed(5)
    for step in range(8):
        now = torch.randn(len(LENS), H, generator=g).half().to(dev)
        want = b.step(now, bb.index, *bb.advance())
        torch.cuda.synchronize()
        x.copy_(now)
        for t, new in zip(static, ba.advance()):
            t.copy_(new)
        out.fill_(9)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), step
    assert torch.equal(a.cache.view(torch.int16), b.cache.view(torch.int16))


def test_padded_batch(dev):
    """Rows of padding (slot -1, no tokens, no adapter) leave the live rows of every
    operator and the cache as they are."""
    res = []
    for pad in (0, 9):
        model, batch = Model(dev), Batch(dev, LENS, pad=pad)
        prefill(model, batch, LENS, 1)
        l, n = model.layers[0], len(LENS)
        g = torch.Generator().manual_seed(6)
        x, h, qkv = (torch.cat((torch.randn(n, w, generator=g).half(),
                                torch.full((pad, w), float("nan")).half())).to(dev)
                     for w in (H, H, WIDE))
        pos, slots, table, lens = batch.advance()
        y, z = ops.residual_norm(h, x, pre_weight=l.norm1)
        qkv = ops.lora_add(qkv, z, *l.lora_qkv, batch.index, model.alpha)
        q, k, v = qkv.view(n + pad, -1, D).split((HQ, HKV, HKV), 1)
        kc, vc = model.kv(0)
        q = ops.rope_append(q, k, v, kc, vc, slots, pos, model.cos_sin)
        a = ops.paged_attention(q, kc, vc, table, lens)
        assert (a[n:] == 0).all()
        res.append([t[:n] for t in (y, z, qkv, q, a)] + [model.cache])
    for one, two in zip(*res):
        assert torch.equal(one.contiguous().view(torch.int16), two.contiguous().view(torch.int16))


def test_capture_needs_its_workspace(dev):
    """Without a call before it, a captured paged_attention or lora_add is refused and the
    capture goes on; after one, it is recorded, and works when the buffers are new again."""
    g = torch.Generator().manual_seed(9)
    q = torch.randn(2, HQ, D, generator=g).half().to(dev)
    kc, vc = (torch.randn(80, HKV, PAGE, D, generator=g).half().to(dev) for _ in range(2))
    table = torch.randperm(80, generator=g).int().view(2, 40).to(dev)
    lens = torch.tensor([640, 600], dtype=torch.int32, device=dev)
    y, x = (torch.randn(300, w, generator=g).half().to(dev) for w in (256, H))
    A, B = (torch.randn(2, a, b, generator=g).half().to(dev) * 0.1 for a, b in ((R, H), (256, R)))
    index = (torch.arange(300, device=dev) % 3 - 1).int()
    calls = [lambda out: ops.paged_attention(q, kc, vc, table, lens, out=out),
             lambda out: ops.lora_add(y, x, A, B, index, out=out)]
    outs = [torch.empty_like(q), torch.empty_like(y)]
    want = [f(None).clone() for f in calls]
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    assert hxm.lib.hxm_release_cache() == 0
    for f, out in zip(calls, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            with pytest.raises(hxm.HxmError, match="workspace-budget"):
                f(out)
            out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        assert (out == 3).all()
    for f, out, w in zip(calls, outs, want):
        with torch.cuda.stream(s):
            f(out)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            f(out)
        for _ in range(3):
            out.fill_(3)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, w)


def test_stream_argument(dev):
    """With stream=, copies of parameters that are not contiguous and new outputs belong to that
    stream: a call does not wait for, nor race with, what the current stream still does."""
    g = torch.Generator().manual_seed(11)
    wide = torch.randn(H, 2, generator=g).half().to(dev)
    h, x = (torch.randn(40, H, generator=g).half().to(dev) for _ in range(2))
    q = torch.randn(2, HQ, D, generator=g).half().to(dev)
    kc, vc = (torch.randn(8, HKV, PAGE, D, generator=g).half().to(dev) for _ in range(2))
    table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
    lens = torch.tensor([60, 33], dtype=torch.int32, device=dev)
    none = torch.full_like(lens, -1)
    A, B = (torch.randn(2, a, b, generator=g).half().to(dev) * 0.1 for a, b in ((R, H), (H, R)))
    scale = torch.rand(2, 3, generator=g).to(dev)[:, 1]
    index = (torch.arange(40, device=dev) % 3 - 1).int()
    calls = [lambda s: ops.residual_norm(h, x, pre_weight=wide[:, 1], post="rms",
                                         post_weight=wide[:, 0], gate=wide.t(), stream=s)[1],
             lambda s: ops.rope_append(q, kc[:2, :, 0], vc[:2, :, 0], kc, vc,
                                       none, stream=s),
             lambda s: ops.paged_attention(q, kc, vc, table, lens, stream=s),
             lambda s: ops.lora_add(h, x, A, B, index, scale, stream=s)]
    want = [f(None).clone() for f in calls]
    s = torch.cuda.Stream()
    big = torch.randn(4096, 4096, device=dev)
    for f, w in zip(calls, want):
        f(s)                                     # workspaces, before the current stream is busy
        torch.cuda.synchronize()
        for _ in range(20):
            big @ big
        with torch.cuda.stream(s):
            same = torch.equal(f(s), w)          # waits for s alone
        assert same
        torch.cuda.synchronize()


def test_host_threads(dev):
    """Four host threads, each with a stream, a model and a batch of its own, give what one
    thread gives."""
    import threading

    def loop(seed, stream):
        lens = [90 + 7 * seed, 0, 300 - 40 * seed, 1]
        with torch.cuda.stream(stream):
            model, batch = Model(dev, seed=seed), Batch(dev, lens, seed=seed)
            prefill(model, batch, lens, 1, seed=seed)
            g = torch.Generator().manual_seed(seed)
            outs = [model.step(torch.randn(len(lens), H, generator=g).half().to(dev), batch.index,
                               *batch.advance()) for _ in range(5)]
            stream.synchronize()
        return outs

    streams = [torch.cuda.Stream() for _ in range(4)]
    want = [loop(i, streams[0]) for i in range(4)]
    got = [None] * 4

    def run(i):
        torch.cuda.set_device(0)
        got[i] = loop(i, streams[i])
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert a is not None and all(torch.equal(x, y) for x, y in zip(a, b))
