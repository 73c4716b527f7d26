"""The attention half of a decode step and what surrounds it, as cases.

The operators a decoder layer needs next to the int8 projections, the SwiGLU
block and the row norms of hxm.ops:

* ``residual_norm``: the norm after a block, its gate and scale, the residual
  add and the norm before the next block, in one pass over the rows;
* ``rope_append``: rotary position embedding of queries and keys, the rotated
  keys and the values stored into a paged cache on the way;
* ``paged_attention``: attention of one new token per sequence over that cache;
* ``lora_add``: the low-rank adapters of many requests added to the output of
  a projection they share.

``own`` chooses between plain torch operations and the framework's kernels.
Run from the repository's root.
"""
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # One decoding sequence: the block's output joins the residual stream
        # and the next block's RMSNorm follows (latency only).
        {"name": "residual_norm_1x4096_f16", "op": "residual_norm", "rows": 1, "cols": 4096,
         "dtype": "f16", "post": "none", "pre": "rms", "gates": 0},
        # Prefill of 2048 tokens, norms on both sides of the block and a
        # learned gate per channel.
        {"name": "residual_norm_2048x4096_bf16", "op": "residual_norm", "rows": 2048,
         "cols": 4096, "dtype": "bf16", "post": "rms", "pre": "rms", "gates": 1},
        # f32 stream of an odd width, LayerNorms, one gate row for each of
        # three sequences (a gate made from a conditioning vector).
        {"name": "residual_norm_1023x5003_f32", "op": "residual_norm", "rows": 1023,
         "cols": 5003, "dtype": "f32", "post": "layer", "pre": "layer", "gates": 3},
        # A decode step of 64 sequences whose batch is padded by three rows;
        # q, k and v are slices of one fused projection.
        {"name": "rope_append_64_f16", "op": "rope_append", "T": 64, "pad": 3, "Hq": 32, "Hkv": 8,
         "D": 128, "rot": 128, "style": "half", "page": 16, "layout": "hnd", "far": 131072,
         "dtype": "f16"},
        # The prefill of 8192 tokens, several prompts in one batch.
        {"name": "rope_append_8192_bf16", "op": "rope_append", "T": 8192, "pad": 0, "Hq": 32,
         "Hkv": 8, "D": 128, "rot": 128, "style": "half", "page": 16, "layout": "nhd",
         "far": 8192, "dtype": "bf16"},
        # Odd token count, partial rotation of neighbouring pairs, pages whose
        # size is no power of two.
        {"name": "rope_append_333_f16", "op": "rope_append", "T": 333, "pad": 5, "Hq": 28,
         "Hkv": 4, "D": 80, "rot": 40, "style": "pairs", "page": 24, "layout": "nhd",
         "far": 1 << 20, "dtype": "f16"},
        # One short sequence, every query head with its own key head (latency).
        {"name": "attention_1x300_f16", "op": "paged_attention", "B": 1, "L": 300, "Hkv": 32,
         "G": 1, "D": 128, "page": 16, "layout": "hnd", "window": 0, "pad": 0, "dtype": "f16"},
        # A serving batch of mixed lengths with two padded rows, shared heads.
        {"name": "attention_64x4096_f16", "op": "paged_attention", "B": 64, "L": 4096, "Hkv": 8,
         "G": 4, "D": 128, "page": 16, "layout": "nhd", "window": 0, "pad": 2, "dtype": "f16"},
        # A few long contexts.
        {"name": "attention_8x32768_bf16", "op": "paged_attention", "B": 8, "L": 32768, "Hkv": 8,
         "G": 4, "D": 128, "page": 64, "layout": "hnd", "window": 0, "pad": 0, "dtype": "bf16"},
        # A sliding window over long contexts, one key head for all queries.
        {"name": "attention_16x16384_w1000_bf16", "op": "paged_attention", "B": 16, "L": 16384,
         "Hkv": 1, "G": 12, "D": 64, "page": 32, "layout": "hnd", "window": 1000, "pad": 0,
         "dtype": "bf16"},
        # A decode step of 48 requests over 16 adapters, some without one.
        {"name": "lora_48x4096x4096_r16_f16", "op": "lora_add", "M": 48, "K": 4096, "N": 4096,
         "R": 16, "L": 16, "run": 1, "none": 0.2, "dtype": "f16"},
        # Prompts of 2048 tokens under four adapters at an up projection.
        {"name": "lora_2048x4096x11008_r64_bf16", "op": "lora_add", "M": 2048, "K": 4096,
         "N": 11008, "R": 64, "L": 4, "run": 300, "none": 0.1, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))
    return max(lo, min(hi, v) // step * step)


def draw(rng):
    op = rng.choice(("residual_norm", "rope_append", "paged_attention", "paged_attention",
                     "lora_add"))
    dtype = rng.choice(("f16", "bf16"))
    if op == "residual_norm":
        rows = _log_int(rng, 1, 8192)
        cols = _log_int(rng, 64, min(32768, 8192 * 4096 // rows))
        if cols > 64 and rng.random() < 0.5:
            cols -= cols % 64
        post = rng.choice(("none", "rms", "layer"))
        return {"op": op, "rows": rows, "cols": cols, "dtype": rng.choice(("f16", "bf16", "f32")),
                "post": post, "pre": rng.choice(("rms", "layer", "rms", "none")),
                "gates": rng.choice((0, 1, rows))}
    heads = rng.choice((1, 2, 4, 5, 8, 16, 32))
    group = rng.choice((1, 2, 3, 4, 6, 8, 16))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    layout = rng.choice(("hnd", "nhd"))
    if op == "rope_append":
        T = _log_int(rng, 1, min(8192, (8192 * 48 * 128) // ((group + 2) * heads * dim)))
        return {"op": op, "T": T, "pad": rng.randrange(4) if T > 8 else 0, "Hq": heads * group,
                "Hkv": heads, "D": dim, "rot": rng.choice((dim, dim, dim // 2)),
                "style": rng.choice(("half", "pairs")), "page": page, "layout": layout,
                "far": _log_int(rng, 8192, 1 << 20), "dtype": dtype}
    if op == "paged_attention":
        L = _log_int(rng, 1, 32768)
        top = 8 * 32768 * 8 * 128 // (L * heads * dim)
        B = _log_int(rng, 1, max(1, min(256, top)))
        return {"op": op, "B": B, "L": L, "Hkv": heads, "G": group, "D": dim, "page": page,
                "layout": layout, "window": rng.choice((0, 0, 0, _log_int(rng, 1, 4096))),
                "pad": rng.randrange(3) if B > 4 else 0, "dtype": dtype}
    return {"op": op, "M": _log_int(rng, 1, 2048), "K": _log_int(rng, 256, 4096, 16),
            "N": _log_int(rng, 64, 11008), "R": rng.choice((8, 16, 16, 32, 64)),
            "L": _log_int(rng, 1, 16), "run": rng.choice((1, 7, 64, 300)),
            "none": rng.choice((0.0, 0.2)), "dtype": dtype}


# ---- what a case fixes beyond its sizes ---------------------------------------

def _lens(case):
    """Tokens in the cache of each sequence: spread over the logarithm up to L
    (which one has), the padded rows empty."""
    rng = random.Random("%(B)d %(L)d %(D)d %(Hkv)d" % case)
    n = [_log_int(rng, max(1, case["L"] // 8), case["L"]) for _ in range(case["B"] - case["pad"])]
    n[rng.randrange(len(n))] = case["L"]
    return n + [0] * case["pad"]


def _adapters(case):
    """The adapter of each row (-1: none): runs of rows of one request."""
    rng = random.Random("%(M)d %(K)d %(N)d %(R)d" % case)
    out = []
    while len(out) < case["M"]:
        a = -1 if rng.random() < case["none"] else rng.randrange(case["L"])
        out += [a] * case["run"]
    return out[:case["M"]]


# ---- inputs -------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def _cache(g, pages, case):
    """A key or value cache [pages, heads, page, D]: heads first in memory
    ("hnd") or tokens first ("nhd")."""
    h, p, d = case["Hkv"], case["page"], case["D"]
    if case["layout"] == "hnd":
        return _randn(g, pages, h, p, d, dtype=DTYPES[case["dtype"]])
    return _randn(g, pages, p, h, d, dtype=DTYPES[case["dtype"]]).transpose(1, 2)


def _norm_params(g, kind, cols, dt):
    if kind == "none":
        return None, None
    w = (1 + _randn(g, cols, scale=0.1)).to(dt)
    return w, _randn(g, cols, scale=0.1).to(dt) if kind == "layer" else None


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "residual_norm":
        rows, cols = case["rows"], case["cols"]
        s["h"] = (_randn(g, rows, cols, scale=0.7) + 0.05).to(dt)
        s["x"] = _randn(g, rows, cols, scale=2.0).to(dt)
        s["post_w"], s["post_b"] = _norm_params(g, case["post"], cols, dt)
        s["pre_w"], s["pre_b"] = _norm_params(g, case["pre"], cols, dt)
        s["gate"] = _randn(g, case["gates"], cols, scale=0.5).to(dt) if case["gates"] else None
    elif case["op"] == "rope_append":
        T, hq, hkv, d = case["T"], case["Hq"], case["Hkv"], case["D"]
        qkv = _randn(g, T, hq + 2 * hkv, d).to(dt)      # the fused projection's output
        s["q"], s["k"], s["v"] = qkv.split((hq, hkv, hkv), dim=1)
        pages = T // case["page"] + 9
        s["k_cache"], s["v_cache"] = _cache(g, pages, case), _cache(g, pages, case)
        slots = torch.randperm(pages * case["page"], generator=g, device="cuda")[:T]
        slots[T - case["pad"]:] = -1                     # padded rows store nothing
        s["slots"] = slots.int()
        s["positions"] = torch.randint(0, case["far"], (T,), generator=g, device="cuda").int()
        half = case["rot"] // 2
        inv = 10000.0 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
        ang = torch.arange(case["far"], device="cuda", dtype=torch.float64)[:, None] * inv
        s["cos_sin"] = torch.cat((ang.cos(), ang.sin()), dim=1).float()
    elif case["op"] == "paged_attention":
        B, page = case["B"], case["page"]
        lens = _lens(case)
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g, device="cuda").int()
        table = torch.full((B, max(need)), -1, device="cuda", dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"], s["lens"] = table, torch.tensor(lens, device="cuda", dtype=torch.int32)
        s["k_cache"], s["v_cache"] = _cache(g, pages, case), _cache(g, pages, case)
        s["q"] = _randn(g, B, case["Hkv"] * case["G"], case["D"], scale=1.5).to(dt)
    else:
        M, K, N, R, L = (case[k] for k in "MKNRL")
        s["x"] = _randn(g, M, K).to(dt)
        s["y"] = _randn(g, M, N).to(dt)
        s["A"] = _randn(g, L, R, K, scale=K ** -0.5).to(dt)
        s["B"] = _randn(g, L, N, R, scale=R ** -0.5).to(dt)
        s["scale"] = torch.rand(L, generator=g, device="cuda") + 0.5
        s["index"] = torch.tensor(_adapters(case), device="cuda", dtype=torch.int32)
    return s


EPS = 1e-5
X_SCALE, H_SCALE = 0.9, 1.25      # of the residual stream and of the block's output


# ---- plain forms --------------------------------------------------------------

def _plain_norm(x, kind, w, b):
    if kind == "none":
        return x
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    return x if b is None else x + b.float()


def _plain_residual_norm(s):
    c = s["case"]
    p = _plain_norm(s["h"].float(), c["post"], s["post_w"], s["post_b"])
    if s["gate"] is not None:
        p = (p.view(c["gates"], -1, c["cols"]) * s["gate"].float()[:, None]).view_as(p)
    y = X_SCALE * s["x"].float() + H_SCALE * p
    if c["pre"] == "none":
        return [y.to(s["h"].dtype)]
    z = _plain_norm(y, c["pre"], s["pre_w"], s["pre_b"])
    return [y.to(s["h"].dtype), z.to(s["h"].dtype)]


def _plain_rotate(x, cos, sin, rot, style):
    f = x.float()
    r = f[..., :rot]
    a, b = (r[..., :rot // 2], r[..., rot // 2:]) if style == "half" else (r[..., 0::2],
                                                                          r[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    r = torch.cat((u, v), -1) if style == "half" else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((r, f[..., rot:]), -1).to(x.dtype)


def _plain_rope_append(s):
    c = s["case"]
    cs = s["cos_sin"][s["positions"]][:, None]
    cos, sin = cs[..., :c["rot"] // 2], cs[..., c["rot"] // 2:]
    q = _plain_rotate(s["q"], cos, sin, c["rot"], c["style"])
    k = _plain_rotate(s["k"], cos, sin, c["rot"], c["style"])
    n = c["T"] - c["pad"]                                # the rows that are no padding
    page, off = s["slots"][:n] // c["page"], s["slots"][:n] % c["page"]
    s["k_cache"][page, :, off] = k[:n]
    s["v_cache"][page, :, off] = s["v"][:n]
    return [q, s["k_cache"], s["v_cache"]]


def _plain_attention(s):
    c = s["case"]
    n = min(c["L"], c["window"] or c["L"])
    pos = s["lens"][:, None] - n + torch.arange(n, device="cuda", dtype=torch.int32)
    live = pos >= 0                                      # the last n tokens, right-aligned
    at = pos.clamp(min=0)
    page = s["table"].gather(1, (at // c["page"]).long()).clamp(min=0)
    k = s["k_cache"][page, :, at % c["page"]].float().permute(0, 2, 3, 1)    # [B, H, D, n]
    v = s["v_cache"][page, :, at % c["page"]].float().transpose(1, 2)        # [B, H, n, D]
    q = s["q"].float().view(c["B"], c["Hkv"], c["G"], c["D"])
    sc = q @ k.contiguous() * c["D"] ** -0.5
    sc = sc.masked_fill(~live[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True).clamp(min=-1e30)
    p = (sc - m).exp()
    z = p.sum(-1, keepdim=True)
    out = (p @ v.contiguous()) / z.clamp(min=1e-30)      # a row without tokens gives zeros
    lse = m + z.log()
    lse = lse.masked_fill(z == 0, -math.inf)
    return [out.reshape(s["q"].shape).to(s["q"].dtype), lse.reshape(c["B"], -1)]


def _plain_lora(s):
    c = s["case"]
    # Every row against every adapter, its own kept: two products over the
    # stacked adapters.
    t = s["x"].float() @ s["A"].float().view(-1, c["K"]).t()
    mine = s["index"][:, None] == torch.arange(c["L"], device="cuda")
    t = t.view(c["M"], c["L"], c["R"]) * (mine * s["scale"])[..., None]
    d = t.view(c["M"], -1) @ s["B"].float().transpose(1, 2).reshape(-1, c["N"])
    return [(s["y"].float() + d).to(s["y"].dtype)]


# ---- the framework's calls ----------------------------------------------------

def _ops():
    path = os.path.join(os.getcwd(), "hexagon-mlir_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import hxm.ops as ops
    return ops


def _own(s):
    ops, c = _ops(), s["case"]
    if c["op"] == "residual_norm":
        y, z = ops.residual_norm(
            s["h"], s["x"], post=c["post"], post_weight=s["post_w"], post_bias=s["post_b"],
            post_eps=EPS, pre=c["pre"], pre_weight=s["pre_w"], pre_bias=s["pre_b"], pre_eps=EPS,
            gate=s["gate"], residual_scale=X_SCALE, block_scale=H_SCALE)
        return [y] if z is None else [y, z]
    if c["op"] == "rope_append":
        q = ops.rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"],
                            s["positions"], s["cos_sin"], interleaved=c["style"] == "pairs")
        return [q, s["k_cache"], s["v_cache"]]
    if c["op"] == "paged_attention":
        return list(ops.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                        window=c["window"], return_lse=True))
    return [ops.lora_add(s["y"], s["x"], s["A"], s["B"], s["index"], s["scale"])]


PLAIN = {"residual_norm": _plain_residual_norm, "rope_append": _plain_rope_append,
         "paged_attention": _plain_attention, "lora_add": _plain_lora}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---- the least a pass moves and computes --------------------------------------

def work(case):
    eb = BYTES[case["dtype"]]
    if case["op"] == "residual_norm":
        rows, cols = case["rows"], case["cols"]
        streams = 3 if case["pre"] == "none" else 4      # h and x in, y and z out
        params = (2 * ((case["post"] != "none") + (case["pre"] != "none")) + case["gates"]) * cols
        return {"bytes": (streams * rows * cols + params) * eb, "flops": 10 * rows * cols}
    if case["op"] == "rope_append":
        T, n, d = case["T"], case["T"] - case["pad"], case["D"]
        moved = 2 * T * case["Hq"] * d + 4 * n * case["Hkv"] * d
        return {"bytes": moved * eb + 4 * T * (case["rot"] + 2),
                "flops": 3 * T * (case["Hq"] + case["Hkv"]) * case["rot"]}
    if case["op"] == "paged_attention":
        lens = [min(n, case["window"] or n) for n in _lens(case)]
        hq = case["Hkv"] * case["G"]
        return {"bytes": (2 * sum(lens) * case["Hkv"] * case["D"]
                          + 2 * case["B"] * hq * case["D"]) * eb
                + sum(-(-n // case["page"]) for n in lens) * 4 + case["B"] * (4 + 4 * hq),
                "flops": 4 * sum(lens) * hq * case["D"]}
    rows = [a for a in _adapters(case) if a >= 0]
    M, K, N, R = (case[k] for k in "MKNR")
    return {"bytes": (2 * M * N + len(rows) * K + len(set(rows)) * R * (K + N)) * eb + 4 * M,
            "flops": 2 * len(rows) * R * (K + N)}


# ---- the definition, in 64 bits -----------------------------------------------

def _norm64(x, kind, w, b):
    if kind == "none":
        return x
    mean = x.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(x[:, :1])
    var = (x - mean).pow(2).sum(1, keepdim=True) / x.shape[1]
    y = (x - mean) / (var + EPS).sqrt() * w.double()
    return y if b is None else y + b.double()


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "residual_norm":
        p = _norm64(s["h"].double(), case["post"], s["post_w"], s["post_b"])
        if case["gates"]:
            p = p * s["gate"].double().repeat_interleave(case["rows"] // case["gates"], 0)
        y = X_SCALE * s["x"].double() + H_SCALE * p
        if case["pre"] == "none":
            return [y]
        return [y, _norm64(y, case["pre"], s["pre_w"], s["pre_b"])]
    if case["op"] == "rope_append":
        rot, half = case["rot"], case["rot"] // 2
        first = torch.arange(half, device="cuda")
        if case["style"] == "half":
            i, j = first, first + half
        else:
            i, j = 2 * first, 2 * first + 1
        cs = s["cos_sin"].double()[s["positions"].long()].unsqueeze(1)

        def turn(x):
            x = x.double()
            y = x.clone()
            y[..., i] = x[..., i] * cs[..., :half] - x[..., j] * cs[..., half:]
            y[..., j] = x[..., i] * cs[..., half:] + x[..., j] * cs[..., :half]
            return y
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        live = s["slots"] >= 0
        slot = s["slots"][live].long()
        kc.transpose(1, 2)[slot // case["page"], slot % case["page"]] = turn(s["k"])[live]
        vc.transpose(1, 2)[slot // case["page"], slot % case["page"]] = s["v"][live].double()
        return [turn(s["q"]), kc, vc]
    if case["op"] == "paged_attention":
        lens, page = _lens(case), case["page"]
        out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        lse = torch.full(s["q"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
        for b, n in enumerate(lens):
            if not n:
                continue
            first = max(0, n - case["window"]) if case["window"] else 0
            pages = s["table"][b, first // page:-(-n // page)].long()
            skip = first - first // page * page
            k, v = (s[w][pages].transpose(1, 2).flatten(0, 1)[skip:skip + n - first].double()
                    for w in ("k_cache", "v_cache"))
            q = s["q"][b].double().view(case["Hkv"], case["G"], case["D"])
            for h in range(case["Hkv"]):
                sc = q[h].matmul(k[:, h].t().contiguous()) / math.sqrt(case["D"])    # [G, n]
                heads = slice(h * case["G"], (h + 1) * case["G"])
                lse[b, heads] = torch.logsumexp(sc, 1)
                out[b, heads] = (sc - lse[b, heads, None]).exp().matmul(v[:, h].contiguous())
        return [out, lse]
    y = s["y"].double()
    for a in range(case["L"]):
        rows = (s["index"] == a).nonzero()[:, 0]
        t = s["x"][rows].double().matmul(s["A"][a].double().t().contiguous())
        y[rows] += s["scale"][a].double() * t.matmul(s["B"][a].double().t().contiguous())
    return [y]
