"""A decode step with drafted tokens, as cases.

Next to the one-token step of ``perf/operators.py``, a serving program that
drafts several tokens per sequence (a chain of them, or a tree) needs:

* ``norm_rope_append``: the norm of each query and key head, the rotary
  positions and the append to the paged cache, in one pass;
* ``tree_attention``: attention of a tree of drafted tokens per sequence over
  that cache, every token over the context and its own ancestors;
* ``verify_draft``: which drafted tokens the target's probabilities keep, from
  given random numbers, and the token that follows them;
* ``compact_cache``: the rows of the kept tokens moved to the end of the
  context, in every layer's cache;
* ``copy_pages``: pages of the cache copied for sequences that fork.

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
        # Four sequences of 16 drafted tokens, three rows of padding; q, k and v
        # are slices of one fused projection (latency).
        {"name": "norm_rope_64_f16", "op": "norm_rope_append", "T": 64, "pad": 3, "Hq": 32,
         "Hkv": 8, "D": 128, "rot": 128, "style": "half", "norm": "rms", "each": False,
         "page": 16, "layout": "hnd", "far": 131072, "dtype": "f16"},
        # The prefill of 8192 tokens, several prompts in one batch.
        {"name": "norm_rope_8192_bf16", "op": "norm_rope_append", "T": 8192, "pad": 0, "Hq": 32,
         "Hkv": 8, "D": 128, "rot": 128, "style": "half", "norm": "rms", "each": False,
         "page": 16, "layout": "nhd", "far": 8192, "dtype": "bf16"},
        # Odd token count, LayerNorms with weights for each head, partial
        # rotation of neighbouring pairs, pages whose size is no power of two.
        {"name": "norm_rope_333_f16", "op": "norm_rope_append", "T": 333, "pad": 5, "Hq": 28,
         "Hkv": 4, "D": 80, "rot": 40, "style": "pairs", "norm": "layer", "each": True,
         "page": 24, "layout": "nhd", "far": 1 << 20, "dtype": "f16"},
        # One short sequence with a chain of seven drafted tokens behind its
        # last one, every query head with its own key head (latency).
        {"name": "tree_1x8x300_f16", "op": "tree_attention", "B": 1, "T": 8, "L": 300, "Hkv": 32,
         "G": 1, "D": 128, "page": 16, "layout": "hnd", "window": 0, "tree": "chain", "pad": 0,
         "dtype": "f16"},
        # A serving batch of mixed lengths with two padded rows, trees of up to
        # 16 tokens, shared heads.
        {"name": "tree_16x16x4096_f16", "op": "tree_attention", "B": 16, "T": 16, "L": 4096,
         "Hkv": 8, "G": 4, "D": 128, "page": 16, "layout": "nhd", "window": 0, "tree": "ragged",
         "pad": 2, "dtype": "f16"},
        # Large trees over a few long contexts.
        {"name": "tree_4x64x32768_bf16", "op": "tree_attention", "B": 4, "T": 64, "L": 32768,
         "Hkv": 8, "G": 4, "D": 128, "page": 64, "layout": "hnd", "window": 0, "tree": "full",
         "pad": 0, "dtype": "bf16"},
        # A sliding window over long contexts, one key head for all queries.
        {"name": "tree_5x25x16384_w1000_bf16", "op": "tree_attention", "B": 5, "T": 25,
         "L": 16384, "Hkv": 1, "G": 12, "D": 64, "page": 32, "layout": "hnd", "window": 1000,
         "tree": "full", "pad": 0, "dtype": "bf16"},
        # One sequence's tree over a vocabulary of 32000 (latency).
        {"name": "verify_1x26x32000_f32", "op": "verify_draft", "B": 1, "T": 26, "V": 32000,
         "tree": "full", "pad": 0, "dtype": "f32"},
        # A batch of chains of five with the draft's own probabilities, a large
        # vocabulary.
        {"name": "verify_64x5x128000_f32", "op": "verify_draft", "B": 64, "T": 5, "V": 128000,
         "tree": "chain", "pad": 3, "dtype": "f32"},
        # The accepted rows of eight sequences, moved in 32 layers.
        {"name": "compact_8x32_l32_f16", "op": "compact_cache", "B": 8, "T": 32, "L": 600,
         "layers": 32, "Hkv": 8, "D": 128, "page": 16, "layout": "hnd", "dtype": "f16"},
        # A sequence forks: its last page, in 32 layers (latency).
        {"name": "copy_1_l32_f16", "op": "copy_pages", "N": 1, "layers": 32, "Hkv": 8, "D": 128,
         "page": 16, "layout": "nhd", "part": True, "dtype": "f16"},
        # Whole pages of long contexts copied, some of the list padding.
        {"name": "copy_300_l16_bf16", "op": "copy_pages", "N": 300, "layers": 16, "Hkv": 8,
         "D": 128, "page": 64, "layout": "hnd", "part": False, "dtype": "bf16"},
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))
    return max(lo, min(hi, v) // step * step)


def draw(rng):
    op = rng.choice(("norm_rope_append", "tree_attention", "tree_attention", "verify_draft",
                     "compact_cache", "copy_pages"))
    dtype = rng.choice(("f16", "bf16"))
    if op == "verify_draft":
        V = _log_int(rng, 1000, 160000)
        T = _log_int(rng, 1, 64)
        B = _log_int(rng, 1, max(1, min(128, 64 * 5 * 128000 // (V * T))))
        return {"op": op, "B": B, "T": T, "V": V, "tree": rng.choice(("chain", "ragged", "full")),
                "pad": rng.randrange(3) if B > 4 else 0,
                "dtype": rng.choice(("f32", "f32", "f16", "bf16"))}
    heads = rng.choice((1, 2, 4, 5, 8, 16, 32))
    group = rng.choice((1, 2, 3, 4, 6, 8, 16))
    dim = rng.choice((64, 80, 96, 128, 128, 256))
    page = rng.choice((8, 16, 16, 24, 32, 64, 128))
    layout = rng.choice(("hnd", "nhd"))
    if op == "norm_rope_append":
        T = _log_int(rng, 1, min(8192, (8192 * 48 * 128) // ((group + 2) * heads * dim)))
        return {"op": op, "T": T, "pad": rng.randrange(4) if T > 8 else 0, "Hq": heads * group,
                "Hkv": heads, "D": dim, "rot": rng.choice((dim, dim, dim // 2)),
                "style": rng.choice(("half", "pairs")), "norm": rng.choice(("rms", "rms", "layer")),
                "each": rng.random() < 0.3, "page": page, "layout": layout,
                "far": _log_int(rng, 8192, 1 << 20), "dtype": dtype}
    if op == "tree_attention":
        T = _log_int(rng, 1, 64)
        L = _log_int(rng, T, 32768)
        top = 4 * 32768 * 8 * 128 // (L * heads * dim)
        top = min(top, 4 * 64 * 32768 * 32 * 128 // (T * L * heads * group * dim))
        B = _log_int(rng, 1, max(1, min(64, top)))
        return {"op": op, "B": B, "T": T, "L": L, "Hkv": heads, "G": group, "D": dim, "page": page,
                "layout": layout, "window": rng.choice((0, 0, 0, _log_int(rng, 1, 4096))),
                "tree": rng.choice(("chain", "ragged", "full")),
                "pad": rng.randrange(3) if B > 4 else 0, "dtype": dtype}
    layers = _log_int(rng, 1, 48)
    if op == "compact_cache":
        T = _log_int(rng, 2, 64)
        L = _log_int(rng, T, 2048)
        top = 8 * 640 * 32 * 8 * 128 // ((L + page) * layers * heads * dim)
        return {"op": op, "B": _log_int(rng, 1, max(1, min(128, top))), "T": T, "L": L,
                "layers": layers, "Hkv": heads, "D": dim, "page": page, "layout": layout,
                "dtype": dtype}
    top = 300 * 16 * 8 * 64 * 128 // (layers * heads * page * dim)
    return {"op": op, "N": _log_int(rng, 1, max(1, min(1024, top))), "layers": layers,
            "Hkv": heads, "D": dim, "page": page, "layout": layout, "part": rng.random() < 0.4,
            "dtype": dtype}


# ---- what a case fixes beyond its sizes ---------------------------------------

def _lens(case):
    """Tokens in the cache of each sequence, the drafted ones included: spread over
    the logarithm up to L (which one has), the padded rows empty."""
    rng = random.Random("%(B)d %(T)d %(L)d %(D)d %(Hkv)d" % case)
    live = case["B"] - case.get("pad", 0)
    n = [_log_int(rng, max(case["T"], case["L"] // 8), case["L"]) for _ in range(live)]
    n[rng.randrange(live)] = case["L"]
    return n + [0] * case.get("pad", 0)


def _parents(case):
    """The parent of each drafted token: -1 the first one's (the last token that was
    sampled), -2 marks padding.  "chain": one after the other, "full": trees that use
    every place, "ragged": trees of up to T."""
    rng = random.Random("tree %(B)d %(T)d" % case)
    rows = []
    for b in range(case["B"]):
        T = case["T"]
        n = 0 if b >= case["B"] - case.get("pad", 0) else (
            rng.randint(max(1, T // 4), T) if case["tree"] == "ragged" else T)
        row = [-1] if n else []
        while len(row) < n:
            i = len(row)
            # Nodes of a level lie together, each with one to four children.
            row.append(i - 1 if case["tree"] == "chain"
                       else max(row[-1], 0) if rng.random() < 0.6 and row.count(row[-1]) < 4
                       else min(i - 1, max(row[-1], 0) + 1))
        rows.append(row + [-2] * (T - n))
    return rows


def _paths(case):
    """The nodes of each sequence that were kept, in order: the first few where they
    lie already, the others behind the last of their places."""
    rng = random.Random("path %(B)d %(T)d %(L)d" % case)
    rows = []
    for _ in range(case["B"]):
        n = min(case["T"], 1 + min(rng.randrange(9), rng.randrange(9)))
        keep = rng.randint(1, min(2, n))
        rest = range(n, case["T"])
        moved = sorted(rng.sample(rest, min(n - keep, len(rest))))
        rows.append(list(range(n - len(moved))) + moved)
    return rows


def _copies(case):
    """(source, destination, rows) of each pair, every eighth of many pairs padding."""
    rng = random.Random("copy %(N)d %(page)d %(Hkv)d" % case)
    pages = list(range(2 * case["N"] + 1))               # the last page stays out of it
    rng.shuffle(pages)
    out = []
    for i in range(case["N"]):
        pad = case["N"] > 8 and i % 8 == 7
        out.append((-1 if pad else pages[i], -1 if pad else pages[case["N"] + i],
                    rng.randint(1, case["page"]) if case["part"] else case["page"]))
    return out


# ---- inputs -------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype).mul_(scale)


def _int(v):
    return torch.tensor(v, device="cuda", dtype=torch.int32)


def _cache(g, pages, case, *layers):
    """A key or value cache [pages, heads, page, D] (with the layers before): heads first
    in memory ("hnd") or tokens first ("nhd")."""
    h, p, d = case["Hkv"], case["page"], case["D"]
    if case["layout"] == "hnd":
        return _randn(g, *layers, pages, h, p, d, dtype=DTYPES[case["dtype"]])
    return _randn(g, *layers, pages, p, h, d, dtype=DTYPES[case["dtype"]]).transpose(-3, -2)


def _table(g, lens, page):
    """(block table, pages): each sequence's pages in random order, -1 behind them."""
    need = [-(-n // page) for n in lens]
    order = torch.randperm(sum(need) + 3, generator=g, device="cuda").int()
    table = torch.full((len(lens), max(need)), -1, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(need) + 3


def _drafts(g, case):
    """Target probabilities [B, T, V], drafted tokens, uniforms, parents, and for chains
    the draft's probabilities.  A node's children are tokens that the target finds
    likely at it (of a chain: a sample of the draft's distribution, a near one)."""
    B, T, V, dt = case["B"], case["T"], case["V"], DTYPES[case["dtype"]]
    parents = _int(_parents(case))
    logits = _randn(g, B, T, V, scale=1.5)
    likely = torch.randint(0, V, (B, T, 6), generator=g, device="cuda")
    logits.scatter_add_(2, likely, 9.0 + _randn(g, B, T, 6, scale=1.5))
    at = parents.clamp(min=0).long()
    draft = None
    if case["tree"] == "chain":
        logits_d = logits + _randn(g, B, T, V, scale=0.6)
        draft = logits_d.softmax(-1).to(dt)
        noise = -torch.empty_like(logits_d).exponential_(generator=g).log_()
        tokens = logits_d.add_(noise).argmax(-1).gather(1, at)
    else:
        # The i-th child takes the i-th of its parent's likely tokens.
        older = (parents[:, :, None] == parents[:, None, :]).tril(-1).sum(-1) % 6
        tokens = likely.gather(1, at[..., None].expand(B, T, 6)).gather(2, older[..., None])[..., 0]
    return {"tokens": tokens.int(), "target": logits.softmax(-1).to(dt), "draft": draft,
            "parents": parents,
            "uniform": torch.rand(B, T, generator=g, device="cuda")}


def prepare(case, seed):
    g, dt = _gen(seed), DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "verify_draft":
        s.update(_drafts(g, case))
    elif case["op"] == "norm_rope_append":
        T, hq, hkv, d = case["T"], case["Hq"], case["Hkv"], case["D"]
        qkv = (_randn(g, T, hq + 2 * hkv, d, scale=1.7) + 0.1).to(dt)   # the fused projection
        s["q"], s["k"], s["v"] = qkv.split((hq, hkv, hkv), dim=1)
        for w, h in (("q", hq), ("k", hkv)):
            shape = (h, d) if case["each"] else (d,)
            s[w + "_w"] = (1 + _randn(g, *shape, scale=0.1)).to(dt)
            s[w + "_b"] = _randn(g, *shape, scale=0.1).to(dt) if case["norm"] == "layer" else None
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
    elif case["op"] == "tree_attention":
        lens = _lens(case)
        s["table"], pages = _table(g, lens, case["page"])
        s["lens"], s["parents"] = _int(lens), _int(_parents(case))
        s["k_cache"], s["v_cache"] = _cache(g, pages, case), _cache(g, pages, case)
        s["q"] = _randn(g, case["B"], case["T"], case["Hkv"] * case["G"], case["D"],
                        scale=1.5).to(dt)
    elif case["op"] == "compact_cache":
        lens = _lens(case)
        s["table"], pages = _table(g, lens, case["page"])
        s["lens"] = _int(lens)
        s["k_cache"], s["v_cache"] = (_cache(g, pages, case, case["layers"]) for _ in "kv")
        paths = _paths(case)
        s["path"] = _int([p + [-1] * (case["T"] - len(p)) for p in paths])
        s["counts"] = _int([len(p) for p in paths])
    else:
        pages = 2 * case["N"] + 2
        s["k_cache"], s["v_cache"] = (_cache(g, pages, case, case["layers"]) for _ in "kv")
        src, dst, rows = zip(*_copies(case))
        s["src"], s["dst"] = _int(src), _int(dst)
        s["rows"] = _int(rows) if case["part"] else None
    return s


EPS = 1e-6


# ---- plain forms --------------------------------------------------------------

def _plain_norm(x, kind, w, b):
    x = x.float()
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.float()
    return x if b is None else x + b.float()


def _plain_rotate(f, cos, sin, rot, style):
    r = f[..., :rot]
    a, b = (r[..., :rot // 2], r[..., rot // 2:]) if style == "half" else (r[..., 0::2],
                                                                          r[..., 1::2])
    u, v = a * cos - b * sin, b * cos + a * sin
    r = torch.cat((u, v), -1) if style == "half" else torch.stack((u, v), -1).flatten(-2)
    return torch.cat((r, f[..., rot:]), -1)


def _plain_norm_rope_append(s):
    c, dt = s["case"], s["q"].dtype
    cs = s["cos_sin"][s["positions"]][:, None]
    cos, sin = cs[..., :c["rot"] // 2], cs[..., c["rot"] // 2:]
    q, k = (_plain_rotate(_plain_norm(s[w], c["norm"], s[w + "_w"], s[w + "_b"]), cos, sin,
                          c["rot"], c["style"]).to(dt) for w in "qk")
    n = c["T"] - c["pad"]                                # the rows that are no padding
    page, off = s["slots"][:n] // c["page"], s["slots"][:n] % c["page"]
    s["k_cache"][page, :, off] = k[:n]
    s["v_cache"][page, :, off] = s["v"][:n]
    return [q, s["k_cache"], s["v_cache"]]


def _ancestors(parents):
    """Bool [B, T, T]: whether node j is node i or above it; False for padded i."""
    T = parents.shape[1]
    node = torch.arange(T, device=parents.device)
    up = (parents[..., None] == node).float()            # one step
    up = up + torch.eye(T, device=parents.device)
    for _ in range(6):                                   # 64 steps
        up = (up @ up.contiguous()).clamp(max=1)
    return (up > 0) & (parents >= -1)[..., None]


def _plain_tree_attention(s):
    c = s["case"]
    B, T, w = c["B"], c["T"], c["window"]
    n = min(c["L"], w + T - 1 if w else c["L"])          # the last n tokens, right-aligned
    pos = s["lens"][:, None] - n + torch.arange(n, device="cuda", dtype=torch.int32)
    at = pos.clamp(min=0)
    page = s["table"].gather(1, (at // c["page"]).long()).clamp(min=0)
    k = s["k_cache"][page, :, at % c["page"]].float().permute(0, 2, 3, 1)    # [B, H, D, n]
    v = s["v_cache"][page, :, at % c["page"]].float().transpose(1, 2)        # [B, H, n, D]
    # What each node sees: of the context what its window holds, of the drafted
    # tokens its ancestors and itself (those too by their depth).
    up = _ancestors(s["parents"])
    depth = up.sum(-1) - 1
    first = s["lens"][:, None] - T + depth - (w - 1 if w else 1 << 30)       # [B, T]
    ctx = s["lens"][:, None] - T
    tok = torch.minimum(pos, ctx - 1)[:, None]                               # [B, 1, n]
    see = (pos >= 0)[:, None] & (tok >= first[..., None]) & (s["parents"] >= -1)[..., None]
    m = min(n, T)
    drafted = up & (ctx[..., None] + depth[:, None, :] >= first[..., None])
    see[..., n - m:] = drafted[..., T - m:]
    q = s["q"].float().view(B, T, c["Hkv"], c["G"], c["D"]).transpose(1, 2)
    q = q.reshape(B, c["Hkv"], T * c["G"], c["D"])
    sc = (q @ k.contiguous() * c["D"] ** -0.5).view(B, c["Hkv"], T, c["G"], n)
    sc.masked_fill_(~see[:, None, :, None], -math.inf)
    top = sc.amax(-1, keepdim=True).clamp(min=-1e30)
    p = sc.sub_(top).exp_()
    z = p.sum(-1, keepdim=True)
    out = (p.view(B, c["Hkv"], T * c["G"], n) @ v.contiguous()).view(B, c["Hkv"], T, c["G"], -1)
    out = out / z.clamp(min=1e-30)                       # a row that sees nothing gives zeros
    lse = (top + z.log()).masked_fill(z == 0, -math.inf)[..., 0]
    return [out.transpose(1, 2).reshape(s["q"].shape).to(s["q"].dtype),
            lse.transpose(1, 2).reshape(B, T, -1)]


def _plain_verify_draft(s):
    c, parents = s["case"], s["parents"]
    B, T, V = c["B"], c["T"], c["V"]
    at, token = parents.clamp(min=0).long(), s["tokens"].long()
    rows = torch.arange(B, device="cuda")[:, None]
    p = s["target"][rows, at, token].double()            # of each token, at its parent
    brothers = (parents[:, :, None] == parents[:, None, :]) & (parents >= 0)[..., None]
    older = brothers.tril(-1)
    if s["draft"] is not None:
        bound = s["uniform"].double() * s["draft"][rows, at, token].double()
        ok = ~older.any(-1)                              # a chain: the first child
    else:
        # Brothers in turn: what is left when the older ones are not kept.
        same = (token[:, :, None] == token[:, None, :]) & older
        fresh = ~same.any(-1)                            # the first brother of its token
        left = 1 - ((older & fresh[:, None, :]) * p[:, None, :]).sum(-1)
        bound, p = s["uniform"].double() * left, p * fresh
        ok = torch.ones_like(fresh)
    ok = ok & (bound < p) & (parents >= 0)
    ok = ok & ~(older & ok[:, None, :]).any(-1)          # the first that is kept
    ok[:, 0] = parents[:, 0] == -1
    kept = (_ancestors(parents) <= ok[:, None, :]).all(-1) & (parents >= -1)
    counts = kept.sum(-1)
    path = torch.where(kept, torch.arange(T, device="cuda"), T).sort(-1).values
    path = path.masked_fill(path == T, -1)
    # The token after the last kept one: from what the target leaves there.
    last = path.gather(1, (counts - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    row = torch.arange(B, device="cuda")
    w = s["target"][row, last].double()
    tried = parents == last[:, None]
    if s["draft"] is not None:
        rest = (w - s["draft"][row, last].double()).clamp(min=0)
        w_left = torch.where(tried.any(-1, keepdim=True), rest, w)
    else:
        gone = torch.zeros(B, V + 1, device="cuda", dtype=torch.bool)
        gone.scatter_(1, torch.where(tried, token, V), True)
        w_left = w.masked_fill(gone[:, :V], 0)
    w = torch.where(w_left.sum(-1, keepdim=True) > 0, w_left, w)
    run = w.cumsum(-1)
    nth = (run <= s["uniform"][:, :1].double() * w.sum(-1, keepdim=True)).sum(-1)
    end = torch.where(w > 0, torch.arange(V, device="cuda"), -1).amax(-1)
    following = torch.minimum(nth, end).masked_fill(counts == 0, -1)
    return [path.int(), counts.int(), following.int()]


def _plain_compact_cache(s):
    c = s["case"]
    ctx = (s["lens"] - c["T"])[:, None]
    k = torch.arange(c["T"], device="cuda")
    live = k < s["counts"][:, None]
    frm, to = ctx + torch.where(live, s["path"], k), ctx + k       # the others stay
    fp = s["table"].gather(1, (frm // c["page"]).long()).long()
    tp = s["table"].gather(1, (to // c["page"]).long()).long()
    fo, to = (frm % c["page"]).long(), (to % c["page"]).long()
    for x in (s["k_cache"], s["v_cache"]):
        moved = x[:, fp, :, fo]                          # read whole before it is written
        x[:, tp, :, to] = torch.where(live[..., None, None, None], moved, x[:, tp, :, to])
    return [s["k_cache"], s["v_cache"], (ctx[:, 0] + s["counts"]).int()]


def _plain_copy_pages(s):
    c = s["case"]
    live = s["src"] >= 0
    # A padded pair copies the last page onto itself.
    src = torch.where(live, s["src"], s["k_cache"].shape[1] - 1)
    dst = torch.where(live, s["dst"], s["k_cache"].shape[1] - 1)
    for x in (s["k_cache"], s["v_cache"]):
        if s["rows"] is None:
            x[:, dst] = x[:, src]
        else:
            keep = torch.arange(c["page"], device="cuda") < s["rows"][:, None]
            x[:, dst] = torch.where(keep[:, None, :, None], x[:, src], x[:, dst])
    return [s["k_cache"], s["v_cache"]]


# ---- the framework's calls ----------------------------------------------------

def _ops():
    path = os.path.join(os.getcwd(), "hexagon-mlir_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    import hxm.ops as ops
    return ops


def _own(s):
    ops, c = _ops(), s["case"]
    if c["op"] == "norm_rope_append":
        q = ops.norm_rope_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"],
                                 s["positions"], s["cos_sin"], norm=c["norm"], q_weight=s["q_w"],
                                 k_weight=s["k_w"], q_bias=s["q_b"], k_bias=s["k_b"], eps=EPS,
                                 interleaved=c["style"] == "pairs")
        return [q, s["k_cache"], s["v_cache"]]
    if c["op"] == "tree_attention":
        return list(ops.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"],
                                       None if c["tree"] == "chain" and not c["pad"]
                                       else s["parents"], window=c["window"], return_lse=True))
    if c["op"] == "verify_draft":
        return list(ops.verify_draft(s["tokens"], s["target"], s["uniform"], s["parents"],
                                     s["draft"]))
    if c["op"] == "compact_cache":
        lens = ops.compact_cache(s["k_cache"], s["v_cache"], s["table"], s["lens"], s["path"],
                                 s["counts"])
        return [s["k_cache"], s["v_cache"], lens]
    ops.copy_pages(s["k_cache"], s["v_cache"], s["src"], s["dst"], s["rows"])
    return [s["k_cache"], s["v_cache"]]


PLAIN = {"norm_rope_append": _plain_norm_rope_append, "tree_attention": _plain_tree_attention,
         "verify_draft": _plain_verify_draft, "compact_cache": _plain_compact_cache,
         "copy_pages": _plain_copy_pages}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


# ---- the least a pass moves and computes --------------------------------------

def work(case):
    eb = BYTES[case["dtype"]]
    if case["op"] == "verify_draft":
        B, T, live = case["B"], case["T"], case["B"] - case["pad"]
        tables = 2 if case["tree"] == "chain" else 1
        # A row of the vocabulary (of the draft's too), the drafted tokens' own values.
        return {"bytes": live * tables * (case["V"] + T) * eb + B * T * 16 + 8 * B,
                "flops": 2 * live * tables * case["V"]}
    if case["op"] == "norm_rope_append":
        T, n, d = case["T"], case["T"] - case["pad"], case["D"]
        moved = 2 * T * case["Hq"] * d + 4 * n * case["Hkv"] * d
        return {"bytes": moved * eb + 4 * T * (case["rot"] + 2),
                "flops": T * (case["Hq"] + case["Hkv"]) * (4 * d + 3 * case["rot"])}
    if case["op"] == "tree_attention":
        T, w, hq = case["T"], case["window"], case["Hkv"] * case["G"]
        lens = _lens(case)
        read = [min(n, w + T - 1 if w else n) for n in lens]
        seen = sum(min(n - T + 1, w or n) for n in lens if n)
        nodes = sum(p > -2 for row in _parents(case) for p in row) / (case["B"] - case["pad"])
        return {"bytes": (2 * sum(read) * case["Hkv"] * case["D"]
                          + 2 * case["B"] * T * hq * case["D"]) * eb
                + sum(-(-n // case["page"]) for n in read) * 4 + case["B"] * (4 + 4 * T * (hq + 1)),
                "flops": 4 * seen * nodes * hq * case["D"]}
    row = 2 * case["layers"] * case["Hkv"] * case["D"] * eb        # of keys and values
    if case["op"] == "compact_cache":
        moved = sum(n != i for p in _paths(case) for i, n in enumerate(p))
        return {"bytes": 2 * moved * row + 4 * case["B"] * (case["T"] + 3), "flops": 0}
    rows = sum(r for a, _, r in _copies(case) if a >= 0)
    return {"bytes": 2 * rows * row + 12 * case["N"], "flops": 0}


# ---- the definition, in 64 bits -----------------------------------------------

def _norm64(x, kind, w, b):
    mean = x.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(x[..., :1])
    var = (x - mean).pow(2).sum(-1, keepdim=True) / x.shape[-1]
    y = (x - mean) / (var + EPS).sqrt() * w.double()
    return y if b is None else y + b.double()


def _walk64(case, s, b):
    """(path, the following token) of one sequence, node by node."""
    parents, tokens = s["parents"][b].tolist(), s["tokens"][b].tolist()
    u = s["uniform"][b].double().tolist()
    if parents[0] != -1:
        return [], -1
    path, V = [0], case["V"]
    while True:
        p = s["target"][b, path[-1]].double()
        children = [i for i in range(path[-1] + 1, case["T"]) if parents[i] == path[-1]]
        if s["draft"] is not None:
            children = children[:1]
        left, w, chosen = 1.0, p, None
        for i in children:
            x = tokens[i]
            q = 1.0 if s["draft"] is None else float(s["draft"][b, path[-1], x])
            if u[i] * q * left < float(w[x]):
                chosen = i
                break
            if s["draft"] is None:
                left -= float(w[x])
                w = w.clone()
                w[x] = 0
            else:
                w = (p - s["draft"][b, path[-1]].double()).clamp(min=0)
        if chosen is not None:
            path.append(chosen)
            continue
        if not float(w.sum()) > 0:
            w = p
        passed = (w.cumsum(0) > u[0] * w.sum()) & (w > 0)
        first = int(passed.int().argmax()) if bool(passed.any()) else int((w > 0).nonzero()[-1])
        assert 0 <= first < V
        return path, first


def _above(parents, i):
    out = []
    while i >= 0:
        out.append(i)
        i = parents[i]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "verify_draft":
        got = [_walk64(case, s, b) for b in range(case["B"])]
        return [_int([p + [-1] * (case["T"] - len(p)) for p, _ in got]),
                _int([len(p) for p, _ in got]), _int([x for _, x in got])]
    if case["op"] == "norm_rope_append":
        rot, half = case["rot"], case["rot"] // 2
        first = torch.arange(half, device="cuda")
        if case["style"] == "half":
            i, j = first, first + half
        else:
            i, j = 2 * first, 2 * first + 1
        cs = s["cos_sin"].double()[s["positions"].long()].unsqueeze(1)

        def turn(w):
            x = _norm64(s[w].double(), case["norm"], s[w + "_w"], s[w + "_b"])
            y = x.clone()
            y[..., i] = x[..., i] * cs[..., :half] - x[..., j] * cs[..., half:]
            y[..., j] = x[..., i] * cs[..., half:] + x[..., j] * cs[..., :half]
            return y
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        live = s["slots"] >= 0
        slot = s["slots"][live].long()
        kc.transpose(1, 2)[slot // case["page"], slot % case["page"]] = turn("k")[live]
        vc.transpose(1, 2)[slot // case["page"], slot % case["page"]] = s["v"][live].double()
        return [turn("q"), kc, vc]
    if case["op"] == "tree_attention":
        T, page, G, w = case["T"], case["page"], case["G"], case["window"]
        out = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
        lse = torch.full(s["q"].shape[:3], -math.inf, device="cuda", dtype=torch.float64)
        for b, n in enumerate(_lens(case)):
            if not n:
                continue
            parents = s["parents"][b].tolist()
            lo = max(0, n - (w + T - 1)) if w else 0
            pages = s["table"][b, lo // page:-(-n // page)].long()
            skip = lo - lo // page * page
            k, v = (s[x][pages].transpose(1, 2).flatten(0, 1)[skip:skip + n - lo].double()
                    for x in ("k_cache", "v_cache"))
            see = torch.zeros(T, n - lo, dtype=torch.bool)
            for i in range(T):
                if parents[i] < -1:
                    continue
                up = _above(parents, i)
                depth = len(up) - 1
                first = max(lo, n - T + depth - w + 1) if w else lo
                see[i, first - lo:n - T - lo] = True
                for j in up:
                    if not w or len(_above(parents, j)) - 1 > depth - w:
                        see[i, n - T + j - lo] = True
            see = see.cuda()
            live = see.any(1)
            for h in range(case["Hkv"]):
                q = s["q"][b, :, h * G:(h + 1) * G].double().reshape(T * G, -1)
                sc = q.matmul(k[:, h].t().contiguous()) / math.sqrt(case["D"])
                sc = sc.view(T, G, -1).masked_fill(~see[:, None], -math.inf)
                at = slice(h * G, (h + 1) * G)
                lse[b, :, at] = torch.logsumexp(sc, 2)
                e = (sc - lse[b, :, at, None]).masked_fill(~see[:, None], -math.inf).exp()
                o = e.view(T * G, -1).matmul(v[:, h].contiguous()).view(T, G, -1)
                out[b, :, at] = o.masked_fill(~live[:, None, None], 0)
        return [out, lse]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    if case["op"] == "compact_cache":
        page, table, lens = case["page"], s["table"].tolist(), _lens(case)
        for x in (kc, vc):
            old = x.clone()
            for b, path in enumerate(_paths(case)):
                for i, node in enumerate(path):
                    a, z = lens[b] - case["T"] + node, lens[b] - case["T"] + i
                    x[:, table[b][z // page], :, z % page] = old[:, table[b][a // page], :,
                                                                 a % page]
        return [kc, vc, _int([n - case["T"] + len(p) for n, p in zip(lens, _paths(case))])]
    for x in (kc, vc):
        for a, z, rows in _copies(case):
            if a >= 0:
                x[:, z, :, :rows] = x[:, a, :, :rows]
    return [kc, vc]
