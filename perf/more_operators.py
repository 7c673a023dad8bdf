"""The operators of speculative serving over a quantised paged cache, as cases that can be timed and checked.

Six kinds, each one call of the package (qwen3_tts_amd.hip, declared in include/qwen_tts_hip.h):

  append8   qwen_hip_op_page_append into a cache of e4m3 codes: rows of q, k, v -> per-head RMSNorm, RoPE, q out, k and v
            as codes with one power-of-two scale a row.
  attn8     qwen_hip_op_page_attention over such a cache.
  treeplan  qwen_hip_op_tree_plan: the parents of drafted tokens -> positions and bit masks of their ancestors.
  tree      qwen_hip_op_tree_attention: a tree of drafted tokens a request over its paged cache.
  verify    qwen_hip_op_tree_verify: drafted trees against the target's probabilities, by given random numbers.
  commit    qwen_hip_op_tree_commit: the accepted path's rows moved together in every layer's cache, lengths, pages given back.

`own` false: the same results from elementary torch operations.
"""
import ctypes
import importlib.util
import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-6
THETA = 1e6
E4M3_MAX = 448.0
MIN_EXP = -64        # smallest exponent of a row's scale


def listed():
    return [
        # 32 streams' step in the Talker's head layout and activation type
        {"name": "append8-decode-T32-f32", "kind": "append8", "T": 32, "nh": 16, "nkv": 8, "hd": 128, "type": "f32", "page": 16, "norm": 1,
         "layout": "head"},
        # a step's worth of long prompts
        {"name": "append8-prompts-T8190-bf16", "kind": "append8", "T": 8190, "nh": 16, "nkv": 8, "hd": 128, "type": "bf16", "page": 64,
         "norm": 1, "layout": "slot"},
        # a busy server with long utterances: bound by the cache's bytes
        {"name": "attn8-decode-B64-bf16", "kind": "attn8", "B": 64, "lo": 1000, "hi": 8000, "new_lo": 1, "new_hi": 1, "nh": 16, "nkv": 8,
         "hd": 128, "type": "bf16", "cache": "e4m3", "page": 64, "window": 0, "layout": "head"},
        # chunks of prompts that continue a cached prefix: bound by the products
        {"name": "attn8-chunk-B6-bf16", "kind": "attn8", "B": 6, "lo": 0, "hi": 6000, "new_lo": 100, "new_hi": 1024, "nh": 16, "nkv": 8,
         "hd": 128, "type": "bf16", "cache": "e4m3", "page": 16, "window": 0, "layout": "slot"},
        # a few streams with short drafts
        {"name": "treeplan-B8", "kind": "treeplan", "B": 8, "lo": 100, "hi": 3000, "new_lo": 5, "new_hi": 16, "width": 4},
        # a large server, trees of all sizes
        {"name": "treeplan-B512", "kind": "treeplan", "B": 512, "lo": 0, "hi": 6000, "new_lo": 1, "new_hi": 61, "width": 9},
        # a handful of streams, f32 queries over the bf16 cache
        {"name": "tree-B4-f32", "kind": "tree", "B": 4, "lo": 200, "hi": 1500, "new_lo": 7, "new_hi": 13, "width": 4, "nh": 16, "nkv": 8,
         "hd": 128, "type": "f32", "cache": "bf16", "page": 16, "window": 0, "layout": "head"},
        # large trees of many streams over the quantised cache
        {"name": "tree-B32-bf16-e4m3", "kind": "tree", "B": 32, "lo": 500, "hi": 6000, "new_lo": 33, "new_hi": 64, "width": 12, "nh": 16,
         "nkv": 8, "hd": 128, "type": "bf16", "cache": "e4m3", "page": 64, "window": 0, "layout": "head"},
        # a few streams' codec tokens, drafted as chains by a small model
        {"name": "verify-B6-V2048-f32", "kind": "verify", "B": 6, "V": 2048, "new_lo": 3, "new_hi": 6, "width": 1, "type": "f32", "draft": 1},
        # a text vocabulary of odd size, trees drawn from a draft model's probabilities
        {"name": "verify-B64-V128003-bf16", "kind": "verify", "B": 64, "V": 128003, "new_lo": 5, "new_hi": 13, "width": 3, "type": "bf16",
         "draft": 1},
        # one layer's cache, a few streams
        {"name": "commit-B8-bf16", "kind": "commit", "B": 8, "lo": 30, "hi": 300, "new_lo": 6, "new_hi": 16, "width": 4, "nkv": 8, "hd": 128,
         "cache": "bf16", "page": 16, "layout": "head", "layers": 1},
        # all 28 layers of the Talker, many streams, quantised
        {"name": "commit-B64-L28-e4m3", "kind": "commit", "B": 64, "lo": 60, "hi": 400, "new_lo": 17, "new_hi": 64, "width": 8, "nkv": 8,
         "hd": 128, "cache": "e4m3", "page": 16, "layout": "head", "layers": 28},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("append8", "attn8", "attn8", "treeplan", "tree", "tree", "verify", "verify", "commit"))
    page = rng.choice((8, 16, 16, 32, 64, 100))
    layout = rng.choice(("head", "slot"))
    nh, nkv, hd = rng.choice(((16, 8, 128), (16, 8, 128), (16, 16, 64), (32, 4, 128), (12, 2, 64)))
    heads = {"nh": nh, "nkv": nkv, "hd": hd}
    if kind == "append8":
        return {"kind": kind, "T": _log(rng, 1, 8000), **heads, "type": rng.choice(("f32", "bf16", "f16")), "page": page,
                "norm": rng.randint(0, 1), "layout": layout}
    if kind == "attn8":
        lo = rng.randint(0, 300)
        one = rng.randint(0, 1)
        return {"kind": kind, "B": _log(rng, 1, 64 if one else 8), "lo": lo, "hi": lo + _log(rng, 1, 7500), "new_lo": 1,
                "new_hi": 1 if one else _log(rng, 1, 600), **heads, "type": rng.choice(("f32", "bf16", "f16")), "cache": "e4m3", "page": page,
                "window": rng.choice((0, 0, 72, 1000)), "layout": layout}
    n = rng.randint(1, 20)
    new = {"new_lo": n, "new_hi": n + rng.randint(0, 40), "width": rng.choice((1, 2, 4, 10))}
    if kind == "treeplan":
        lo = rng.randint(0, 500)
        return {"kind": kind, "B": _log(rng, 1, 600), "lo": lo, "hi": lo + _log(rng, 1, 6000), **new, "width": rng.choice((2, 4, 10))}
    if kind == "tree":
        t, cache = rng.choice((("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "e4m3"), ("bf16", "e4m3"), ("f16", "e4m3")))
        lo = rng.randint(0, 300)
        return {"kind": kind, "B": _log(rng, 1, 32), "lo": lo, "hi": lo + _log(rng, 1, 6000), **new, **heads, "type": t, "cache": cache,
                "page": page, "window": rng.choice((0, 0, 0, 200)), "layout": layout}
    if kind == "verify":
        n = rng.randint(1, 8)
        return {"kind": kind, "B": _log(rng, 1, 64), "V": _log(rng, 1000, 128000), "new_lo": n, "new_hi": n + rng.randint(0, 5),
                "width": rng.choice((1, 2, 4)), "type": rng.choice(("f32", "bf16", "f16")), "draft": rng.choice((0, 1, 1))}
    lo = rng.randint(0, 60)
    return {"kind": kind, "B": _log(rng, 1, 64), "lo": lo, "hi": lo + _log(rng, 1, 400), **new, "nkv": nkv, "hd": hd,
            "cache": rng.choice(("bf16", "f16", "e4m3", "e4m3")), "page": page, "layout": layout, "layers": _log(rng, 1, 16)}


# ---- lengths, from the case alone --------------------------------------------------------------


def _spread(lo, hi, n, phase=0):
    """n whole numbers evenly from lo to hi, in an order with no trend."""
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, n) == 1)
    return [v[(i * step + phase) % n] for i in range(n)]


def _requests(c):
    """(tokens in the cache before, new tokens) of each request."""
    return _spread(c.get("lo", 0), c.get("hi", 0), c["B"]), _spread(c["new_lo"], c["new_hi"], c["B"], 1)


def _blocks(n, page):
    return (n + page - 1) // page


def _cu(lens):
    v = [0]
    for n in lens:
        v.append(v[-1] + n)
    return v


# ---- inputs, from a seed -----------------------------------------------------------------------


def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFFFFFF)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (std * torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)).to(dtype)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _shuffled(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)).to(torch.int32)


def _tables(need, pages, width):
    """Block tables of `need` pages a request out of the shuffled `pages`, -1 past them."""
    t = torch.full((len(need), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = pages[at:at + n]
        at += n
    return t.to(DEV)


def _seen(x, layout):
    """A pool [...][page][head][slot] (and [hd]) whatever the order in memory: `slot` has [page][slot][head]."""
    return x if layout == "head" else x.transpose(-3, -2)


def _pool(c, seed, n_pages, layers=None):
    """A cache's pages, filled: K about N(0, 1) (normed per head), V a projection's N(0, 0.7), as values of the cache's
    type or as e4m3 codes with a scale's exponent byte a row. All seen as [layer][page][kv head][slot][head_dim]."""
    a, b = (c["nkv"], c["page"]) if c["layout"] == "head" else (c["page"], c["nkv"])
    shape = ((layers,) if layers else ()) + (n_pages, a, b, c["hd"])
    s = {}
    for at, (n, std) in enumerate((("k", 1.0), ("v", 0.7))):
        x = std * torch.randn(shape, generator=_gen(seed, 11 + at), device=DEV, dtype=torch.float32)
        if c["cache"] != "e4m3":
            s[n] = _seen(x.to(TYPES[c["cache"]]), c["layout"])
            continue
        codes, e = _quantised(x)
        s[n] = _seen(codes.view(torch.uint8), c["layout"])
        s[n + "s"] = e if c["layout"] == "head" else e.transpose(-2, -1)
    return s


def _two(e):
    """2^e in 32 bits, -126 <= e <= 127."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantised(x):
    """e4m3 codes and the exponent byte of each row's scale: the least 2^e, e >= MIN_EXP, with max |x| <= 448 2^e."""
    m = x.abs().amax(-1)
    f, e = torch.frexp(m / E4M3_MAX)                            # m / 448 = f 2^e, f in [1/2, 1): 2^e is enough, 2^(e-1) if f = 1/2
    e = torch.where(m > 0, torch.where(f == 0.5, e - 1, e), MIN_EXP).clamp(min=MIN_EXP)
    e = e + (m > E4M3_MAX * _two(e)).int()                      # (the quotient was rounded)
    return (x * _two(-e)[..., None]).to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _values(codes, scale):
    """Values of codes (as bytes) under their rows' exponent bytes."""
    return codes.view(torch.float8_e4m3fn).float() * _two(scale.int() - 127)[..., None]


def _trees(c, seed, lens):
    """Parents within each request, packed: a token's parent is one of the `width` before it, the last one most often."""
    g = torch.Generator().manual_seed((int(seed) * 31 + 7) & 0x7FFFFFFF)
    parents = []
    for n in lens:
        back = (torch.rand(n, generator=g).square() * c["width"]).to(torch.int32)
        i = torch.arange(n, dtype=torch.int32)
        parents.append(torch.where(i > 0, (i - 1 - back).clamp(min=0), -1))
    return torch.cat(parents).to(torch.int32).to(DEV)


def prepare(case, seed):
    c = dict(case)
    return globals()["_prepare_" + c["kind"]](c, seed)


def _rope(n, hd):
    inv = THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _prepare_append8(c, seed):
    T, page, t = c["T"], c["page"], TYPES[c["type"]]
    n_pages = _blocks(T, page) + 8
    g = _gen(seed, 1)
    rows = _randn(g, T, (c["nh"] + 2 * c["nkv"]) * c["hd"], dtype=t)
    slot = _shuffled(n_pages * page, seed)[:T].to(DEV)
    pos = torch.randint(0, 8192, (T,), generator=g, device=DEV, dtype=torch.int32)
    cos, sin = _rope(8192, c["hd"])
    return {"case": c, "rows": rows, **_pool({**c, "cache": "e4m3"}, seed, n_pages), "slot": slot, "pos": pos, "cos": cos, "sin": sin,
            "n_pages": n_pages, "qn": 1 + _randn(g, c["hd"], std=0.1), "kn": 1 + _randn(g, c["hd"], std=0.1),
            "q_out": torch.zeros(T, c["nh"] * c["hd"], dtype=t, device=DEV)}


def _prepare_attn8(c, seed):
    old, new = _requests(c)
    kv = [o + n for o, n in zip(old, new)]
    need = [_blocks(n, c["page"]) for n in kv]
    n_pages = sum(need) + 5
    q = _randn(_gen(seed, 1), sum(new), c["nh"], c["hd"], dtype=TYPES[c["type"]], std=1.5)
    return {"case": c, "q": q, **_pool(c, seed, n_pages), "n_pages": n_pages, "table": _tables(need, _shuffled(n_pages, seed), max(need) + 3),
            "kv_len": _int(kv), "cu": _int(_cu(new)), "out": torch.zeros_like(q), "max_q": max(new), "max_kv": max(kv)}


def _prepare_treeplan(c, seed):
    old, new = _requests(c)
    words = _blocks(max(new), 32)
    T = sum(new)
    more = torch.randint(0, 64, (c["B"],), generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)).tolist()
    return {"case": c, "parent": _trees(c, seed, new), "cu": _int(_cu(new)), "kv_len": _int([o + n + m for o, n, m in zip(old, new, more)]), "T": T,
            "words": words, "max_q": max(new), "pos": _int([0] * T), "mask": torch.zeros(T, words, dtype=torch.int32, device=DEV)}


def _prepare_tree(c, seed):
    s = {**_prepare_treeplan(c, seed), **_prepare_attn8(c, seed)}
    p = _plain_treeplan(s)
    return {**s, **p}


def _prepare_verify(c, seed):
    _, new = _requests(c)
    T, B, V, t = sum(new), c["B"], c["V"], TYPES[c["type"]]
    g = _gen(seed, 1)
    cu, parent = _cu(new), _trees(c, seed, new)
    s = {"case": c, "cu": _int(cu), "parent": parent, "max_q": max(new), "T": T}
    # the target's probabilities after each token, and a draft model's that are near them
    x = _randn(g, T, V, std=3.0)
    s["p"] = x.softmax(-1).to(t)
    x += _randn(g, T, V, std=0.6)
    q = x.softmax(-1)
    del x
    first = torch.repeat_interleave(_int(cu[:-1]).long(), torch.tensor(new, device=DEV))
    at = first + parent.long().clamp(min=0)
    if c["draft"]:
        s["q"] = q.to(t)
        q = s["q"].float()
    # each token drawn from its parent's row; the roots are tokens of before
    cum = q.double().cumsum(-1)
    pick = torch.rand(T, generator=g, device=DEV, dtype=torch.float64) * cum[at, -1]
    s["tok"] = torch.searchsorted(cum[at], pick[:, None], right=True)[:, 0].clamp(max=V - 1).to(torch.int32)
    s["u"] = torch.rand(T, generator=g, device=DEV)
    s["r"] = torch.rand(B, generator=g, device=DEV)
    s.update(path=_int([0] * T), out_tok=_int([0] * T), n_path=_int([0] * B))
    return s


def _prepare_commit(c, seed):
    old, new = _requests(c)
    B, page, T = c["B"], c["page"], sum(new)
    kv = [o + n for o, n in zip(old, new)]
    need = [_blocks(n, page) for n in kv]
    n_free = 40
    n_pages = sum(need) + n_free
    pages = _shuffled(n_pages, seed)
    parent = _trees(c, seed, new).cpu()
    g = torch.Generator().manual_seed((int(seed) * 13 + 5) & 0x7FFFFFFF)
    cu, path, n_path = _cu(new), torch.full((T,), -1, dtype=torch.int32), []
    for b, n in enumerate(new):  # a walk from a random node up to the root, as verification leaves it
        at, up = int(torch.randint(0, n, (1,), generator=g)), []
        while at >= 0:
            up.append(at)
            at = int(parent[cu[b] + at])
        path[cu[b]:cu[b] + len(up)] = torch.tensor(up[::-1], dtype=torch.int32)
        n_path.append(len(up))
    free = torch.full((n_pages,), -1, dtype=torch.int32)
    free[:n_free] = pages[sum(need):]
    return {"case": c, **_pool(c, seed, n_pages, c["layers"]), "n_pages": n_pages, "cu": _int(cu), "kv_len": _int(kv), "path": path.to(DEV),
            "n_path": _int(n_path), "table": _tables(need, pages, max(need) + 2), "free": free.to(DEV), "n_free": _int([n_free]), "T": T,
            "max_q": max(new), "kv_out": _int([0] * B), "n_free_out": _int([0]), "status": _int([0])}


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return globals()["_plain_" + state["case"]["kind"]](state)


def _norm_rope(x, gain, cos, sin, dt):
    """x [T][heads][hd]: RMSNorm over hd times gain (None: none), then the halves rotated by the angles."""
    x = x.to(dt)
    if gain is not None:
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * gain.to(dt)
    h = x.shape[-1] // 2
    c, s = cos.to(dt)[:, None], sin.to(dt)[:, None]
    return torch.cat((x[..., :h] * c - x[..., h:] * s, x[..., h:] * c + x[..., :h] * s), -1)


def _split(s):
    c = s["case"]
    return [x.reshape(x.shape[0], -1, c["hd"]) for x in
            s["rows"].split((c["nh"] * c["hd"], c["nkv"] * c["hd"], c["nkv"] * c["hd"]), 1)]


def _cache(s):
    """The quantised cache's state: codes as e4m3 numbers, scales as powers of two."""
    f8, e8 = torch.float8_e4m3fn, torch.float8_e8m0fnu
    return {"k": s["k"].view(f8), "v": s["v"].view(f8), "ks": s["ks"].view(e8), "vs": s["vs"].view(e8)}


def _plain_append8(s):
    c = s["case"]
    q, k, v = _split(s)
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    q = _norm_rope(q, s["qn"] if c["norm"] else None, cos, sin, torch.float32)
    k = _norm_rope(k, s["kn"] if c["norm"] else None, cos, sin, torch.float32)
    page, off = s["slot"].long() // c["page"], s["slot"].long() % c["page"]
    for n, x in (("k", k), ("v", v.float())):
        codes, e = _quantised(x)
        s[n][page, :, off] = codes.view(torch.uint8)
        s[n + "s"][page, :, off] = e
    return {"q": q.to(s["rows"].dtype).reshape(c["T"], -1), **_cache(s)}


def _softmax_rows(sc, see):
    """exp(sc - max) where seen, 0 elsewhere, and the sums; a row that sees nothing is all 0."""
    m = torch.where(see, sc, -math.inf).amax(-1, keepdim=True)
    p = torch.where(see, (sc - torch.where(m == -math.inf, 0.0, m)).exp(), 0.0)
    return p, p.sum(-1, keepdim=True)


def _attend(q, k, v, see, scale):
    """q [B][n][nh][hd], k and v [B][L][nkv][hd], see [B][n][L] -> [B][n][nh][hd]."""
    B, n, nh, hd = q.shape
    nkv, L = k.shape[2], k.shape[1]
    q = q.reshape(B, n, nkv, nh // nkv, hd).permute(0, 2, 3, 1, 4).reshape(B * nkv, -1, hd)
    kt = k.permute(0, 2, 3, 1).reshape(B * nkv, hd, L).contiguous()
    sc = torch.bmm(q, kt).mul_(scale).view(B, nkv, nh // nkv, n, L)
    p, l = _softmax_rows(sc, see[:, None, None])
    del sc
    o = torch.bmm(p.view(B * nkv, -1, L), v.permute(0, 2, 1, 3).reshape(B * nkv, L, hd).contiguous())
    l = l.view(B * nkv, -1, 1)
    o = torch.where(l > 0, o / l, 0.0)
    return o.view(B, nkv, nh // nkv, n, hd).permute(0, 3, 1, 2, 4).reshape(B, n, nh, hd)


def _padded(cu, n, T):
    """For n rows of each sequence: the rows' places in the packed rows, and each packed row's sequence and place."""
    at = cu[:-1, None] + torch.arange(n, device=DEV)
    t = torch.arange(T, device=DEV)
    b = torch.searchsorted(cu, t, right=True) - 1
    return at.clamp(max=T - 1), b, t - cu[b]


def _paged(s, see, at, b, i):
    """Attention of the padded rows over the requests' keys, in the packed rows' order."""
    c = s["case"]
    j = torch.arange(s["max_kv"], device=DEV)
    page = s["table"].long()[:, j // c["page"]].clamp(min=0)
    off = (j % c["page"]).expand_as(page)
    k, v = s["k"][page, :, off], s["v"][page, :, off]
    k, v = (_values(k, s["ks"][page, :, off]), _values(v, s["vs"][page, :, off])) if c["cache"] == "e4m3" else (k.float(), v.float())
    o = _attend(s["q"].float()[at], k, v, see, c["hd"] ** -0.5)
    return o[b, i].to(s["q"].dtype)


def _plain_attn8(s):
    w, n = s["case"]["window"], s["max_q"]
    cu, kv = s["cu"].long(), s["kv_len"].long()
    at, b, i = _padded(cu, n, s["q"].shape[0])
    pos = (kv - cu.diff())[:, None, None] + torch.arange(n, device=DEV)[:, None]
    j = torch.arange(s["max_kv"], device=DEV)
    see = (j <= pos) & (j < kv[:, None, None])
    return _paged(s, see & (j > pos - w) if w else see, at, b, i)


def _bits(words):
    """[...][32 words] truth values of the words' bits."""
    return ((words[..., None] >> torch.arange(32, device=DEV)) & 1).flatten(-2).bool()


def _plain_treeplan(s):
    cu, N = s["cu"].long(), 32 * s["words"]
    at, b, i = _padded(cu, N, s["T"])
    n = cu.diff()
    up = torch.where(torch.arange(N, device=DEV) < n[:, None], s["parent"].long()[at], -1)
    # ancestors: the paths of 1, 2, 4, .. steps up put together
    see = torch.eye(N, device=DEV, dtype=torch.bool).expand(len(n), N, N)
    for _ in range(max(1, (N - 1).bit_length())):
        to = up.clamp(min=0)
        see = see | (see.gather(1, to[..., None].expand_as(see)) & (up >= 0)[..., None])
        up = torch.where(up >= 0, up.gather(1, to), -1)
    depth = see.sum(-1) - 1
    word = (see.view(len(n), N, -1, 32).long() << torch.arange(32, device=DEV)).sum(-1)
    word = torch.where(word >= 2 ** 31, word - 2 ** 32, word)
    return {"pos": ((s["kv_len"].long() - n)[:, None] + depth)[b, i].to(torch.int32), "mask": word[b, i].to(torch.int32)}


def _plain_tree(s):
    w, n, L = s["case"]["window"], s["max_q"], s["max_kv"]
    cu, kv = s["cu"].long(), s["kv_len"].long()
    at, b, i = _padded(cu, n, s["q"].shape[0])
    first = (kv - cu.diff())[:, None, None]
    j = torch.arange(L, device=DEV)
    mine = _bits(s["mask"][at])
    see = j < first
    if w:
        see = see & (j > s["pos"].long()[at][..., None] - w)
    new = (j - first).expand(-1, n, -1)
    here = (new >= 0) & (j < kv[:, None, None]) & (new < mine.shape[-1])
    see = see | (here & mine.gather(-1, new.clamp(0, mine.shape[-1] - 1)))
    return _paged(s, see, at, b, i)


def _plain_verify(s):
    """A token's children in the order of their places: child i is kept with probability min(1, w(x) / (z q(x))), w the target's
    probabilities at first and z = 1; a child that is not kept takes max(w / z - q, 0) of w, and z is its sum. In 64 bits."""
    c = s["case"]
    B, N, V = c["B"], s["max_q"], c["V"]
    cu = s["cu"].long()
    n = cu.diff()
    at = (cu[:-1, None] + torch.arange(N, device=DEV)).clamp(max=s["T"] - 1)
    parent, tok, u = s["parent"].long()[at], s["tok"].long()[at], s["u"].double()[at]
    cur, z = torch.zeros(B, dtype=torch.long, device=DEV), torch.ones(B, dtype=torch.float64, device=DEV)
    base = s["p"][at[:, 0]].double().clamp(min=0)
    w = base
    q = s["q"][at[:, 0]].double().clamp(min=0) if c["draft"] else None
    keep = torch.zeros(B, N, dtype=torch.bool, device=DEV)
    keep[:, 0] = n > 0
    for i in range(1, N):
        child = (parent[:, i] == cur) & (i < n)
        x = tok[:, i:i + 1]
        wx = w.gather(1, x)[:, 0]
        qx = q.gather(1, x)[:, 0] if c["draft"] else 1.0
        yes = child & (u[:, i] * qx * z < wx)
        no = child & ~yes
        if c["draft"]:
            left = (w / torch.where(z > 0, z, 1.0)[:, None] - q).clamp(min=0)
            zl = torch.where(z > 0, left.sum(1), 0.0)
        else:
            left = w.scatter(1, x, 0.0)
            zl = (z - wx).clamp(min=0)
        base = torch.where(yes[:, None], s["p"][at[:, i]].double().clamp(min=0), base)
        w = torch.where(yes[:, None], base, torch.where(no[:, None], left, w))
        z = torch.where(yes, 1.0, torch.where(no, zl, z))
        if c["draft"]:
            q = torch.where(yes[:, None], s["q"][at[:, i]].double().clamp(min=0), q)
        cur = torch.where(yes, i, cur)
        keep[:, i] = yes
    w = torch.where((w.sum(1) > 0)[:, None], w, base)
    cum = w.cumsum(1)
    over = (cum > (s["r"].double() * cum[:, -1])[:, None]) & (w > 0)
    last = torch.where(over.any(1), over.long().argmax(1), -1)
    # kept places and their tokens, in order, and the new token behind them
    n_path = keep.sum(1)
    order = torch.where(keep, torch.arange(N, device=DEV), N).sort(1).values
    k = torch.arange(N, device=DEV)
    path = torch.where(k < n_path[:, None], order, -1)
    follow = torch.cat((path[:, 1:], torch.full_like(path[:, :1], -1)), 1)
    out = torch.where(k == n_path[:, None] - 1, last[:, None], torch.where(follow >= 0, tok.gather(1, follow.clamp(min=0)), -1))
    live = k < n[:, None]
    return {"path": path[live].to(torch.int32), "out_tok": out[live].to(torch.int32), "n_path": n_path.to(torch.int32)}


def _plain_commit(s):
    c, page = s["case"], s["case"]["page"]
    cu, kv, table = s["cu"].long(), s["kv_len"].long(), s["table"].long()
    n = cu.diff()
    keep = s["n_path"].long()
    first = kv - n
    _, b, k = _padded(cu, s["max_q"], s["T"])
    src = s["path"].long()
    move = k < keep[b]
    src = torch.where(move, src, 0)
    at, to = first[b] + src, first[b] + k
    from_page, to_page = table[b, at // page], table[b, to // page]
    # (rows that stay are written where they were)
    to_page, to_off = torch.where(move, to_page, from_page), torch.where(move, to % page, at % page)
    stay = ~move
    for x in ("k", "v") + (("ks", "vs") if c["cache"] == "e4m3" else ()):
        rows = s[x][:, from_page, :, at % page]
        # row 0 of a request never moves; what stays repeats it, after the moves
        s[x][:, torch.where(stay, from_page, to_page), :, to_off] = rows
    after = first + keep
    have, want = (kv + page - 1) // page, (after + page - 1) // page
    col = torch.arange(table.shape[1], device=DEV)
    back = (col >= want[:, None]) & (col < have[:, None])
    rank = back.reshape(-1).long().cumsum(0) - 1
    n0 = s["n_free"].long()
    free = torch.cat((s["free"].long(), s["free"].long()[:1]))  # one place more for what is not given back
    free[torch.where(back.reshape(-1), n0 + rank, s["n_pages"])] = table.reshape(-1)
    i32 = torch.int32
    pool = _cache(s) if c["cache"] == "e4m3" else {"k": s["k"], "v": s["v"]}
    return {**pool, "kv_len": after.to(i32), "free": free[:-1].to(i32), "n_free": (n0 + back.sum()).to(i32),
            "status": torch.zeros(1, dtype=i32, device=DEV)}


# ---- the framework's calls -----------------------------------------------------------------------


def _hip():
    """qwen3-tts_amd has a hyphen in its folder's name: loaded by path as qwen3_tts_amd."""
    if "qwen3_tts_amd" not in sys.modules:
        d = os.path.join(ROOT, "qwen3-tts_amd")
        spec = importlib.util.spec_from_file_location("qwen3_tts_amd", os.path.join(d, "__init__.py"),
                                                      submodule_search_locations=[d])
        m = importlib.util.module_from_spec(spec)
        sys.modules["qwen3_tts_amd"] = m
        spec.loader.exec_module(m)
    from qwen3_tts_amd import hip
    return hip


def _own(s):
    """The call on the descriptors that a program makes once for its buffers."""
    if "call" not in s:
        s["call"] = globals()["_call_" + s["case"]["kind"]](s, _hip())
    f, args, out = s["call"]
    if f(*args, torch.cuda.current_stream().cuda_stream) != 0:
        raise RuntimeError(_hip().last_error())
    return out


def _pages(s, hip, layer=None):
    c = s["case"]
    k, v = (s["k"], s["v"]) if layer is None else (s["k"][layer], s["v"][layer])
    d = hip.KvPages(k=k.data_ptr(), v=v.data_ptr(), dtype=hip.E4M3 if "ks" in s else hip.DT[c["cache"]], n_pages=s["n_pages"],
                    page_size=c["page"], n_kv_heads=c["nkv"], head_dim=c["hd"], page_stride=k.stride(0), head_stride=k.stride(1),
                    slot_stride=k.stride(2))
    if "ks" in s:
        ks, vs = (s["ks"], s["vs"]) if layer is None else (s["ks"][layer], s["vs"][layer])
        d.k_scale, d.v_scale = ks.data_ptr(), vs.data_ptr()
        d.scale_page_stride, d.scale_head_stride, d.scale_slot_stride = ks.stride()
    return d


def _call_append8(s, hip):
    c, rows = s["case"], s["rows"]
    e, w = rows.element_size(), rows.stride(0)
    q = rows.data_ptr()
    k = q + c["nh"] * c["hd"] * e
    v = k + c["nkv"] * c["hd"] * e
    d = hip.PageAppend(dtype=hip.DT[c["type"]], n_heads=c["nh"], T=c["T"], rope_len=s["cos"].shape[0], eps=EPS, q=q, k=k, v=v,
                       q_stride=w, k_stride=w, v_stride=w, q_out=s["q_out"].data_ptr(), q_out_stride=s["q_out"].stride(0),
                       q_norm=s["qn"].data_ptr() if c["norm"] else None, k_norm=s["kn"].data_ptr() if c["norm"] else None,
                       rope_cos=s["cos"].data_ptr(), rope_sin=s["sin"].data_ptr(), pos=s["pos"].data_ptr(), slot=s["slot"].data_ptr())
    return hip.lib().qwen_hip_op_page_append, (ctypes.byref(_pages(s, hip)), ctypes.byref(d)), {"q": s["q_out"], **_cache(s)}


def _attn(s, hip, kv):
    c, q = s["case"], s["q"]
    d = hip.PageAttn(dtype=hip.DT[c["type"]], n_heads=c["nh"], B=c["B"], T=q.shape[0], max_q=s["max_q"], max_kv=s["max_kv"],
                     window=c["window"], scale=c["hd"] ** -0.5, q=q.data_ptr(), out=s["out"].data_ptr(), q_stride=q.stride(0),
                     out_stride=s["out"].stride(0), cu_q=s["cu"].data_ptr(), kv_len=s["kv_len"].data_ptr(),
                     table=s["table"].data_ptr(), table_cols=s["table"].shape[1], table_stride=s["table"].stride(0))
    n = hip.lib().qwen_hip_op_page_attention_workspace(ctypes.byref(kv), ctypes.byref(d))
    if n < 0:
        raise RuntimeError(hip.last_error())
    s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    d.workspace, d.workspace_bytes = s["workspace"].data_ptr(), n
    return d


def _call_attn8(s, hip):
    kv = _pages(s, hip)
    return hip.lib().qwen_hip_op_page_attention, (ctypes.byref(kv), ctypes.byref(_attn(s, hip, kv))), s["out"]


def _call_treeplan(s, hip):
    d = hip.TreePlan(parent=s["parent"].data_ptr(), cu_q=s["cu"].data_ptr(), kv_len=s["kv_len"].data_ptr(), pos=s["pos"].data_ptr(),
                     mask=s["mask"].data_ptr(), mask_stride=s["mask"].stride(0), B=s["case"]["B"], T=s["T"], mask_words=s["words"])
    return hip.lib().qwen_hip_op_tree_plan, (ctypes.byref(d),), {"pos": s["pos"], "mask": s["mask"]}


def _call_tree(s, hip):
    kv = _pages(s, hip)
    tree = hip.Tree(mask=s["mask"].data_ptr(), pos=s["pos"].data_ptr(), mask_stride=s["mask"].stride(0), mask_words=s["words"])
    return hip.lib().qwen_hip_op_tree_attention, (ctypes.byref(kv), ctypes.byref(_attn(s, hip, kv)), ctypes.byref(tree)), s["out"]


def _call_verify(s, hip):
    c, p = s["case"], s["p"]
    d = hip.TreeVerify(dtype=hip.DT[c["type"]], B=c["B"], T=s["T"], V=c["V"], p=p.data_ptr(), p_stride=p.stride(0),
                       tok=s["tok"].data_ptr(), parent=s["parent"].data_ptr(), cu_q=s["cu"].data_ptr(), u=s["u"].data_ptr(),
                       r=s["r"].data_ptr(), path=s["path"].data_ptr(), out_tok=s["out_tok"].data_ptr(), n_path=s["n_path"].data_ptr())
    if c["draft"]:
        d.q, d.q_stride = s["q"].data_ptr(), s["q"].stride(0)
    n = hip.lib().qwen_hip_op_tree_verify_workspace(ctypes.byref(d))
    if n < 0:
        raise RuntimeError(hip.last_error())
    s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    d.workspace, d.workspace_bytes = s["workspace"].data_ptr(), n
    return hip.lib().qwen_hip_op_tree_verify, (ctypes.byref(d),), {"path": s["path"], "out_tok": s["out_tok"], "n_path": s["n_path"]}


def _call_commit(s, hip):
    c = s["case"]
    d = hip.TreeCommit(path=s["path"].data_ptr(), n_path=s["n_path"].data_ptr(), cu_q=s["cu"].data_ptr(), kv_len=s["kv_len"].data_ptr(),
                       table=s["table"].data_ptr(), table_stride=s["table"].stride(0), table_cols=s["table"].shape[1],
                       kv_len_out=s["kv_out"].data_ptr(), free_pages=s["free"].data_ptr(), n_free=s["n_free"].data_ptr(),
                       n_free_out=s["n_free_out"].data_ptr(), status=s["status"].data_ptr(), layer_stride=s["k"].stride(0),
                       scale_layer_stride=s["ks"].stride(0) if "ks" in s else 0, n_layers=c["layers"], B=c["B"], T=s["T"])
    pool = _cache(s) if "ks" in s else {"k": s["k"], "v": s["v"]}
    out = {**pool, "kv_len": s["kv_out"], "free": s["free"], "n_free": s["n_free_out"], "status": s["status"]}
    return hip.lib().qwen_hip_op_tree_commit, (ctypes.byref(_pages(s, hip, 0)), ctypes.byref(d)), out


# ---- what a pass cannot do without ---------------------------------------------------------------


def _size(t):
    return {"f32": 4, "e4m3": 1}.get(t, 2)


def work(case):
    c = case
    if c["kind"] == "append8":
        e, nh, nkv, hd, T = _size(c["type"]), c["nh"], c["nkv"], c["hd"], c["T"]
        return {"bytes": T * ((2 * nh + 2 * nkv) * hd * e + 2 * nkv * (hd + 1) + 4 * hd + 8), "flops": T * (nh + nkv) * hd * 8}
    old, new = _requests(c)
    T = sum(new)
    if c["kind"] == "treeplan":
        return {"bytes": T * (8 + 4 * _blocks(max(new), 32)) + 8 * c["B"], "flops": 0}
    if c["kind"] == "verify":
        # the row that the new token comes from, of the target and of the draft; each token's own probabilities
        return {"bytes": (1 + c["draft"]) * c["B"] * c["V"] * _size(c["type"]) + 20 * T, "flops": (2 + 2 * c["draft"]) * c["B"] * c["V"]}
    if c["kind"] == "commit":
        # about half of a walk's depth moves: a quarter of the tokens, each row read and written in k and v of every layer
        row = c["nkv"] * (c["hd"] * _size(c["cache"]) + (c["cache"] == "e4m3"))
        return {"bytes": 4 * c["layers"] * row * max(1, T // 4) + 12 * T, "flops": 0}
    e, w, ke = _size(c["type"]), c["window"], _size(c["cache"])
    tree = c["kind"] == "tree"
    pairs = keys = 0
    for o, n in zip(old, new):
        if tree:  # the prefix, and a token itself
            pairs += n * ((min(o, w) if w else o) + 1)
        else:
            pairs += sum(min(p, w) if w else p for p in range(o + 1, o + n + 1))
        keys += min(o + n, n + w - 1) if w else o + n
    row = c["hd"] * ke + (c["cache"] == "e4m3")
    return {"bytes": 2 * T * c["nh"] * c["hd"] * e + 2 * keys * c["nkv"] * row, "flops": 4 * c["hd"] * c["nh"] * pairs}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["case"]["kind"]
    if kind in ("treeplan", "verify", "commit"):  # whole numbers, and rows that are only moved
        return None
    return _exact_append8(s) if kind == "append8" else _exact_rows(s)


def _bytes_as(x, f):
    """A pool of bytes, byte by byte through a table of the 256 numbers they stand for."""
    return torch.tensor([f(i) for i in range(256)], dtype=torch.float64, device=DEV)[x.long()]


def _e4m3(i):
    s, e, m = -1.0 if i & 128 else 1.0, i >> 3 & 15, i & 7
    return math.nan if e == 15 and m == 7 else s * (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))


def _power(i):
    return math.nan if i == 255 else 2.0 ** (i - 127)


def _exact_append8(s):
    """Codes before their rounding: the row over its scale."""
    c, rows = s["case"], s["rows"].double()
    nh, nkv, hd = c["nh"], c["nkv"], c["hd"]
    x = rows.view(c["T"], nh + 2 * nkv, hd).clone()
    if c["norm"]:
        gain = torch.cat((s["qn"].double().expand(nh, hd), s["kn"].double().expand(nkv, hd)))
        x[:, :nh + nkv] *= gain / (x[:, :nh + nkv].pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt()
    z = torch.complex(x[:, :nh + nkv, :hd // 2], x[:, :nh + nkv, hd // 2:])
    p = s["pos"].long()
    z = z * torch.complex(s["cos"].double()[p], s["sin"].double()[p])[:, None]
    x[:, :nh + nkv] = torch.cat((z.real, z.imag), -1)
    out = {"q": x[:, :nh].reshape(c["T"], -1)}
    at = s["slot"].long()
    for n, y in (("k", x[:, nh:nh + nkv]), ("v", x[:, nh + nkv:])):
        scale = 2.0 ** (y.abs().amax(-1) / E4M3_MAX).log2().ceil().clamp(min=MIN_EXP)
        out[n], out[n + "s"] = _bytes_as(s[n], _e4m3), _bytes_as(s[n + "s"], _power)
        out[n].permute(0, 2, 1, 3)[at // c["page"], at % c["page"]] = y / scale[..., None]
        out[n + "s"].permute(0, 2, 1)[at // c["page"], at % c["page"]] = scale
    return out


def _exact_rows(s):
    c = s["case"]
    hd, nh, nkv, w = c["hd"], c["nh"], c["nkv"], c["window"]
    cu, out = s["cu"].tolist(), []
    for b in range(c["B"]):
        n = int(s["kv_len"][b])
        pg = s["table"][b, :_blocks(n, c["page"])].long()
        kv = []
        for x in ("k", "v"):
            y = s[x][pg].transpose(1, 2).reshape(-1, nkv, hd)[:n]
            y = _bytes_as(y, _e4m3) * _bytes_as(s[x + "s"][pg].transpose(1, 2).reshape(-1, nkv)[:n], _power)[..., None] if "ks" in s else y.double()
            kv.append(y)
        q = s["q"][cu[b]:cu[b + 1]].double()
        m = q.shape[0]
        i, j = torch.arange(n - m, n, device=DEV)[:, None], torch.arange(n, device=DEV)[None]
        hidden = j > i
        if c["kind"] == "tree":
            # a token and the chain of its parents
            up = s["parent"][cu[b]:cu[b + 1]].tolist()
            hidden = torch.ones(m, n, dtype=torch.bool)
            hidden[:, :n - m] = False
            depth = []
            for t in range(m):
                a, d = t, -1
                while a >= 0:
                    hidden[t, n - m + a] = False
                    a, d = up[a], d + 1
                depth.append(d)
                if w:
                    hidden[t, :max(0, min(n - m, n - m + d - w + 1))] = True
            hidden = hidden.to(DEV)
        elif w:
            hidden = hidden | (j <= i - w)
        heads = []
        for h in range(nh):
            g = h // (nh // nkv)
            a = (q[:, h] @ kv[0][:, g].T.contiguous()) / math.sqrt(hd)
            heads.append(a.masked_fill_(hidden, -math.inf).softmax(-1) @ kv[1][:, g].contiguous())
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
