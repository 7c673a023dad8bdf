"""The operators of paged, batched serving, as cases that can be timed and checked.

Five kinds, each one call of the package (qwen3_tts_amd.hip, declared in include/qwen_tts_hip.h):

  plan    qwen_hip_op_page_plan: the requests' old and new lengths -> pages taken from and given back to
          the free list, block tables, packed offsets, each new token's position and cache slot.
  append  qwen_hip_op_page_append: rows of q, k, v -> per-head RMSNorm, RoPE, q out, k and v into pages.
  paged   qwen_hip_op_page_attention: new tokens of several requests over their paged caches.
  packed  qwen_hip_op_packed_attention: whole prompts of different lengths in one call, causal.
  rules   qwen_hip_op_logit_rules: repetition, presence and frequency penalties, token biases and an
          allowed-token bit mask on a batch's logits.

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


def listed():
    return [
        # a decode step of a small server: one token each
        {"name": "plan-decode-B8", "kind": "plan", "B": 8, "page": 16, "lo": 100, "hi": 3000, "new_lo": 1, "new_hi": 1, "done": 0},
        # a large server's mixed step: prompts' chunks, single tokens and finished requests
        {"name": "plan-mixed-B512", "kind": "plan", "B": 512, "page": 16, "lo": 0, "hi": 6000, "new_lo": 1, "new_hi": 200, "done": 37},
        # 32 streams' step in the Talker's head layout and activation type
        {"name": "append-decode-T32-f32", "kind": "append", "T": 32, "nh": 16, "nkv": 8, "hd": 128, "type": "f32", "kv": "bf16",
         "page": 16, "norm": 1, "layout": "head"},
        # a step's worth of long prompts
        {"name": "append-prompts-T8190-bf16", "kind": "append", "T": 8190, "nh": 16, "nkv": 8, "hd": 128, "type": "bf16", "kv": "bf16",
         "page": 64, "norm": 1, "layout": "slot"},
        # a handful of streams, f32 queries over the bf16 cache: the smallest attention call
        {"name": "paged-decode-B4-f32", "kind": "paged", "B": 4, "lo": 200, "hi": 1500, "new_lo": 1, "new_hi": 1, "nh": 16, "nkv": 8,
         "hd": 128, "type": "f32", "kv": "bf16", "page": 16, "window": 0, "layout": "head"},
        # a busy server with long utterances: bound by the cache's bytes
        {"name": "paged-decode-B64-bf16", "kind": "paged", "B": 64, "lo": 1000, "hi": 8000, "new_lo": 1, "new_hi": 1, "nh": 16, "nkv": 8,
         "hd": 128, "type": "bf16", "kv": "bf16", "page": 64, "window": 0, "layout": "head"},
        # chunks of prompts that continue a cached prefix: bound by the products
        {"name": "paged-chunk-B6-bf16", "kind": "paged", "B": 6, "lo": 0, "hi": 6000, "new_lo": 100, "new_hi": 1024, "nh": 16, "nkv": 8,
         "hd": 128, "type": "bf16", "kv": "bf16", "page": 16, "window": 0, "layout": "slot"},
        # three short sentences of the Talker at once
        {"name": "packed-B3-f32", "kind": "packed", "B": 3, "lo": 21, "hi": 128, "nh": 16, "nkv": 8, "hd": 128, "type": "f32", "window": 0},
        # sixteen prompts with and without a reference recording
        {"name": "packed-B16-bf16", "kind": "packed", "B": 16, "lo": 40, "hi": 1500, "nh": 16, "nkv": 8, "hd": 128, "type": "bf16", "window": 0},
        # two of the longest prompts: the largest call
        {"name": "packed-long-B2-f16", "kind": "packed", "B": 2, "lo": 5003, "hi": 8191, "nh": 16, "nkv": 8, "hd": 128, "type": "f16", "window": 0},
        # a few streams' codec logits
        {"name": "rules-B6-f32", "kind": "rules", "B": 6, "V": 2048, "type": "f32", "hist_lo": 0, "hist_hi": 300, "bias": 0, "mask": 0},
        # a text vocabulary of odd size, long histories, biases and a grammar's mask
        {"name": "rules-B64-bf16", "kind": "rules", "B": 64, "V": 128003, "type": "bf16", "hist_lo": 10, "hist_hi": 4000, "bias": 50, "mask": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("plan", "append", "paged", "paged", "packed", "packed", "rules"))
    page = rng.choice((8, 16, 16, 32, 64, 100))
    layout = rng.choice(("head", "slot"))
    nh, nkv, hd = rng.choice(((16, 8, 128), (16, 8, 128), (16, 16, 64), (32, 4, 128), (12, 2, 64)))
    if kind == "plan":
        lo = rng.randint(0, 500)
        B = _log(rng, 1, 600)
        return {"kind": kind, "B": B, "page": page, "lo": lo, "hi": lo + _log(rng, 1, 6000), "new_lo": 1,
                "new_hi": _log(rng, 1, 250), "done": rng.randint(0, B // 4)}
    if kind == "append":
        t, kv = rng.choice((("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")))
        return {"kind": kind, "T": _log(rng, 1, 8000), "nh": nh, "nkv": nkv, "hd": hd, "type": t, "kv": kv, "page": page,
                "norm": rng.randint(0, 1), "layout": layout}
    if kind == "paged":
        t, kv = rng.choice((("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")))
        lo = rng.randint(0, 300)
        one = rng.randint(0, 1)
        return {"kind": kind, "B": _log(rng, 1, 64 if one else 8), "lo": lo, "hi": lo + _log(rng, 1, 7500), "new_lo": 1,
                "new_hi": 1 if one else _log(rng, 1, 600), "nh": nh, "nkv": nkv, "hd": hd, "type": t, "kv": kv, "page": page,
                "window": rng.choice((0, 0, 72, 1000)), "layout": layout}
    if kind == "packed":
        lo = _log(rng, 1, 400)
        return {"kind": kind, "B": _log(rng, 1, 12), "lo": lo, "hi": lo + _log(rng, 1, 2500), "nh": nh, "nkv": nkv, "hd": hd,
                "type": rng.choice(("f32", "bf16", "f16")), "window": rng.choice((0, 0, 72, 1000))}
    lo = rng.randint(0, 50)
    return {"kind": kind, "B": _log(rng, 1, 64), "V": _log(rng, 1000, 128000), "type": rng.choice(("f32", "bf16", "f16")),
            "hist_lo": lo, "hist_hi": lo + _log(rng, 1, 4000), "bias": rng.choice((0, 20, 200)), "mask": rng.randint(0, 1)}


# ---- lengths, from the case alone --------------------------------------------------------------


def _spread(lo, hi, n, phase=0):
    """n whole numbers evenly from lo to hi, in an order with no trend."""
    v = [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]
    step = next(s for s in (7, 5, 3, 11, 13, 1) if math.gcd(s, n) == 1)
    return [v[(i * step + phase) % n] for i in range(n)]


def _requests(c):
    """(tokens in the cache before, new tokens) of each request."""
    return _spread(c["lo"], c["hi"], c["B"]), _spread(c["new_lo"], c["new_hi"], c["B"], 1)


def _pairs(n_q, n_kv, w):
    """Visible (query, key) pairs of n_q queries that end at key n_kv."""
    return sum(min(p, w) if w else p for p in range(n_kv - n_q + 1, n_kv + 1))


def _keys(n_q, n_kv, w):
    """Keys that at least one of them sees."""
    return min(n_kv, n_q + w - 1) if w else n_kv


def _blocks(n, page):
    return (n + page - 1) // page


# ---- inputs, from a seed -----------------------------------------------------------------------


def _gen(seed, stream):
    return torch.Generator(device=DEV).manual_seed((int(seed) * 1000003 + stream) & 0x7FFFFFFFFFFF)


def _randn(g, *shape, dtype=torch.float32, std=1.0):
    return (std * torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)).to(dtype)


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _pool(c, seed, n_pages):
    """A cache's pages, filled: K about N(0, 1) (normed per head), V a projection's N(0, 0.7); seen as
    [page][kv head][slot][head_dim] whatever the order in memory."""
    shape = (n_pages, c["nkv"], c["page"], c["hd"]) if c["layout"] == "head" else (n_pages, c["page"], c["nkv"], c["hd"])
    t = TYPES[c["kv"]]
    k = torch.randn(shape, generator=_gen(seed, 11), device=DEV, dtype=torch.float32).to(t)
    v = (0.7 * torch.randn(shape, generator=_gen(seed, 12), device=DEV, dtype=torch.float32)).to(t)
    return (k, v) if c["layout"] == "head" else (k.transpose(1, 2), v.transpose(1, 2))


def _tables(need, pages, width):
    """Block tables of `need` pages a request out of the shuffled `pages`, -1 past them."""
    t = torch.full((len(need), width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = pages[at:at + n]
        at += n
    return t.to(DEV)


def _shuffled(n, seed):
    return torch.randperm(n, generator=torch.Generator().manual_seed(int(seed) & 0x7FFFFFFF)).to(torch.int32)


def _cu(lens):
    v = [0]
    for n in lens:
        v.append(v[-1] + n)
    return v


def prepare(case, seed):
    c = dict(case)
    return globals()["_prepare_" + c["kind"]](c, seed)


def _prepare_plan(c, seed):
    old, new = _requests(c)
    B, page = c["B"], c["page"]
    for i in range(c["done"]):  # finished requests, spread over the batch: their pages go back
        new[i * B // max(1, c["done"])] = -1
    have = [_blocks(n, page) for n in old]
    width = _blocks(max(o + max(n, 0) for o, n in zip(old, new)), page) + 8
    more = sum(_blocks(o + n, page) - _blocks(o, page) for o, n in zip(old, new) if n > 0)
    n_free = more + 64
    n_pages = sum(have) + n_free
    pages = _shuffled(n_pages, seed)
    free = torch.full((n_pages,), -1, dtype=torch.int32)
    free[:n_free] = pages[sum(have):]
    T = sum(max(n, 0) for n in new)
    cap = (T + 63) // 64 * 64
    return {"case": c, "B": B, "page": page, "n_pages": n_pages, "cap": cap, "width": width, "new_len": _int(new),
            "kv_len": _int(old), "table": _tables(have, pages, width), "free": free.to(DEV), "n_free": _int([n_free]),
            "kv_out": _int([0] * B), "cu": _int([0] * (B + 1)), "pos": _int([0] * cap), "slot": _int([0] * cap),
            "n_free_out": _int([0]), "status": _int([0])}


def _rope(n, hd):
    inv = THETA ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
    a = torch.arange(n, device=DEV, dtype=torch.float64)[:, None] * inv
    return a.cos().float(), a.sin().float()


def _prepare_append(c, seed):
    T, page, t = c["T"], c["page"], TYPES[c["type"]]
    n_pages = _blocks(T, page) + 8
    g = _gen(seed, 1)
    rows = _randn(g, T, (c["nh"] + 2 * c["nkv"]) * c["hd"], dtype=t)
    k, v = _pool(c, seed, n_pages)
    slot = _shuffled(n_pages * page, seed)[:T].to(DEV)
    pos = torch.randint(0, 8192, (T,), generator=g, device=DEV, dtype=torch.int32)
    cos, sin = _rope(8192, c["hd"])
    return {"case": c, "rows": rows, "k": k, "v": v, "slot": slot, "pos": pos, "cos": cos, "sin": sin, "n_pages": n_pages,
            "qn": 1 + _randn(g, c["hd"], std=0.1), "kn": 1 + _randn(g, c["hd"], std=0.1),
            "q_out": torch.zeros(T, c["nh"] * c["hd"], dtype=t, device=DEV)}


def _prepare_paged(c, seed):
    old, new = _requests(c)
    kv = [o + n for o, n in zip(old, new)]
    need = [_blocks(n, c["page"]) for n in kv]
    n_pages = sum(need) + 5
    k, v = _pool(c, seed, n_pages)
    T = sum(new)
    q = _randn(_gen(seed, 1), T, c["nh"], c["hd"], dtype=TYPES[c["type"]], std=1.5)
    return {"case": c, "q": q, "k": k, "v": v, "n_pages": n_pages, "table": _tables(need, _shuffled(n_pages, seed), max(need) + 3),
            "kv_len": _int(kv), "cu": _int(_cu(new)), "out": torch.zeros_like(q), "max_q": max(new), "max_kv": max(kv)}


def _prepare_packed(c, seed):
    lens = _spread(c["lo"], c["hi"], c["B"])
    T, t = sum(lens), TYPES[c["type"]]
    g = _gen(seed, 1)
    rows = _randn(g, T, (c["nh"] + 2 * c["nkv"]) * c["hd"], dtype=t)  # q | k | v of a fused projection
    rows[:, :c["nh"] * c["hd"]] *= 1.5
    return {"case": c, "rows": rows, "cu": _int(_cu(lens)), "T": T, "max_len": max(lens),
            "out": torch.zeros(T, c["nh"], c["hd"], dtype=t, device=DEV)}


def _prepare_rules(c, seed):
    B, V = c["B"], c["V"]
    g = _gen(seed, 1)
    hl = _spread(c["hist_lo"], c["hist_hi"], B)
    n = sum(hl)
    # a history repeats itself: tokens drawn from the low quarter of a square law
    hist = (torch.rand(n, generator=g, device=DEV).square() * V).to(torch.int32).clamp_(0, V - 1)
    s = {"case": c, "logits": _randn(g, B, V, dtype=TYPES[c["type"]], std=4.0), "hist": hist, "hist_off": _int(_cu(hl)),
         "n_prompt": _int([h // 3 for h in hl]), "rep": 1.0 + 0.3 * torch.rand(B, generator=g, device=DEV),
         "presence": 0.5 * torch.rand(B, generator=g, device=DEV), "frequency": 0.2 * torch.rand(B, generator=g, device=DEV)}
    s["out"] = torch.zeros_like(s["logits"])
    if c["bias"]:
        s["bias_tok"] = torch.rand(B, V, generator=g, device=DEV).topk(c["bias"], 1).indices.to(torch.int32).reshape(-1)
        s["bias_val"] = _randn(g, B * c["bias"], std=3.0)
        s["bias_off"] = _int([c["bias"] * b for b in range(B + 1)])
    if c["mask"]:
        s["mask"] = torch.randint(-2 ** 31, 2 ** 31, (B, (V + 31) // 32), generator=g, device=DEV, dtype=torch.int64).to(torch.int32)
    return s


# ---- one pass ------------------------------------------------------------------------------------


def run(state):
    if own:
        return _own(state)
    return globals()["_plain_" + state["case"]["kind"]](state)


def _plain_plan(s):
    page = s["page"]
    new, kv, table, n0 = s["new_len"].long(), s["kv_len"].long(), s["table"].long(), s["n_free"].long()
    gone, add = new < 0, new.clamp(min=0)
    have = (kv + page - 1) // page
    after = torch.where(gone, 0, kv + add)
    want = torch.where(gone, 0, (after + page - 1) // page)
    col = torch.arange(s["width"], device=DEV)
    # pages given back, in request order, onto the free list's end
    back = gone[:, None] & (col < have[:, None])
    rank = back.reshape(-1).long().cumsum(0) - 1
    free = torch.cat((s["free"].long(), s["free"].long()[:1]))  # one place more for what is not given back
    free[torch.where(back.reshape(-1), n0 + rank, s["n_pages"])] = table.reshape(-1)
    free = free[:-1]
    n1 = n0 + back.sum()
    # pages taken from its end, in request order
    need = torch.where(gone, 0, want - have)
    first = need.cumsum(0) - need
    idx = first[:, None] + col - have[:, None]
    taken = ~gone[:, None] & (col >= have[:, None]) & (col < want[:, None])
    table = torch.where(taken, free[(n1 - 1 - idx).clamp(0, s["n_pages"] - 1)], table)
    cu = torch.cat((torch.zeros(1, dtype=torch.long, device=DEV), add.cumsum(0)))
    t = torch.arange(s["cap"], device=DEV)
    b = torch.searchsorted(cu, t, right=True).sub(1).clamp(max=s["B"] - 1)
    p = kv[b] + t - cu[b]
    live = t < cu[-1]
    slot = table[b, (p // page).clamp(0, s["width"] - 1)] * page + p % page
    i32 = torch.int32
    return {"kv_len": after.to(i32), "cu": cu.to(i32), "pos": torch.where(live, p, -1).to(i32),
            "slot": torch.where(live, slot, -1).to(i32), "table": table.to(i32), "free": free.to(i32),
            "n_free": (n1 - need.sum()).to(i32), "status": torch.zeros(1, dtype=i32, device=DEV)}


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


def _plain_append(s):
    c = s["case"]
    q, k, v = _split(s)
    cos, sin = s["cos"][s["pos"].long()], s["sin"][s["pos"].long()]
    q = _norm_rope(q, s["qn"] if c["norm"] else None, cos, sin, torch.float32)
    k = _norm_rope(k, s["kn"] if c["norm"] else None, cos, sin, torch.float32)
    page, off = s["slot"].long() // c["page"], s["slot"].long() % c["page"]
    s["k"][page, :, off] = k.to(s["k"].dtype)
    s["v"][page, :, off] = v.float().to(s["v"].dtype)
    return q.to(s["rows"].dtype).reshape(c["T"], -1), s["k"], s["v"]


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


def _see(n_q, n_kv, n, L, w):
    """[B][n][L]: query i of n_q, at position n_kv - n_q + i, sees key j."""
    pos = (n_kv - n_q)[:, None, None] + torch.arange(n, device=DEV)[:, None]
    j = torch.arange(L, device=DEV)
    see = (j <= pos) & (j < n_kv[:, None, None])
    return see & (j > pos - w) if w else see


def _plain_paged(s):
    c = s["case"]
    T, n, L = s["q"].shape[0], s["max_q"], s["max_kv"]
    cu, kv = s["cu"].long(), s["kv_len"].long()
    at, b, i = _padded(cu, n, T)
    j = torch.arange(L, device=DEV)
    page = s["table"].long()[:, j // c["page"]].clamp(min=0)
    off = (j % c["page"]).expand_as(page)
    k, v = s["k"][page, :, off].float(), s["v"][page, :, off].float()
    o = _attend(s["q"].float()[at], k, v, _see(cu.diff(), kv, n, L, c["window"]), c["hd"] ** -0.5)
    return o[b, i].to(s["q"].dtype)


def _plain_packed(s):
    c = s["case"]
    cu, n = s["cu"].long(), s["max_len"]
    at, b, i = _padded(cu, n, s["T"])
    q, k, v = (x.float()[at] for x in _split(s))
    o = _attend(q, k, v, _see(cu.diff(), cu.diff(), n, n, c["window"]), c["hd"] ** -0.5)
    return o[b, i].to(s["rows"].dtype)


def _plain_rules(s):
    c = s["case"]
    B, V = c["B"], c["V"]
    off = s["hist_off"].long()
    e = torch.arange(s["hist"].numel(), device=DEV)
    b = torch.searchsorted(off, e, right=True) - 1
    answer = (e - off[b] >= s["n_prompt"].long()[b]).to(torch.int32)
    at = b * V + s["hist"].long()
    seen = torch.zeros(B * V, dtype=torch.int32, device=DEV).index_add_(0, at, torch.ones_like(answer)).view(B, V)
    n = torch.zeros(B * V, dtype=torch.int32, device=DEV).index_add_(0, at, answer).view(B, V)
    x, r = s["logits"].float(), s["rep"][:, None]
    x = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x)
    x = x - n * s["frequency"][:, None] - (n > 0) * s["presence"][:, None]
    if c["bias"]:
        row = torch.arange(B, device=DEV)[:, None].expand(B, c["bias"]).reshape(-1)
        x = x.index_put((row, s["bias_tok"].long()), s["bias_val"], accumulate=True)
    if c["mask"]:
        t = torch.arange(V, device=DEV)
        x = torch.where((s["mask"][:, t >> 5] >> (t & 31)) & 1 == 1, x, -math.inf)
    return x.to(s["logits"].dtype)


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


def _pages(s, hip):
    c, k = s["case"], s["k"]
    return hip.KvPages(k=k.data_ptr(), v=s["v"].data_ptr(), dtype=hip.DT[c["kv"]], n_pages=s["n_pages"], page_size=c["page"],
                       n_kv_heads=c["nkv"], head_dim=c["hd"], page_stride=k.stride(0), head_stride=k.stride(1), slot_stride=k.stride(2))


def _call_plan(s, hip):
    d = hip.PagePlan(B=s["B"], page_size=s["page"], n_pages=s["n_pages"], table_cols=s["width"], max_tokens=s["cap"],
                     table_stride=s["table"].stride(0), new_len=s["new_len"].data_ptr(), kv_len=s["kv_len"].data_ptr(),
                     n_free=s["n_free"].data_ptr(), table=s["table"].data_ptr(), free_pages=s["free"].data_ptr(),
                     kv_len_out=s["kv_out"].data_ptr(), n_free_out=s["n_free_out"].data_ptr(), cu_q=s["cu"].data_ptr(),
                     pos=s["pos"].data_ptr(), slot=s["slot"].data_ptr(), status=s["status"].data_ptr())
    out = {"kv_len": s["kv_out"], "cu": s["cu"], "pos": s["pos"], "slot": s["slot"], "table": s["table"], "free": s["free"],
           "n_free": s["n_free_out"], "status": s["status"]}
    return hip.lib().qwen_hip_op_page_plan, (ctypes.byref(d),), out


def _call_append(s, hip):
    c, rows = s["case"], s["rows"]
    e, w = rows.element_size(), rows.stride(0)
    q = rows.data_ptr()
    k = q + c["nh"] * c["hd"] * e
    v = k + c["nkv"] * c["hd"] * e
    d = hip.PageAppend(dtype=hip.DT[c["type"]], n_heads=c["nh"], T=c["T"], rope_len=s["cos"].shape[0], eps=EPS, q=q, k=k, v=v,
                       q_stride=w, k_stride=w, v_stride=w, q_out=s["q_out"].data_ptr(), q_out_stride=s["q_out"].stride(0),
                       q_norm=s["qn"].data_ptr() if c["norm"] else None, k_norm=s["kn"].data_ptr() if c["norm"] else None,
                       rope_cos=s["cos"].data_ptr(), rope_sin=s["sin"].data_ptr(), pos=s["pos"].data_ptr(), slot=s["slot"].data_ptr())
    return hip.lib().qwen_hip_op_page_append, (ctypes.byref(_pages(s, hip)), ctypes.byref(d)), (s["q_out"], s["k"], s["v"])


def _call_paged(s, hip):
    c, q, kv = s["case"], s["q"], _pages(s, hip)
    d = hip.PageAttn(dtype=hip.DT[c["type"]], n_heads=c["nh"], B=c["B"], T=q.shape[0], max_q=s["max_q"], max_kv=s["max_kv"],
                     window=c["window"], scale=c["hd"] ** -0.5, q=q.data_ptr(), out=s["out"].data_ptr(), q_stride=q.stride(0),
                     out_stride=s["out"].stride(0), cu_q=s["cu"].data_ptr(), kv_len=s["kv_len"].data_ptr(),
                     table=s["table"].data_ptr(), table_cols=s["table"].shape[1], table_stride=s["table"].stride(0))
    n = hip.lib().qwen_hip_op_page_attention_workspace(ctypes.byref(kv), ctypes.byref(d))
    if n < 0:
        raise RuntimeError(hip.last_error())
    s["workspace"] = torch.empty(max(n, 1), dtype=torch.uint8, device=DEV)
    d.workspace, d.workspace_bytes = s["workspace"].data_ptr(), n
    return hip.lib().qwen_hip_op_page_attention, (ctypes.byref(kv), ctypes.byref(d)), s["out"]


def _call_packed(s, hip):
    c, rows = s["case"], s["rows"]
    e, w = rows.element_size(), rows.stride(0)
    q = rows.data_ptr()
    k = q + c["nh"] * c["hd"] * e
    d = hip.PackedAttn(dtype=hip.DT[c["type"]], n_heads=c["nh"], n_kv_heads=c["nkv"], head_dim=c["hd"], B=c["B"], T=s["T"],
                       window=c["window"], scale=c["hd"] ** -0.5, q=q, k=k, v=k + c["nkv"] * c["hd"] * e, out=s["out"].data_ptr(),
                       q_stride=w, k_stride=w, v_stride=w, out_stride=s["out"].stride(0), cu=s["cu"].data_ptr())
    return hip.lib().qwen_hip_op_packed_attention, (ctypes.byref(d),), s["out"]


def _call_rules(s, hip):
    c, x = s["case"], s["logits"]
    d = hip.LogitRules(dtype=hip.DT[c["type"]], B=c["B"], V=c["V"], logits=x.data_ptr(), out=s["out"].data_ptr(),
                       logits_stride=x.stride(0), out_stride=s["out"].stride(0), hist=s["hist"].data_ptr(),
                       hist_off=s["hist_off"].data_ptr(), hist_cap=s["hist"].numel(), n_prompt=s["n_prompt"].data_ptr(),
                       rep=s["rep"].data_ptr(), presence=s["presence"].data_ptr(), frequency=s["frequency"].data_ptr())
    if c["bias"]:
        d.bias_tok, d.bias_val = s["bias_tok"].data_ptr(), s["bias_val"].data_ptr()
        d.bias_off, d.bias_cap = s["bias_off"].data_ptr(), s["bias_tok"].numel()
    if c["mask"]:
        d.mask, d.mask_stride = s["mask"].data_ptr(), s["mask"].stride(0)
    return hip.lib().qwen_hip_op_logit_rules, (ctypes.byref(d),), s["out"]


# ---- what a pass cannot do without ---------------------------------------------------------------


def _size(t):
    return 4 if t == "f32" else 2


def work(case):
    c = case
    if c["kind"] == "plan":
        old, new = _requests(c)
        for i in range(c["done"]):
            new[i * c["B"] // max(1, c["done"])] = -1
        moved = sum(_blocks(o, c["page"]) if n < 0 else _blocks(o + n, c["page"]) - _blocks(o, c["page"]) for o, n in zip(old, new))
        return {"bytes": 16 * c["B"] + 8 * sum(max(n, 0) for n in new) + 8 * moved, "flops": 0}
    if c["kind"] == "append":
        e, nh, nkv, hd, T = _size(c["type"]), c["nh"], c["nkv"], c["hd"], c["T"]
        return {"bytes": T * ((2 * nh + 2 * nkv) * hd * e + 2 * nkv * hd * 2 + 4 * hd + 8), "flops": T * (nh + nkv) * hd * 7}
    if c["kind"] == "rules":
        B, V = c["B"], c["V"]
        return {"bytes": 2 * B * V * _size(c["type"]) + 4 * sum(_spread(c["hist_lo"], c["hist_hi"], B)) + 8 * B * c["bias"]
                + (B * V // 8 if c["mask"] else 0), "flops": 0}
    e, w = _size(c["type"]), c["window"]
    if c["kind"] == "paged":
        old, new = _requests(c)
        kv, ke = [o + n for o, n in zip(old, new)], 2
    else:
        kv = new = _spread(c["lo"], c["hi"], c["B"])
        ke = e
    keys = sum(_keys(n, k, w) for n, k in zip(new, kv))
    return {"bytes": 2 * sum(new) * c["nh"] * c["hd"] * e + 2 * keys * c["nkv"] * c["hd"] * ke,
            "flops": 4 * c["hd"] * c["nh"] * sum(_pairs(n, k, w) for n, k in zip(new, kv))}


# ---- the definitions in 64 bits ------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["kind"] == "append":
        return _exact_append(s)
    if c["kind"] == "rules":
        return _exact_rules(s)
    if c["kind"] == "plan":
        return None
    hd, nh, nkv = c["hd"], c["nh"], c["nkv"]
    cu = s["cu"].tolist()
    out = []
    for b in range(c["B"]):
        r = slice(cu[b], cu[b + 1])
        if c["kind"] == "paged":
            n = int(s["kv_len"][b])
            pg = s["table"][b, :_blocks(n, c["page"])].long()
            k, v = (s[x][pg].transpose(1, 2).reshape(-1, nkv, hd)[:n].double() for x in ("k", "v"))
            q = s["q"][r].double()
        else:
            q, k, v = (x.double() for x in
                       (s["rows"][r, :nh * hd].reshape(-1, nh, hd), s["rows"][r, nh * hd:(nh + nkv) * hd].reshape(-1, nkv, hd),
                        s["rows"][r, (nh + nkv) * hd:].reshape(-1, nkv, hd)))
            n = q.shape[0]
        i = torch.arange(n - q.shape[0], n, device=DEV)[:, None]
        j = torch.arange(n, device=DEV)[None]
        hidden = (j > i) | (j <= i - c["window"]) if c["window"] else j > i
        heads = []
        for h in range(nh):
            g = h // (nh // nkv)
            a = (q[:, h] @ k[:, g].T.contiguous()) / math.sqrt(hd)
            heads.append(a.masked_fill_(hidden, -math.inf).softmax(-1) @ v[:, g].contiguous())
        out.append(torch.stack(heads, 1))
    return torch.cat(out)


def _exact_append(s):
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
    k, v = s["k"].double(), s["v"].double()
    at = s["slot"].long()
    k.permute(0, 2, 1, 3)[at // c["page"], at % c["page"]] = x[:, nh:nh + nkv]
    v.permute(0, 2, 1, 3)[at // c["page"], at % c["page"]] = x[:, nh + nkv:]
    return x[:, :nh].reshape(c["T"], -1), k, v


def _exact_rules(s):
    c = s["case"]
    off, npr = s["hist_off"].tolist(), s["n_prompt"].tolist()
    rows = []
    for b in range(c["B"]):
        h = s["hist"][off[b]:off[b + 1]].long()
        total = torch.bincount(h, minlength=c["V"])
        said = torch.bincount(h[npr[b]:], minlength=c["V"])
        x, r = s["logits"][b].double(), s["rep"][b].double()
        x = torch.where(total == 0, x, torch.minimum(x, torch.zeros_like(x)) * r + torch.maximum(x, torch.zeros_like(x)) / r)
        x = x - said * s["frequency"][b].double() - (said != 0) * s["presence"][b].double()
        if c["bias"]:
            one = slice(b * c["bias"], (b + 1) * c["bias"])
            x[s["bias_tok"][one].long()] += s["bias_val"][one].double()
        if c["mask"]:
            bits = (s["mask"][b].long() & 0xFFFFFFFF)[:, None] >> torch.arange(32, device=DEV)
            x[(bits & 1).reshape(-1)[:c["V"]] == 0] = -math.inf
        rows.append(x)
    return torch.stack(rows)
