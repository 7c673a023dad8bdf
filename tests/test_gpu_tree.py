"""The quantised cache and trees of drafted tokens against plain implementations in 64 bits on the CPU.

Tolerances.  A rounding to a type is off by at most half a step, eps / 2 of the value.
  append     a row without norm and RoPE is exact in 64 bits, and so are its scale and the ties of its codes: bytes are compared.  With them
             the row's f32 arithmetic is off by at most 16 2^-24 (|y1| + |y2|), the rotation's two terms (test_gpu_pages), and its code by
             half a step more: 2^-4 |y|, and 2^-10 scales for the codes under the smallest normal one.  A magnitude that is off by as
             much may take the neighbouring scale where it is 448 scales.
  attention  as over 16-bit caches (test_gpu_pages): codes and scales are exact, so are their products in f32 and bf16.  f16 rows: a
             probability times its scale relative to the largest, 2^E, is off by 2^-25 2^E where it is under f16's normal range, or dropped under
             2^-24 2^E, and a value widened for the matrix core by 2^-25 2^E: with codes of at most 448 and a largest value of more
             than 224 2^E that is 2 2^-25 and 2 2^-25 of it for each key with probabilities of at most 1 (2^8 at most, the row's sum then as large), next to 2 2^-25 of the
             probability's own rounding: 6 n 2^-25 max|v|.
  verify     whole numbers: equal.  Both sides add in f64; a border is off by 2^18 2^-53 of 1 at most, so the random numbers, multiples of
             2^-24 or drawn once for good, do not fall between.
  plan, commit  whole numbers and moved bytes: equal.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from qwen3_tts_amd import hip  # noqa: E402
from test_gpu_pages import DEV, KINDS, TYPES, cu_of, dp, i32, ok, pages_of, pool, stream  # noqa: E402


def quantised64(x):
    """Codes (as bytes) and scale bytes of rows of finite numbers, exact."""
    x = x.double()
    m = x.abs().amax(-1)
    e = torch.full_like(m, -64)
    big = m > 448 * 2.0 ** -64
    f, at = torch.frexp(m / 7)                                       # m / 7 = f 2^at: 448 = 7 2^6 (m / 7 is within 2^-53 of it: not near a
    e[big] = (torch.where(f == 0.5, at - 1, at).double() - 6)[big]   # power of two unless m is one times 7, and then exact)
    y = x / 2.0 ** e[..., None]
    return y.float().to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)     # (y.float(): x had 24 bits)


def values64(codes, scale):
    s = scale.double()
    s = torch.where(s > 246, math.nan, 2.0 ** (s.clamp(min=63) - 127))
    return codes.contiguous().view(torch.float8_e4m3fn).double() * s[..., None]


def pool8(shape, layout, g, dev=DEV):
    """Codes and scales of a pool, random bytes, seen as [page][head][place]."""
    n, nkv, page, hd = shape
    mem = (n, nkv, page, hd) if layout == "head" else (n, page, nkv, hd)
    c = torch.randint(0, 256, mem, generator=g, dtype=torch.int16).to(torch.uint8).to(dev)
    s = torch.randint(100, 130, mem[:3], generator=g, dtype=torch.int16).to(torch.uint8).to(dev)
    return (c, s) if layout == "head" else (c.transpose(1, 2), s.transpose(1, 2))


def pages8(k, ks, v, vs):
    d = pages_of(k, v, "bf16")
    d.dtype, d.k_scale, d.v_scale = hip.E4M3, dp(ks), dp(vs)
    d.scale_page_stride, d.scale_head_stride, d.scale_slot_stride = ks.stride()
    assert ks.stride() == vs.stride()
    return d


def call_append(kv, d):
    ok(hip.lib().qwen_hip_op_page_append(C.byref(kv), C.byref(d), stream()))
    torch.cuda.synchronize()


# ---- append ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("layout,page", [("head", 16), ("slot", 7)])
@pytest.mark.parametrize("t,nkv,hd,T", [("f32", 8, 128, 33), ("f32", 1, 64, 1), ("bf16", 2, 64, 40), ("f16", 16, 128, 9), ("bf16", 3, 128, 300)])
def test_append_of_rows_as_they_are(t, nkv, hd, T, layout, page):
    """Without norm and RoPE: every byte, with what other places hold left alone."""
    print(f"[case] append8 {t} {nkv}x{hd} T={T} {layout} page={page}", flush=True)
    g = torch.Generator().manual_seed(hd + T)
    n_pages = T // page + 3
    rows = torch.randn(T, 2 * nkv, hd, generator=g) * 2.0 ** torch.randint(-9, 10, (T, 2 * nkv, 1), generator=g)
    rows = (rows * 2.0 ** torch.randint(-12, 1, (T, 2 * nkv, hd), generator=g)).to(TYPES[t])       # codes of all exponents
    rows[T // 2, 0] = 0
    k, ks = pool8((n_pages, nkv, page, hd), layout, g)
    v, vs = pool8((n_pages, nkv, page, hd), layout, g)
    want = [x.cpu().clone() for x in (k, ks, v, vs)]
    slot = torch.randperm(n_pages * page, generator=g)[:T].to(torch.int32)
    slot[T // 3] = -1 if T > 3 else slot[T // 3]
    c, s = quantised64(rows)
    for i, at in enumerate(slot.tolist()):
        if at >= 0:
            want[0][at // page, :, at % page], want[1][at // page, :, at % page] = c[i, :nkv], s[i, :nkv]
            want[2][at // page, :, at % page], want[3][at // page, :, at % page] = c[i, nkv:], s[i, nkv:]
    r, sl, E = rows.to(DEV), slot.to(DEV), rows.element_size()
    call_append(pages8(k, ks, v, vs), hip.PageAppend(dtype=hip.DT[t], T=T, k=dp(r), v=dp(r) + nkv * hd * E, k_stride=2 * nkv * hd,
                                                     v_stride=2 * nkv * hd, slot=dp(sl)))
    for got, exp in zip((k, ks, v, vs), want):
        assert torch.equal(got.cpu(), exp)


@pytest.mark.parametrize("t,nh,nkv,hd,T,norm,rope", [("f32", 16, 8, 128, 33, 1, 1), ("bf16", 12, 2, 64, 40, 1, 0), ("f16", 16, 16, 128, 9, 0, 1), ("f32", 4, 4, 64, 70, 1, 1)])
def test_append_with_norm_and_rope(t, nh, nkv, hd, T, norm, rope):
    g = torch.Generator().manual_seed(hd + T)
    page, n_pages = 16, T // 16 + 2
    rows = (2 * torch.randn(T, nh + 2 * nkv, hd, generator=g)).to(TYPES[t])
    slot = torch.randperm(n_pages * page, generator=g)[:T].to(torch.int32)
    pos = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32)
    ang = torch.randn(50, hd // 2, generator=g, dtype=torch.float64)
    cos, sin = ang.cos().float(), ang.sin().float()
    qn, kn = 1 + 0.3 * torch.randn(hd, generator=g), 1 + 0.3 * torch.randn(hd, generator=g)
    k, ks = pool8((n_pages, nkv, page, hd), "head", g)
    v, vs = pool8((n_pages, nkv, page, hd), "head", g)
    dev = [x.to(DEV) for x in (rows, slot, pos, cos, sin, qn, kn)]
    q_out = torch.zeros(T, nh * hd, dtype=TYPES[t], device=DEV)
    E, w, base = rows.element_size(), (nh + 2 * nkv) * hd, dp(dev[0])
    call_append(pages8(k, ks, v, vs), hip.PageAppend(
        dtype=hip.DT[t], n_heads=nh, T=T, rope_len=50, eps=1e-6, q=base, k=base + nh * hd * E, v=base + (nh + nkv) * hd * E, q_stride=w, k_stride=w,
        v_stride=w, q_out=dp(q_out), q_out_stride=nh * hd, q_norm=dp(dev[5]) if norm else None, k_norm=dp(dev[6]) if norm else None,
        rope_cos=dp(dev[3]) if rope else None, rope_sin=dp(dev[4]) if rope else None, pos=dp(dev[2]), slot=dp(dev[1])))
    x = rows[:, :nh + nkv].double()
    if norm:
        x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * torch.cat((qn.double().expand(nh, hd), kn.double().expand(nkv, hd)))
    mag = x.abs()
    if rope:
        c, s = cos.double()[pos.long()][:, None], sin.double()[pos.long()][:, None]
        a, b = x[..., :hd // 2], x[..., hd // 2:]
        x = torch.cat((a * c - b * s, b * c + a * s), -1)
        m = (a.abs() * c.abs() + b.abs() * s.abs(), b.abs() * c.abs() + a.abs() * s.abs())
        mag = torch.cat(m, -1)
    off = 16 * 2.0 ** -24 * mag
    eps = torch.finfo(TYPES[t]).eps
    got = q_out.double().cpu().view(T, nh, hd)
    assert bool(((got - x[:, :nh]).abs() <= off[:, :nh] + eps / 2 * (x[:, :nh].abs() + off[:, :nh]) + 2.0 ** -25).all())
    at = slot.long()
    kb, sb = k.cpu()[at // page, :, at % page], ks.cpu()[at // page, :, at % page]
    kx, err = x[:, nh:], off[:, nh:]
    scale = 2.0 ** (sb.double() - 127)
    m, me = kx.abs().amax(-1), err.amax(-1)
    assert bool((m - me <= 448 * scale).all()) and bool((m + me > 224 * scale).all())
    assert bool(((values64(kb, sb) - kx).abs() <= err + 2.0 ** -4 * (kx.abs() + err) + 2.0 ** -10 * scale[..., None]).all())
    c, s = quantised64(rows[:, nh + nkv:])
    assert torch.equal(v.cpu()[at // page, :, at % page], c) and torch.equal(vs.cpu()[at // page, :, at % page], s)


def test_append_of_edges():
    """Magnitudes at a scale's border, tiny and huge ones, zeros, ties, and rows that are not finite."""
    hd = 64
    up = lambda x: float(np.nextafter(np.float32(x), np.float32(np.inf)))  # noqa: E731
    tops = [448.0, up(448.0), 224.0, up(224.0), 448 * 2.0 ** -64, up(448 * 2.0 ** -64), 2.0 ** -64, 2.0 ** -75, 1e-45, 0.0, 448 * 2.0 ** 118, up(448 * 2.0 ** 118),
            float(np.nextafter(np.float32(2.0 ** 127), np.float32(0))), 17.0, 19.0, 240.0, 247.9]
    rows = torch.zeros(len(tops) + 5, 2, hd)
    spread = torch.linspace(-1, 1, hd)
    for i, m in enumerate(tops):
        rows[i, 0] = spread * m
        rows[i, 0, -1] = m
        rows[i, 1, 5] = -m
        rows[i, 1, 6:40] = m / 448 * torch.arange(34) / 16           # halves of small codes' steps
    want_c, want_s = quantised64(rows[:len(tops)])
    for i, bad in enumerate((math.inf, -math.inf, math.nan, 2.0 ** 127, -3e38)):
        rows[len(tops) + i] = 1.5
        rows[len(tops) + i, :, 7 * i] = bad
    n = rows.shape[0]
    g = torch.Generator().manual_seed(1)
    k, ks = pool8((n, 1, 1, hd), "head", g)
    v, vs = pool8((n, 1, 1, hd), "head", g)
    r, slot = rows.to(DEV), i32(list(range(n)))
    call_append(pages8(k, ks, v, vs), hip.PageAppend(dtype=0, T=n, k=dp(r), v=dp(r) + 4 * hd, k_stride=2 * hd, v_stride=2 * hd, slot=dp(slot)))
    for j, (x, s) in enumerate(((k, ks), (v, vs))):
        x, s = x.cpu().view(n, hd), s.cpu().view(n)
        assert torch.equal(s[:len(tops)], want_s[:, j]) and torch.equal(x[:len(tops)], want_c[:, j])
        assert bool((s[len(tops):] == 255).all()) and bool(values64(x[len(tops):], s[len(tops):]).isnan().all())
    assert want_s[0, 0] == 127 and want_s[1, 0] == 128 and want_s.min() == 63 and want_s.max() == 246


def test_append_codes_and_scales_in_one_buffer():
    """A page's codes of k and v and its scales behind each other; and heads outermost."""
    n, nkv, page, hd, T = 5, 2, 4, 64, 11
    g = torch.Generator().manual_seed(6)
    rows = torch.randn(T, 2 * nkv * hd, generator=g).to(torch.bfloat16).to(DEV)
    slot = i32([3, 5, 7, 9, 11, 0, 15, 8, 1, 19, 18])
    d = hip.PageAppend(dtype=1, T=T, k=dp(rows), v=dp(rows) + nkv * hd * 2, k_stride=2 * nkv * hd, v_stride=2 * nkv * hd, slot=dp(slot))
    sep = [torch.zeros(n, nkv, page, hd, dtype=torch.uint8, device=DEV) for _ in range(2)] + [torch.zeros(n, nkv, page, dtype=torch.uint8, device=DEV) for _ in range(2)]
    call_append(pages8(sep[0], sep[2], sep[1], sep[3]), d)
    one = nkv * page * hd
    stride = 2 * one + 2 * nkv * page
    buf = torch.zeros(n * stride, dtype=torch.uint8, device=DEV)
    k, v = (buf[o:].as_strided((n, nkv, page, hd), (stride, page * hd, hd, 1)) for o in (0, one))
    ks, vs = (buf[2 * one + o:].as_strided((n, nkv, page), (stride, page, 1)) for o in (0, nkv * page))
    call_append(pages8(k, ks, v, vs), d)
    heads = [torch.zeros(nkv, page, n, hd, dtype=torch.uint8, device=DEV).permute(2, 0, 1, 3) for _ in range(2)] + \
            [torch.zeros(nkv, n, page, dtype=torch.uint8, device=DEV).permute(1, 0, 2) for _ in range(2)]
    call_append(pages8(heads[0], heads[2], heads[1], heads[3]), d)
    for a, b, c in zip(sep, (k, v, ks, vs), heads):
        assert torch.equal(a, b) and torch.equal(a, c) and bool(a.any())


# ---- attention -------------------------------------------------------------------------------------


def see_of(n, L, window, tree=None):
    """[n][L]: what each new token sees; tree: (truth values [n][n], depths)."""
    pos, j = torch.arange(L - n, L)[:, None], torch.arange(L)[None]
    if tree is None:
        return (j <= pos) & ((j > pos - window) if window else torch.ones_like(j, dtype=torch.bool))
    mask, depth = tree
    see = torch.zeros(n, L, dtype=torch.bool)
    first = L - n
    if first > 0:
        see[:, :first] = (j[:, :first] > (first + depth[:, None] - window)) if window else True
    see[:, max(first, 0):] = mask[:, max(-first, 0):n]
    return see


def attend_see(q, k, v, see, scale):
    """The rows, and sum p |v| / sum p; rows that see nothing are 0."""
    n, nh, hd = q.shape
    nkv = k.shape[1]
    out, mag = torch.zeros(n, nh, hd, dtype=torch.float64), torch.zeros(n, nh, hd, dtype=torch.float64)
    some = see.any(1)
    for h in range(nh):
        kk, vv = k[:, h // (nh // nkv)].double(), v[:, h // (nh // nkv)].double()
        s = (q[:, h].double() @ kk.T * scale).masked_fill(~see, -math.inf)
        p = torch.zeros_like(s)
        p[some] = s[some].softmax(-1)
        hidden = ~see.any(0)
        vv = vv.masked_fill(hidden[:, None], 0.0)
        out[:, h], mag[:, h] = p @ vv, p @ vv.abs()
    return out, mag


def close(got, exact, mag, t, n_max, vmax):
    got, eps = got.double().cpu(), torch.finfo(TYPES[t]).eps
    if t == "f32":
        off = float((got - exact).norm() / exact.norm().clamp(min=1e-30))
        assert off <= 8e-6, off
        assert bool(((got - exact).abs() <= 5e-5 * vmax).all())
        return
    tol = eps / 2 * 1.01 * (2 * exact.abs() + mag) + 5e-5 * vmax + (6 * n_max * 2.0 ** -25 * vmax + 2.0 ** -25 if t == "f16" else 0.0)
    bad = ((got - exact).abs() / tol).max()
    assert bool(bad <= 1), float(bad)


def random_tree(n, width, g):
    """Parents, each among the `width` before; one in seven a root of its own."""
    up = [-1]
    for i in range(1, n):
        up.append(-1 if float(torch.rand((), generator=g)) < 1 / 7 else max(0, i - 1 - int(width * float(torch.rand((), generator=g)) ** 2)))
    return up[:n]


def closure(up):
    n = len(up)
    see, depth = torch.zeros(n, n, dtype=torch.bool), torch.zeros(n, dtype=torch.long)
    for i, p in enumerate(up):
        p = p if 0 <= p < i else -1
        if p >= 0:
            see[i] = see[p]
            depth[i] = depth[p] + 1
        see[i, i] = True
    return see, depth


def words_of(see, words):
    """[n][n] truth values as int32 words."""
    n = see.shape[0]
    b = torch.zeros(n, 32 * words, dtype=torch.long)
    b[:, :n] = see.long()
    w = (b.view(n, words, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


class Steps:
    """Requests of (tokens before, new tokens) over a shuffled pool in which what no request holds is NaN.  cache: a 16-bit type, or
    e4m3.  masks: for each request the truth values of its new tokens and their depths, or None for a chain; words 0: no trees at all."""

    def __init__(self, reqs, nh, nkv, hd, t, cache, page, layout, seed=0, T=None, window=0, max_q=None, max_kv=None, words=0, masks=None, ke=(-2, 1), ve=(-3, 4),
                 scale=None):
        g = torch.Generator().manual_seed(seed)
        self.reqs, self.t, self.window, self.scale, self.words = reqs, t, window, scale or hd ** -0.5, words
        self.nh, self.hd = nh, hd
        lens = [a + n for a, n in reqs]
        h = lambda n: -(-n // page)  # noqa: E731
        need = [h(n) for n in lens]
        n_pages, cols = sum(need) + 3, max(need + [1]) + 2
        perm = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((len(reqs), cols + 1), -1, dtype=torch.int32)
        shape = (n_pages, nkv, page, hd)
        if cache == "e4m3":
            both = []
            for lo, hi in (ke, ve):
                x = torch.randn(shape, generator=g) * 2.0 ** torch.randint(lo, hi, shape[:3], generator=g)[..., None]
                both.append(quantised64(x))
            (k, ks), (v, vs) = both
            kv = values64(k, ks), values64(v, vs)
            empty = lambda: (torch.full(shape, 0x7F, dtype=torch.uint8), torch.full(shape[:3], 255, dtype=torch.uint8))  # noqa: E731
            pools, src = [*empty(), *empty()], (k, ks, v, vs)
        else:
            k, v = (torch.randn(shape, generator=g).to(TYPES[cache]) for _ in range(2))
            kv, src = (k, v), (k, v)
            pools = [torch.full(shape, math.nan, dtype=TYPES[cache]) for _ in range(2)]
        self.kv, self.rows = [], []
        for b, n in enumerate(lens):
            mine, perm = perm[:need[b]], perm[need[b]:]
            table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
            p, o = torch.tensor([mine[i // page] for i in range(n)], dtype=torch.long), torch.tensor([i % page for i in range(n)], dtype=torch.long)
            for x, y in zip(pools, src):
                x[p, :, o] = y[p, :, o]
            self.rows.append((p, o))
            self.kv.append((kv[0][p, :, o], kv[1][p, :, o]))
        put = lambda x: x.to(DEV) if layout == "head" else x.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)  # noqa: E731
        self.pools = [put(x) for x in pools]
        self.pages = pages8(*self.pools) if cache == "e4m3" else pages_of(*self.pools, cache)
        new = [n for _, n in reqs]
        self.cu = cu_of(new)
        self.T = self.cu[-1] if T is None else T
        self.q = (1.5 * torch.randn(self.T, nh, hd, generator=g)).to(TYPES[t])
        q = torch.zeros(self.T, nh * hd + 16).to(TYPES[t])
        q[:, :nh * hd] = self.q.reshape(self.T, -1)
        self.qd, self.table, self.cud, self.kvl = q.to(DEV), table.to(DEV), i32(self.cu), i32(lens)
        self.out = torch.full((self.T, nh * hd + 8), 7.0, dtype=TYPES[t], device=DEV)
        self.d = hip.PageAttn(dtype=hip.DT[t], n_heads=nh, B=len(reqs), T=self.T, table_cols=cols, max_q=max(new + [0]) if max_q is None else max_q,
                              max_kv=max(lens + [0]) if max_kv is None else max_kv, window=window, scale=self.scale, q=dp(self.qd), out=dp(self.out),
                              q_stride=q.stride(0), out_stride=self.out.stride(0), cu_q=dp(self.cud), kv_len=dp(self.kvl), table=dp(self.table),
                              table_stride=self.table.stride(0))
        self.masks = masks
        if words:
            if masks is None:
                self.masks = [closure(random_tree(n, 5, g)) if n <= 32 * words else None for n in new]
            m, pos = torch.full((self.T, words + 1), -1, dtype=torch.int32), torch.full((self.T,), 12345, dtype=torch.int32)
            for b, mk in enumerate(self.masks):
                if mk is not None:
                    m[self.cu[b]:self.cu[b + 1], :words] = words_of(mk[0], words)
                    pos[self.cu[b]:self.cu[b + 1]] = (reqs[b][0] + mk[1]).to(torch.int32)
            self.m, self.pos = m.to(DEV), pos.to(DEV)
            self.tree = hip.Tree(mask=dp(self.m), pos=dp(self.pos) if window else None, mask_stride=words + 1, mask_words=words)

    def call(self):
        L, kv, d = hip.lib(), C.byref(self.pages), C.byref(self.d)
        ok(L.qwen_hip_op_tree_attention(kv, d, C.byref(self.tree), stream()) if self.words else L.qwen_hip_op_page_attention(kv, d, stream()))

    def run(self):
        n = hip.lib().qwen_hip_op_page_attention_workspace(C.byref(self.pages), C.byref(self.d))
        assert n >= 0, hip.last_error()
        self.ws = torch.full((n + 64,), 255, dtype=torch.uint8, device=DEV)      # NaN bits; 64 bytes that stay
        self.d.workspace, self.d.workspace_bytes = dp(self.ws), n
        self.call()
        torch.cuda.synchronize()
        assert bool((self.ws[n:] == 255).all())
        w = self.nh * self.hd
        assert bool((self.out[:, w:] == 7).all()) and bool((self.out[self.cu[-1]:] == 7).all())
        return self.out[:self.cu[-1], :w].view(-1, self.nh, self.hd)

    def want(self):
        both = []
        for b, ((_, n), (k, v)) in enumerate(zip(self.reqs, self.kv)):
            see = see_of(n, k.shape[0], self.window, self.masks[b] if self.words else None)
            both.append(attend_see(self.q[self.cu[b]:self.cu[b + 1]], k, v, see, self.scale))
        return torch.cat([o for o, _ in both]), torch.cat([m for _, m in both])

    def check(self):
        got = self.run()
        exact, mag = self.want()
        close(got, exact, mag, self.t, max(a + n for a, n in self.reqs), float(max(v.abs().max() for _, v in self.kv if v.numel())))


# No bound on the keys lets requests of several rows take the kernel for many rows however little there is to do.
HINTS = pytest.mark.parametrize("max_kv", [None, 0])
HEADS = [(16, 8, 128), (16, 16, 64), (12, 2, 64), (32, 4, 128), (7, 1, 128), (128, 2, 64)]
ROWS = ["f32", "bf16", "f16"]
CACHES = KINDS + [(t, "e4m3") for t in ROWS]


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_codes_single_tokens(t, nh, nkv, hd):
    print(f"[case] codes single tokens {t} {nh}/{nkv}x{hd}", flush=True)
    reqs = [(0, 1), (1, 1), (30, 1), (31, 1), (32, 1), (15, 1), (700, 1), (255, 1), (256, 1), (333, 1)]
    Steps(reqs, nh, nkv, hd, t, "e4m3", 16, "head", seed=1).check()
    Steps(reqs[:3], nh, nkv, hd, t, "e4m3", 5, "slot", seed=2, window=17).check()
    Steps(reqs, nh, nkv, hd, t, "e4m3", 16, "slot", seed=2, max_kv=100000).check()      # many ranges, streamed
    Steps(reqs, nh, nkv, hd, t, "e4m3", 16, "slot", seed=2, max_kv=512).check()


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("nh,nkv,hd,page,layout,window", [(16, 8, 128, 16, "head", 0), (16, 16, 64, 7, "slot", 72), (12, 2, 64, 64, "head", 5),
                                                          (32, 4, 128, 1, "slot", 0), (7, 1, 128, 100, "head", 200)])
def test_codes_chunks(t, nh, nkv, hd, page, layout, window):
    print(f"[case] codes chunks {t} {nh}/{nkv}x{hd} page={page} {layout} window={window}", flush=True)
    reqs = [(0, 1), (0, 45), (130, 3), (0, 0), (60, 65), (17, 0), (250, 131), (5, 2), (1, 33)]
    for max_q, max_kv in ((None, None), (1, 10), (0, 0), (10, 4000)):
        Steps(reqs, nh, nkv, hd, t, "e4m3", page, layout, seed=3, window=window, max_q=max_q, max_kv=max_kv).check()


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("nh,nkv,hd,page,layout,window", [(16, 8, 128, 16, "head", 0), (16, 16, 64, 24, "slot", 72), (6, 2, 128, 3, "slot", 300)])
def test_codes_long_chunks(t, nh, nkv, hd, page, layout, window):
    reqs = [(0, 300), (513, 257), (64, 128), (1, 191)]
    Steps(reqs, nh, nkv, hd, t, "e4m3", page, layout, seed=4, window=window, T=900).check()
    Steps(reqs, nh, nkv, hd, t, "e4m3", page, layout, seed=5, window=window, max_kv=6000).check()
    Steps(reqs, nh, nkv, hd, t, "e4m3", page, layout, seed=6, window=window, max_kv=0).check()


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("reqs", [[(700, 1), (30, 1), (0, 1)], [(0, 300), (400, 140)]])
@pytest.mark.parametrize("ke,ve", [((-1, 1), (-60, -55)), ((-1, 1), (55, 60)), ((-20, 1), (-20, 12)), ((-62, 0), (-62, -30))])
@HINTS
def test_scales_of_any_size(t, reqs, ke, ve, max_kv):
    """Values under f16's range, past it, and of scales that differ by more than it holds."""
    if t == "f16" and ve[1] > 20:
        pytest.skip("f16 rows hold no such values")
    s = Steps(reqs, 16, 8, 128, t, "e4m3", 16, "head", seed=8, ke=ke, ve=ve, max_kv=max_kv)
    s.check()


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("reqs", [[(40, 1), (100, 1)], [(0, 40), (90, 45)], [(200, 150)]])
@pytest.mark.parametrize("what", ["code", "scale"])
@HINTS
def test_codes_that_are_nan_reach_those_who_see_them(t, reqs, what, max_kv):
    """A key's scale byte over 246, or a code that is NaN: NaN for the rows that see it, the others exact."""
    s = Steps(reqs, 4, 2, 64, t, "e4m3", 16, "head", seed=9, max_kv=max_kv)
    clean = s.run().clone()
    b = len(reqs) - 1
    L = sum(reqs[b])
    at = L - 1 if reqs[b][1] > 1 else L - 2                                   # the last new token, or one that its row sees
    p, o = s.rows[b][0][at], s.rows[b][1][at]
    for which in (0, 2):                                                      # of k, of v
        before = [x.clone() for x in s.pools]
        if what == "code":
            s.pools[which][p, 0, o, 5] = 0xFF
        else:
            s.pools[which + 1][p, 0, o] = 247 + which
        got = s.run()
        hit = torch.zeros(clean.shape, dtype=torch.bool)
        hit[-1, :2] = True                                                    # query heads 0 and 1 read kv head 0
        if what == "code" and which == 2:
            hit[-1, :2, :5] = hit[-1, :2, 6:] = False
        assert torch.equal(got.isnan().cpu(), hit)
        exact, mag = s.want()
        keep = ~hit
        vmax = float(max(v.abs().max() for _, v in s.kv))
        e = torch.finfo(TYPES[t]).eps
        tol = e / 2 * 1.01 * (2 * exact.abs() + mag) + 5e-5 * vmax + 6 * L * 2.0 ** -25 * vmax
        assert bool(((got.double().cpu() - exact).abs() <= tol)[keep].all())
        for x, y in zip(s.pools, before):
            x.copy_(y)


@HINTS
def test_codes_in_bad_pages_hold_no_keys(max_kv):
    for t, n in (("f32", 1), ("bf16", 1), ("bf16", 60), ("f16", 60)):
        s = Steps([(96, n)], 4, 2, 64, t, "e4m3", 16, "head", seed=10, max_kv=max_kv)
        s.table[0, 2], s.table[0, 4] = 10 ** 6, -1
        got = s.run()
        see = see_of(n, 96 + n, 0)
        see[:, 32:48] = see[:, 64:80] = False
        exact, mag = attend_see(s.q, *s.kv[0], see, s.scale)
        close(got, exact, mag, t, 96 + n, float(s.kv[0][1].abs().max()))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 70])
@HINTS
def test_a_quantised_cache_past_32_bits(t, n, max_kv):
    """Codes and scales whose offsets pass 2^32."""
    s = Steps([(50, n)], 2, 1, 64, t, "e4m3", 16, "head", seed=11, max_kv=max_kv)
    n_pages = s.pools[0].shape[0]
    far = (5 << 30) // (n_pages - 1) // 64 * 64
    big = []
    for x in s.pools:
        y = torch.zeros(far * (n_pages - 1) + 4096, dtype=torch.uint8, device=DEV).as_strided(x.shape, (far, *x.stride()[1:]))
        y.copy_(x)
        big.append(y)
    s.pools, s.pages = big, pages8(*big)
    assert far * (n_pages - 1) > 1 << 32
    s.check()


# ---- plan ------------------------------------------------------------------------------------------


def tree_plan(up, cu, kv, T, words, stride):
    """The plan's positions and masks over buffers that hold 7 before."""
    pos, mask = torch.full((T,), 7, dtype=torch.int32, device=DEV), torch.full((T, stride), 7, dtype=torch.int32, device=DEV)
    keep = [i32(up + [0] * (T - len(up))), i32(cu), i32(kv), pos, mask]
    d = hip.TreePlan(parent=dp(keep[0]), cu_q=dp(keep[1]), kv_len=dp(keep[2]), pos=dp(pos), mask=dp(mask), mask_stride=stride, B=len(kv), T=T, mask_words=words)
    ok(hip.lib().qwen_hip_op_tree_plan(C.byref(d), stream()))
    torch.cuda.synchronize()
    return pos.cpu(), mask.cpu()


@pytest.mark.parametrize("lens,words,extra", [([1], 1, 0), ([7, 0, 1, 32, 31], 1, 2), ([33, 5, 64], 2, 0), ([40, 3], 1, 0), ([1024, 1025, 100], 32, 1), ([200] * 70, 7, 3),
                                              ([3] * 1000, 1, 0)])
def test_tree_plan(lens, words, extra):
    g = torch.Generator().manual_seed(sum(lens))
    ups = [random_tree(n, 1 if i == 0 else 40, g) for i, n in enumerate(lens)]
    ups[-1] = [u if i % 5 else (i, i + 3, -7)[i % 3] for i, u in enumerate(ups[-1])]      # its own, a later one, none: roots
    kv = [n + 11 * b for b, n in enumerate(lens)]
    cu, T = cu_of(lens), sum(lens) + 4
    pos, mask = tree_plan(sum(ups, []), cu, kv, T, words, words + extra)
    for b, up in enumerate(ups):
        p, m = pos[cu[b]:cu[b + 1]], mask[cu[b]:cu[b + 1]]
        if lens[b] > 32 * words:
            assert p.tolist() == list(range(kv[b] - lens[b], kv[b])) and bool((m == 7).all())
            continue
        see, depth = closure(up)
        assert torch.equal(p.long(), kv[b] - lens[b] + depth)
        assert torch.equal(m[:, :words], words_of(see, words)) and bool((m[:, words:] == 7).all())
    assert bool((pos[cu[-1]:] == 7).all()) and bool((mask[cu[-1]:] == 7).all())


def test_tree_plan_offsets_out_of_range_stay_inside():
    pos, mask = tree_plan([-1, 0, 1, 1], [-5, 2, 2, 1 << 30], [10, 3, -4], 4, 1, 1)
    assert pos.tolist() == [8, 9, -2, -2] and mask[:, 0].tolist() == [1, 3, 1, 2]


# ---- trees -----------------------------------------------------------------------------------------


@pytest.mark.parametrize("t,cache", CACHES)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_trees(t, cache, nh, nkv, hd):
    print(f"[case] trees {t} {cache} {nh}/{nkv}x{hd}", flush=True)
    reqs = [(0, 1), (0, 13), (1, 5), (30, 9), (31, 2), (0, 0), (33, 32), (700, 7), (255, 16), (90, 31)]
    Steps(reqs, nh, nkv, hd, t, cache, 16, "head", seed=1, words=1).check()
    Steps(reqs, nh, nkv, hd, t, cache, 7, "slot", seed=2, words=3, max_kv=100000, T=130).check()
    Steps(reqs[:5], nh, nkv, hd, t, cache, 16, "slot", seed=2, words=1, window=20, max_q=1).check()


@pytest.mark.parametrize("t,cache", CACHES)
@pytest.mark.parametrize("nh,nkv,hd,page,window", [(16, 8, 128, 16, 0), (16, 16, 64, 7, 0), (12, 2, 64, 64, 40), (32, 4, 128, 100, 150)])
def test_large_trees_and_chunks(t, cache, nh, nkv, hd, page, window):
    """Trees past a word and a block of keys, beside chunks of text that are longer than any mask."""
    print(f"[case] large trees {t} {cache} {nh}/{nkv}x{hd} page={page} window={window}", flush=True)
    reqs = [(300, 64), (0, 61), (129, 33), (63, 64), (64, 50), (500, 130), (0, 70)]
    Steps(reqs, nh, nkv, hd, t, cache, page, "head", seed=3, words=2, window=window).check()
    Steps(reqs, nh, nkv, hd, t, cache, page, "slot", seed=4, words=5, window=window, max_kv=5000).check()
    Steps(reqs, nh, nkv, hd, t, cache, page, "slot", seed=5, words=3, window=window, max_kv=0).check()


@pytest.mark.parametrize("t,cache", CACHES)
@pytest.mark.parametrize("reqs", [[(0, 9), (40, 12), (3, 5)], [(0, 60), (100, 64), (5, 40)]])
@HINTS
def test_any_mask(t, cache, reqs, max_kv):
    """Masks that are no trees: bits after a token, none at all, all; rows that see nothing are 0."""
    g = torch.Generator().manual_seed(2)
    masks = []
    for _, n in reqs:
        m = torch.rand(n, n, generator=g) < 0.3
        m[0] = False
        m[n // 2] = True
        m[-1] = False
        masks.append((m, torch.zeros(n, dtype=torch.long)))
    s = Steps(reqs, 4, 2, 64, t, cache, 16, "head", seed=5, words=2, masks=masks, max_kv=max_kv)
    s.check()
    assert bool((s.run()[0] == 0).all()) and bool((s.run()[reqs[0][1] - 1] == 0).all())


@pytest.mark.parametrize("t,cache", CACHES)
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("reqs", [[(20, 9)], [(70, 64)]])
@HINTS
def test_what_a_mask_hides_never_reaches_a_row(t, cache, value, reqs, max_kv):
    """Token 4 is no number in k, then in v: only its descendants and itself are touched."""
    n = reqs[0][1]
    g = torch.Generator().manual_seed(3)
    up = random_tree(n, 3, g)
    see, depth = closure(up)
    s = Steps(reqs, 4, 2, 64, t, cache, 16, "head", seed=6, words=2, masks=[(see, depth)], max_kv=max_kv)
    clean = s.run().clone()
    p, o = s.rows[0][0][reqs[0][0] + 4], s.rows[0][1][reqs[0][0] + 4]
    hidden = ~see[:, 4]
    assert bool(hidden.any()) and not bool(hidden.all())
    for which in range(2):
        before = [x.clone() for x in s.pools]
        if cache == "e4m3":
            s.pools[2 * which + 1][p, :, o] = 255
        else:
            s.pools[which][p, :, o] = value
        got = s.run()
        exact, mag = s.want()
        vmax = float(s.kv[0][1].abs().max())
        e = torch.finfo(TYPES[t]).eps
        tol = e / 2 * 1.01 * (2 * exact.abs() + mag) + 5e-5 * vmax + 6 * sum(reqs[0]) * 2.0 ** -25 * vmax
        assert bool(((got.double().cpu() - exact).abs() <= tol)[hidden].all())
        for x, y in zip(s.pools, before):
            x.copy_(y)
    assert bool(torch.isfinite(clean).all())


@pytest.mark.parametrize("t,cache", CACHES)
@HINTS
def test_chains_are_what_causal_attention_gives(t, cache, max_kv):
    """A chain's masks, and a mask too short for its requests: the same rows as without trees."""
    for reqs in ([(40, 9), (200, 13), (0, 30)], [(100, 64), (0, 50), (300, 40)]):
        chain = [(torch.ones(n, n).tril().bool(), torch.arange(n)) for _, n in reqs]
        for window in (0, 25):
            a = Steps(reqs, 8, 4, 128, t, cache, 16, "head", seed=7, window=window, max_kv=max_kv)
            got = a.run().clone()
            b = Steps(reqs, 8, 4, 128, t, cache, 16, "head", seed=7, words=2, masks=chain, max_kv=max_kv)
            c = Steps([(x, n + 33) for x, n in reqs], 8, 4, 128, t, cache, 16, "head", seed=7, words=1, window=window, max_kv=max_kv)
            c.masks = [None] * 3
            c.check()
            if not window:                              # (a window's end moves over new tokens too; a mask's does not)
                assert float((b.run().double() - got.double()).abs().max()) <= 2 * torch.finfo(TYPES[t]).eps * float(got.abs().max())


@HINTS
def test_trees_with_lengths_that_do_not_hold_their_tokens(max_kv):
    """kv_len under the number of new tokens: the last tokens' keys are what there is."""
    for t, n in (("f32", 9), ("bf16", 60)):
        s = Steps([(0, n), (20, n)], 4, 2, 64, t, "bf16", 16, "head", seed=12, words=2, max_kv=max_kv)
        s.kvl.copy_(i32([n - 4, 20 + n]))
        got = s.run()
        see = see_of(n, n - 4, 0, s.masks[0])
        exact, mag = attend_see(s.q[:n], s.kv[0][0][:n - 4], s.kv[0][1][:n - 4], see, s.scale)
        close(got[:n], exact, mag, t, n, float(s.kv[0][1].abs().max()))


# ---- verification ----------------------------------------------------------------------------------


def verify_model(p, q, tok, up, cu, u, r):
    """One request after the other, in f64."""
    V = p.shape[1]
    pos = lambda x: np.where(x > 0, x, 0.0)  # noqa: E731  (NaN: 0)
    path, out, n_path = [-1] * len(tok), [-1] * len(tok), []
    for b in range(len(cu) - 1):
        q0, n = cu[b], cu[b + 1] - cu[b]
        if n == 0:
            n_path.append(0)
            continue
        cur, kept, w, z = 0, [0], pos(p[q0]), 1.0
        toks = []
        for c in range(1, n):
            if up[q0 + c] != cur or not 0 <= tok[q0 + c] < V:
                continue
            x = tok[q0 + c]
            qr = pos(q[q0 + cur]) if q is not None else None
            qx = qr[x] if q is not None else 1.0
            if u[q0 + c] < 0 or u[q0 + c] * qx * z < w[x]:
                cur, w, z = c, pos(p[q0 + c]), 1.0
                kept.append(c)
                toks.append(int(x))
            elif q is not None:
                w = np.maximum(w / z - qr, 0.0) if z > 0 else w * 0
                z = float(w.sum())
            else:
                z = max(z - w[x], 0.0)
                w = w.copy()
                w[x] = 0.0
        if not w.sum() > 0:
            w = pos(p[q0 + cur])
        cum = np.cumsum(w)
        over = np.flatnonzero((cum > r[b] * cum[-1]) & (w > 0))
        last = int(over[0]) if len(over) else int(np.flatnonzero(w > 0)[-1]) if (w > 0).any() else -1
        path[q0:q0 + len(kept)] = kept
        out[q0:q0 + len(kept)] = toks + [last]
        n_path.append(len(kept))
    return path, out, n_path


class Verify:
    def __init__(self, lens, V, t, draft, seed=0, width=4, noise=0.7, pad=0, children=0, T=None):
        g = torch.Generator().manual_seed(seed)
        self.cu, self.V, n = cu_of(lens), V, sum(lens)
        self.T = n if T is None else T
        self.up = []
        for m in lens:
            self.up += random_tree(m, width, g)[:m]
        x = 2 * torch.randn(self.T, V, generator=g)
        y = x + noise * torch.randn(self.T, V, generator=g)
        self.p, self.q = x.softmax(-1).to(TYPES[t]), y.softmax(-1).to(TYPES[t]) if draft else None
        src = self.q if draft else y.softmax(-1)
        first = [self.cu[b] for b in range(len(lens)) for _ in range(lens[b])]
        self.tok = [int(torch.multinomial(src[f + max(a, 0)].float(), 1, generator=g)) for f, a in zip(first, self.up)]
        self.u, self.r = torch.rand(n, generator=g), torch.rand(len(lens), generator=g)
        self.t, self.lens, self.pad, self.children = t, lens, pad, children

    def run(self):
        more = self.T - len(self.tok)
        wide = lambda x: torch.nn.functional.pad(x, (0, self.pad)).to(DEV) if x is not None else None  # noqa: E731
        p, q = wide(self.p), wide(self.q)
        E = p.element_size()
        if self.pad:                                    # rows that begin at an element, not at a word
            p, q = (None if x is None else torch.nn.functional.pad(x.view(-1), (1, 0)) for x in (p, q))
        tok, up = i32(self.tok + [0] * more), i32(self.up + [0] * more)
        u, r, cu = torch.nn.functional.pad(self.u, (0, more)).to(DEV), self.r.to(DEV), i32(self.cu)
        path, out = (torch.full((self.T,), 77, dtype=torch.int32, device=DEV) for _ in range(2))
        n_path = i32([77] * len(self.lens))
        at = E if self.pad else 0
        d = hip.TreeVerify(dtype=hip.DT[self.t], B=len(self.lens), T=self.T, V=self.V, p=dp(p) + at, p_stride=self.V + self.pad, q=dp(q) + at if q is not None else None,
                           q_stride=self.V + self.pad, tok=dp(tok), parent=dp(up), cu_q=dp(cu), u=dp(u), r=dp(r), path=dp(path), out_tok=dp(out), n_path=dp(n_path),
                           max_children=self.children)
        n = hip.lib().qwen_hip_op_tree_verify_workspace(C.byref(d))
        ws = torch.full((n + 64,), 255, dtype=torch.uint8, device=DEV)
        d.workspace, d.workspace_bytes = dp(ws), n
        ok(hip.lib().qwen_hip_op_tree_verify(C.byref(d), stream()))
        torch.cuda.synchronize()
        assert bool((ws[n:] == 255).all())
        m = len(self.tok)
        assert bool((path[m:] == 77).all()) and bool((out[m:] == 77).all())
        return path[:m].tolist(), out[:m].tolist(), n_path.tolist()

    def want(self):
        f = lambda x: None if x is None else x.double().numpy()  # noqa: E731
        return verify_model(f(self.p), f(self.q), self.tok, self.up, self.cu, self.u.double().numpy(), self.r.double().numpy())

    def check(self):
        assert self.run() == self.want()


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("draft", [0, 1])
@pytest.mark.parametrize("V,pad", [(1, 0), (5, 3), (1000, 1), (4096, 0), (4097, 0), (20011, 0), (128003, 0)])
def test_verify(t, draft, V, pad):
    print(f"[case] verify {t} draft={draft} V={V}", flush=True)
    lens = [1, 5, 0, 13, 2, 9, 30][:4 if V > 100000 else 7]
    for width, children in ((1, 0), (4, 0), (9, 9)):
        Verify(lens, V, t, draft, seed=V + width, width=width, pad=pad, children=children, T=sum(lens) + 3).check()


@pytest.mark.parametrize("draft", [0, 1])
@pytest.mark.parametrize("V", [40, 9000])
def test_verify_many_children(draft, V):
    """Up to 150 children of one token, most of them turned down, the same tokens among them."""
    for seed in range(6):
        v = Verify([150, 70, 200], V, "f32", draft, seed=seed, width=1, noise=3.0)
        for b in range(3):
            for i in range(1, v.lens[b]):
                v.up[v.cu[b] + i] = 0 if i < 100 + seed else v.up[v.cu[b] + i]
        v.u = 0.9 + 0.1 * v.u if seed % 2 else v.u
        v.check()


@pytest.mark.parametrize("draft", [0, 1])
@pytest.mark.parametrize("V", [50, 12000])
def test_verify_edges(draft, V):
    v = Verify([6, 6, 6, 6, 6, 6, 6, 6], V, "f32", draft, seed=5, width=1)
    c = v.cu
    for b in range(8):
        v.up[c[b]:c[b + 1]] = [-1, 0, 0, 0, 1, 1]
    v.tok[c[0] + 1], v.tok[c[0] + 2] = -1, V                            # no tokens: passed over
    v.u[c[1] + 1] = v.u[c[1] + 4] = -1.0                                # kept for certain
    v.p[c[2]] = 0.0                                                     # nothing can follow
    v.p[c[3]] = math.nan
    v.p[c[4], ::2] = -1.0                                               # not greater than 0: 0
    if draft:
        v.q[c[5]] = v.p[c[5]]                                           # nothing is left after a rejection (w = max(p / 1 - p, 0)): p's row
        v.u[c[5] + 1] = 1.0                                             # (1 q(x) < p(x): false)
    v.u[c[6] + 1:c[6] + 4] = math.nan                                   # never kept
    v.r[7] = float(np.nextafter(np.float32(1), np.float32(0)))
    v.u[c[7]:] = 0.0
    v.check()
    got = v.run()
    assert got[1][c[2]] == -1 and got[1][c[3]] == -1


@pytest.mark.parametrize("what", ["one-hot", "roots"])
def test_verify_greedy_and_other_roots(what):
    """One-hot rows keep exactly the drafts that agree; a token that is no descendant of the first is never looked at."""
    v = Verify([7] * 5, 300, "bf16", 0, seed=3, width=2)
    if what == "one-hot":
        best = torch.randint(0, 300, (35,))
        v.p = torch.nn.functional.one_hot(best, 300).to(torch.bfloat16)
        for b in range(5):
            for i in range(1, 7):
                if i != 3:
                    v.tok[v.cu[b] + i] = int(best[v.cu[b] + max(v.up[v.cu[b] + i], 0)])
    else:
        for b in range(5):
            v.up[v.cu[b]:v.cu[b] + 7] = [-1, -1, 1, 2, 9, 5, 0]
    v.check()


@pytest.mark.parametrize("draft", [0, 1])
def test_tokens_that_come_out_are_distributed_as_the_targets(draft):
    """100 000 requests of a root and three drafts of it, drawn from q (or certain): the first token out against p, each count within 5
    standard deviations."""
    g = torch.Generator().manual_seed(17)
    B, V = 100_000, 6
    p = torch.tensor([0.3, 0.05, 0.25, 0.1, 0.2, 0.1])
    q = torch.tensor([0.1, 0.3, 0.2, 0.2, 0.15, 0.05])
    n = 4
    tok = torch.multinomial(q.expand(B, V), n, replacement=True, generator=g) if draft else torch.tensor([0, 4, 0, 2]).expand(B, n)
    pd = p.expand(B * n, V).contiguous().to(DEV)
    qd = q.expand(B * n, V).contiguous().to(DEV)
    bufs = [tok.reshape(-1).to(torch.int32).to(DEV), i32([-1, 0, 0, 0] * B), i32(list(range(0, B * n + 1, n))), torch.rand(B * n, generator=g).to(DEV),
            torch.rand(B, generator=g).to(DEV)]
    path, out, n_path = (torch.zeros(m, dtype=torch.int32, device=DEV) for m in (B * n, B * n, B))
    for b0 in range(0, B, 50_000):                      # 65535 requests at most
        d = hip.TreeVerify(dtype=0, B=50_000, T=B * n, V=V, p=dp(pd), p_stride=V, q=dp(qd) if draft else None, q_stride=V, tok=dp(bufs[0]), parent=dp(bufs[1]),
                           cu_q=dp(bufs[2]) + 4 * b0, u=dp(bufs[3]), r=dp(bufs[4]) + 4 * b0, path=dp(path), out_tok=dp(out), n_path=dp(n_path) + 4 * b0)
        m = hip.lib().qwen_hip_op_tree_verify_workspace(C.byref(d))
        ws = torch.zeros(m, dtype=torch.uint8, device=DEV)
        d.workspace, d.workspace_bytes = dp(ws), m
        ok(hip.lib().qwen_hip_op_tree_verify(C.byref(d), stream()))
    torch.cuda.synchronize()
    first = out.view(B, n)[:, 0].cpu().long()
    count = torch.bincount(first, minlength=V).double()
    want = B * p.double()
    assert bool(((count - want).abs() <= 5 * (want * (1 - p.double())).sqrt()).all()), count.tolist()
    assert 0 < int((n_path == 2).sum()) < B


def test_verify_offsets_out_of_range_stay_inside():
    v = Verify([4, 3], 30, "f32", 1, seed=2)
    v.cu = [-9, 4, 1 << 30]
    path, out, n_path = v.run()
    v.cu = [0, 4, 7]
    assert (path, out, n_path) == v.want()


def test_steps_without_new_tokens():
    """All requests idle, and buffers for no tokens at all."""
    for T in (0, 5):
        n_path, cu, r, kv = i32([7, 7, 7]), i32([0] * 4), torch.zeros(3, device=DEV), i32([0, 4, 9])
        buf = [torch.full((max(T, 1),), 7, dtype=torch.int32, device=DEV) for _ in range(6)]
        p = torch.zeros(max(T, 1), 9, device=DEV)
        d = hip.TreeVerify(dtype=0, B=3, T=T, V=9, p=dp(p), p_stride=9, tok=dp(buf[0]), parent=dp(buf[1]), cu_q=dp(cu), u=dp(buf[2]), r=dp(r), path=dp(buf[3]),
                           out_tok=dp(buf[4]), n_path=dp(n_path))
        ws = torch.zeros(hip.lib().qwen_hip_op_tree_verify_workspace(C.byref(d)), dtype=torch.uint8, device=DEV)
        d.workspace, d.workspace_bytes = dp(ws), ws.numel()
        ok(hip.lib().qwen_hip_op_tree_verify(C.byref(d), stream()))
        plan = hip.TreePlan(parent=dp(buf[1]), cu_q=dp(cu), kv_len=dp(kv), pos=dp(buf[5]), mask=dp(buf[0]), mask_stride=1, B=3, T=T, mask_words=1)
        ok(hip.lib().qwen_hip_op_tree_plan(C.byref(plan), stream()))
        torch.cuda.synchronize()
        assert n_path.tolist() == [0, 0, 0] and all(bool((b == 7).all()) for b in buf)
    Commit([(5, 0, 0), (0, 0, 0), (17, 0, 3)], "e4m3", 2, 2, 64, 4, "head", seed=1).check()


# ---- commit ----------------------------------------------------------------------------------------


class Commit:
    def __init__(self, reqs, cache, layers, nkv, hd, page, layout, seed=0, free=5, keep=None):
        """reqs: (tokens before, new tokens, kept)."""
        g = torch.Generator().manual_seed(seed)
        self.reqs, self.page, self.layers = reqs, page, layers
        h = lambda n: -(-n // page)  # noqa: E731
        need = [h(a + n) for a, n, _ in reqs]
        self.n_pages, cols = sum(need) + free, max(need + [1]) + 1
        perm = torch.randperm(self.n_pages, generator=g).tolist()
        self.table = []
        for m in need:
            self.table.append(perm[:m] + [-1] * (cols + 1 - m))
            perm = perm[m:]
        self.free, self.n_free, self.cols = perm + [-9] * (self.n_pages - len(perm)), len(perm), cols
        mem = (layers, self.n_pages, nkv, page, hd) if layout == "head" else (layers, self.n_pages, page, nkv, hd)
        see = lambda x: x if layout == "head" else x.transpose(2, 3)  # noqa: E731
        if cache == "e4m3":
            mk = lambda s: see(torch.randint(0, 256, s, generator=g, dtype=torch.int16).to(torch.uint8).to(DEV))  # noqa: E731
            self.pools = [mk(mem), mk(mem[:4]), mk(mem), mk(mem[:4])]
            self.kv = pages8(*(x[0] for x in self.pools))
        else:
            self.pools = [see(torch.randn(mem, generator=g).to(TYPES[cache]).to(DEV)) for _ in range(2)]
            self.kv = pages_of(self.pools[0][0], self.pools[1][0], cache)
        self.cu = cu_of([n for _, n, _ in reqs])
        self.path = []
        for _, n, k in reqs:
            some = sorted(torch.randperm(n, generator=g)[:max(k, 0)].tolist()) if n else []
            self.path += some + [-1] * (n - len(some))
        self.kvl, self.n_path = [a + n for a, n, _ in reqs], [k for _, _, k in reqs]

    def run(self, in_place=False, lengths=True, layers=None, split=False):
        B, T = len(self.reqs), self.cu[-1]
        path, n_path, cu, kvl, table, free, nf = (i32(x) for x in (self.path + [5, 5], self.n_path, self.cu, self.kvl, self.table, self.free, [self.n_free]))
        kv2, nf2 = (kvl, nf) if in_place else (i32([7] * B), i32([7]))
        status = i32([7])
        sl = self.pools[1].stride(0) if len(self.pools) == 4 else 0
        d = hip.TreeCommit(path=dp(path), n_path=dp(n_path), cu_q=dp(cu), kv_len=dp(kvl), table=dp(table), table_stride=table.stride(0), table_cols=self.cols,
                           kv_len_out=dp(kv2) if lengths else None, free_pages=dp(free), n_free=dp(nf), n_free_out=dp(nf2), status=dp(status),
                           layer_stride=self.pools[0].stride(0), scale_layer_stride=sl, B=B, T=T + 2, n_layers=self.layers if layers is None else layers)
        if split:                                       # a call a layer, lengths with the last
            for l in range(self.layers):
                kv = pages8(*(x[l] for x in self.pools)) if len(self.pools) == 4 else pages_of(self.pools[0][l], self.pools[1][l], "bf16")
                kv.dtype, d.n_layers = self.kv.dtype, 1
                d.kv_len_out = dp(kv2) if l == self.layers - 1 else None
                ok(hip.lib().qwen_hip_op_tree_commit(C.byref(kv), C.byref(d), stream()))
        else:
            ok(hip.lib().qwen_hip_op_tree_commit(C.byref(self.kv), C.byref(d), stream()))
        torch.cuda.synchronize()
        return dict(kv=kv2.tolist(), n_free=int(nf2), free=free.tolist(), status=int(status), table=table.tolist())

    def want(self, bad=False):
        pools = [x.cpu().clone() for x in self.pools]
        free, nf, kv2 = list(self.free), self.n_free, []
        h = lambda n: -(-n // self.page)  # noqa: E731
        at = lambda b, p: (self.table[b][p // self.page], p % self.page)  # noqa: E731
        for b, (a, n, k) in enumerate(self.reqs):
            k = min(max(k, 0), n)
            for i in range(k):
                src = self.path[self.cu[b] + i]
                if i < src < n:
                    (p, o), (p2, o2) = at(b, a + src), at(b, a + i)
                    for x in pools:
                        x[:, p2, :, o2] = x[:, p, :, o]
            for c in range(h(a + k), h(a + n)):
                free[nf] = self.table[b][c]
                nf += 1
            kv2.append(a + k)
        return pools, dict(kv=kv2, n_free=nf, free=free, status=0, table=[r for r in self.table])

    def check(self, **kw):
        pools, want = self.want()
        got = self.run(**kw)
        if not kw.get("lengths", True):
            got = want                                  # not written
        assert got == want
        for x, y in zip(self.pools, pools):
            assert torch.equal(x.cpu(), y)


COMMITS = [[(5, 9, 4)], [(0, 1, 1), (7, 13, 13), (16, 16, 3), (30, 0, 0), (15, 40, 0), (100, 61, 20), (3, 300, 270)], [(20 + b, 1 + b % 17, (1 + b % 17) // 2) for b in range(200)]]


@pytest.mark.parametrize("cache", ["bf16", "f16", "e4m3"])
@pytest.mark.parametrize("layers,nkv,hd,page,layout", [(1, 8, 128, 16, "head"), (3, 2, 64, 7, "slot"), (2, 1, 64, 1, "head"), (2, 20, 128, 64, "slot")])
def test_commit(cache, layers, nkv, hd, page, layout):
    print(f"[case] commit {cache} L={layers} {nkv}x{hd} page={page} {layout}", flush=True)
    for i, reqs in enumerate(COMMITS[:3 if nkv * hd <= 128 else 2]):
        for in_place in (False, True):
            Commit(reqs, cache, layers, nkv, hd, page, layout, seed=i).check(in_place=in_place)


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_commit_rows_or_lengths_alone(cache):
    c = Commit(COMMITS[1], cache, 3, 2, 64, 8, "head", seed=4)
    c.check(lengths=False)
    c = Commit(COMMITS[1], cache, 3, 2, 64, 8, "head", seed=4)
    c.check(split=True, in_place=True)
    c = Commit(COMMITS[1], cache, 3, 2, 64, 8, "head", seed=4)
    before, (_, want) = [x.clone() for x in c.pools], c.want()
    assert c.run(layers=0) == want and all(torch.equal(x, y) for x, y in zip(c.pools, before))


def test_commit_of_2048_requests():
    Commit([(b % 40, b % 7, (b % 7) // 2) for b in range(2048)], "bf16", 1, 1, 64, 4, "head", seed=6).check(in_place=True)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("what", ["n_free", "full", "negative", "short", "long"])
def test_commit_of_lengths_that_cannot_be(what, in_place):
    c = Commit([(5, 9, 4), (20, 12, 2), (0, 3, 3)], "bf16", 1, 2, 64, 4, "head", seed=7)
    if what == "n_free":
        c.n_free = c.n_pages + 1
    elif what == "full":
        c.n_free = c.n_pages
    else:
        c.kvl[1] = {"negative": -3, "short": 11, "long": c.cols * 4 + 1}[what]
    got = c.run(in_place=in_place)
    assert got == dict(kv=c.kvl, n_free=c.n_free, free=c.free, status=hip.PLAN_INVALID, table=c.table)


def test_commit_of_paths_that_are_none():
    """Entries before their place, past the tokens, or in pages there are not, move nothing; counts are brought into range."""
    c = Commit([(5, 9, 9), (20, 12, 40), (8, 6, -3)], "e4m3", 2, 2, 64, 4, "head", seed=8)
    c.path[:9] = [0, 5, 1, -4, 99, 8, 6, 1 << 30, 8]
    c.path[9:21] = [2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 11, 11]
    c.check()
    c = Commit([(0, 9, 3)], "bf16", 1, 2, 64, 2, "head", seed=9)
    c.path[:3] = [0, 4, 8]
    c.table[0][2] = 10 ** 6                               # holds 4 and 5
    before = [x.clone() for x in c.pools]
    c.run()
    for x, y in zip(c.pools, before):
        y[:, c.table[0][1], :, 0] = y[:, c.table[0][4], :, 0]
        assert torch.equal(x, y)


# ---- a run of them together ------------------------------------------------------------------------


class Decoder:
    """One attention layer as a language model: a token's q | k | v rows are looked up, its logits a product of what attention
    gives. Tokens come one at a time, or several a step from a tree of drafts. Everything stays on the device."""

    NH, NKV, HD, V, PAGE, COLS = 4, 2, 64, 50, 4, 30

    def __init__(self, B, cache, t="f32", max_tokens=64, words=2, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.B, self.t, self.T, self.words, self.cache = B, t, max_tokens, words, cache
        nh, nkv, hd = self.NH, self.NKV, self.HD
        self.table_e = torch.randn(self.V, (nh + 2 * nkv) * hd, generator=g).to(TYPES[t]).to(DEV)
        self.w = torch.randn(nh * hd, self.V, generator=g).to(DEV)
        self.n_pages = B * self.COLS
        ang = torch.arange(self.PAGE * self.COLS, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
        z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
        self.cos, self.sin, self.norm = ang.cos().float().to(DEV), ang.sin().float().to(DEV), torch.ones(hd, device=DEV)
        shape = (self.n_pages, nkv, self.PAGE, hd)
        if cache == "e4m3":
            self.pools = [torch.zeros(s, dtype=torch.uint8, device=DEV) for s in (shape, shape[:3], shape, shape[:3])]
            self.pages = pages8(*self.pools)
        else:
            self.pools = [torch.zeros(shape, dtype=TYPES[cache], device=DEV) for _ in range(2)]
            self.pages = pages_of(*self.pools, cache)
        self.new, self.kv, self.table, self.free, self.n_free = z(B), z(B), z(B, self.COLS) - 1, i32(list(range(self.n_pages))), i32([self.n_pages])
        self.cu, self.pos, self.slot, self.status, self.status2 = z(B + 1), z(self.T), z(self.T), z(1), z(1)
        self.parent, self.tok, self.mask, self.tpos = z(self.T), z(self.T), z(self.T, words), z(self.T) - 1
        self.u, self.r = torch.zeros(self.T, device=DEV), torch.zeros(B, device=DEV)
        self.q = torch.zeros(self.T, nh * hd, dtype=TYPES[t], device=DEV)
        self.out, self.rows = torch.zeros_like(self.q), torch.zeros(self.T, (nh + 2 * nkv) * hd, dtype=TYPES[t], device=DEV)
        self.p = torch.zeros(self.T, self.V, device=DEV)
        self.path, self.out_tok, self.n_path = z(self.T), z(self.T), z(B)
        E, W = self.rows.element_size(), self.rows.stride(0)
        self.plan = hip.PagePlan(new_len=dp(self.new), kv_len=dp(self.kv), n_free=dp(self.n_free), table=dp(self.table), free_pages=dp(self.free),
                                 kv_len_out=dp(self.kv), n_free_out=dp(self.n_free), cu_q=dp(self.cu), pos=dp(self.pos), slot=dp(self.slot), status=dp(self.status),
                                 table_stride=self.COLS, B=B, page_size=self.PAGE, n_pages=self.n_pages, table_cols=self.COLS, max_tokens=self.T)
        self.tplan = hip.TreePlan(parent=dp(self.parent), cu_q=dp(self.cu), kv_len=dp(self.kv), pos=dp(self.tpos), mask=dp(self.mask), mask_stride=words, B=B, T=self.T,
                                  mask_words=words)
        self.app = hip.PageAppend(dtype=hip.DT[t], n_heads=nh, T=self.T, rope_len=self.cos.shape[0], eps=1e-6, q=dp(self.rows), k=dp(self.rows) + nh * hd * E,
                                  v=dp(self.rows) + (nh + nkv) * hd * E, q_stride=W, k_stride=W, v_stride=W, q_out=dp(self.q), q_out_stride=nh * hd, q_norm=dp(self.norm),
                                  k_norm=dp(self.norm), rope_cos=dp(self.cos), rope_sin=dp(self.sin), pos=dp(self.tpos), slot=dp(self.slot))
        self.att = hip.PageAttn(dtype=hip.DT[t], n_heads=nh, B=B, T=self.T, table_cols=self.COLS, max_q=0, max_kv=self.PAGE * self.COLS, scale=hd ** -0.5, q=dp(self.q),
                                out=dp(self.out), q_stride=nh * hd, out_stride=nh * hd, cu_q=dp(self.cu), kv_len=dp(self.kv), table=dp(self.table), table_stride=self.COLS)
        n = hip.lib().qwen_hip_op_page_attention_workspace(C.byref(self.pages), C.byref(self.att))
        self.ws = torch.zeros(max(n, 16), dtype=torch.uint8, device=DEV)
        self.att.workspace, self.att.workspace_bytes = dp(self.ws), n
        self.tree = hip.Tree(mask=dp(self.mask), pos=dp(self.tpos), mask_stride=words, mask_words=words)
        self.ver = hip.TreeVerify(dtype=0, B=B, T=self.T, V=self.V, p=dp(self.p), p_stride=self.V, tok=dp(self.tok), parent=dp(self.parent), cu_q=dp(self.cu), u=dp(self.u),
                                  r=dp(self.r), path=dp(self.path), out_tok=dp(self.out_tok), n_path=dp(self.n_path))
        n = hip.lib().qwen_hip_op_tree_verify_workspace(C.byref(self.ver))
        self.ws2 = torch.zeros(n, dtype=torch.uint8, device=DEV)
        self.ver.workspace, self.ver.workspace_bytes = dp(self.ws2), n
        self.com = hip.TreeCommit(path=dp(self.path), n_path=dp(self.n_path), cu_q=dp(self.cu), kv_len=dp(self.kv), table=dp(self.table), table_stride=self.COLS,
                                  kv_len_out=dp(self.kv), free_pages=dp(self.free), n_free=dp(self.n_free), n_free_out=dp(self.n_free), status=dp(self.status2), B=B,
                                  T=self.T, table_cols=self.COLS, n_layers=1)

    def step(self):
        """A step on the tokens that `put` has left; the model's own arithmetic is torch's."""
        L, s, kv = hip.lib(), stream(), C.byref(self.pages)
        ok(L.qwen_hip_op_page_plan(C.byref(self.plan), s))
        ok(L.qwen_hip_op_tree_plan(C.byref(self.tplan), s))
        self.rows.copy_(self.table_e[self.tok.long()])
        ok(L.qwen_hip_op_page_append(kv, C.byref(self.app), s))
        ok(L.qwen_hip_op_tree_attention(kv, C.byref(self.att), C.byref(self.tree), s))
        logits = self.out.float() @ self.w
        self.p.copy_((logits == logits.amax(-1, keepdim=True)).float())           # greedy
        ok(L.qwen_hip_op_tree_verify(C.byref(self.ver), s))
        ok(L.qwen_hip_op_tree_commit(kv, C.byref(self.com), s))

    def put(self, trees):
        """(parents, tokens) for each request."""
        pad = self.T - sum(len(u) for u, _ in trees)
        self.new.copy_(i32([len(u) for u, _ in trees]))
        self.parent.copy_(i32(sum([u for u, _ in trees], []) + [-1] * pad))
        self.tok.copy_(i32(sum([x for _, x in trees], []) + [0] * pad))

    def took(self, trees):
        """Each request's tokens of the step."""
        torch.cuda.synchronize()
        assert int(self.status) == 0 and int(self.status2) == 0
        out, n, at, got = self.out_tok.tolist(), self.n_path.tolist(), 0, []
        for b, (u, _) in enumerate(trees):
            got.append(out[at:at + n[b]])
            at += len(u)
        used = sum(-(-k // self.PAGE) for k in self.kv.tolist())
        assert used + int(self.n_free) == self.n_pages
        live = [p for b, k in enumerate(self.kv.tolist()) for p in self.table[b, :-(-k // self.PAGE)].tolist()]
        assert sorted(live + self.free[:int(self.n_free)].tolist()) == list(range(self.n_pages))
        return got


def draft_tree(truth, g, V):
    """A tree behind the last token: the true continuation now and then, other tokens beside it; each with siblings."""
    up, tok, at = [-1], [truth[0]], 0
    for t in truth[1:]:
        right = float(torch.rand((), generator=g)) < 0.8
        kids = int(torch.randint(1, 4, (), generator=g))
        which = int(torch.randint(0, kids, (), generator=g))
        first = len(up)
        for i in range(kids):
            up.append(at)
            tok.append(t if right and i == which else int(torch.randint(0, V, (), generator=g)))
        at = first + which
    return up, tok


@pytest.mark.parametrize("t,cache", [("f32", "bf16"), ("f32", "e4m3"), ("bf16", "bf16")])
@pytest.mark.parametrize("replayed", [False, True])
def test_drafted_steps_give_the_tokens_of_single_ones(t, cache, replayed):
    """Greedy tokens of three requests one at a time, and the same tokens in fewer steps from drafts, eager and from a graph: lengths, pages and
    what each step keeps follow."""
    print(f"[case] drafted steps {t} {cache} replayed={replayed}", flush=True)
    B, n = 3, 40
    one = Decoder(B, cache, t, max_tokens=3, words=1)
    seqs = [[7], [11], [49]]
    for _ in range(n):
        trees = [([-1], [s[-1]]) for s in seqs]
        one.put(trees)
        one.step()
        for s, x in zip(seqs, one.took(trees)):
            s += x
    assert all(len(s) == n + 1 for s in seqs)
    many = Decoder(B, cache, t)
    g = torch.Generator().manual_seed(4)
    if replayed:
        trees = [([-1], [0])] * B
        many.put(trees)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            many.step()                                 # (the library's products set themselves up)
            side.synchronize()
            many.kv.zero_()
            many.n_free.fill_(many.n_pages)
            many.free.copy_(i32(list(range(many.n_pages))))
            many.table.fill_(-1)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            many.step()
    at, steps, most = [0] * B, 0, 0
    while min(at) < n - 6:
        trees = [draft_tree(s[a:a + 1 + (steps + b) % 5], g, Decoder.V) for b, (s, a) in enumerate(zip(seqs, at))]
        many.put(trees)
        graph.replay() if replayed else many.step()
        for b, x in enumerate(many.took(trees)):
            assert x == seqs[b][at[b] + 1:at[b] + 1 + len(x)][:len(x)] or at[b] + len(x) > n, (b, at[b], x)
            at[b] = min(at[b] + len(x), n - 1)
            most = max(most, len(x))
        assert many.kv.tolist() == at or max(at) >= n - 1
        if max(at) >= n - 6:
            break
        steps += 1
    assert most >= 3 and steps < 30


@pytest.mark.parametrize("what", ["attention", "verify"])
def test_two_calls_at_once_have_their_own_workspaces(what):
    """Two calls on two streams, each with its workspace, twenty times over."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    if what == "attention":
        reqs = [(700, 9), (300, 13), (90, 5)]
        x = [Steps(reqs, 8, 4, 128, "bf16", "e4m3", 16, "head", seed=s, words=1) for s in (1, 2)]
        want = [s.run().clone() for s in x]
        for s in x:
            s.out.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(20):
            for s, st in zip(x, (a, b)):
                with torch.cuda.stream(st):
                    s.call()
        torch.cuda.synchronize()
        assert all(torch.equal(s.out[:, :1024].view(-1, 8, 128), w) for s, w in zip(x, want))
        return
    x = [Verify([5, 9, 13], 60_000, "bf16", 1, seed=s) for s in (1, 2)]
    want = [v.want() for v in x]
    got = []
    for _ in range(5):
        for v, st in zip(x, (a, b)):
            with torch.cuda.stream(st):
                got.append(v.run())
    assert all(g == want[i % 2] for i, g in enumerate(got))


# ---- what a row does not see, in finite numbers ------------------------------------------------------


def rows_close(got, s, rows):
    """The rows of truth values `rows` against 64 bits."""
    exact, mag = s.want()
    close(got.cpu()[rows], exact[rows], mag[rows], s.t, max(a + n for a, n in s.reqs), float(max(v.abs().max() for _, v in s.kv)))


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("n", [9, 64])
@pytest.mark.parametrize("what", ["later", "sibling", "window", "bad page"])
@HINTS
def test_codes_of_large_scales_that_a_row_does_not_see(t, n, what, max_kv):
    """A key with the largest scale there is, finite, that rows do not see, or at the place that stands in for keys in bad pages: in
    k, then in v, those rows stay as they are."""
    print(f"[case] hidden scales {t} n={n} {what} max_kv={max_kv}", flush=True)
    rows = torch.ones(n, dtype=torch.bool)
    if what == "sibling":
        g = torch.Generator().manual_seed(3)
        see, depth = closure(random_tree(n, 3, g))
        s = Steps([(70, n)], 4, 2, 64, t, "e4m3", 16, "head", seed=6, words=2, masks=[(see, depth)], max_kv=max_kv)
        p, o, rows = s.rows[0][0][74], s.rows[0][1][74], ~see[:, 4]
    elif what == "bad page":
        s = Steps([(200, n)], 4, 2, 64, t, "e4m3", 16, "head", seed=0, max_kv=max_kv)
        p, o = 0, 0
        assert not bool((s.rows[0][0] == 0).any())                           # page 0 is no request's
        for x, y in zip(s.pools, (0x30, 127, 0x30, 127)):
            x[0, :, 0] = y
        s.table[0, 4:8] = -1
        see = see_of(n, 200 + n, 0)
        see[:, 64:128] = False
        s.want = lambda: attend_see(s.q, *s.kv[0], see, s.scale)
    else:
        s = Steps([(90, n)], 4, 2, 64, t, "e4m3", 16, "head", seed=7, max_kv=max_kv, window=80 if what == "window" else 0)
        at = 5 if what == "window" else 89 + n
        p, o = s.rows[0][0][at], s.rows[0][1][at]
        if what == "later":
            rows[-1] = False
    assert bool(rows.any())
    for which in (1, 3):                                                      # of k, of v
        before = s.pools[which].clone()
        s.pools[which][p, :, o] = 246
        rows_close(s.run(), s, rows)
        s.pools[which].copy_(before)


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("reqs", [[(700, 1), (30, 1)], [(200, 9), (64, 64)], [(0, 300)]])
@HINTS
def test_keys_of_large_scales_that_weigh_nothing(t, reqs, max_kv):
    """A key whose score is far under the others' and whose scales are 2^40 and 2^60 times theirs: the others keep their scores and values."""
    s = Steps(reqs, 4, 2, 64, t, "e4m3", 16, "head", seed=12, max_kv=max_kv)
    s.q = s.q.abs()
    s.qd[:, :4 * 64] = s.q.reshape(s.T, -1).to(DEV)
    for b in range(len(reqs)):
        (p, o), (k, v) = s.rows[b], s.kv[b]
        for at in (1, min(70, sum(reqs[b]) - 2)):
            s.pools[0][p[at], :, o[at]], s.pools[1][p[at], :, o[at]] = 0xB8, 167   # -1 times 2^40
            s.pools[2][p[at], :, o[at]], s.pools[3][p[at], :, o[at]] = 0x38, 187   # 1 times 2^60
            k[at], v[at] = -2.0 ** 40, 2.0 ** 60
    got = s.run()
    exact, mag = s.want()
    rows = torch.cat([torch.arange(n) + a > 1 for a, n in reqs])               # (the first two rows of a request see little else)
    vmax = max(float(v[v.abs() < 2.0 ** 59].abs().max()) for _, v in s.kv)
    close(got.cpu()[rows], exact[rows], mag[rows], t, max(a + n for a, n in reqs), vmax)


# ---- windows and trees -------------------------------------------------------------------------------


@pytest.mark.parametrize("lens,words,window", [([7, 1, 30], 1, 1), ([64, 33, 5], 2, 4), ([64, 40], 2, 31), ([300], 10, 33), ([40], 2, 1000), ([33], 1, 2)])
def test_tree_plan_with_a_window(lens, words, window):
    """Masks leave out ancestors `window` tokens back and further; positions and chunks are as without."""
    g = torch.Generator().manual_seed(sum(lens))
    ups = [random_tree(n, 2, g) for n in lens]
    kv, cu, T = [n + 7 for n in lens], cu_of(lens), sum(lens)
    plain, keep = tree_plan(sum(ups, []), cu, kv, T, words, words), hip.TreePlan
    try:
        hip.TreePlan = lambda **kw: keep(window=window, **kw)
        pos, mask = tree_plan(sum(ups, []), cu, kv, T, words, words)
    finally:
        hip.TreePlan = keep
    assert torch.equal(pos, plain[0])
    for b, up in enumerate(ups):
        if lens[b] > 32 * words:
            assert bool((mask[cu[b]:cu[b + 1]] == 7).all())
            continue
        see, depth = closure(up)
        see &= depth[:, None] - depth[None] < window
        assert torch.equal(mask[cu[b]:cu[b + 1]], words_of(see, words))


@pytest.mark.parametrize("t,cache", CACHES)
@pytest.mark.parametrize("window", [1, 5, 25])
@HINTS
def test_windows_over_planned_chains_are_those_of_causal_attention(t, cache, window, max_kv):
    """Chains longer than the window: the plan's masks and positions give what attention without trees gives."""
    for reqs in ([(40, 9), (200, 30), (0, 30)], [(100, 64), (0, 50), (300, 40)]):
        got = Steps(reqs, 8, 4, 128, t, cache, 16, "head", seed=7, window=window, max_kv=max_kv).run().clone()
        chain = [(torch.ones(n, n).tril().bool(), torch.arange(n)) for _, n in reqs]
        s = Steps(reqs, 8, 4, 128, t, cache, 16, "head", seed=7, window=window, max_kv=max_kv, words=2, masks=chain)
        up = i32(sum([list(range(-1, n - 1)) for _, n in reqs], []))
        s.m.fill_(-1)
        s.pos.fill_(-1)
        d = hip.TreePlan(parent=dp(up), cu_q=dp(s.cud), kv_len=dp(s.kvl), pos=dp(s.pos), mask=dp(s.m), mask_stride=3, B=len(reqs), T=s.T, mask_words=2, window=window)
        ok(hip.lib().qwen_hip_op_tree_plan(C.byref(d), stream()))
        assert float((s.run().double() - got.double()).abs().max()) <= 2 * torch.finfo(TYPES[t]).eps * float(got.abs().max())


# ---- a commit is whole or not at all -----------------------------------------------------------------


@pytest.mark.parametrize("what,how", [(w, h) for h in ("apart", "in place", "count in place") for w in ("n_free", "full", "negative", "short", "long")] +
                         [(w, "rows only") for w in ("negative", "short", "long")])
@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_a_commit_that_cannot_be_moves_nothing(cache, what, how):
    c = Commit([(5, 9, 4), (20, 12, 2), (0, 3, 3)] + [(9, 5, 2)] * 300, cache, 2, 2, 64, 4, "head", seed=7)
    if what == "n_free":
        c.n_free = c.n_pages + 1
    elif what == "full":
        c.n_free = c.n_pages
    else:
        c.kvl[290] = {"negative": -3, "short": 4, "long": c.cols * 4 + 1}[what]
    before = [x.clone() for x in c.pools]
    if how == "count in place":                         # the free count is replaced, the lengths are not
        keep = hip.TreeCommit

        def one(**kw):
            kw["n_free_out"] = kw["n_free"]
            return keep(**kw)
        try:
            hip.TreeCommit = one
            got = c.run()
        finally:
            hip.TreeCommit = keep
        assert got["kv"] == c.kvl and got["status"] == hip.PLAN_INVALID
    else:
        got = c.run(in_place=how == "in place", lengths=how != "rows only")
        if how != "rows only":
            assert got == dict(kv=c.kvl, n_free=c.n_free, free=c.free, status=hip.PLAN_INVALID, table=c.table)
    assert all(torch.equal(x, y) for x, y in zip(c.pools, before))


@pytest.mark.parametrize("cache", ["bf16", "e4m3"])
def test_a_commit_whose_free_count_is_replaced(cache):
    """The count in place, lengths apart: rows, lengths and pages as ever, many requests and layers."""
    for seed in range(4):
        c = Commit([(20 + b % 50, 1 + b % 17, (1 + b % 17) // 3) for b in range(150)], cache, 4, 2, 64, 4, "head", seed=seed)
        pools, want = c.want()
        keep = hip.TreeCommit
        out = {}

        def one(**kw):
            kw["n_free_out"] = kw["n_free"]
            out["d"] = kw["n_free"]
            return keep(**kw)
        try:
            hip.TreeCommit = one
            got = c.run()
        finally:
            hip.TreeCommit = keep
        assert {k: v for k, v in got.items() if k != "n_free"} == {k: v for k, v in want.items() if k != "n_free"}
        for x, y in zip(c.pools, pools):
            assert torch.equal(x.cpu(), y)

@pytest.mark.parametrize("layers", [1, 3])
@pytest.mark.parametrize("in_place", [False, True])
def test_commits_of_many_requests(layers, in_place):
    """Enough of them that lengths are made before the rows are moved: whole, and one that cannot be."""
    reqs = [(b % 40, 1 + b % 7, (1 + b % 7) // 2) for b in range(1500)]
    Commit(reqs, "e4m3", layers, 1, 64, 4, "head", seed=6).check(in_place=in_place)
    c = Commit(reqs, "e4m3", layers, 1, 64, 4, "head", seed=6)
    c.kvl[1400] = -1
    before = [x.clone() for x in c.pools]
    got = c.run(in_place=in_place)
    assert got == dict(kv=c.kvl, n_free=c.n_free, free=c.free, status=hip.PLAN_INVALID, table=c.table)
    assert all(torch.equal(x, y) for x, y in zip(c.pools, before))


# ---- layers' codes and scales in one buffer ----------------------------------------------------------


@pytest.mark.parametrize("order", ["layers", "pages", "apart", "between"])
def test_commits_over_layers_in_one_buffer(order):
    """Codes and scales of several layers beside each other: what separate pools give."""
    L, nkv, page, hd = 3, 2, 4, 64
    reqs = [(5, 9, 4), (20, 12, 2), (0, 3, 3), (9, 30, 17)]
    c = Commit(reqs, "e4m3", L, nkv, hd, page, "head", seed=5)
    n, code, scale = c.n_pages, nkv * page * hd, nkv * page
    pools, want = c.want()
    buf = torch.zeros(16 * L * n * (code + scale), dtype=torch.uint8, device=DEV)
    one = 2 * code + 2 * scale                          # a page: codes of k and v, scales of k and v
    if order == "layers":                               # [layer][k codes | v codes | k scales | v scales], pages within each
        at = [(0, (n * one, code)), (2 * n * code, (n * one, scale)), (n * code, (n * one, code)), (2 * n * code + n * scale, (n * one, scale))]
    elif order == "pages":                              # [page][layer][the same]
        at = [(o, (one, L * one)) for o in (0, 2 * code, code, 2 * code + scale)]
    elif order == "apart":
        at = [(0, (n * code, code)), (2 * L * n * code, (n * scale, scale)), (L * n * code, (n * code, code)), (2 * L * n * code + L * n * scale, (n * scale, scale))]
    else:                                               # all scales between the first two layers' codes
        far = 4 * n * code
        at = [(0, (far, code)), (2 * n * code, (n * scale, scale)), (n * code, (far, code)), (3 * n * code, (n * scale, scale))]
    new = []
    for x, (o, (layer, pg)) in zip(c.pools, at):
        inner = (page * hd, hd, 1) if x.dim() == 5 else (page, 1)
        y = buf[o:].as_strided(x.shape, (layer, pg, *inner))
        y.copy_(x)
        new.append(y)
    c.pools, c.kv = new, pages8(*(x[0] for x in new))
    assert c.run() == want
    for x, y in zip(c.pools, pools):
        assert torch.equal(x.cpu(), y)


def test_buffers_of_no_tokens_overlap_nothing():
    """No tokens at all: buffers of no length inside others are no overlap."""
    n_path, cu, r, kv = i32([7, 7, 7, 7]), i32([0] * 4), torch.zeros(3, device=DEV), i32([0, 4, 9])
    p = torch.zeros(16, device=DEV)
    d = hip.TreeVerify(dtype=0, B=3, T=0, V=9, p=dp(p), p_stride=9, tok=dp(n_path) + 4, parent=dp(n_path) + 4, cu_q=dp(cu), u=dp(n_path) + 4, r=dp(r), path=dp(n_path) + 4,
                       out_tok=dp(n_path) + 8, n_path=dp(n_path))
    ws = torch.zeros(hip.lib().qwen_hip_op_tree_verify_workspace(C.byref(d)), dtype=torch.uint8, device=DEV)
    d.workspace, d.workspace_bytes = dp(ws), ws.numel()
    ok(hip.lib().qwen_hip_op_tree_verify(C.byref(d), stream()))
    torch.cuda.synchronize()
    assert n_path.tolist() == [0, 0, 0, 7]


# ---- verification in several launches ----------------------------------------------------------------


@pytest.mark.parametrize("draft", [0, 1])
def test_verify_edges_of_large_vocabularies(draft):
    test_verify_edges(draft, 50_001)


@pytest.mark.parametrize("draft", [0, 1])
@pytest.mark.parametrize("children", [0, 1])
def test_verify_many_children_of_large_vocabularies(draft, children):
    """More rejections than launches, requests of more than 64 tokens, and a bound on the children that does not hold."""
    for seed in range(4):
        v = Verify([90, 6, 130], 50_001, "f32", draft, seed=seed, width=2, noise=3.0, children=children)
        for b in (0, 2):
            for i in range(1, v.lens[b]):
                v.up[v.cu[b] + i] = 0 if i < 66 + seed else v.up[v.cu[b] + i]
        v.u = 0.9 + 0.1 * v.u if seed % 2 else v.u
        if seed == 3:
            v.u[v.cu[0] + 70] = v.u[v.cu[2] + 100] = -1.0                    # kept for certain, if it is looked at
        v.check()


class VerifyCall(Verify):
    """The same call on buffers that stay, so that several are under way at once."""

    def build(self):
        dev = lambda x: None if x is None else x.to(DEV)  # noqa: E731
        n, T = len(self.lens), self.T
        self.buf = [dev(self.p), dev(self.q), i32(self.tok), i32(self.up), i32(self.cu), dev(self.u), dev(self.r)]
        self.res = [torch.full((m,), 77, dtype=torch.int32, device=DEV) for m in (T, T, n)]
        p, q, tok, up, cu, u, r = (dp(x) if x is not None else None for x in self.buf)
        self.d = hip.TreeVerify(dtype=hip.DT[self.t], B=n, T=T, V=self.V, p=p, p_stride=self.V, q=q, q_stride=self.V, tok=tok, parent=up, cu_q=cu, u=u, r=r,
                                path=dp(self.res[0]), out_tok=dp(self.res[1]), n_path=dp(self.res[2]), max_children=self.children)
        self.ws = torch.full((hip.lib().qwen_hip_op_tree_verify_workspace(C.byref(self.d)),), 255, dtype=torch.uint8, device=DEV)
        self.d.workspace, self.d.workspace_bytes = dp(self.ws), self.ws.numel()
        return self

    def call(self):
        ok(hip.lib().qwen_hip_op_tree_verify(C.byref(self.d), stream()))


@pytest.mark.parametrize("V", [3000, 60_000])
def test_verifications_under_way_at_once(V):
    """Two verifications on two streams, issued in turn without a wait, each with its workspace."""
    st = [torch.cuda.Stream(), torch.cuda.Stream()]
    x = [VerifyCall([5, 9, 13], V, "bf16", 1, seed=s).build() for s in (1, 2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for v, s in zip(x, st):
            with torch.cuda.stream(s):
                v.call()
    torch.cuda.synchronize()
    for v in x:
        assert tuple(r.tolist() for r in v.res) == v.want()


@pytest.mark.parametrize("V", [3000, 60_000])
def test_verifications_replayed(V):
    """A captured verification follows what its buffers hold at each replay."""
    v = VerifyCall([5, 9, 13, 0, 70], V, "bf16", 1, seed=3).build()
    v.call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        v.call()
    for seed in range(3):
        w = Verify([13, 5, 0, 70, 9], V, "bf16", 1, seed=10 + seed)
        for a, b in zip(v.buf, (w.p, w.q, torch.tensor(w.tok), torch.tensor(w.up), torch.tensor(w.cu), w.u, w.r)):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert tuple(r.tolist() for r in v.res) == w.want()


# ---- the largest there are ---------------------------------------------------------------------------


@pytest.mark.parametrize("t,cache", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "e4m3"), ("bf16", "e4m3"), ("f16", "e4m3")])
@pytest.mark.parametrize("window", [0, 100])
def test_trees_of_as_many_tokens_as_masks_hold(t, cache, window):
    s = Steps([(70, 1024), (5, 1000), (40, 1025), (300, 7)], 4, 2, 64, t, cache, 16, "head", seed=31, words=32, window=window)
    s.check()


@pytest.mark.parametrize("draft", [0, 1])
def test_verify_the_largest_vocabulary(draft):
    Verify([3, 1, 4], 1 << 20, "bf16", draft, seed=9, width=3).check()


@pytest.mark.parametrize("draft", [0, 1])
@pytest.mark.parametrize("V", [300, 50_001])
def test_verify_a_chunk_of_text(draft, V):
    """A long chain that is given, kept for certain up to its drafts at the end, beside a tree."""
    v = Verify([400, 9], V, "bf16", draft, seed=4, width=3)
    v.up[:400] = list(range(-1, 399))
    v.u[:395] = -1.0
    v.check()
    assert v.run()[2][0] >= 395
