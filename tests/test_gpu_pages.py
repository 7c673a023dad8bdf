"""The paged, batched operators against plain implementations in 64 bits on the CPU.

Tolerances.  A rounding to a type is off by at most half a step, eps / 2 of the value.
  append     f32 arithmetic: the sum of squares 12 roundings (a lane's 8 terms, 4 exchanges), each counting half in the
             root, then division, root, two products and the rotation's three: under 16 roundings of 2^-24 on |y1| + |y2|
             (the rotation's two terms); then one rounding to the stored type.
  attention  16-bit: every probability rounded once, p' = p (1 + d) with |d| <= eps / 2, in the sum over v and in the sum of
             the row.  sum p' v is off by at most eps / 2 sum p |v|, sum p' by at most eps / 2 of itself, so their quotient o
             by eps / 2 (sum p |v| / sum p + |o|), to first order in eps (1 % covers the second); the output's own
             rounding is another eps / 2 |o|.  f16: a p below its normal range is off by 2^-25 absolutely, n 2^-25 max|v| over
             the row's sum, which is 1 at least, and as much of o through the sum.  And the f32 part below.
             f32 part, in the 2-norm over all outputs: each score is a sum of head_dim exact plane products in at most
             6 head_dim / 16 f32 additions of partial sums that stay near its standard size: with scores up to about 8
             (in units of their softmax) sqrt(48) 2^-24 8 = 3.3e-6, and the sums over keys add the same order of 2^-24
             sqrt(6 n / 16 / 4) < 1e-6 for n <= 700: 8e-6 in all.  16-bit element by element: 5e-5 max|v|, 6 times the same.
  rules      at most 3 roundings after the penalty's own, of values up to the largest stage's: 4 2^-24 of it, then one to the
             stored type; rep_each: one more for each entry.
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

from qwen3_tts_amd import hip  # noqa: E402

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


def dp(t):
    return None if t is None else t.data_ptr()


def stream():
    return torch.cuda.current_stream().cuda_stream


def ok(rc):
    assert rc == 0, hip.last_error()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def cu_of(lens):
    return [0] + np.cumsum(lens).tolist()


# ---- plan ------------------------------------------------------------------------------------------


def plan_model(new, kv, table, free, n_free, page, n_pages, cols, cap):
    """The plan, one request after the other."""
    table, free, B = [list(r) for r in table], list(free), len(new)
    h = lambda n: -(-n // page)  # noqa: E731
    status, total = 0, 0
    if not 0 <= n_free <= n_pages:
        status |= hip.PLAN_INVALID
    stack, need = [], 0
    for b in range(B):
        if kv[b] < 0 or kv[b] > cols * page:
            status |= hip.PLAN_INVALID
        elif new[b] < 0:
            stack += table[b][:h(kv[b])]
        elif kv[b] + new[b] > cols * page:
            status |= hip.PLAN_TABLE_FULL
        else:
            total += new[b]
            need += h(kv[b] + new[b]) - h(kv[b])
    if total > cap:
        status |= hip.PLAN_TOO_MANY
    if n_free + len(stack) > n_pages:
        status |= hip.PLAN_INVALID
    if need > n_free + len(stack):
        status |= hip.PLAN_NO_PAGES
    if status:
        return dict(kv=list(kv), n_free=n_free, cu=[0] * (B + 1), pos=[-1] * cap, slot=[-1] * cap, table=table, free=free, status=status)
    free[n_free:n_free + len(stack)] = stack
    avail, kv2, pos, slot = free[:n_free + len(stack)], [], [], []
    for b in range(B):
        if new[b] < 0:
            kv2.append(0)
            continue
        for c in range(h(kv[b]), h(kv[b] + new[b])):
            table[b][c] = avail.pop()
        for p in range(kv[b], kv[b] + new[b]):
            pg = table[b][p // page]
            pos.append(p)
            slot.append(pg * page + p % page if 0 <= pg < n_pages else -1)
        kv2.append(kv[b] + new[b])
    cu = cu_of([max(n, 0) for n in new])
    pad = [-1] * (cap - len(pos))
    return dict(kv=kv2, n_free=len(avail), cu=cu, pos=pos + pad, slot=slot + pad, table=table, free=free, status=0)


class Plan:
    def __init__(self, new, kv, table, free, n_free, page, n_pages, cols, cap, in_place=False):
        B = len(new)
        self.new, self.kv, self.table, self.free, self.nf = i32(new), i32(kv), i32(table), i32(free), i32([n_free])
        self.kv2 = self.kv if in_place else i32([7] * B)
        self.nf2 = self.nf if in_place else i32([7])
        self.cu, self.pos, self.slot, self.status = i32([7] * (B + 1)), i32([7] * (cap + 3)), i32([7] * (cap + 3)), i32([7])
        self.d = hip.PagePlan(new_len=dp(self.new), kv_len=dp(self.kv), n_free=dp(self.nf), table=dp(self.table), free_pages=dp(self.free),
                              kv_len_out=dp(self.kv2), n_free_out=dp(self.nf2), cu_q=dp(self.cu), pos=dp(self.pos), slot=dp(self.slot),
                              status=dp(self.status), table_stride=self.table.stride(0), B=B, page_size=page, n_pages=n_pages,
                              table_cols=cols, max_tokens=cap)
        self.cap = cap

    def run(self):
        ok(hip.lib().qwen_hip_op_page_plan(C.byref(self.d), stream()))
        torch.cuda.synchronize()
        assert self.pos[self.cap:].tolist() == [7] * 3 and self.slot[self.cap:].tolist() == [7] * 3
        return dict(kv=self.kv2.tolist(), n_free=int(self.nf2), cu=self.cu.tolist(), pos=self.pos[:self.cap].tolist(),
                    slot=self.slot[:self.cap].tolist(), table=self.table.tolist(), free=self.free.tolist(), status=int(self.status))


def plan_case(rng, B, page, lo, hi, new_hi, done, spare=5, cap=None):
    kv = rng.integers(lo, hi + 1, B).tolist()
    new = rng.integers(0, new_hi + 1, B).tolist()
    for b in rng.permutation(B)[:done]:
        new[b] = -int(rng.integers(1, 4))
    h = lambda n: -(-n // page)  # noqa: E731
    cols = max(h(k + max(n, 0)) for k, n in zip(kv, new)) + 1
    more = sum(h(k + n) - h(k) for k, n in zip(kv, new) if n >= 0)
    back = sum(h(k) for k, n in zip(kv, new) if n < 0)
    n_free = max(more - back, 0) + spare
    n_pages = sum(map(h, kv)) + n_free
    pages = rng.permutation(n_pages).tolist()
    table = []
    for k in kv:
        table.append(pages[:h(k)] + [-1] * (cols + 2 - h(k)))
        pages = pages[h(k):]
    free = pages + [-7] * (n_pages - n_free)
    total = sum(max(n, 0) for n in new)
    return new, kv, table, free, n_free, page, n_pages, cols, total + 3 if cap is None else cap


@pytest.mark.parametrize("B,page,lo,hi,new_hi,done", [
    (1, 16, 0, 0, 1, 0), (1, 16, 31, 33, 40, 0), (7, 1, 0, 9, 3, 2), (8, 16, 100, 300, 1, 0), (65, 7, 0, 50, 30, 20), (3, 100, 0, 500, 250, 3),
    (1100, 16, 0, 60, 2, 100), (2048, 24, 0, 40, 7, 500), (64, 16, 0, 100, 300, 5), (33, 64, 0, 3, 0, 0)])
def test_plan(B, page, lo, hi, new_hi, done):
    print(f"[case] plan B={B} page={page} {lo}..{hi} +{new_hi} done={done}", flush=True)
    rng = np.random.default_rng(B * 1000 + page)
    for cap in (None, 9000):                            # 9000: past the tokens that the first launch takes
        case = plan_case(rng, B, page, lo, hi, new_hi, done, cap=cap)
        if cap is not None and sum(max(n, 0) for n in case[0]) > cap:
            continue
        want = plan_model(*case)
        assert want["status"] == 0
        p = Plan(*case)
        assert p.run() == want
        assert p.run() == want                          # separate outputs: the call can be repeated
        assert Plan(*case, in_place=True).run() == want


def test_plan_takes_and_gives_back_exactly_everything():
    rng = np.random.default_rng(5)
    case = plan_case(rng, 40, 8, 1, 60, 50, 20, spare=0)
    want = plan_model(*case)
    assert want["status"] == 0
    assert Plan(*case).run() == want


@pytest.mark.parametrize("cap", [None, 9000])
@pytest.mark.parametrize("what", ["pages", "table", "tokens", "negative", "n_free", "twice", "long", "overflow"])
def test_plan_that_cannot_be_made_changes_nothing(what, cap):
    rng = np.random.default_rng(9)
    new, kv, table, free, n_free, page, n_pages, cols, cap = plan_case(rng, 20, 16, 20, 90, 60, 4, spare=0, cap=cap)
    if what == "pages":
        b = next(b for b in range(20) if new[b] >= 0 and (kv[b] + new[b]) // page + 1 < cols)
        new[b] += 2 * page
        cap += 2 * page
        cols += 2
    elif what == "table":
        cols = max(-(-k // page) for k in kv)
    elif what == "tokens":
        cap = sum(max(n, 0) for n in new) - 1
    elif what == "negative":
        kv[3] = -1
    elif what == "n_free":
        n_free = n_pages + 1
    elif what == "twice":
        n_free = n_pages
        free = list(range(n_pages))
    elif what == "long":
        kv[2] = 2 ** 31 - 1
    elif what == "overflow":
        new[1] = new[2] = 2 ** 31 - 1
    case = (new, kv, table, free, n_free, page, n_pages, cols, cap)
    want = plan_model(*case)
    assert want["status"] != 0
    assert Plan(*case).run() == want


def test_plan_makes_no_slot_of_a_bad_page():
    """Page numbers are passed on as they are; one outside the pool makes no slot."""
    new, kv, table = [3, -1, 20], [5, 40, 0], [[99, -1, -1], [2, -4, 7], [-1, -1, -1]]
    free = [10, -9] + [0] * 8
    case = (new, kv, table, free, 2, 16, 10, 3, 30)
    want = plan_model(*case)
    assert want["slot"][:3] == [-1] * 3 and want["table"][2][:2] == [7, -4] and want["slot"][3] == 7 * 16
    assert want["slot"][3 + 16:3 + 20] == [-1] * 4
    assert Plan(*case).run() == want


# ---- append ----------------------------------------------------------------------------------------


def pool(shape, t, layout, g, dev=DEV):
    """[page][head][place][hd] filled with what must not change, in the given order of memory."""
    n_pages, nkv, page, hd = shape
    mem = (n_pages, nkv, page, hd) if layout == "head" else (n_pages, page, nkv, hd)
    x = torch.randn(mem, generator=g).to(t).to(dev)
    return x if layout == "head" else x.transpose(1, 2)


def pages_of(k, v, name):
    return hip.KvPages(k=dp(k), v=dp(v), dtype=hip.DT[name], n_pages=k.shape[0], page_size=k.shape[2], n_kv_heads=k.shape[1],
                       head_dim=k.shape[3], page_stride=k.stride(0), head_stride=k.stride(1), slot_stride=k.stride(2))


@pytest.mark.parametrize("layout,page", [("head", 16), ("slot", 7)])
@pytest.mark.parametrize("norm,rope", [(1, 1), (0, 1), (1, 0), (0, 0)])
@pytest.mark.parametrize("t,kv,nh,nkv,hd,T", [("f32", "bf16", 16, 8, 128, 33), ("f32", "f16", 5, 1, 64, 1), ("bf16", "bf16", 12, 2, 64, 40),
                                              ("f16", "f16", 16, 16, 128, 9)])
def test_append(t, kv, nh, nkv, hd, T, norm, rope, layout, page):
    print(f"[case] append {t}->{kv} {nh}/{nkv}x{hd} T={T} norm={norm} rope={rope} {layout} page={page}", flush=True)
    g = torch.Generator().manual_seed(hd + T)
    n_pages = T // page + 3
    pad = 8                                             # elements between the parts of a row
    rows = (2 * torch.randn(T, (nh + 2 * nkv) * hd + 3 * pad, generator=g)).to(TYPES[t])
    k0, v0 = pool((n_pages, nkv, page, hd), TYPES[kv], layout, g), pool((n_pages, nkv, page, hd), TYPES[kv], layout, g)
    slot = torch.randperm(n_pages * page, generator=g)[:T].to(torch.int32)
    pos = torch.randint(0, 50, (T,), generator=g, dtype=torch.int32)
    skipped = [i for i in range(T) if i % 5 == 3]
    for i in skipped:                                   # outside the cache, or outside the tables
        if rope and i % 2:
            pos[i] = 50 if i % 4 == 1 else -1
        else:
            slot[i] = -1 if i % 4 else n_pages * page
    ang = torch.randn(50, hd // 2, generator=g, dtype=torch.float64)
    cos, sin = ang.cos().float(), ang.sin().float()
    qn, kn = 1 + 0.3 * torch.randn(hd, generator=g), 1 + 0.3 * torch.randn(hd, generator=g)
    dev = [x.to(DEV) for x in (rows, slot, pos, cos, sin, qn, kn)]
    E = rows.element_size()
    q_at, k_at, v_at = 0, nh * hd + pad, (nh + nkv) * hd + 2 * pad
    q_out = torch.full((T, nh * hd + 16), 7.0, dtype=TYPES[t], device=DEV)
    k, v = k0.clone(memory_format=torch.preserve_format), v0.clone(memory_format=torch.preserve_format)
    assert k.stride() == k0.stride()
    base = dp(dev[0])
    d = hip.PageAppend(dtype=hip.DT[t], n_heads=nh, T=T, rope_len=50, eps=1e-6, q=base + q_at * E, k=base + k_at * E, v=base + v_at * E,
                       q_stride=dev[0].stride(0), k_stride=dev[0].stride(0), v_stride=dev[0].stride(0), q_out=dp(q_out),
                       q_out_stride=q_out.stride(0), q_norm=dp(dev[5]) if norm else None, k_norm=dp(dev[6]) if norm else None,
                       rope_cos=dp(dev[3]) if rope else None, rope_sin=dp(dev[4]) if rope else None, pos=dp(dev[2]) if rope else None,
                       slot=dp(dev[1]))
    ok(hip.lib().qwen_hip_op_page_append(C.byref(pages_of(k, v, kv)), C.byref(d), stream()))
    torch.cuda.synchronize()

    def want(x, gain):
        x = x.double().view(T, -1, hd)
        y = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * gain.double() if norm else x
        if not rope:
            return y, y.abs()
        p = pos.long().clamp(0, 49)
        c, s = cos.double()[p][:, None], sin.double()[p][:, None]
        a, b = y[..., :hd // 2], y[..., hd // 2:]
        big = torch.cat((a.abs() + b.abs(),) * 2, -1)
        return torch.cat((a * c - b * s, b * c + a * s), -1), big

    def close(got, exact, big, name):
        eps = torch.finfo(TYPES[name]).eps
        tiny = 2.0 ** -25 if name == "f16" else 0.0     # half of f16's last step below its normal range
        tol = 16 * 2.0 ** -24 * big * (1 if norm or rope else 0) + eps / 2 * 1.001 * (exact.abs() + 16 * 2.0 ** -24 * big) + tiny
        assert bool(((got.double() - exact).abs() <= tol).all()), float(((got.double() - exact).abs() / tol).max())

    live = [i for i in range(T) if i not in skipped]
    qw, qb = want(rows[:, q_at:q_at + nh * hd], qn)
    kw, kb = want(rows[:, k_at:k_at + nkv * hd], kn)
    vw = rows[:, v_at:v_at + nkv * hd].double().view(T, nkv, hd)
    got = q_out.cpu()
    close(got[live, :nh * hd].view(-1, nh, hd), qw[live], qb[live], t)
    assert bool((got[skipped] == 7).all()) and bool((got[:, nh * hd:] == 7).all())
    k, v, k0, v0 = k.cpu(), v.cpu(), k0.cpu(), v0.cpu()
    for i in live:
        p, o = int(slot[i]) // page, int(slot[i]) % page
        close(k[p, :, o], kw[i], kb[i], kv)
        close(v[p, :, o], vw[i], torch.zeros(nkv, hd, dtype=torch.float64), kv)
        k[p, :, o], v[p, :, o] = k0[p, :, o], v0[p, :, o]
    assert torch.equal(k, k0) and torch.equal(v, v0)    # nothing else was written


def test_append_in_place_and_without_q():
    g = torch.Generator().manual_seed(3)
    rows = torch.randn(6, 4 * 64, generator=g).to(DEV)
    k, v = pool((4, 1, 4, 64), torch.bfloat16, "head", g), pool((4, 1, 4, 64), torch.bfloat16, "head", g)
    slot = i32([3, 5, 7, 9, 11, 0])
    gain = torch.full((64,), 2.0, device=DEV)
    kv = pages_of(k, v, "bf16")
    d = dict(dtype=0, n_heads=2, T=6, eps=0.0, k=dp(rows) + 2 * 64 * 4, v=dp(rows) + 3 * 64 * 4, q_stride=256, k_stride=256, v_stride=256,
             slot=dp(slot), k_norm=dp(gain))
    a = hip.PageAppend(**d)
    ok(hip.lib().qwen_hip_op_page_append(C.byref(kv), C.byref(a), stream()))
    torch.cuda.synchronize()
    k1, before = k.clone(), rows.clone()
    # the same with q: normed in place, k not read before or after it is not q's
    a = hip.PageAppend(**d, q=dp(rows), q_out=dp(rows), q_out_stride=256, q_norm=dp(gain))
    ok(hip.lib().qwen_hip_op_page_append(C.byref(kv), C.byref(a), stream()))
    torch.cuda.synchronize()
    assert torch.equal(k, k1) and torch.equal(rows[:, 128:], before[:, 128:])
    x = before[:, :128].double().view(6, 2, 64)
    y = 2 * x / x.square().mean(-1, keepdim=True).sqrt()
    assert float(((rows[:, :128].double().view(6, 2, 64) - y).abs() / y.abs().clamp(min=1e-30)).max()) < 16 * 2.0 ** -24



def test_append_writes_q_beside_the_rows_it_reads():
    """q_out as further columns of the rows' own buffer, and one token in place with a stride of its own."""
    g = torch.Generator().manual_seed(5)
    rows = torch.randn(6, 6 * 64 + 16, generator=g).to(DEV)                 # q (2 heads), k, v, q_out (2 heads)
    before, W = rows.clone(), rows.shape[1]
    k, v = (pool((4, 1, 4, 64), torch.bfloat16, "head", g) for _ in range(2))
    slot, gain = i32([3, 5, 7, 9, 11, 0]), torch.full((64,), 2.0, device=DEV)
    d = hip.PageAppend(dtype=0, n_heads=2, T=6, eps=0.0, q=dp(rows), k=dp(rows) + 128 * 4, v=dp(rows) + 192 * 4, q_out=dp(rows) + 256 * 4, q_stride=W,
                       k_stride=W, v_stride=W, q_out_stride=W, slot=dp(slot), q_norm=dp(gain))
    ok(hip.lib().qwen_hip_op_page_append(C.byref(pages_of(k, v, "bf16")), C.byref(d), stream()))
    torch.cuda.synchronize()
    keep = [*range(256), *range(384, W)]
    assert torch.equal(rows[:, keep], before[:, keep])
    x = before[:, :128].double().view(6, 2, 64)
    y = 2 * x / x.square().mean(-1, keepdim=True).sqrt()
    assert float(((rows[:, 256:384].double().view(6, 2, 64) - y).abs() / y.abs().clamp(min=1e-30)).max()) < 16 * 2.0 ** -24
    for i, s in enumerate(slot.tolist()):
        assert torch.equal(k[s // 4, 0, s % 4], before[i, 128:192].bfloat16()) and torch.equal(v[s // 4, 0, s % 4], before[i, 192:256].bfloat16())
    d.T, d.q_out, d.q_out_stride = 1, dp(rows), 128
    ok(hip.lib().qwen_hip_op_page_append(C.byref(pages_of(k, v, "bf16")), C.byref(d), stream()))
    torch.cuda.synchronize()
    assert torch.equal(rows[0, :128], rows[0, 256:384]) and torch.equal(rows[1:, :128], before[1:, :128])



@pytest.mark.parametrize("order", ["page k/v head place", "page place head k/v", "head page place k/v", "k/v place head page", "page place, gap"])
def test_append_into_caches_of_any_order(order):
    """k and v in one buffer, interleaved at any level: what separate pools hold."""
    n, nkv, page, hd = 4, 2, 4, 64
    g = torch.Generator().manual_seed(6)
    rows = torch.randn(9, 2 * nkv * hd, generator=g).to(torch.bfloat16).to(DEV)
    slot = i32([3, 5, 7, 9, 11, 0, 15, 8, 1])
    axes = {"page k/v head place": (1, 0, 2, 3), "page place head k/v": (3, 0, 2, 1), "head page place k/v": (3, 1, 0, 2), "k/v place head page": (0, 3, 2, 1)}
    if order in axes:                                           # where k/v, page, head and place stand
        at = axes[order]
        dims = [0] * 4
        for i, d in zip(at, (2, n, nkv, page)):
            dims[i] = d
        both = torch.zeros(*dims, hd, dtype=torch.bfloat16, device=DEV).permute(*at, 4)
        k, v = both[0], both[1]
    else:                                                       # v in the gaps that k's pages leave
        buf = torch.zeros(n * 2 * page * nkv * hd, dtype=torch.bfloat16, device=DEV)
        k, v = (buf[o * page * nkv * hd:].as_strided((n, nkv, page, hd), (2 * page * nkv * hd, hd, nkv * hd, 1)) for o in (0, 1))
    ks, vs = (torch.zeros(n, nkv, page, hd, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    d = hip.PageAppend(dtype=1, T=9, k=dp(rows), v=dp(rows) + nkv * hd * 2, k_stride=2 * nkv * hd, v_stride=2 * nkv * hd, slot=dp(slot))
    for a, b in ((k, v), (ks, vs)):
        ok(hip.lib().qwen_hip_op_page_append(C.byref(pages_of(a, b, "bf16")), C.byref(d), stream()))
    torch.cuda.synchronize()
    assert torch.equal(k, ks) and torch.equal(v, vs) and bool(ks.any())
    assert torch.equal(ks[1, :, 1], rows[1, :nkv * hd].view(nkv, hd)) and torch.equal(vs[1, :, 1], rows[1, nkv * hd:].view(nkv, hd))


def far_pool(n_pages, nkv, page, hd, total):
    """bf16 pages `total` bytes from the first to the end, far apart."""
    far = total // 2 // n_pages // 64 * 64
    return torch.zeros(total // 2, dtype=torch.bfloat16, device=DEV).as_strided((n_pages, nkv, page, hd), (far, page * hd, hd, 1))


def test_append_past_32_bits():
    """Slots whose byte offsets pass 2^32."""
    rows = torch.randn(2, 192, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(DEV)
    slot = i32([5, 2])
    k, v = far_pool(3, 1, 2, 64, 8 << 30), far_pool(3, 1, 2, 64, 8 << 30)
    assert 2 * k.stride(0) * 2 > 1 << 32
    d = hip.PageAppend(dtype=1, n_heads=1, T=2, eps=0.0, k=dp(rows), v=dp(rows) + 128, k_stride=192, v_stride=192, slot=dp(slot))
    ok(hip.lib().qwen_hip_op_page_append(C.byref(pages_of(k, v, "bf16")), C.byref(d), stream()))
    torch.cuda.synchronize()
    for x, at in ((k, 0), (v, 64)):
        assert torch.equal(x[2, 0, 1], rows[0, at:at + 64]) and torch.equal(x[1, 0, 0], rows[1, at:at + 64])


# ---- attention -------------------------------------------------------------------------------------


def attend64(q, k, v, first, window, scale):
    """q [n][nh][hd] at positions first .., k and v [L][nkv][hd]: the rows, and sum p |v| / sum p."""
    n, nh, hd = q.shape
    L, nkv = k.shape[:2]
    out, mag = torch.zeros(n, nh, hd, dtype=torch.float64), torch.zeros(n, nh, hd, dtype=torch.float64)
    pos, j = torch.arange(first, first + n)[:, None], torch.arange(L)[None]
    see = (j <= pos) & ((j > pos - window) if window else torch.ones_like(j, dtype=torch.bool))
    some = see.any(1)
    for h in range(nh):
        kk, vv = k[:, h // (nh // nkv)].double(), v[:, h // (nh // nkv)].double()
        s = (q[:, h].double() @ kk.T * scale).masked_fill(~see, -math.inf)
        p = torch.zeros_like(s)
        p[some] = s[some].softmax(-1)
        out[:, h], mag[:, h] = p @ vv, p @ vv.abs()
    return out, mag


def close_attention(got, exact, mag, t, n_max, vmax):
    got, eps = got.double().cpu(), torch.finfo(TYPES[t]).eps
    if t == "f32":
        off = float((got - exact).norm() / exact.norm().clamp(min=1e-30))
        assert off <= 8e-6, off
        assert bool(((got - exact).abs() <= 5e-5 * vmax).all())
        return
    tol = eps / 2 * 1.01 * (2 * exact.abs() + mag) + 5e-5 * vmax + (2 * n_max * 2.0 ** -25 * vmax + 2.0 ** -25 if t == "f16" else 0.0)
    bad = ((got - exact).abs() / tol).max()
    assert bool(bad <= 1), float(bad)


class Paged:
    """Requests of (tokens before, new tokens) over a shuffled pool; what no request holds is NaN."""

    def __init__(self, reqs, nh, nkv, hd, t, kv, page, layout, seed=0, T=None, window=0, max_q=None, max_kv=None, scale=None):
        g = torch.Generator().manual_seed(seed)
        self.reqs, self.t, self.window, self.scale = reqs, t, window, scale or hd ** -0.5
        lens = [a + n for a, n in reqs]
        h = lambda n: -(-n // page)  # noqa: E731
        need = [h(n) for n in lens]
        n_pages, cols = sum(need) + 3, max(need + [1]) + 2
        perm = torch.randperm(n_pages, generator=g).tolist()
        table = torch.full((len(reqs), cols + 1), -1, dtype=torch.int32)
        k, v = (pool((n_pages, nkv, page, hd), TYPES[kv], layout, g, "cpu") for _ in range(2))
        self.kv = []
        fill = torch.full((), math.nan)
        kc, vc = torch.empty_like(k).fill_(fill), torch.empty_like(v).fill_(fill)
        for b, n in enumerate(lens):
            mine, perm = perm[:need[b]], perm[need[b]:]
            table[b, :need[b]] = torch.tensor(mine, dtype=torch.int32)
            rows = [(mine[p // page], p % page) for p in range(n)]
            for p, o in rows:
                kc[p, :, o], vc[p, :, o] = k[p, :, o], v[p, :, o]
            ix = (torch.tensor([p for p, _ in rows], dtype=torch.long), torch.tensor([o for _, o in rows], dtype=torch.long))
            self.kv.append((k[ix[0], :, ix[1]], v[ix[0], :, ix[1]]))
        new = [n for _, n in reqs]
        self.cu = cu_of(new)
        self.T = self.cu[-1] if T is None else T
        self.q = (1.5 * torch.randn(self.T, nh, hd + 8, generator=g)).to(TYPES[t])[..., :hd]
        q = torch.zeros(self.T, nh * hd + 16).to(TYPES[t])
        q[:, :nh * hd] = self.q.reshape(self.T, -1)
        self.kc, self.vc, self.qd = kc.to(DEV), vc.to(DEV), q.to(DEV)
        self.table, self.cud, self.kvl = table.to(DEV), i32(self.cu), i32(lens)
        self.out = torch.full((self.T, nh * hd + 8), 7.0, dtype=TYPES[t], device=DEV)
        self.pages = pages_of(self.kc, self.vc, kv)
        self.d = hip.PageAttn(dtype=hip.DT[t], n_heads=nh, B=len(reqs), T=self.T, table_cols=cols, max_q=max(new + [0]) if max_q is None else max_q,
                              max_kv=max(lens + [0]) if max_kv is None else max_kv, window=window, scale=self.scale, q=dp(self.qd), out=dp(self.out),
                              q_stride=q.stride(0), out_stride=self.out.stride(0), cu_q=dp(self.cud), kv_len=dp(self.kvl), table=dp(self.table),
                              table_stride=self.table.stride(0))
        self.shape = (nh, hd)

    def run(self):
        n = hip.lib().qwen_hip_op_page_attention_workspace(C.byref(self.pages), C.byref(self.d))
        assert n >= 0, hip.last_error()
        self.ws = torch.full((n + 64,), 255, dtype=torch.uint8, device=DEV)      # NaN bits; 64 bytes that stay
        self.d.workspace, self.d.workspace_bytes = dp(self.ws), n
        ok(hip.lib().qwen_hip_op_page_attention(C.byref(self.pages), C.byref(self.d), stream()))
        torch.cuda.synchronize()
        assert bool((self.ws[n:] == 255).all())
        nh, hd = self.shape
        assert bool((self.out[:, nh * hd:] == 7).all()) and bool((self.out[self.cu[-1]:] == 7).all())
        return self.out[:self.cu[-1], :nh * hd].view(-1, nh, hd)

    def want(self):
        both = [attend64(self.q[self.cu[b]:self.cu[b + 1]], k, v, k.shape[0] - n, self.window, self.scale)
                for b, ((_, n), (k, v)) in enumerate(zip(self.reqs, self.kv))]
        return torch.cat([o for o, _ in both]), torch.cat([m for _, m in both])

    def check(self):
        got = self.run()
        exact, mag = self.want()
        close_attention(got, exact, mag, self.t, max(a + n for a, n in self.reqs), float(max(v.abs().max() for _, v in self.kv if v.numel())))


HEADS = [(16, 8, 128), (16, 16, 64), (12, 2, 64), (32, 4, 128), (7, 1, 128), (128, 2, 64)]
KINDS = [("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")]


@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_page_attention_single_tokens(t, kv, nh, nkv, hd):
    print(f"[case] paged single tokens {t} {nh}/{nkv}x{hd}", flush=True)
    reqs = [(0, 1), (1, 1), (30, 1), (31, 1), (32, 1), (15, 1), (700, 1), (255, 1), (256, 1), (333, 1)]
    Paged(reqs, nh, nkv, hd, t, kv, 16, "head", seed=1).check()
    Paged(reqs[:3], nh, nkv, hd, t, kv, 5, "slot", seed=2, window=17).check()
    # as if the longest held 10^5 keys: many ranges, streamed; of 256 keys, and the last range takes what is left
    Paged(reqs, nh, nkv, hd, t, kv, 16, "slot", seed=2, max_kv=100000).check()
    Paged(reqs, nh, nkv, hd, t, kv, 16, "slot", seed=2, max_kv=512).check()


@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("nh,nkv,hd,page,layout,window", [(16, 8, 128, 16, "head", 0), (16, 16, 64, 7, "slot", 72), (12, 2, 64, 64, "head", 5),
                                                          (32, 4, 128, 1, "slot", 0), (7, 1, 128, 100, "head", 200)])
def test_page_attention_chunks(t, kv, nh, nkv, hd, page, layout, window):
    print(f"[case] paged chunks {t} {nh}/{nkv}x{hd} page={page} {layout} window={window}", flush=True)
    reqs = [(0, 1), (0, 45), (130, 3), (0, 0), (60, 65), (17, 0), (250, 131), (5, 2), (1, 33)]
    p = Paged(reqs, nh, nkv, hd, t, kv, page, layout, seed=3, window=window)
    p.check()
    # a hint that is too small, or none, changes the launch and not the result
    for max_q, max_kv in ((1, 10), (0, 0), (10, 4000)):
        q = Paged(reqs, nh, nkv, hd, t, kv, page, layout, seed=3, window=window, max_q=max_q, max_kv=max_kv)
        q.check()


@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("nh,nkv,hd,page,layout,window", [(16, 8, 128, 16, "head", 0), (16, 16, 64, 24, "slot", 72), (8, 4, 64, 64, "head", 5),
                                                          (6, 2, 128, 3, "slot", 300)])
def test_page_attention_long_chunks(t, kv, nh, nkv, hd, page, layout, window):
    """Chunks of many rows: whole tiles, the first and last rows of tiles, keys that end inside a block."""
    print(f"[case] paged long chunks {t} {nh}/{nkv}x{hd} page={page} {layout} window={window}", flush=True)
    reqs = [(0, 257), (63, 128), (300, 64), (1, 0), (0, 191), (128, 129)]
    Paged(reqs, nh, nkv, hd, t, kv, page, layout, seed=14, window=window).check()
    Paged(reqs, nh, nkv, hd, t, kv, page, layout, seed=14, window=window, max_q=20, max_kv=6000).check()


@pytest.mark.parametrize("t,kv", KINDS)
def test_page_attention_many_requests_and_padding(t, kv):
    """More requests than a ballot looks at, empty ones among them, and rows behind the last one."""
    reqs = [((b * 37) % 90, (b * 5) % 4 * (b % 3)) for b in range(150)]
    Paged(reqs, 4, 2, 64, t, kv, 8, "head", seed=5, T=sum(n for _, n in reqs) + 9).check()


@pytest.mark.parametrize("t,kv", KINDS)
def test_page_attention_one_long_request(t, kv):
    """One request: its keys are split over many workgroups and joined."""
    p = Paged([(3000, 1)], 16, 8, 128, t, kv, 16, "head", seed=6)
    assert hip.lib().qwen_hip_op_page_attention_workspace(C.byref(p.pages), C.byref(p.d)) > 0
    p.check()
    Paged([(2900, 40)], 2, 1, 128, t, kv, 16, "slot", seed=7).check()


@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("reqs", [[(40, 1), (600, 1), (33, 1)], [(40, 50), (200, 90)]])
def test_rows_before_the_first_request_stay(t, kv, reqs):
    p = Paged(reqs, 4, 2, 64, t, kv, 16, "head", seed=22, T=sum(n for _, n in reqs))
    exact, mag = p.want()
    lead = 5                                                    # the same rows five tokens later
    q, out = p.qd, p.out
    p.qd, p.out = torch.cat((torch.full((lead, q.shape[1]), math.nan, dtype=q.dtype, device=DEV), q)), torch.full((q.shape[0] + lead, out.shape[1]), 7.0, dtype=out.dtype, device=DEV)
    p.cud.copy_(i32([c + lead for c in p.cu]))
    p.d.q, p.d.out, p.d.T = dp(p.qd), dp(p.out), q.shape[0] + lead
    n = hip.lib().qwen_hip_op_page_attention_workspace(C.byref(p.pages), C.byref(p.d))
    ws = torch.full((n + 1,), 255, dtype=torch.uint8, device=DEV)
    p.d.workspace, p.d.workspace_bytes = dp(ws), n
    ok(hip.lib().qwen_hip_op_page_attention(C.byref(p.pages), C.byref(p.d), stream()))
    torch.cuda.synchronize()
    assert bool((p.out[:lead] == 7).all())
    close_attention(p.out[lead:, :256].reshape(-1, 4, 64), exact, mag, t, 700, 6.0)


@pytest.mark.parametrize("t,kv", KINDS)
def test_two_calls_at_once(t, kv):
    """Two streams, a workspace each, the same cache."""
    ps = [Paged([(900, 1), (50, 1), (300, 1)], 4, 2, 64, t, kv, 16, "head", seed=23) for _ in range(2)]
    ps[1].d.q = dp(ps[0].qd)
    ps[1].pages, ps[1].d.table = ps[0].pages, dp(ps[0].table)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ws = []
    for p in ps:
        n = hip.lib().qwen_hip_op_page_attention_workspace(C.byref(p.pages), C.byref(p.d))
        ws.append(torch.full((n + 1,), 255, dtype=torch.uint8, device=DEV))
        p.d.workspace, p.d.workspace_bytes = dp(ws[-1]), n
    torch.cuda.synchronize()
    for _ in range(20):
        for p, st in zip(ps, streams):
            ok(hip.lib().qwen_hip_op_page_attention(C.byref(p.pages), C.byref(p.d), st.cuda_stream))
    torch.cuda.synchronize()
    exact, mag = ps[0].want()
    assert torch.equal(ps[0].out[:3], ps[1].out[:3])
    close_attention(ps[0].out[:, :256].reshape(3, 4, 64), exact, mag, t, 901, 6.0)


@pytest.mark.parametrize("t,kv", KINDS)
def test_rows_that_see_nothing_are_zero(t, kv):
    """Fewer keys than new tokens (the first rows lie before position 0), no keys, a negative length, no pages."""
    p = Paged([(0, 40), (0, 3), (0, 5), (9, 4)], 4, 2, 64, t, kv, 16, "head", seed=8)
    p.kvl.copy_(i32([25, 0, -3, 13]))
    p.table[3] = -1
    got = p.run()
    assert bool((got[:15] == 0).all()) and bool((got[40:] == 0).all())
    k, v = p.kv[0]
    exact, mag = attend64(p.q[15:40], k[:25], v[:25], 0, 0, p.scale)
    close_attention(got[15:40], exact, mag, t, 25, float(v.abs().max()))


@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 2, 64), (16, 2, 128)])
def test_hidden_values_never_reach_a_row(t, kv, value, nh, nkv, hd):
    """Keys and values that only later rows see hold NaN or infinities: the earlier rows do not change."""
    reqs = [(40, 50), (2000, 6)]
    p = Paged(reqs, nh, nkv, hd, t, kv, 16, "head", seed=9)
    exact, mag = p.want()
    for b, bad in ((0, 70), (1, 2003)):
        pg = int(p.table[b, bad // 16])
        p.kc[pg, :, bad % 16] = value
        p.vc[pg, :, bad % 16] = value
    got = p.run().cpu()
    fine = list(range(30)) + [50, 51, 52]                       # tokens at positions before the bad ones
    vmax = float(max(v.abs().max() for _, v in p.kv))
    close_attention(got[fine], exact[fine], mag[fine], t, 2006, vmax)
    after = got[[30, 49, 53, 55]].float()
    if math.isnan(value):
        assert bool(after.isnan().all())
    else:
        assert not bool(after.isfinite().all())


def test_bad_pages_hold_no_keys():
    p = Paged([(100, 3), (64, 1)], 4, 2, 64, "bf16", "bf16", 16, "head", seed=10)
    keep = torch.ones(103, dtype=torch.bool)
    p.table[0, 1], p.table[0, 4] = p.pages.n_pages, -5
    keep[16:32] = keep[64:80] = False
    got = p.run().cpu()
    k, v = p.kv[0]
    for i in range(3):
        m = keep & (torch.arange(103) <= 100 + i)
        exact, mag = attend64(p.q[i:i + 1], k[m], v[m], 10 ** 6, 0, p.scale)
        close_attention(got[i:i + 1], exact, mag, "bf16", 103, float(v.abs().max()))


def test_f32_keeps_the_differences_of_large_scores():
    """Scores near 1000 that differ by little, over many blocks of keys: the softmax is one of differences, so only the
    scores' own rounding counts, 64 terms of an f32 sum around 1000 (2^-24 1000 a term at most, 8 of them by chance)."""
    p = Paged([(900, 1), (0, 40)], 2, 1, 64, "f32", "bf16", 16, "head", seed=19)
    k0 = torch.full((64,), 4.0)
    p.q[:] = 30.0
    p.qd[:, :128] = 30.0
    for b, (k, v) in enumerate(p.kv):
        k[:] = (k0 + 0.02 * torch.randn(k.shape, generator=torch.Generator().manual_seed(b))).to(torch.bfloat16)
        n, pg = k.shape[0], p.table[b].cpu()
        for i in range(n):
            p.kc[int(pg[i // 16]), :, i % 16] = k[i].to(DEV)
    got, (exact, _) = p.run().double().cpu(), p.want()
    off = float((got - exact).norm() / exact.norm())
    assert off < 8 * 1000 * 2.0 ** -24, off


def test_large_scores_do_not_overflow():
    """Scores of thousands: the softmax is one of differences."""
    for t, kv in KINDS:
        p = Paged([(50, 2)], 4, 2, 64, t, kv, 16, "head", seed=11, scale=200.0)
        got, (exact, mag) = p.run().double().cpu(), p.want()
        assert bool(got.isfinite().all())
        # one key outweighs the rest: its row, to the rounding of the scores (2^-22 of thousands) and the type's
        assert float((got - exact).norm() / exact.norm()) < 0.02



@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("reqs,packed_too", [([(0, 40), (30, 3)], True), ([(700, 1), (30, 1), (0, 1)], False), ([(0, 900)], True), ([(500, 130), (64, 200)], False)])
def test_scores_past_f32_once_scaled(t, kv, reqs, packed_too, sign):
    """Scores that are finite, but not times the scale: still the softmax of their differences.  q and k are whole numbers up
    to 7 times 2^13 (q negative: scores all below), so every score is a whole number under 64 49 2^26, exact in f32 in any order;
    scores that differ do so by 2^26 1e30, so a row is the mean of v over its keys of the largest score, to the tolerances above."""
    nh, nkv, hd = 16, 8, 64
    p = Paged(reqs, nh, nkv, hd, t, kv, 16, "head", seed=34, scale=1e30)
    g = torch.Generator().manual_seed(35)
    p.q[:] = (sign * torch.randint(1, 8, p.q.shape, generator=g) * 2.0 ** 13).to(TYPES[t])
    p.qd[:, :nh * hd] = p.q.reshape(p.T, -1).to(DEV)
    for b, (k, _) in enumerate(p.kv):
        k[:] = (torch.randint(1, 8, k.shape, generator=g) * 2.0 ** 13).to(k.dtype)
        at = torch.arange(k.shape[0])
        p.kc[p.table[b].cpu().long()[at // 16].to(DEV), :, (at % 16).to(DEV)] = k.to(DEV)
    exact, mag = p.want()
    vmax = float(max(v.abs().max() for _, v in p.kv))
    close_attention(p.run(), exact, mag, t, 1000, vmax)
    if not packed_too:
        return
    n = reqs[0][1]
    rows = torch.cat((p.q[:n].reshape(n, -1), p.kv[0][0].reshape(n, -1).to(TYPES[t]), p.kv[0][1].reshape(n, -1).to(TYPES[t])), 1).to(DEV)
    out, cu, E = torch.full((n, nh * hd), 7.0, dtype=TYPES[t], device=DEV), i32([0, n]), rows.element_size()
    d = hip.PackedAttn(dtype=hip.DT[t], n_heads=nh, n_kv_heads=nkv, head_dim=hd, B=1, T=n, scale=1e30, q=dp(rows), k=dp(rows) + nh * hd * E,
                       v=dp(rows) + (nh + nkv) * hd * E, out=dp(out), q_stride=rows.stride(0), k_stride=rows.stride(0), v_stride=rows.stride(0),
                       out_stride=nh * hd, cu=dp(cu))
    ok(hip.lib().qwen_hip_op_packed_attention(C.byref(d), stream()))
    torch.cuda.synchronize()
    close_attention(out.view(n, nh, hd), exact[:n], mag[:n], t, 1000, vmax)


def test_one_key_returns_its_value():
    """With one visible key the output is that key's value to the bit, in every type (f32: its planes sum to it)."""
    for t, kv in KINDS:
        p = Paged([(0, 1), (7, 4)], 4, 2, 128, t, kv, 16, "head", seed=12, window=1)
        got = p.run()
        for b, ((a, n), (_, v)) in enumerate(zip(p.reqs, p.kv)):
            want = v[a:a + n].repeat_interleave(2, 1).to(TYPES[t])
            assert torch.equal(got[p.cu[b]:p.cu[b + 1]].cpu(), want)
    q = torch.randn(5, 6 * 64, generator=torch.Generator().manual_seed(1)).to(DEV)
    out = torch.empty(5, 2 * 64, device=DEV)
    ok(packed(q, [5], 2, 2, 64, "f32", out, window=1))
    torch.cuda.synchronize()
    assert torch.equal(out, q[:, 256:])


def test_cache_past_32_bits():
    """Keys in pages whose byte offsets pass 2^32."""
    p = Paged([(70, 1)], 2, 1, 64, "bf16", "bf16", 16, "head", seed=13)
    k, v = (far_pool(p.pages.n_pages, 1, 16, 64, 6 << 30) for _ in range(2))
    k.copy_(p.kc)
    v.copy_(p.vc)
    p.pages.k, p.pages.v, p.pages.page_stride = dp(k), dp(v), k.stride(0)
    assert int(p.table.max()) * k.stride(0) * 2 > 1 << 32
    p.check()


@pytest.mark.parametrize("t,kv", KINDS)
def test_chunk_over_a_cache_past_32_bits(t, kv):
    """The same for chunks of many rows."""
    p = Paged([(70, 120), (0, 90)], 4, 1, 128, t, kv, 16, "head", seed=15)
    total = 7 << 30
    far = total // 2 // p.pages.n_pages // 128 * 128
    k, v = (torch.zeros(total // 2, dtype=TYPES[kv], device=DEV).as_strided((p.pages.n_pages, 1, 16, 128), (far, 2048, 128, 1)) for _ in range(2))
    k.copy_(p.kc)
    v.copy_(p.vc)
    p.pages.k, p.pages.v, p.pages.page_stride = dp(k), dp(v), far
    assert int(p.table.max()) * far * 2 > 1 << 32
    p.check()


@pytest.mark.parametrize("t,kv", KINDS)
@pytest.mark.parametrize("far", ["page", "place", "head"])
@pytest.mark.parametrize("reqs", [[(70, 120), (0, 90)], [(150, 1), (31, 1), (0, 1)]])
def test_a_cache_between_2_and_4_gib(t, kv, far, reqs):
    """Byte offsets past 2^31 that stay under 2^32, by pages, by places of a page and by heads."""
    p = Paged(reqs, 8, 2, 128, t, kv, 16, "head", seed=36)
    n, total = p.pages.n_pages, (1 << 31) - 500000
    step = {"page": total // n, "place": total // 16, "head": total - (1 << 18)}[far] // 128 * 128
    assert n <= 64                                              # the rest of a place's offset: under 2^18 elements
    strides = {"page": (step, 2048, 128), "place": (256, 128, step), "head": (2048, step, 128)}[far]
    k, v = (torch.zeros(total, dtype=TYPES[kv], device=DEV).as_strided((n, 2, 16, 128), strides + (1,)) for _ in range(2))
    k.copy_(p.kc)
    v.copy_(p.vc)
    last = {"page": int(p.table.max()), "place": 15, "head": 1}[far] * step * 2
    assert (1 << 31) <= last < 1 << 32
    p.pages.k, p.pages.v, p.pages.page_stride, p.pages.head_stride, p.pages.slot_stride = dp(k), dp(v), *strides
    p.check()



@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_many_long_requests(t):
    """More requests than the order by length looks at (256), of many rows each."""
    lens = [(b * 13) % 40 + 20 * (b % 2) for b in range(300)]
    T, g = sum(lens), torch.Generator().manual_seed(16)
    rows = torch.randn(T, 6 * 64, generator=g).to(TYPES[t])
    out = torch.full((T, 256), 7.0, dtype=TYPES[t], device=DEV)
    ok(packed(rows.to(DEV), lens, 4, 1, 64, t, out))
    exact, mag = packed_want(rows, lens, 4, 1, 64, 0)
    close_attention(out.cpu().view(T, 4, 64), exact, mag, t, 60, float(rows.abs().max()))
    Paged([(b % 7, n) for b, n in enumerate(lens)], 4, 1, 64, t, "bf16", 8, "slot", seed=17).check()


def test_most_requests():
    """65535 requests, most of them empty, in every launch that finds them by their rows."""
    B, g = 65535, torch.Generator().manual_seed(18)
    lens = [0] * B
    for b, n in ((0, 3), (1, 40), (63, 1), (64, 2), (1023, 33), (1024, 5), (40000, 70), (65534, 17)):
        lens[b] = n
    T = sum(lens)
    for t, nh in (("f32", 2), ("bf16", 2)):
        rows = torch.randn(T, (nh + 2) * 64, generator=g).to(TYPES[t])
        out = torch.full((T, nh * 64), 7.0, dtype=TYPES[t], device=DEV)
        ok(packed(rows.to(DEV), lens, nh, 1, 64, t, out))
        exact, mag = packed_want(rows, [n for n in lens if n], nh, 1, 64, 0)
        close_attention(out.cpu().view(T, nh, 64), exact, mag, t, 70, float(rows.abs().max()))


def packed(rows, lens, nh, nkv, hd, t, out, window=0, cu=None, T=None):
    E = rows.element_size()
    cu = i32(cu_of(lens)) if cu is None else cu
    d = hip.PackedAttn(dtype=hip.DT[t], n_heads=nh, n_kv_heads=nkv, head_dim=hd, B=len(lens), T=rows.shape[0] if T is None else T,
                       window=window, scale=hd ** -0.5, q=dp(rows), k=dp(rows) + nh * hd * E, v=dp(rows) + (nh + nkv) * hd * E, out=dp(out),
                       q_stride=rows.stride(0), k_stride=rows.stride(0), v_stride=rows.stride(0), out_stride=out.stride(0), cu=dp(cu))
    rc = hip.lib().qwen_hip_op_packed_attention(C.byref(d), stream())
    torch.cuda.synchronize()                                    # cu lives this long
    return rc


def packed_want(rows, lens, nh, nkv, hd, window):
    out = []
    for a, b in zip(cu_of(lens), cu_of(lens)[1:]):
        q, k, v = rows[a:b].split((nh * hd, nkv * hd, nkv * hd), 1)
        out.append(attend64(q.reshape(-1, nh, hd), k.reshape(-1, nkv, hd), v.reshape(-1, nkv, hd), 0, window, hd ** -0.5))
    return torch.cat([o for o, _ in out]), torch.cat([m for _, m in out])


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("nh,nkv,hd,lens,window", [
    (16, 8, 128, [1], 0), (16, 8, 128, [45, 1, 128, 0, 33], 0), (16, 16, 64, [200, 31, 32, 64, 65], 72), (12, 2, 64, [301, 17], 0),
    (7, 1, 128, [100, 0, 0, 50], 30), (32, 4, 128, [513], 0), (4, 2, 64, [3] * 130 + [0] * 20 + [40], 0), (16, 8, 128, [600, 90], 1000),
    (16, 8, 128, [129, 63, 64, 65, 0, 1, 256], 0), (6, 2, 64, [43, 171, 300], 65)])
def test_packed_attention(t, nh, nkv, hd, lens, window):
    print(f"[case] packed {t} {nh}/{nkv}x{hd} {lens[:6]} window={window}", flush=True)
    g = torch.Generator().manual_seed(len(lens) + hd)
    T = sum(lens)
    rows = torch.randn(T + 5, (nh + 2 * nkv) * hd + 8, generator=g).to(TYPES[t])
    rows[T:] = math.nan                                         # rows of no sequence
    out = torch.full((T + 5, nh * hd + 8), 7.0, dtype=TYPES[t], device=DEV)
    ok(packed(rows.to(DEV), lens, nh, nkv, hd, t, out, window))
    out = out.cpu()
    assert bool((out[T:] == 7).all()) and bool((out[:, nh * hd:] == 7).all())
    w = rows[:T, :(nh + 2 * nkv) * hd]
    exact, mag = packed_want(w, lens, nh, nkv, hd, window)
    close_attention(out[:T, :nh * hd].view(T, nh, hd), exact, mag, t, max(lens), float(w.abs().max()))


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("n,nh,nkv", [(50, 4, 2), (900, 16, 8)])
def test_out_beside_the_rows_it_is_made_of(t, n, nh, nkv):
    """out as further columns of q, k and v's own buffer, and k and v the same rows of it."""
    hd, g = 64, torch.Generator().manual_seed(24)
    W = (2 * nh + nkv) * hd
    rows = torch.randn(n, W, generator=g).to(TYPES[t])
    dev, cu, E = rows.to(DEV), i32([0, n]), rows.element_size()
    d = hip.PackedAttn(dtype=hip.DT[t], n_heads=nh, n_kv_heads=nkv, head_dim=hd, B=1, T=n, scale=hd ** -0.5, q=dp(dev), k=dp(dev) + nh * hd * E,
                       v=dp(dev) + nh * hd * E, out=dp(dev) + (nh + nkv) * hd * E, q_stride=W, k_stride=W, v_stride=W, out_stride=W, cu=dp(cu))
    ok(hip.lib().qwen_hip_op_packed_attention(C.byref(d), stream()))
    torch.cuda.synchronize()
    kv = rows[:, nh * hd:(nh + nkv) * hd]
    exact, mag = packed_want(torch.cat((rows[:, :nh * hd], kv, kv), 1), [n], nh, nkv, hd, 0)
    assert torch.equal(dev[:, :(nh + nkv) * hd].cpu(), rows[:, :(nh + nkv) * hd])
    close_attention(dev[:, (nh + nkv) * hd:].cpu().view(n, nh, hd), exact, mag, t, n, float(rows.abs().max()))



@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("where", ["v", "k", "q", "all"])
def test_values_that_are_not_finite(t, where):
    """An infinity in one value of one early token, or in everything: each row and dim as the formula has it, and a long
    prompt of such rows ends soon (each of them passes its keys 64 at a time, and no further once it is NaN)."""
    g = torch.Generator().manual_seed(20)
    n, nh, nkv, hd = 1500, 4, 2, 64
    rows = torch.randn(n, 8 * 64, generator=g).to(TYPES[t])
    clean = rows.clone()
    if where == "v":
        rows[3, 6 * 64 + 5] = math.inf                          # dim 5 of kv head 0
    elif where == "k":
        rows[3, 4 * 64:5 * 64] = math.nan                       # kv head 0
    elif where == "q":
        rows[700, 64:128] = math.inf                            # head 1 of one token
    else:
        rows[:] = math.nan
    out = torch.empty(n, 256, dtype=TYPES[t], device=DEV)
    ok(packed(rows.to(DEV), [n], nh, nkv, hd, t, out))
    out = out.cpu().view(n, nh, hd)
    exact, mag = packed_want(clean, [n], nh, nkv, hd, 0)
    bad = torch.zeros(n, nh, hd, dtype=torch.bool)
    if where == "v":
        bad[3:, :2, 5] = True
        # the infinite value times a probability: infinite, or NaN where that is 0 in f32
        assert bool((out[bad].isinf() & (out[bad] > 0) | out[bad].isnan()).all())
    elif where == "k":
        bad[3:, :2] = True
        assert bool(out[bad].isnan().all())
    elif where == "q":
        bad[700, 1] = True
        assert not bool(out[bad].isfinite().any())
    else:
        assert bool(out.isnan().all())
        return
    vmax = float(clean.abs().max())
    close_attention(torch.where(bad, exact.to(out.dtype), out), exact, mag, t, n, vmax)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("lens", [[90], [40, 75, 33], [600, 700, 690, 512, 800, 640, 720, 555]])
def test_scores_of_minus_infinity(t, lens):
    """The first 30 keys of each prompt score -infinity against every row: they count for nothing, and a row that has
    no others is 0."""
    g = torch.Generator().manual_seed(23)
    T, nh, nkv, hd = sum(lens), 8, 4, 64
    rows = torch.randn(T, (nh + 2 * nkv) * hd, generator=g).to(TYPES[t])
    rows[:, 0:nh * hd:hd] = rows[:, 0:nh * hd:hd].abs() + 0.25
    only = torch.zeros(T, dtype=torch.bool)
    for a in cu_of(lens)[:-1]:
        rows[a:a + 30, nh * hd:(nh + nkv) * hd:hd] = -math.inf
        only[a:a + 30] = True
    out = torch.empty(T, nh * hd, dtype=TYPES[t], device=DEV)
    ok(packed(rows.to(DEV), lens, nh, nkv, hd, t, out))
    out = out.cpu().view(T, nh, hd)
    exact, mag = packed_want(rows, lens, nh, nkv, hd, 0)
    assert bool(exact[only].isnan().all()) and bool(exact[~only].isfinite().all())
    assert bool((out[only] == 0).all())
    close_attention(out[~only], exact[~only], mag[~only], t, max(lens), float(rows[:, (nh + nkv) * hd:].abs().max()))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_packed_hidden_values_never_reach_a_row(t):
    g = torch.Generator().manual_seed(2)
    lens, nh, nkv, hd = [90, 40], 4, 2, 64
    rows = torch.randn(130, 8 * 64, generator=g).to(TYPES[t])
    exact, mag = packed_want(rows, lens, nh, nkv, hd, 0)
    rows[57, 4 * 64:] = math.inf
    rows[100, 4 * 64:6 * 64] = math.nan
    out = torch.empty(130, 256, dtype=TYPES[t], device=DEV)
    ok(packed(rows.to(DEV), lens, nh, nkv, hd, t, out))
    out = out.cpu().view(130, 4, 64)
    fine = list(range(57)) + list(range(90, 100))
    close_attention(out[fine], exact[fine], mag[fine], t, 90, float(rows[:50].abs().max()))
    assert bool(out[100:].isnan().all()) and not bool(out[57:90].isfinite().any())


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("T,nh", [(20, 4), (400, 4), (2000, 16)])
def test_packed_offsets_out_of_range_stay_inside(t, T, nh):
    """Offsets past T or backwards write nothing outside the tensors (16-row, 32-row and 128-row tiles)."""
    rows = torch.randn(T, 8 * nh // 4 * 64, device=DEV).to(TYPES[t])
    out = torch.full((T + 24, nh * 64), 7.0, dtype=TYPES[t], device=DEV)
    for cu in ([0, T // 2, 25 * T], [0, T - 5, T // 2], [-4, 6, T], [2 ** 31 - 1, -2 ** 31, 7], [T, 0, T], [T - 1, 3, T - 1]):
        ok(packed(rows, [0, 0], nh, nh // 2, 64, t, out[12:], cu=i32(cu)))
    assert bool((out[:12] == 7).all()) and bool((out[12 + T:] == 7).all())


def test_packed_matches_the_prefill_attention():
    """One f32 prompt: the packed call and the framework's own prefill attention, both f32 products."""
    g = np.random.default_rng(3)
    S, nh, nkv = 150, 16, 8
    qkv = g.standard_normal((S, (nh + 2 * nkv) * 128)).astype(np.float32)
    want = np.empty((S, nh * 128), np.float32)
    ok(hip.lib().qwen_hip_op_prefill_attention(want.ctypes.data, qkv.ctypes.data, S, nh, nkv, 128 ** -0.5))
    out = torch.empty(S, nh * 128, device=DEV)
    ok(packed(torch.from_numpy(qkv).to(DEV), [S], nh, nkv, 128, "f32", out))
    out = out.cpu().numpy()
    assert np.linalg.norm(out - want) / np.linalg.norm(want) < 2 * 8e-6


# ---- rules -----------------------------------------------------------------------------------------


def rules64(x, hist, npr, rep, pres, freq, bias, mask, each):
    """One row, f64, token by token; also the largest stage and the number of roundings."""
    x, V = x.double().numpy().copy(), x.numel()
    big, n_round = np.abs(x), np.zeros(V)
    for t in range(V):
        c, o = hist.count(t), hist[npr:].count(t)
        for _ in range((c if each else 1) if c and rep is not None else 0):
            x[t] = x[t] / rep if x[t] > 0 else x[t] * rep
            big[t] = max(big[t], abs(x[t]))
            n_round[t] += 1
        if o and freq is not None:
            x[t] -= o * freq
            big[t] = max(big[t], abs(x[t]), abs(o * freq))
            n_round[t] += 2
        if o and pres is not None:
            x[t] -= pres
            big[t] = max(big[t], abs(x[t]))
            n_round[t] += 1
        if t in bias:
            x[t] += bias[t]
            big[t] = max(big[t], abs(x[t]))
            n_round[t] += 1
        if mask is not None and not mask[t]:
            x[t] = -math.inf
    return torch.from_numpy(x), torch.from_numpy(big), torch.from_numpy(n_round)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("V,on,each", [(1, "rpfbm", 0), (7, "rpfbm", 0), (1000, "rpfbm", 1), (4099, "rpfbm", 0), (4099, "m", 0), (513, "b", 0),
                                       (513, "f", 0), (513, "p", 0), (513, "r", 1), (100, "", 0), (8192, "rm", 0), (8193, "rpfbm", 0), (16385, "rpfb", 1)])
def test_logit_rules(t, V, on, each):
    print(f"[case] rules {t} V={V} {on} each={each}", flush=True)
    rng = np.random.default_rng(V + len(on))
    B, pad = 5, 3
    x = torch.from_numpy(4 * rng.standard_normal((B, V + pad))).to(TYPES[t])
    x[1, :V // 2] = -math.inf
    hists = [rng.integers(0, V, n).tolist() + [V, -1, 2 ** 31 - 1, -2 ** 31] for n in (0, 3, 40, 200, 50)]
    hists[4] = [V // 2] * 300
    npr = [0, 1, 40, 150, 5]
    rep, pres, freq = (rng.uniform(a, b, B).astype(np.float32) for a, b in ((1.0, 1.4), (-0.5, 1.0), (0.0, 0.3)))
    listed = [[(int(rng.integers(0, V)), float(v)) for v in 3 * rng.standard_normal(n)] + [(V, 1.0), (-1, 1.0)] for n in (0, 1, 30, 5, 300)]
    listed[2] += [(0, 1.5), (0, -2.25), (V - 1, 0.75)]          # a token listed again: the last entry counts
    allowed = rng.random((B, V)) < 0.6
    allowed[3] = False                                          # a row that may say nothing
    words = (V + 31) // 32 + 1
    bits = np.zeros((B, words * 32), np.uint64)
    bits[:, :V] = allowed
    mask = torch.from_numpy((bits.reshape(B, words, 32) << np.arange(32, dtype=np.uint64)).sum(2).astype(np.uint32).view(np.int32)).to(DEV)
    dev = {"x": x.to(DEV), "hist": i32(sum(hists, [])), "hoff": i32(cu_of([len(h) for h in hists])), "npr": i32(npr),
           "rep": torch.from_numpy(rep).to(DEV), "pres": torch.from_numpy(pres).to(DEV), "freq": torch.from_numpy(freq).to(DEV),
           "btok": i32([a for r in listed for a, _ in r]), "bval": torch.tensor([v for r in listed for _, v in r], device=DEV),
           "boff": i32(cu_of([len(r) for r in listed]))}
    out = torch.full((B + 1, V + pad), 7.0, dtype=TYPES[t], device=DEV)

    def call(dst, stride):
        d = hip.LogitRules(dtype=hip.DT[t], B=B, V=V, logits=dp(dev["x"]), out=dp(dst), logits_stride=V + pad, out_stride=stride, rep_each=each)
        if set(on) & set("rpf"):
            d.hist, d.hist_off, d.hist_cap, d.n_prompt = dp(dev["hist"]), dp(dev["hoff"]), dev["hist"].numel(), dp(dev["npr"])
        d.rep, d.presence, d.frequency = (dp(dev[n]) if c in on else None for c, n in (("r", "rep"), ("p", "pres"), ("f", "freq")))
        if "b" in on:
            d.bias_tok, d.bias_val, d.bias_off, d.bias_cap = dp(dev["btok"]), dp(dev["bval"]), dp(dev["boff"]), dev["btok"].numel()
        if "m" in on:
            d.mask, d.mask_stride = dp(mask), words
        ok(hip.lib().qwen_hip_op_logit_rules(C.byref(d), stream()))
        torch.cuda.synchronize()

    call(out, V + pad)
    got = out.cpu()
    assert bool((got[:, V:] == 7).all()) and bool((got[B] == 7).all())
    eps = torch.finfo(TYPES[t]).eps
    for b in range(B):
        want, big, n = rules64(x[b, :V], hists[b], npr[b], float(rep[b]) if "r" in on else None, float(pres[b]) if "p" in on else None,
                               float(freq[b]) if "f" in on else None, {a: np.float32(v) for a, v in listed[b]} if "b" in on else {},
                               allowed[b] if "m" in on else None, each)
        if t == "f16":                                          # past half a step over its largest value f16 rounds to infinity
            want = torch.where(want.abs() >= 65520, want.sign() * math.inf, want)
        g, inf = got[b, :V].double(), want.isinf()
        assert torch.equal(g.isinf(), inf) and bool((g[inf] == want[inf]).all())
        tol = n * 2.0 ** -24 * big
        tol = tol + (0 if t == "f32" else eps / 2 * (want.abs() + tol) + 2.0 ** -25)
        assert bool(((g - want).abs() <= tol)[~inf].all()), (b, float((g - want).abs()[~inf].max()))
    call(dev["x"], V + pad)                                     # in place: the same bits
    assert torch.equal(dev["x"][:, :V].cpu(), got[:B, :V])


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_logit_rules_of_long_lists(t):
    """A history past 65535 entries, one token in it more often than a count goes, and more biases than one a thread."""
    V, n = 9001, 70000
    rng = np.random.default_rng(8)
    h = np.concatenate([np.full(66000, 7), rng.integers(0, V, n - 66000)])
    rng.shuffle(h)
    x = torch.from_numpy(rng.standard_normal(V)).to(TYPES[t])
    btok, bval = rng.integers(0, V, 5000), rng.standard_normal(5000).astype(np.float32)
    dev = [x.to(DEV), i32(h.tolist()), i32([0, n]), torch.tensor([1.2], device=DEV), torch.tensor([0.001], device=DEV), i32(btok.tolist()),
           torch.from_numpy(bval).to(DEV), i32([0, 5000]), torch.empty(V, dtype=TYPES[t], device=DEV)]
    d = hip.LogitRules(dtype=hip.DT[t], B=1, V=V, logits=dp(dev[0]), out=dp(dev[8]), logits_stride=V, out_stride=V, hist=dp(dev[1]),
                       hist_off=dp(dev[2]), hist_cap=n, rep=dp(dev[3]), frequency=dp(dev[4]), bias_tok=dp(dev[5]), bias_val=dp(dev[6]),
                       bias_off=dp(dev[7]), bias_cap=5000)
    ok(hip.lib().qwen_hip_op_logit_rules(C.byref(d), stream()))
    torch.cuda.synchronize()
    c = np.minimum(np.bincount(h, minlength=V), 65535)
    rep, freq = float(np.float32(1.2)), float(np.float32(0.001))
    w = x.double().numpy()
    w = np.where(c > 0, np.where(w > 0, w / rep, w * rep), w) - c * freq
    last = np.zeros(V)
    last[btok] = bval                                           # the last entry of a token counts
    w = torch.from_numpy(w + last)
    tol = 4 * 2.0 ** -24 * (w.abs() + torch.from_numpy(c * freq) + 8) + (0 if t == "f32" else 2.0 ** -8 * w.abs() * 1.01)
    assert bool(((dev[8].double().cpu() - w).abs() <= tol).all())


@pytest.mark.parametrize("V", [300, 9000])
@pytest.mark.parametrize("each", [0, 1])
def test_logit_rules_offsets_out_of_range_stay_inside(V, each):
    """Offsets past the lists, negative, falling and at both ends of their type are brought into the lists; what lies next to
    a list, tokens that would change every row, is not read.  A cap of 2^31 - 1 over sane offsets changes nothing."""
    rng = np.random.default_rng(V + each)
    cap, far = 50, 2 ** 31 - 1
    tok, btok = rng.integers(0, V - 3, cap), rng.integers(0, V - 3, cap)
    bval = (3 * rng.standard_normal(cap)).astype(np.float32)
    around = lambda v, g: torch.cat((torch.full((8192,), g, dtype=v.dtype), v, torch.full((8192,), g, dtype=v.dtype))).to(DEV)  # noqa: E731
    dev = [around(torch.from_numpy(tok.astype(np.int32)), V - 2), around(torch.from_numpy(btok.astype(np.int32)), V - 1),
           around(torch.from_numpy(bval), 99.0)]
    at = [dp(d) + 8192 * 4 for d in dev]
    wild = [0, 20, far, -far - 1, 30, cap + 3, 5, far - 100, far - 4000, cap, -1, far - 4096, cap + 1, far, far, 3, cap]
    sane = [0, 13, 13, 40, cap]
    for off, hold in ((wild, cap), (wild, 0), (sane, cap), (sane, far)):
        B = len(off) - 1
        x = torch.from_numpy(4 * rng.standard_normal((B, V))).float()
        xd, out, offd = x.to(DEV), torch.full((B, V), 7.0, device=DEV), i32(off)
        rep, pres, freq = (torch.full((B,), v, device=DEV) for v in (1.25, 0.5, 0.125))
        npr = i32([2] * B)
        d = hip.LogitRules(dtype=0, B=B, V=V, logits=dp(xd), out=dp(out), logits_stride=V, out_stride=V, rep_each=each, hist=at[0], hist_off=dp(offd),
                           hist_cap=hold, n_prompt=dp(npr), rep=dp(rep), presence=dp(pres), frequency=dp(freq), bias_tok=at[1], bias_val=at[2],
                           bias_off=dp(offd), bias_cap=hold)
        print(f"[case] rules V={V} each={each} offsets {off[:4]}.. of {hold}", flush=True)
        ok(hip.lib().qwen_hip_op_logit_rules(C.byref(d), stream()))
        got = out.cpu().double()
        for b in range(B):
            i0 = min(max(off[b], 0), hold)
            i1 = min(max(off[b + 1], i0), hold)
            want, big, n = rules64(x[b], tok[i0:i1].tolist(), 2, 1.25, 0.5, 0.125, dict(zip(btok[i0:i1].tolist(), bval[i0:i1])), None, each)
            assert bool(((got[b] - want).abs() <= n * 2.0 ** -24 * big).all()), (b, off[b], off[b + 1])


def test_rules_then_argmax_is_the_sampler_of_one_stream():
    """rep_each on one f32 row: the token that qwen_hip_op_sample picks greedily with its penalty."""
    rng = np.random.default_rng(4)
    for n in (0, 5, 60):
        lg = (3 * rng.standard_normal(2000)).astype(np.float32)
        prev = rng.choice(np.argsort(-lg)[:30], n).astype(np.int32)
        seed = np.array([1], np.uint32)
        want = hip.lib().qwen_hip_op_sample(lg.ctypes.data, 2000, 0.0, 0, 1.0, 1.3, prev.ctypes.data if n else None, n, seed.ctypes.data)
        x, h, o, r = torch.from_numpy(lg).to(DEV), i32(prev.tolist() + [0]), i32([0, n]), torch.tensor([1.3], device=DEV)
        d = hip.LogitRules(dtype=0, B=1, V=2000, logits=dp(x), out=dp(x), logits_stride=2000, out_stride=2000, hist=dp(h), hist_off=dp(o),
                           hist_cap=n + 1, rep=dp(r), rep_each=1)
        ok(hip.lib().qwen_hip_op_logit_rules(C.byref(d), stream()))
        assert int(x.argmax()) == want


# ---- together --------------------------------------------------------------------------------------


class Server:
    """A few requests over one pool, as a server runs them: plan, append, attention, with the f32 rows of all their
    tokens drawn beforehand; the plan works in place, so that a captured step can be replayed."""
    nh, nkv, hd, page, cols, n_pages = 4, 2, 64, 16, 8, 20

    def __init__(self, t, B, cap):
        g = torch.Generator().manual_seed(21)
        self.t, self.B, self.cap = t, B, cap
        kv = "bf16" if t == "f32" else t
        w = (self.nh + 2 * self.nkv) * self.hd
        self.all = torch.randn(B, 120, w, generator=g).to(TYPES[t])
        self.rows = torch.zeros(cap, w, dtype=TYPES[t], device=DEV)
        self.q = torch.zeros(cap, self.nh * self.hd, dtype=TYPES[t], device=DEV)
        self.out = torch.full((cap, self.nh * self.hd), 7.0, dtype=TYPES[t], device=DEV)
        self.k, self.v = (torch.full((self.n_pages, self.nkv, self.page, self.hd), math.nan, dtype=TYPES[kv], device=DEV) for _ in range(2))
        ang = torch.randn(128, self.hd // 2, generator=g)
        self.cos, self.sin = ang.cos().to(DEV), ang.sin().to(DEV)
        self.p = Plan([0] * B, [0] * B, [[-1] * self.cols for _ in range(B)], list(range(self.n_pages)), self.n_pages, self.page,
                      self.n_pages, self.cols, cap, in_place=True)
        self.pages = pages_of(self.k, self.v, kv)
        E, W = self.rows.element_size(), w
        self.a = hip.PageAppend(dtype=hip.DT[t], n_heads=self.nh, T=cap, rope_len=128, eps=1e-6, q=dp(self.rows),
                                k=dp(self.rows) + self.nh * self.hd * E, v=dp(self.rows) + (self.nh + self.nkv) * self.hd * E, q_stride=W, k_stride=W,
                                v_stride=W, q_out=dp(self.q), q_out_stride=self.q.stride(0), rope_cos=dp(self.cos), rope_sin=dp(self.sin),
                                pos=dp(self.p.pos), slot=dp(self.p.slot))
        self.d = hip.PageAttn(dtype=hip.DT[t], n_heads=self.nh, B=B, T=cap, table_cols=self.cols, max_q=cap, max_kv=128, scale=self.hd ** -0.5,
                              q=dp(self.q), out=dp(self.out), q_stride=self.q.stride(0), out_stride=self.out.stride(0), cu_q=dp(self.p.cu),
                              kv_len=dp(self.p.kv2), table=dp(self.p.table), table_stride=self.cols)
        n = hip.lib().qwen_hip_op_page_attention_workspace(C.byref(self.pages), C.byref(self.d))
        self.ws = torch.empty(n + 1, dtype=torch.uint8, device=DEV)
        self.d.workspace, self.d.workspace_bytes = dp(self.ws), n
        self.done = [0] * B

    def launch(self):
        L = hip.lib()
        ok(L.qwen_hip_op_page_plan(C.byref(self.p.d), stream()))
        ok(L.qwen_hip_op_page_append(C.byref(self.pages), C.byref(self.a), stream()))
        ok(L.qwen_hip_op_page_attention(C.byref(self.pages), C.byref(self.d), stream()))

    def feed(self, new):
        at = 0
        for b, n in enumerate(new):
            if n > 0:
                self.rows[at:at + n] = self.all[b, self.done[b]:self.done[b] + n].to(DEV)
                at += n
            self.done[b] = 0 if n < 0 else self.done[b] + n
        self.p.new.copy_(i32(new))
        return at

    def want(self, new):
        """The new tokens' rows from the whole histories, in 64 bits, K and V as the cache rounds them."""
        out, mag = [], []
        kvt = self.k.dtype
        for b, n in enumerate(new):
            if n <= 0:
                continue
            x = self.all[b, :self.done[b]].double().view(self.done[b], -1, self.hd).clone()
            c, s = self.cos.cpu().double()[:self.done[b], None], self.sin.cpu().double()[:self.done[b], None]
            qk, h = x[:, :self.nh + self.nkv], self.hd // 2
            x[:, :self.nh + self.nkv] = torch.cat((qk[..., :h] * c - qk[..., h:] * s, qk[..., h:] * c + qk[..., :h] * s), -1)
            q, k, v = x.split((self.nh, self.nkv, self.nkv), 1)
            o, m = attend64(q[-n:].to(TYPES[self.t]), k.float().to(kvt), v.float().to(kvt), self.done[b] - n, 0, self.hd ** -0.5)
            out.append(o)
            mag.append(m)
        return torch.cat(out), torch.cat(mag)

    def check(self, new, at):
        exact, mag = self.want(new)
        got = self.out[:at].cpu().double().view(at, self.nh, self.hd)
        # k and q pass one more rounding, whose f32 input is off by a few 2^-24: where that lands next to a tie an
        # element moves by a whole step of its type (2^-8 of one of 64 terms of a score), so a score by
        # 2 * 2^-8 * 5 * 5 / 8 = 0.025 and a row by as much of max|v| in a few keys' weight; the 2-norm says the rest
        assert float((got - exact).norm() / exact.norm()) < (2e-3 if self.t == "f32" else 8e-3)
        assert bool((self.out[at:] == 7).all())


STEPS = [[30, 17, 0], [1, 1, 45], [1, 0, 1], [1, -1, 1], [20, 33, 1], [1, 1, 1], [-1, 1, 1], [3, 1, 40]]


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_requests_come_grow_and_go(t):
    s = Server(t, 3, 64)
    for new in STEPS:
        print(f"[case] server {t} step {new}", flush=True)
        at = s.feed(new)
        s.out.fill_(7.0)
        s.launch()
        torch.cuda.synchronize()
        assert int(s.p.status) == 0 and s.p.kv2.tolist() == s.done
        s.check(new, at)
    held = sum(-(-n // 16) for n in s.done)
    assert int(s.p.nf2) == s.n_pages - held
    assert sorted(s.p.free[:int(s.p.nf2)].tolist() + [int(s.p.table[b, c]) for b in range(3) for c in range(-(-s.done[b] // 16))]) == list(range(20))


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_a_captured_step_is_replayed(t):
    """The whole step in one graph, replayed with other lengths and with eager work in between, equals the eager step
    to the bit; on a stream other than the current one."""
    eager, s = Server(t, 3, 64), Server(t, 3, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.launch()                                              # no new tokens: nothing changes
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        s.launch()
    for new in STEPS:
        print(f"[case] replay {t} step {new}", flush=True)
        at = eager.feed(new)
        assert s.feed(new) == at
        eager.out.fill_(7.0)
        s.out.fill_(7.0)
        eager.launch()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(s.out, eager.out)
        assert s.p.kv2.tolist() == eager.p.kv2.tolist() and s.p.table.tolist() == eager.p.table.tolist()
        s.check(new, at)


@pytest.mark.parametrize("handle", [None, 1, 2], ids=["null", "legacy", "per-thread"])
def test_the_handles_that_are_no_streams_of_the_callers(handle, monkeypatch):
    """NULL, hipStreamLegacy and hipStreamPerThread, for a step, a packed call and the rules."""
    s = Server("bf16", 3, 64)
    at = s.feed([30, 17, 0])
    s.out.fill_(7.0)
    rows = torch.randn(30, 4 * 64, generator=torch.Generator().manual_seed(4))
    dev, out, x, y = rows.to(DEV), torch.zeros(30, 128, device=DEV), torch.arange(100, dtype=torch.float32, device=DEV), torch.zeros(100, device=DEV)
    d = hip.LogitRules(dtype=0, B=1, V=100, logits=dp(x), out=dp(y), logits_stride=100, out_stride=100)
    cu = i32([0, 30])
    torch.cuda.synchronize()
    monkeypatch.setitem(globals(), "stream", lambda: handle)
    s.launch()
    torch.cuda.synchronize()
    s.check([30, 17, 0], at)
    ok(packed(dev, [30], 2, 1, 64, "f32", out, cu=cu))
    ok(hip.lib().qwen_hip_op_logit_rules(C.byref(d), handle))
    torch.cuda.synchronize()
    exact, mag = packed_want(rows, [30], 2, 1, 64, 0)
    close_attention(out.cpu().view(30, 2, 64), exact, mag, "f32", 30, float(rows.abs().max()))
    assert torch.equal(x, y)



def test_a_step_that_cannot_be_planned_leaves_everything():
    s = Server("f32", 3, 64)
    s.feed([30, 17, 0])
    s.launch()
    torch.cuda.synchronize()
    k, done = s.k.clone(), list(s.done)
    s.p.new.copy_(i32([200, 1, 1]))                             # past its table
    s.out.fill_(7.0)
    s.launch()
    torch.cuda.synchronize()
    assert int(s.p.status) & hip.PLAN_TABLE_FULL and s.p.kv2.tolist() == done
    assert torch.equal(s.k.isnan(), k.isnan()) and torch.equal(s.k[~k.isnan()], k[~k.isnan()])
    assert bool((s.out == 7).all())


def test_prompts_packed_or_from_the_cache_agree():
    """The same tokens through the packed call and, appended without norm or RoPE, through the cache (bf16 all through)."""
    g = torch.Generator().manual_seed(31)
    lens, nh, nkv, hd = [70, 33, 128], 16, 8, 128
    T = sum(lens)
    rows = torch.randn(T, (nh + 2 * nkv) * hd, generator=g).to(torch.bfloat16).to(DEV)
    out = torch.empty(T, nh * hd, dtype=torch.bfloat16, device=DEV)
    ok(packed(rows, lens, nh, nkv, hd, "bf16", out))
    p = Paged([(0, n) for n in lens], nh, nkv, hd, "bf16", "bf16", 16, "slot", seed=32)
    slot = torch.cat([p.table[b, torch.arange(n, device=DEV) // 16] * 16 + torch.arange(n, device=DEV) % 16 for b, n in enumerate(lens)]).to(torch.int32)
    p.qd = torch.empty(T, nh * hd, dtype=torch.bfloat16, device=DEV)
    a = hip.PageAppend(dtype=1, n_heads=nh, T=T, eps=0.0, q=dp(rows), k=dp(rows) + nh * hd * 2, v=dp(rows) + (nh + nkv) * hd * 2,
                       q_stride=rows.stride(0), k_stride=rows.stride(0), v_stride=rows.stride(0), q_out=dp(p.qd), q_out_stride=nh * hd, slot=dp(slot))
    ok(hip.lib().qwen_hip_op_page_append(C.byref(p.pages), C.byref(a), stream()))
    p.d.q, p.d.q_stride = dp(p.qd), nh * hd
    got = p.run().reshape(T, -1)
    assert torch.equal(p.qd, rows[:, :nh * hd])
    exact, mag = packed_want(rows.cpu(), lens, nh, nkv, hd, 0)
    for x in (got, out):
        close_attention(x.view(T, nh, hd), exact, mag, "bf16", 128, float(rows.abs().max()))


@pytest.mark.parametrize("what", ["plan", "plan of two launches", "append", "attention", "attention of two launches", "packed", "rules"])
def test_an_error_that_was_left_is_not_the_calls(what):
    """A failed HIP call of the caller's (a device that there is not), whose error nobody has read: the operators launch, say
    so, and leave it."""
    L = hip.lib()
    H = C.CDLL(hip.LIB_PATH)                                    # its own HIP runtime
    if what.startswith("plan"):
        rng = np.random.default_rng(1)
        case = plan_case(rng, 20, 16, 20, 90, 60, 4, cap=9000 if "two" in what else 1000)
        p, want = Plan(*case, in_place=True), plan_model(*case)
        call = lambda st: L.qwen_hip_op_page_plan(C.byref(p.d), st)  # noqa: E731
    elif what == "append":
        g = torch.Generator().manual_seed(3)
        rows, slot = torch.randn(2, 192, generator=g).to(DEV), i32([5, 2])
        k, v = (pool((3, 1, 2, 64), torch.bfloat16, "head", g) for _ in range(2))
        pages, d = pages_of(k, v, "bf16"), hip.PageAppend(dtype=0, T=2, k=dp(rows), v=dp(rows) + 256, k_stride=192, v_stride=192, slot=dp(slot))
        call = lambda st: L.qwen_hip_op_page_append(C.byref(pages), C.byref(d), st)  # noqa: E731
    elif what.startswith("attention"):
        p = Paged([(900, 1), (40, 1)] if "two" in what else [(40, 1), (3, 1)], 4, 2, 64, "bf16", "bf16", 16, "head", seed=33)
        n = L.qwen_hip_op_page_attention_workspace(C.byref(p.pages), C.byref(p.d))
        assert (n > 0) == ("two" in what)
        ws = torch.zeros(n + 1, dtype=torch.uint8, device=DEV)
        p.d.workspace, p.d.workspace_bytes = dp(ws), n
        call = lambda st: L.qwen_hip_op_page_attention(C.byref(p.pages), C.byref(p.d), st)  # noqa: E731
    elif what == "packed":
        rows = torch.randn(30, 4 * 64, generator=torch.Generator().manual_seed(4))
        dev, out, cu = rows.to(DEV), torch.zeros(30, 128, device=DEV), i32([0, 30])
        d = hip.PackedAttn(dtype=0, n_heads=2, n_kv_heads=1, head_dim=64, B=1, T=30, scale=0.125, q=dp(dev), k=dp(dev) + 512, v=dp(dev) + 768,
                           out=dp(out), q_stride=256, k_stride=256, v_stride=256, out_stride=128, cu=dp(cu))
        call = lambda st: L.qwen_hip_op_packed_attention(C.byref(d), st)  # noqa: E731
    else:
        x = torch.arange(100, dtype=torch.float32, device=DEV)
        out = torch.zeros(100, device=DEV)
        d = hip.LogitRules(dtype=0, B=1, V=100, logits=dp(x), out=dp(out), logits_stride=100, out_stride=100)
        call = lambda st: L.qwen_hip_op_logit_rules(C.byref(d), st)  # noqa: E731
    st = stream()
    torch.cuda.synchronize()
    assert H.hipGetLastError() == 0
    left = H.hipSetDevice(1000)
    rc, stays = call(st), H.hipGetLastError()                   # read before torch's next launch, which would report it
    assert left != 0
    assert rc == 0, hip.last_error()
    assert stays == left and H.hipGetLastError() == 0
    torch.cuda.synchronize()
    if what.startswith("plan"):
        assert p.kv.tolist() == want["kv"] and int(p.nf) == want["n_free"] and p.slot[:p.cap].tolist() == want["slot"]
    elif what == "append":
        assert torch.equal(k[2, 0, 1], rows[0, :64].bfloat16()) and torch.equal(v[1, 0, 0], rows[1, 64:128].bfloat16())
    elif what.startswith("attention"):
        exact, mag = p.want()
        close_attention(p.out[:, :256].reshape(2, 4, 64), exact, mag, "bf16", 901, 6.0)
    elif what == "packed":
        exact, mag = packed_want(rows, [30], 2, 1, 64, 0)
        close_attention(out.cpu().view(30, 2, 64), exact, mag, "f32", 30, float(rows.abs().max()))
    else:
        assert torch.equal(out, x)
