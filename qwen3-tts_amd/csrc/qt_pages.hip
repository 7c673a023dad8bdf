// qt_pages.hip — a paged cache's bookkeeping for one step (qwen_hip_op_page_plan) and its writer
// (qwen_hip_op_page_append).
#include "qt_ops.h"

// ---- the plan --------------------------------------------------------------------------------
// With h(n) = ceil(n / page_size): an ended request gives back its h(kv) pages, a continued one takes
// h(kv + new) - h(kv).  In request order, exclusive sums of the pages given back, of those taken and of the new
// tokens say where each request's entries lie; then every page and every token finds its request by a search
// in those sums, independently of the others.  Page i of all taken is the free list's entry n_free + R - 1 - i, R
// pages having been given back: entries n_free .. n_free + R - 1 are those pages themselves, read from the tables,
// so nothing written is read again and everything is checked before anything is written.
//
// One workgroup does it all: three sums over at most 2048 requests need no second launch and no
// global scratch, and a step's work is a few hundred KB at most.  Bound by the latency of its dependent loads
// (lengths, then free list and tables) and of the launch.  Past PLAN_ONE tokens the slots go to a grid of their own,
// which reads what the workgroup wrote.
#define PLAN_T 1024
#define PLAN_MAX_B 2048        // 32 KB of LDS
#define PLAN_ONE 8192
#define PLAN_SAT (1u << 30)     // sums stop here: under 2^31 in any order, over every limit they are held to

struct PlanArgs {
    const int *new_len, *kv_len, *n_free;
    int *table, *free_pages, *kv_out, *n_free_out, *cu, *pos, *slot, *status;
    long long ts;
    int B, ps, n_pages, cols, cap, slots_here;
    QtDiv div;
};

__device__ __forceinline__ unsigned plan_add(unsigned a, unsigned b) { return min(a + b, PLAN_SAT); }

// the last b with first[b] <= i (first[0] = 0, ascending): of requests that begin at the same place all but the
// last are empty
__device__ __forceinline__ int plan_find(const unsigned *first, int B, unsigned i) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= i) lo = mid; else hi = mid;
    }
    return lo;
}
__global__ __launch_bounds__(PLAN_T) void k_page_plan(PlanArgs a) {
    extern __shared__ unsigned sh[];
    unsigned *tok = sh, *take = tok + a.B + 1, *back = take + a.B + 1;     // exclusive sums, [B + 1] each
    int *kv = reinterpret_cast<int *>(back + a.B + 1);                     // lengths before, [B]
    __shared__ unsigned wsum[3][PLAN_T / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_free = a.n_free[0];
    int flags = n_free < 0 || n_free > a.n_pages ? QWEN_HIP_PLAN_INVALID : 0;
    const int per = (a.B + PLAN_T - 1) / PLAN_T, b0 = tid * per, b1 = min(b0 + per, a.B);
    const long long room = (long long)a.cols * a.ps;
    unsigned s[3] = {0u, 0u, 0u};
    for (int b = b0; b < b1; b++) {
        const int n = a.new_len[b];
        int len = a.kv_len[b];
        unsigned t = 0, p = 0, r = 0;
        if (len < 0 || (long long)len > room) {
            flags |= QWEN_HIP_PLAN_INVALID;
            len = 0;
        } else if (n < 0) {
            r = qt_quot(len, a.div) + (len % a.ps != 0);
        } else if ((long long)len + n > room) {
            flags |= QWEN_HIP_PLAN_TABLE_FULL;
        } else {
            t = n;
            p = (unsigned)(((long long)len + n + a.ps - 1) / a.ps) - (qt_quot(len, a.div) + (len % a.ps != 0));
        }
        kv[b] = len;
        tok[b] = s[0]; take[b] = s[1]; back[b] = s[2];
        s[0] = plan_add(s[0], t); s[1] = plan_add(s[1], p); s[2] = plan_add(s[2], r);
    }
    // exclusive sums over the threads
    unsigned inc[3], tot[3], base[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        unsigned x = s[k];
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned y = __shfl_up(x, o, 64);
            if (lane >= o) x = plan_add(x, y);
        }
        inc[k] = x;
        if (lane == 63) wsum[k][wave] = x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; k++) {
        unsigned before = 0, all = 0;
        for (int w = 0; w < PLAN_T / 64; w++) {
            if (w == wave) before = all;
            all = plan_add(all, wsum[k][w]);
        }
        const unsigned up = __shfl_up(inc[k], 1, 64);
        base[k] = lane == 0 ? before : plan_add(before, up);
        tot[k] = all;
    }
    for (int b = b0; b < b1; b++) {
        tok[b] = plan_add(tok[b], base[0]);
        take[b] = plan_add(take[b], base[1]);
        back[b] = plan_add(back[b], base[2]);
    }
    if (tid == 0) { tok[a.B] = tot[0]; take[a.B] = tot[1]; back[a.B] = tot[2]; }
    const unsigned R = tot[2], N = tot[1], T = tot[0];
    if (T > (unsigned)a.cap) flags |= QWEN_HIP_PLAN_TOO_MANY;
    if (n_free + (long long)R > a.n_pages) flags |= QWEN_HIP_PLAN_INVALID;   // pages given back twice
    if ((long long)N > n_free + (long long)R) flags |= QWEN_HIP_PLAN_NO_PAGES;
    __syncthreads();
    // page j of those given back, and page i of those taken
    const auto given = [&](unsigned j) {
        const int b = plan_find(back, a.B, j);
        return a.table[(long long)b * a.ts + (j - back[b])];
    };
    const auto taken = [&](unsigned i) {
        const long long at = (long long)n_free + R - 1 - i;
        return at >= n_free ? given((unsigned)(at - n_free)) : a.free_pages[at];
    };
    int any = 0;
    for (int k = 0; k < 4; k++) any |= __syncthreads_or(flags & (1 << k)) ? 1 << k : 0;
    if (any == 0) {                                                          // the sums are in range: look at the pages
        bool bad = false;
        for (unsigned j = tid; j < R; j += PLAN_T) bad |= (unsigned)given(j) >= (unsigned)a.n_pages;
        for (unsigned i = tid; i < N; i += PLAN_T) bad |= (unsigned)taken(i) >= (unsigned)a.n_pages;
        any = __syncthreads_or(bad) ? QWEN_HIP_PLAN_INVALID : 0;
    }
    if (any) {
        for (int b = tid; b < a.B; b += PLAN_T) a.kv_out[b] = a.kv_len[b];
        for (int b = tid; b <= a.B; b += PLAN_T) a.cu[b] = 0;
        if (a.slots_here)
            for (int t = tid; t < a.cap; t += PLAN_T) { a.pos[t] = -1; a.slot[t] = -1; }
        if (tid == 0) { a.n_free_out[0] = n_free; a.status[0] = any; }
        return;
    }
    const auto have = [&](int b) { return (unsigned)(qt_quot(kv[b], a.div) + (kv[b] % a.ps != 0)); };
    for (unsigned j = tid; j < R; j += PLAN_T) a.free_pages[n_free + j] = given(j);
    for (unsigned i = tid; i < N; i += PLAN_T) {
        const int b = plan_find(take, a.B, i);
        a.table[(long long)b * a.ts + have(b) + (i - take[b])] = taken(i);
    }
    if (a.slots_here)
        for (unsigned t = tid; t < (unsigned)a.cap; t += PLAN_T) {
            int p = -1, at = -1;
            if (t < T) {
                const int b = plan_find(tok, a.B, t);
                p = kv[b] + (int)(t - tok[b]);
                const unsigned c = (unsigned)qt_quot(p, a.div), hb = have(b);
                const int page = c < hb ? a.table[(long long)b * a.ts + c] : taken(take[b] + c - hb);
                // an old page's number is the caller's: one out of range makes no slot
                at = (unsigned)page < (unsigned)a.n_pages ? page * a.ps + (p - (int)c * a.ps) : -1;
            }
            a.pos[t] = p;
            a.slot[t] = at;
        }
    for (int b = b0; b < b1; b++) {
        const int n = a.new_len[b];
        a.kv_out[b] = n < 0 ? 0 : kv[b] + n;
    }
    for (int b = tid; b <= a.B; b += PLAN_T) a.cu[b] = (int)tok[b];
    if (tid == 0) { a.n_free_out[0] = (int)(n_free + R - N); a.status[0] = 0; }
}

// positions and slots of a large step: the plan's tables and offsets are written
__global__ __launch_bounds__(256) void k_page_slots(PlanArgs a) {
    extern __shared__ unsigned cu[];
    for (int b = threadIdx.x; b <= a.B; b += 256) cu[b] = (unsigned)a.cu[b];
    __syncthreads();
    const unsigned T = cu[a.B];
    for (int k = 0; k < 4; k++) {
        const unsigned t = blockIdx.x * 1024 + k * 256 + threadIdx.x;
        if (t >= (unsigned)a.cap) return;
        int p = -1, at = -1;
        if (t < T) {
            const int b = plan_find(cu, a.B, t);
            p = a.kv_out[b] - (int)(cu[b + 1] - t);
            const int c = qt_quot(p, a.div), page = a.table[(long long)b * a.ts + c];
            at = (unsigned)page < (unsigned)a.n_pages ? page * a.ps + (p - c * a.ps) : -1;
        }
        a.pos[t] = p;
        a.slot[t] = at;
    }
}

extern "C" int qwen_hip_op_page_plan(const qwen_hip_page_plan_t *p, void *stream) {
    QT_REFUSE(!p, "page_plan: null descriptor");
    QT_REFUSE(!p->new_len || !p->kv_len || !p->n_free || !p->table || !p->free_pages || !p->kv_len_out || !p->n_free_out ||
                  !p->cu_q || !p->status || (p->max_tokens > 0 && (!p->pos || !p->slot)),
              "page_plan: null pointer");
    QT_REFUSE(p->B < 1 || p->B > PLAN_MAX_B, "page_plan: B %d out of range (1..%d)", p->B, PLAN_MAX_B);
    QT_REFUSE(p->n_pages < 1 || p->page_size < 1 || (long long)p->n_pages * p->page_size > 0x7FFFFFFFll,
              "page_plan: %d pages of %d (both at least 1, 2^31 - 1 slots at most)", p->n_pages, p->page_size);
    QT_REFUSE(p->table_cols < 1 || (long long)p->table_cols * p->page_size > (1 << 30),
              "page_plan: table_cols %d (at least 1, 2^30 positions at most)", p->table_cols);
    QT_REFUSE(p->table_stride < p->table_cols, "page_plan: table_stride %lld under table_cols %d", p->table_stride, p->table_cols);
    QT_REFUSE(p->max_tokens < 0 || p->max_tokens > (1 << 28), "page_plan: max_tokens %d out of range (0..2^28)", p->max_tokens);
    hipStream_t st = (hipStream_t)stream;
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "page_plan: the stream's device: %s", hipGetErrorString(on.err));
    PlanArgs a = {p->new_len, p->kv_len, p->n_free, p->table, p->free_pages, p->kv_len_out, p->n_free_out, p->cu_q, p->pos,
                  p->slot, p->status, p->table_stride, p->B, p->page_size, p->n_pages, p->table_cols, p->max_tokens,
                  p->max_tokens <= PLAN_ONE, qt_div_of(p->page_size)};
    hipLaunchKernelGGL(k_page_plan, dim3(1), dim3(PLAN_T), (size_t)(4 * p->B + 3) * 4, st, a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && !a.slots_here) {
        hipLaunchKernelGGL(k_page_slots, dim3((p->max_tokens + 1023) / 1024), dim3(256), (size_t)(p->B + 1) * 4, st, a);
        e = hipGetLastError();
    }
    QT_REFUSE(e != hipSuccess, "page_plan: launch failed: %s", hipGetErrorString(e));
    return 0;
}

// ---- the append --------------------------------------------------------------------------------
// y = x / sqrt(mean x^2 + eps) g, then (y1, y2) -> (y1 c - y2 s, y2 c + y1 s) on a head's halves, all in f32,
// rounded once.  A head's row is HD / 8 lanes of 8 elements (16-byte loads); its sum of squares and its rotation's
// other half are lane exchanges.  A workgroup takes one token: its lanes' angles and gains are loaded once
// and serve every head.  Bound by the rows' bytes for prompts, by the latency of slot, angles and rows for a step.
struct AppendArgs {
    const uint8_t *q, *k, *v;
    uint8_t *qo, *kc, *vc;
    long long qs, ks, vs, os, ps_page, ps_head, ps_slot;
    const float *qn, *kn, *rc, *rs;
    const int *pos, *slot;
    int T, nh, nkv, rope_len, n_slots, page;
    float eps;
    QtDiv div;
};

template <typename QT, typename KT, int HD>
__global__ __launch_bounds__(256) void k_page_append(AppendArgs a) {
    constexpr int E = sizeof(typename QT::elem), L = HD / 8;       // lanes a row
    const int t = blockIdx.x, slot = a.slot[t];
    if ((unsigned)slot >= (unsigned)a.n_slots) return;
    const int pos = a.rc ? a.pos[t] : 0;
    if (a.rc && (unsigned)pos >= (unsigned)a.rope_len) return;
    const int l = threadIdx.x % L, grp = threadIdx.x / L;
    float c[8], s[8], gq[8], gk[8];
    if (a.rc) {
        const int at = (8 * l) % (HD / 2);
        qt_load8<QtF32>(a.rc + (size_t)pos * (HD / 2) + at, c);
        qt_load8<QtF32>(a.rs + (size_t)pos * (HD / 2) + at, s);
    }
    if (a.qn) qt_load8<QtF32>(a.qn + 8 * l, gq);
    if (a.kn) qt_load8<QtF32>(a.kn + 8 * l, gk);
    const int page = qt_quot(slot, a.div);
    const long long dst = page * a.ps_page + (slot - page * a.page) * a.ps_slot + 8 * l;
    const int nq = a.q ? a.nh : 0;
    for (int r = grp; r < nq + 2 * a.nkv; r += 256 / L) {
        const bool isq = r < nq, isv = r >= nq + a.nkv;
        const int h = isq ? r : isv ? r - nq - a.nkv : r - nq;
        const uint8_t *src = isq ? a.q + (size_t)(t * a.qs) * E : isv ? a.v + (size_t)(t * a.vs) * E : a.k + (size_t)(t * a.ks) * E;
        float x[8];
        qt_load8<QT>(src + ((size_t)h * HD + 8 * l) * E, x);
        if (!isv) {
            if (isq ? a.qn != nullptr : a.kn != nullptr) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) ss = fmaf(x[e], x[e], ss);
#pragma unroll
                for (int o = 1; o < L; o <<= 1) ss += __shfl_xor(ss, o, L);
                const float inv = 1.0f / sqrtf(ss / HD + a.eps);
#pragma unroll
                for (int e = 0; e < 8; e++) x[e] = x[e] * inv * (isq ? gq[e] : gk[e]);
            }
            if (a.rc) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float y = __shfl_xor(x[e], L / 2, L);
                    x[e] = l < L / 2 ? fmaf(x[e], c[e], -(y * s[e])) : fmaf(x[e], c[e], y * s[e]);
                }
            }
        }
        if (isq) qt_store8<QT>(a.qo + ((size_t)(t * a.os) + (size_t)h * HD + 8 * l) * E, x);
        else qt_store8<KT>((isv ? a.vc : a.kc) + (dst + h * a.ps_head) * 2, x);
    }
}

extern "C" int qwen_hip_op_page_append(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_append_t *p, void *stream) {
    if (qt_check_pages("page_append", kv)) return -1;
    QT_REFUSE(!p, "page_append: null descriptor");
    const int E = qt_dt_size(p->dtype);
    QT_REFUSE(!E || (p->dtype != QWEN_HIP_DT_F32 && p->dtype != kv->dtype),
              "page_append: rows of dtype %d into a cache of dtype %d (f32, or the cache's own)", p->dtype, kv->dtype);
    QT_REFUSE(p->T < 0 || p->T > (1 << 28), "page_append: T %d out of range (0..2^28)", p->T);
    if (p->T == 0) return 0;
    QT_REFUSE(!p->k || !p->v || !p->slot || (p->q && !p->q_out), "page_append: null pointer");
    QT_REFUSE(!p->rope_cos != !p->rope_sin || (p->rope_cos && (!p->pos || p->rope_len < 1)),
              "page_append: RoPE needs both tables, pos and rope_len");
    QT_REFUSE(p->q && (p->n_heads < 1 || p->n_heads > 65535), "page_append: n_heads %d out of range (1..65535)", p->n_heads);
    QT_REFUSE(!(p->eps >= 0.f), "page_append: eps is negative or NaN");
    const long long qw = (long long)p->n_heads * kv->head_dim;
    const int A = 16 / E;
    QT_REFUSE(qt_off16(p->q) || qt_off16(p->k) || qt_off16(p->v) || qt_off16(p->q_out) || qt_off16(p->q_norm) ||
                  qt_off16(p->k_norm) || qt_off16(p->rope_cos) || qt_off16(p->rope_sin),
              "page_append: pointers have to be aligned to 16 bytes");
    QT_REFUSE((p->q && (p->q_stride % A || p->q_stride < 0 || p->q_out_stride % A || p->q_out_stride < qw)) || p->k_stride % A ||
                  p->k_stride < 0 || p->v_stride % A || p->v_stride < 0,
              "page_append: strides have to be multiples of 16 bytes, not negative, q_out's at least a token's %lld elements", qw);
    hipStream_t st = (hipStream_t)stream;
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "page_append: the stream's device: %s", hipGetErrorString(on.err));
    const AppendArgs a = {(const uint8_t *)p->q, (const uint8_t *)p->k, (const uint8_t *)p->v, (uint8_t *)p->q_out,
                          (uint8_t *)kv->k, (uint8_t *)kv->v, p->q_stride, p->k_stride, p->v_stride, p->q_out_stride,
                          kv->page_stride, kv->head_stride, kv->slot_stride, p->q_norm, p->k_norm, p->rope_cos, p->rope_sin,
                          p->pos, p->slot, p->T, p->n_heads, kv->n_kv_heads, p->rope_len, kv->n_pages * kv->page_size,
                          kv->page_size, p->eps, qt_div_of(kv->page_size)};
#define APPEND(QT, KT) do { \
        if (kv->head_dim == 128) hipLaunchKernelGGL((k_page_append<QT, KT, 128>), dim3(p->T), dim3(256), 0, st, a); \
        else hipLaunchKernelGGL((k_page_append<QT, KT, 64>), dim3(p->T), dim3(256), 0, st, a); } while (0)
    if (p->dtype == QWEN_HIP_DT_BF16) APPEND(QtBf16, QtBf16);
    else if (p->dtype == QWEN_HIP_DT_F16) APPEND(QtF16, QtF16);
    else if (kv->dtype == QWEN_HIP_DT_BF16) APPEND(QtF32, QtBf16);
    else APPEND(QtF32, QtF16);
#undef APPEND
    const hipError_t e = hipGetLastError();
    QT_REFUSE(e != hipSuccess, "page_append: launch failed: %s", hipGetErrorString(e));
    return 0;
}
