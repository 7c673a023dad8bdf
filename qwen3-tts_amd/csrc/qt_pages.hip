// qt_pages.hip — a paged cache's bookkeeping for one step (qwen_hip_op_page_plan) and its writer
// (qwen_hip_op_page_append).
#include "qt_ops.h"

// ---- the plan --------------------------------------------------------------------------------
// With h(n) = ceil(n / page_size): an ended request gives back its h(kv) pages, a continued one takes
// h(kv + new) - h(kv).  In request order, exclusive sums of the pages given back, of those taken and of the new
// tokens say where each request's entries lie; then every page and every token finds its request by a search
// in those sums, independently of the others.  Page i of all taken is the free list's entry n_free + R - 1 - i, R
// pages having been given back: entries n_free .. n_free + R - 1 are those pages themselves, read from the tables.
// So nothing that is written is read again, and any number of workgroups can share the pages and tokens when each makes the sums
// over the (at most 2048) requests for itself; only the lengths and the free count, which may be replaced in place, are
// written by one of them, and in a launch of their own where the others may still read what they replace.
// Bound by the latency of its dependent loads (lengths, then free list and tables) and of the launch: 8 requests of one
// token 6 us a pass, 512 requests, 37 of them ended, 47 680 tokens 8.9 (one workgroup for all pages, a second launch for
// the slots: 30).
#define PLAN_T 256
#define PLAN_MAX_B 2048         // 32 KB of LDS
#define PLAN_SAT (1u << 30)     // sums stop here: under 2^31 in any order, over every limit they are held to

struct PlanArgs {
    const int *new_len, *kv_len, *n_free;
    int *table, *free_pages, *kv_out, *n_free_out, *cu, *pos, *slot, *status;
    long long ts;
    int B, ps, n_pages, cols, cap;
    int share, finish;          // this launch writes pages and tokens; offsets, lengths, the free count and status
    QtDiv div;
};

__device__ __forceinline__ unsigned plan_add(unsigned a, unsigned b) { return min(a + b, PLAN_SAT); }

// The last b with first[b] <= i (first[0] = 0, ascending), for four i at once: of requests that begin at the same
// place all but the last are empty.  Fixed steps, so the four searches' LDS reads overlap.
__device__ __forceinline__ void plan_find(const unsigned *first, int B, const unsigned (&i)[4], int (&b)[4]) {
#pragma unroll
    for (int k = 0; k < 4; k++) b[k] = 0;
    for (int s = 1 << (31 - __clz(B)); s; s >>= 1)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int p = b[k] + s;
            if (first[min(p, B - 1)] <= i[k] && p < B) b[k] = p;
        }
}

__global__ __launch_bounds__(PLAN_T) void k_page_plan(PlanArgs a) {
    extern __shared__ unsigned sh[];
    unsigned *tok = sh, *take = tok + a.B + 1, *back = take + a.B + 1;     // exclusive sums, [B + 1] each
    int *kv = reinterpret_cast<int *>(back + a.B + 1);                     // lengths before, [B]
    __shared__ unsigned wsum[3][PLAN_T / 64];
    __shared__ int bad;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n_free = a.n_free[0];
    if (tid == 0) bad = n_free < 0 || n_free > a.n_pages ? QWEN_HIP_PLAN_INVALID : 0;
    __syncthreads();
    const long long room = (long long)a.cols * a.ps;
    int flags = 0;
    for (int b = tid; b < a.B; b += PLAN_T) {
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
            p = (qt_quot(len + n, a.div) + ((len + n) % a.ps != 0)) - (qt_quot(len, a.div) + (len % a.ps != 0));
        }
        kv[b] = len; tok[b] = t; take[b] = p; back[b] = r;
    }
    if (flags) atomicOr(&bad, flags);
    __syncthreads();
    // exclusive sums: a thread's requests, the wave's threads, the waves
    const int per = (a.B + PLAN_T - 1) / PLAN_T, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    unsigned s[3] = {0u, 0u, 0u}, x[3];
    for (int b = b0; b < b1; b++) { s[0] = plan_add(s[0], tok[b]); s[1] = plan_add(s[1], take[b]); s[2] = plan_add(s[2], back[b]); }
#pragma unroll
    for (int k = 0; k < 3; k++) x[k] = s[k];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
#pragma unroll
        for (int k = 0; k < 3; k++) {
            const unsigned y = __shfl_up(x[k], o, 64);
            if (lane >= o) x[k] = plan_add(x[k], y);
        }
    if (lane == 63)
#pragma unroll
        for (int k = 0; k < 3; k++) wsum[k][wave] = x[k];
    __syncthreads();
    unsigned tot[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {
        unsigned before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < PLAN_T / 64; w++) {
            if (w == wave) before = all;
            all = plan_add(all, wsum[k][w]);
        }
        const unsigned up = __shfl_up(x[k], 1, 64);
        s[k] = lane == 0 ? before : plan_add(before, up);
        tot[k] = all;
    }
    for (int b = b0; b < b1; b++) {
        const unsigned t = tok[b], p = take[b], r = back[b];
        tok[b] = s[0]; take[b] = s[1]; back[b] = s[2];
        s[0] = plan_add(s[0], t); s[1] = plan_add(s[1], p); s[2] = plan_add(s[2], r);
    }
    const unsigned T = tot[0], N = tot[1], R = tot[2];
    int any = bad;
    if (T > (unsigned)a.cap) any |= QWEN_HIP_PLAN_TOO_MANY;
    if (n_free + (long long)R > a.n_pages) any |= QWEN_HIP_PLAN_INVALID;     // pages given back twice
    if ((long long)N > n_free + (long long)R) any |= QWEN_HIP_PLAN_NO_PAGES;
    __syncthreads();
    const unsigned at0 = blockIdx.x * 4 * PLAN_T, stride = gridDim.x * 4 * PLAN_T;
    // pages given back begin at the last workgroup, pages taken at the middle one: few have two kinds of work
    const unsigned at_given = stride - 4 * PLAN_T - at0, at_taken = (blockIdx.x + gridDim.x / 2) % gridDim.x * 4 * PLAN_T;
    const auto have = [&](int b) { return (unsigned)(qt_quot(kv[b], a.div) + (kv[b] % a.ps != 0)); };
    const auto four = [&](unsigned (&i)[4], unsigned at) {
#pragma unroll
        for (int k = 0; k < 4; k++) i[k] = at + k * PLAN_T + tid;
    };
    // pages j of those given back, and pages i of those taken, four at once
    const auto given = [&](const unsigned (&j)[4], int (&v)[4]) {
        int b[4];
        plan_find(back, a.B, j, b);
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = j[k] < R ? a.table[(long long)b[k] * a.ts + (j[k] - back[b[k]])] : -1;
    };
    const auto taken = [&](const unsigned (&i)[4], int (&v)[4]) {
        unsigned j[4];                                                       // i < R: the j-th given back
        bool some = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            j[k] = i[k] < N ? R - 1 - i[k] : ~0u;
            some |= j[k] < R;
            v[k] = i[k] < N && i[k] >= R ? a.free_pages[n_free - 1 - (int)(i[k] - R)] : -1;
        }
        if (some) {
            int g[4];
            given(j, g);
#pragma unroll
            for (int k = 0; k < 4; k++) v[k] = j[k] < R ? g[k] : v[k];
        }
    };
    unsigned i[4];
    int v[4], b[4];
    if (a.share && !any) {
        for (unsigned at = at_given; at < R; at += stride) {
            four(i, at);
            given(i, v);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i[k] < R) a.free_pages[n_free + (int)i[k]] = v[k];
        }
        for (unsigned at = at_taken; at < N; at += stride) {
            four(i, at);
            plan_find(take, a.B, i, b);
            taken(i, v);
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i[k] < N) a.table[(long long)b[k] * a.ts + have(b[k]) + (i[k] - take[b[k]])] = v[k];
        }
    }
    if (a.share)
        for (unsigned at = at0; at < (unsigned)a.cap; at += stride) {
            unsigned f[4];
            int p[4], c[4], page[4];
            bool some = false;
            four(i, at);
            plan_find(tok, a.B, i, b);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool live = !any && i[k] < T;
                p[k] = live ? kv[b[k]] + (int)(i[k] - tok[b[k]]) : -1;
                c[k] = live ? qt_quot(p[k], a.div) : 0;
                const unsigned hb = have(b[k]);
                f[k] = live && (unsigned)c[k] >= hb ? take[b[k]] + c[k] - hb : ~0u;      // a new page, or one of before
                some |= f[k] != ~0u;
                page[k] = live && f[k] == ~0u ? a.table[(long long)b[k] * a.ts + c[k]] : -1;
            }
            if (some) {
                taken(f, v);
#pragma unroll
                for (int k = 0; k < 4; k++) page[k] = f[k] != ~0u ? v[k] : page[k];
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                if (i[k] >= (unsigned)a.cap) continue;
                a.pos[i[k]] = p[k];
                a.slot[i[k]] = (unsigned)page[k] < (unsigned)a.n_pages ? page[k] * a.ps + (p[k] - c[k] * a.ps) : -1;
            }
        }
    if (!a.finish || blockIdx.x) return;
    for (int r = tid; r < a.B; r += PLAN_T) {
        const int n = a.new_len[r];
        a.kv_out[r] = any ? a.kv_len[r] : n < 0 ? 0 : kv[r] + n;
    }
    for (int r = tid; r <= a.B; r += PLAN_T) a.cu[r] = any ? 0 : r == a.B ? (int)T : (int)tok[r];
    if (tid == 0) { a.n_free_out[0] = any ? n_free : (int)(n_free + R - N); a.status[0] = any; }
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
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "page_plan: the stream's device: %s", hipGetErrorString(on.err));
    PlanArgs a = {p->new_len, p->kv_len, p->n_free, p->table, p->free_pages, p->kv_len_out, p->n_free_out, p->cu_q, p->pos,
                  p->slot, p->status, p->table_stride, p->B, p->page_size, p->n_pages, p->table_cols, p->max_tokens, 1, 1,
                  qt_div_of(p->page_size)};
    // A workgroup for every 512 tokens, or 16 requests: pages given back, whose number the host does not know, may be
    // many a request.
    const int most = p->max_tokens > p->B * 32 ? p->max_tokens : p->B * 32;
    const int wgs = most <= 1024 ? 1 : most >= (128 << 10) ? 256 : (most + 511) / 512;
    const bool in_place = p->kv_len_out == p->kv_len || p->n_free_out == p->n_free;
    a.finish = wgs == 1 || !in_place;
    const size_t lds = (size_t)(4 * p->B + 3) * 4;
    hipError_t e = qt_launch(k_page_plan, dim3(wgs), dim3(PLAN_T), lds, st, a);
    if (e == hipSuccess && !a.finish) {
        a.share = 0;
        a.finish = 1;
        e = qt_launch(k_page_plan, dim3(1), dim3(PLAN_T), lds, st, a);
    }
    QT_REFUSE(e != hipSuccess, "page_plan: launch failed: %s", hipGetErrorString(e));
    return 0;
}

// ---- the append --------------------------------------------------------------------------------
// y = x / sqrt(mean x^2 + eps) g, then (y1, y2) -> (y1 c - y2 s, y2 c + y1 s) on a head's halves, all in f32,
// rounded once.  A head's row is HD / 8 lanes of 8 elements (16-byte loads); its sum of squares and its rotation's
// other half are lane exchanges.  A workgroup takes one token: its lanes' angles and gains are loaded once
// and serve every head.  Bound by the rows' bytes for prompts (8190 tokens bf16, 16 query and 8 kv heads of 128: 33 us, 4.2 TB/s,
// the copy rate being 4.9), by the launch and the latency of slot, angles and rows for a step (32 tokens f32: 6.4 us).
//
// Into a quantised cache a row's lanes also exchange its largest magnitude, as bits, whose order is that of the magnitudes with
// infinities and NaN last; it gives the scale's exponent by one addition (qt_scale_byte), the division by the scale is an exact product, and
// the conversion rounds once.  8190 tokens bf16: 30.6 us, 3.9 TB/s; 32 tokens f32: 6.3.
struct AppendArgs {
    const uint8_t *q, *k, *v;
    uint8_t *qo, *kc, *vc, *ksc, *vsc;
    long long qs, ks, vs, os, ps_page, ps_head, ps_slot, ss_page, ss_head, ss_slot;
    const float *qn, *kn, *rc, *rs;
    const int *pos, *slot;
    int T, nh, nkv, rope_len, n_slots, page;
    float eps;
    QtDiv div;
};

template <typename QT, typename KT, int HD>
__global__ __launch_bounds__(256) void k_page_append(AppendArgs a) {
    constexpr int E = sizeof(typename QT::elem), EK = sizeof(typename KT::elem), L = HD / 8;       // L: lanes a row
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
    const long long sdst = EK == 1 ? page * a.ss_page + (slot - page * a.page) * a.ss_slot : 0;
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
        else if constexpr (EK == 1) {
            uint32_t m = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) m = max(m, __float_as_uint(x[e]) & 0x7FFFFFFFu);
#pragma unroll
            for (int o = 1; o < L; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, L));
            const uint32_t byte = qt_scale_byte(m);
            const float inv = __uint_as_float((254u - byte) << 23);             // of a NaN row: not used
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] *= inv;
            const uint2 c = byte == 255u ? make_uint2(0x7F7F7F7Fu, 0x7F7F7F7Fu) : qt_codes_e4m3(x);
            *reinterpret_cast<uint2 *>((isv ? a.vc : a.kc) + dst + h * a.ps_head) = c;
            if (l == 0) (isv ? a.vsc : a.ksc)[sdst + h * a.ss_head] = (uint8_t)byte;
        } else qt_store8<KT>((isv ? a.vc : a.kc) + (dst + h * a.ps_head) * EK, x);
    }
}

extern "C" int qwen_hip_op_page_append(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_append_t *p, void *stream) {
    if (qt_check_pages("page_append", kv)) return -1;
    QT_REFUSE(!p, "page_append: null descriptor");
    const int E = qt_dt_size(p->dtype);
    const bool codes = kv->dtype == QWEN_HIP_DT_E4M3;
    QT_REFUSE(!E || (p->dtype != QWEN_HIP_DT_F32 && p->dtype != kv->dtype && !codes),
              "page_append: rows of dtype %d into a cache of dtype %d (f32, or the cache's own)", p->dtype, kv->dtype);
    QT_REFUSE(p->T < 0 || p->T >= 1 << 24, "page_append: T %d out of range (0..2^24 - 1)", p->T);
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
    // a token's workgroup writes its q after reading its own rows, at no known time before or after the others read theirs
    const bool in_place = p->q && p->q_out == p->q;
    QT_REFUSE(in_place && p->T > 1 && p->q_stride != p->q_out_stride, "page_append: q in place with two strides, %lld and %lld", p->q_stride,
              p->q_out_stride);
    const long long kw = (long long)kv->n_kv_heads * kv->head_dim * E;
    QT_REFUSE(p->q && ((!in_place && qt_rows_meet(p->q_out, p->q_out_stride * E, qw * E, p->q, p->q_stride * E, qw * E, p->T)) ||
                       qt_rows_meet(p->q_out, p->q_out_stride * E, qw * E, p->k, p->k_stride * E, kw, p->T) ||
                       qt_rows_meet(p->q_out, p->q_out_stride * E, qw * E, p->v, p->v_stride * E, kw, p->T)),
              "page_append: q_out overlaps rows that are read (it may be q itself)");
    if (qt_check_pages_apart("page_append", kv)) return -1;
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "page_append: the stream's device: %s", hipGetErrorString(on.err));
    const AppendArgs a = {(const uint8_t *)p->q, (const uint8_t *)p->k, (const uint8_t *)p->v, (uint8_t *)p->q_out,
                          (uint8_t *)kv->k, (uint8_t *)kv->v, codes ? kv->k_scale : nullptr, codes ? kv->v_scale : nullptr,
                          p->q_stride, p->k_stride, p->v_stride, p->q_out_stride, kv->page_stride, kv->head_stride, kv->slot_stride,
                          codes ? kv->scale_page_stride : 0, codes ? kv->scale_head_stride : 0, codes ? kv->scale_slot_stride : 0, p->q_norm, p->k_norm, p->rope_cos, p->rope_sin,
                          p->pos, p->slot, p->T, p->n_heads, kv->n_kv_heads, p->rope_len, kv->n_pages * kv->page_size,
                          kv->page_size, p->eps, qt_div_of(kv->page_size)};
#define APPEND(QT, KT) (kv->head_dim == 128 ? k_page_append<QT, KT, 128> : k_page_append<QT, KT, 64>)
    void (*const kernel)(AppendArgs) = codes && p->dtype == QWEN_HIP_DT_F32    ? APPEND(QtF32, QtE4m3)
                                       : codes && p->dtype == QWEN_HIP_DT_BF16 ? APPEND(QtBf16, QtE4m3)
                                       : codes                                 ? APPEND(QtF16, QtE4m3)
                                       : p->dtype == QWEN_HIP_DT_BF16    ? APPEND(QtBf16, QtBf16)
                                       : p->dtype == QWEN_HIP_DT_F16   ? APPEND(QtF16, QtF16)
                                       : kv->dtype == QWEN_HIP_DT_BF16 ? APPEND(QtF32, QtBf16)
                                                                       : APPEND(QtF32, QtF16);
#undef APPEND
    const hipError_t e = qt_launch(kernel, dim3(p->T), dim3(256), 0, st, a);
    QT_REFUSE(e != hipSuccess, "page_append: launch failed: %s", hipGetErrorString(e));
    return 0;
}
