// qt_pattn.hip — the host side of attention over paged caches and packed prompts, and the kernels over 16-bit and f32
// operands.
#include "qt_pattn.h"

// ---- host side -------------------------------------------------------------------------------------

// The kernel, its launch slots and key ranges.  Launch slots: by request (max_q as far as known) or by rows, whichever is
// fewer.  Key ranges: enough workgroups to fill the CUs, 256 keys each at least.
static AttPlan att_plan(AttArgs &a, int dtype, bool paged, int max_q, int max_kv, bool tree, bool codes) {
    AttPlan p = {ATT_ONE, 0, false};
    a.gdiv = qt_div_of(a.G);
    a.tps = 0;
    const long long rows = (long long)a.T * a.G;
    const bool more = tree || codes, little = more && max_kv > 0 && rows * a.nkv * max_kv < 4ll << 20;
    if (dtype == QWEN_HIP_DT_F32) {
        // 32-row tiles for prompts while they give every CU work (one of 512 positions 23.7 us against 25.4 in 16-row tiles,
        // 16 of 64 16.6 against 20.4; three of 21 to 128 11.9 against 8.9)
        if (!paged && (rows / 32 + a.B) * a.nkv >= 256) p.kind = ATT_F32;
    } else if (rows >= (codes ? 56ll : 32ll) * a.B && !little && (paged || (rows / 128 + a.B) * a.nkv >= 96)) {
        // 128-row tiles from 32 rows a request on (64 requests of 32 tokens 42 us against 79 in 16-row tiles, 8 of 16 over
        // 3000 keys 27.3 against 27.8, 32 of 4 70 against 60); prompts, whose keys are not split, while there are tiles
        // enough (8 of 100 to 300 13.1 us against 20.3; one of 512 15.9 against 13.0, three of 21 to 128 9.2 against 8.4).
        // Those are equal requests.  The rule goes by a call's mean, so a step of single tokens and a chunk takes one kernel
        // for both (bf16, 16 over 8 heads, a chunk over 2000 keys: 64 streams of 1000 to 8000 keys and 512 tokens in 16-row tiles
        // 259 us, 198 and 33 in a call each; 32 of them and 1024 tokens in 128-row tiles 160, 110 and 49)
        // Over codes, which 16-row tiles read half as fast again, from 56 rows on (32 trees over 3000 keys, 48 rows: 128-row tiles 99.5 us, 16-row
        // 91.7; 64 rows 102 and 111; over bf16 48 rows 112 and 139, 32 rows 107 and 111); codes and trees, while there is work for two
        // launches (64 rows each over 1000 keys, 16 heads on 8: 4 requests 18.9 to 19.7 and 15.7 to 16.9, 8 requests 24.7 to 25.7 and 24.2 to 25.5; one of
        // 128 rows over 1000 keys 19.7 and 14, over 6000 28 and 30).
        p.kind = ATT_TILE;
    }
    if (p.kind == ATT_ONE) {
        const long long by_rows = rows / 16 + a.B, tps = ((long long)max_q * a.G + 15) / 16, by_req = tps * a.B;
        if (max_q > 0 && by_req <= by_rows) a.tps = (int)tps;
        p.slots = a.tps > 0 ? by_req : by_rows;
    } else {
        p.slots = rows / (p.kind == ATT_TILE ? 128 : 32) + a.B;
    }
    // Single tokens want many ranges (64 streams of up to 8000 keys: 2 of them 217 us, 8 199, 16 200), since a workgroup
    // only reads; a tile's sums are large, and two workgroups a CU are enough (chunks over up to 7000 keys: 2 ranges
    // 171 us, 1 226, 3 190, 4 205).  Over codes, and for trees, requests of one tile each take up to four a CU, since their lengths
    // differ by more than a tile's.  Two, three, four, five and six a CU over codes: 32 trees of 33 to 64 tokens over 500 to 6000 keys 124, 125, 115,
    // 115, 129 us; 32 of 64 over 3000 each 105, 86, 85, 103, 103; 16 of 40 to 64 over 1000 to 8000 116, 91, 79, 105, 100; 24 of 33 to 60 over 100
    // to 2500 61, 50, 50, 50, 57; 48 of 30 to 64 over 200 to 4000 137, 102, 102, 102, 121; 20 chunks of 40 to 64 over 500 to 7000 136, 96, 82, 93,
    // 92.  Chunks of several tiles, ranges 2 to 5: 168, 171, 182, 180.
    const bool one_tile = more && max_q > 0 && (long long)max_q * a.G <= 128;
    const long long wgs = p.slots * a.nkv, blocks = ((long long)max_kv + 31) / 32;
    long long n = wgs > 0 && paged ? ((p.kind == ATT_TILE ? (one_tile ? 1024 : 512) : 4096) + wgs - 1) / wgs : 1;
    if (n > (blocks + 7) / 8) n = (blocks + 7) / 8;
    if (n > 64) n = 64;
    if (n < 1) n = 1;
    a.splits = (int)n;
    a.chunk = (int)((blocks + n - 1) / n + 1) & ~1;
    if (a.chunk < 2) a.chunk = 2;
    // One tile a request: K and V are read once.  Past the 256 MB that the last-level cache holds they are not kept
    // there (64 streams of up to 8000 keys 210 -> 200 us; 4 of 1500, whose 14 MB stay, 12.5 -> 13.8).
    p.stream = a.tps == 1;
    return p;
}

static int check_rows(const char *who, int dtype, int n_heads, int nkv, int hd, int B, int T, int window, float scale) {
    QT_REFUSE(!qt_dt_size(dtype), "%s: dtype %d (f32, bf16 or f16)", who, dtype);
    QT_REFUSE(hd != 64 && hd != 128, "%s: head_dim %d (64 or 128)", who, hd);
    QT_REFUSE(nkv < 1 || nkv > 65535 || n_heads < nkv || n_heads % nkv || n_heads / nkv > 64,
              "%s: %d query heads over %d kv heads (a multiple, 64 a kv head at most)", who, n_heads, nkv);
    QT_REFUSE(B < 0 || B > 65535, "%s: B %d out of range (0..65535)", who, B);
    QT_REFUSE(T < 0 || (long long)T * n_heads > 0x3FFFFFFll, "%s: %d tokens of %d heads (2^26 - 1 rows at most)", who, T, n_heads);
    QT_REFUSE(window < 0, "%s: window %d is negative", who, window);
    QT_REFUSE(!(scale > 0.f) || scale > 1e30f, "%s: scale has to be positive and finite", who);
    return 0;
}

static int paged_args(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p, bool tree, AttArgs &a, AttPlan &plan) {
    const char *const who = tree ? "tree_attention" : "page_attention";
    if (qt_check_pages(who, kv)) return -1;
    QT_REFUSE(!p, "%s: null descriptor", who);
    if (check_rows(who, p->dtype, p->n_heads, kv->n_kv_heads, kv->head_dim, p->B, p->T, p->window, p->scale)) return -1;
    QT_REFUSE(kv->dtype != QWEN_HIP_DT_E4M3 && (p->dtype == QWEN_HIP_DT_F32 ? kv->dtype != QWEN_HIP_DT_BF16 : p->dtype != kv->dtype),
              "%s: rows of dtype %d over a cache of dtype %d (f32 over bf16, else the cache's own; any over e4m3)", who, p->dtype, kv->dtype);
    QT_REFUSE(p->max_q < 0 || p->max_kv < 0, "%s: max_q %d, max_kv %d", who, p->max_q, p->max_kv);
    QT_REFUSE(p->table_cols < 1 || (long long)p->table_cols * kv->page_size > ATT_MAX_KEYS || p->table_stride < p->table_cols,
              "%s: table_cols %d of stride %lld (at least 1, 2^30 positions at most)", who, p->table_cols, p->table_stride);
    a = AttArgs{};
    a.B = p->B; a.T = p->T; a.nkv = kv->n_kv_heads; a.G = p->n_heads / kv->n_kv_heads;
    plan = att_plan(a, p->dtype, true, p->max_q < p->T ? p->max_q : p->T, p->max_kv, tree, kv->dtype == QWEN_HIP_DT_E4M3);
    plan.stream = plan.stream && 2ll * qt_kv_size(kv->dtype) * p->B * p->max_kv * kv->n_kv_heads * kv->head_dim > 256ll << 20;
    return 0;
}

extern "C" long long qwen_hip_op_page_attention_workspace(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p) {
    AttArgs a, t;                                     // with and without trees
    AttPlan plan;
    if (paged_args(kv, p, false, a, plan) || paged_args(kv, p, true, t, plan)) return -1;
    const long long n = a.splits > t.splits ? a.splits : t.splits;
    return n > 1 ? n * a.T * p->n_heads * (kv->head_dim + 2) * 4 : 0;
}

template <typename QT, int HD, bool PAGED>
static hipError_t att_launch(const AttArgs &a, const AttPlan &plan, hipStream_t st) {
    typedef typename std::conditional<PAGED && std::is_same<QT, QtF32>::value, QtBf16, QT>::type KT;
    const dim3 grid((unsigned)(plan.slots * a.nkv), a.splits);
    if (plan.kind == ATT_ONE && PAGED && plan.stream) return qt_launch(k_att_one<QT, KT, HD, PAGED, PAGED>, grid, dim3(64 * ATT_WV), 0, st, a);
    if (plan.kind == ATT_ONE) return qt_launch(k_att_one<QT, KT, HD, PAGED, false>, grid, dim3(64 * ATT_WV), 0, st, a);
    if constexpr (sizeof(typename QT::elem) == 2) return qt_launch(k_att_tile<QT, HD, PAGED>, grid, dim3(256), 0, st, a);
    else return qt_launch(k_att_f32<HD>, grid, dim3(64 * ATT_WV), 0, st, a);
}
template <bool PAGED> static hipError_t att_launch_rows(const AttArgs &a, const AttPlan &plan, int dtype, int hd, hipStream_t st) {
    if (dtype == QWEN_HIP_DT_F32) return hd == 128 ? att_launch<QtF32, 128, PAGED>(a, plan, st) : att_launch<QtF32, 64, PAGED>(a, plan, st);
    if (dtype == QWEN_HIP_DT_BF16) return hd == 128 ? att_launch<QtBf16, 128, PAGED>(a, plan, st) : att_launch<QtBf16, 64, PAGED>(a, plan, st);
    return hd == 128 ? att_launch<QtF16, 128, PAGED>(a, plan, st) : att_launch<QtF16, 64, PAGED>(a, plan, st);
}
static hipError_t att_merge(const AttArgs &a, int dtype, int hd, hipStream_t st) {
    const long long rows = (long long)a.T * a.nkv * a.G;
    void (*const kernel)(AttArgs) = dtype == QWEN_HIP_DT_F32    ? (hd == 128 ? k_att_merge<QtF32, 128> : k_att_merge<QtF32, 64>)
                                    : dtype == QWEN_HIP_DT_BF16 ? (hd == 128 ? k_att_merge<QtBf16, 128> : k_att_merge<QtBf16, 64>)
                                                                : (hd == 128 ? k_att_merge<QtF16, 128> : k_att_merge<QtF16, 64>);
    return qt_launch(kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
}

static int paged_attention(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p, const qwen_hip_tree_t *tree, void *stream) {
    const char *const who = tree ? "tree_attention" : "page_attention";
    AttArgs a;
    AttPlan plan;
    if (paged_args(kv, p, tree != nullptr, a, plan)) return -1;
    if (p->B == 0 || p->T == 0) return 0;
    if (tree) {
        QT_REFUSE(tree->mask_words < 1 || tree->mask_words > 32 || tree->mask_stride < tree->mask_words,
                  "tree_attention: mask_words %d of stride %lld (1..32, the stride at least as many)", tree->mask_words, tree->mask_stride);
        QT_REFUSE(!tree->mask || (p->window > 0 && !tree->pos), "tree_attention: null pointer (a window needs pos)");
    }
    QT_REFUSE(!p->q || !p->out || !p->cu_q || !p->kv_len || !p->table, "%s: null pointer", who);
    QT_REFUSE(p->out == p->q, "%s: out must not be q", who);
    const int A = 16 / qt_dt_size(p->dtype);
    QT_REFUSE(qt_off16(p->q) || qt_off16(p->out) || qt_off16(p->workspace), "%s: pointers have to be aligned to 16 bytes", who);
    QT_REFUSE(p->q_stride % A || p->q_stride < 0 || p->out_stride % A || p->out_stride < (long long)p->n_heads * kv->head_dim,
              "%s: strides %lld, %lld (multiples of 16 bytes, out's at least a token's)", who, p->q_stride, p->out_stride);
    const long long need = a.splits > 1 ? (long long)a.splits * a.T * p->n_heads * (kv->head_dim + 2) * 4 : 0;
    QT_REFUSE(need > 0 && (!p->workspace || p->workspace_bytes < need), "%s: a workspace of %lld bytes is needed, %lld given", who,
              need, p->workspace ? p->workspace_bytes : 0ll);
    QT_REFUSE(plan.slots * a.nkv > 0xFFFFFFll, "%s: too many tiles for one launch", who);
    const long long E = qt_dt_size(p->dtype), row = (long long)p->n_heads * kv->head_dim * E;
    QT_REFUSE(qt_rows_meet(p->out, p->out_stride * E, row, p->q, p->q_stride * E, row, p->T), "%s: out overlaps q", who);
    if (tree) {
        const int *const pos = p->window > 0 ? tree->pos : nullptr;
        QT_REFUSE(qt_rows_meet(p->out, p->out_stride * E, row, tree->mask, tree->mask_stride * 4, 4ll * tree->mask_words, p->T) ||
                      (pos && qt_rows_meet(p->out, p->out_stride * E, row, pos, 4, 4, p->T)),
                  "tree_attention: out overlaps mask or pos");
        const QtMem ws[] = {{p->workspace, need, "workspace", nullptr}};
        const QtMem in[] = {{tree->mask, 4 * ((p->T - 1) * tree->mask_stride + tree->mask_words), 0, 0}, {pos, 4ll * p->T, 0, 0}};
        QT_REFUSE(need > 0 && qt_meets(ws, 1, in, 2), "tree_attention: the workspace overlaps mask or pos");
    }
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "%s: the stream's device: %s", who, hipGetErrorString(on.err));
    a.q = (const uint8_t *)p->q; a.k = (const uint8_t *)kv->k; a.v = (const uint8_t *)kv->v; a.out = (uint8_t *)p->out;
    a.qs = p->q_stride; a.os = p->out_stride;
    a.ks_page = kv->page_stride; a.ks_head = kv->head_stride; a.ks_slot = a.vs_slot = kv->slot_stride;
    a.cu = p->cu_q; a.kv_len = p->kv_len; a.table = p->table; a.ts = p->table_stride;
    a.cols = p->table_cols; a.n_pages = kv->n_pages; a.ps = kv->page_size; a.div = qt_div_of(kv->page_size);
    a.window = p->window <= ATT_MAX_KEYS ? p->window : 0;
    a.near = (kv->n_pages - 1.0) * kv->page_stride + (kv->n_kv_heads - 1.0) * kv->head_stride + (kv->page_size - 1.0) * kv->slot_stride < 2147000000.0;
    a.c = p->scale * QT_LOG2E;
    a.po = (float *)p->workspace;
    a.pm = a.po + (size_t)a.splits * a.T * p->n_heads * kv->head_dim;
    const bool codes = kv->dtype == QWEN_HIP_DT_E4M3;
    if (codes) {
        a.ksc = kv->k_scale; a.vsc = kv->v_scale;
        a.ss_page = kv->scale_page_stride; a.ss_head = kv->scale_head_stride; a.ss_slot = kv->scale_slot_stride;
        a.near = a.near && (kv->n_pages - 1.0) * kv->scale_page_stride + (kv->page_size - 1.0) * kv->scale_slot_stride < 2147000000.0;
    }
    if (tree) { a.mask = tree->mask; a.pos = tree->pos; a.mstride = tree->mask_stride; a.mwords = tree->mask_words; }
    hipError_t e = codes  ? att_launch_codes(a, plan, p->dtype, kv->head_dim, tree != nullptr, st)
                   : tree ? att_launch_tree(a, plan, p->dtype, kv->head_dim, st)
                          : att_launch_rows<true>(a, plan, p->dtype, kv->head_dim, st);
    if (e == hipSuccess && a.splits > 1) e = att_merge(a, p->dtype, kv->head_dim, st);
    QT_REFUSE(e != hipSuccess, "%s: launch failed: %s", who, hipGetErrorString(e));
    return 0;
}

extern "C" int qwen_hip_op_page_attention(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p, void *stream) {
    return paged_attention(kv, p, nullptr, stream);
}

extern "C" int qwen_hip_op_tree_attention(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p, const qwen_hip_tree_t *tree, void *stream) {
    QT_REFUSE(!tree, "tree_attention: null tree");
    return paged_attention(kv, p, tree, stream);
}

extern "C" int qwen_hip_op_packed_attention(const qwen_hip_packed_attn_t *p, void *stream) {
    QT_REFUSE(!p, "packed_attention: null descriptor");
    if (check_rows("packed_attention", p->dtype, p->n_heads, p->n_kv_heads, p->head_dim, p->B, p->T, p->window, p->scale)) return -1;
    if (p->B == 0 || p->T == 0) return 0;
    QT_REFUSE(!p->q || !p->k || !p->v || !p->out || !p->cu, "packed_attention: null pointer");
    QT_REFUSE(p->out == p->q || p->out == p->k || p->out == p->v, "packed_attention: out must not be q, k or v");
    const int A = 16 / qt_dt_size(p->dtype);
    QT_REFUSE(qt_off16(p->q) || qt_off16(p->k) || qt_off16(p->v) || qt_off16(p->out), "packed_attention: pointers have to be aligned to 16 bytes");
    QT_REFUSE(p->q_stride % A || p->k_stride % A || p->v_stride % A || p->out_stride % A || p->q_stride < 0 || p->k_stride < 0 ||
                  p->v_stride < 0 || p->out_stride < (long long)p->n_heads * p->head_dim || p->k_stride >= 1 << 24 || p->v_stride >= 1 << 24,
              "packed_attention: strides %lld, %lld, %lld, %lld (multiples of 16 bytes, out's at least a token's, k's and v's under 2^24)", p->q_stride,
              p->k_stride, p->v_stride, p->out_stride);
    AttArgs a = {};
    a.B = p->B; a.T = p->T; a.nkv = p->n_kv_heads; a.G = p->n_heads / p->n_kv_heads;
    const AttPlan plan = att_plan(a, p->dtype, false, 0, 0, false, false);
    QT_REFUSE(plan.slots * a.nkv > 0xFFFFFFll, "packed_attention: too many tiles for one launch");
    const long long E = qt_dt_size(p->dtype), row = (long long)p->n_heads * p->head_dim * E, kw = (long long)p->n_kv_heads * p->head_dim * E;
    QT_REFUSE(qt_rows_meet(p->out, p->out_stride * E, row, p->q, p->q_stride * E, row, p->T) ||
                  qt_rows_meet(p->out, p->out_stride * E, row, p->k, p->k_stride * E, kw, p->T) ||
                  qt_rows_meet(p->out, p->out_stride * E, row, p->v, p->v_stride * E, kw, p->T),
              "packed_attention: out overlaps q, k or v");
    a.q = (const uint8_t *)p->q; a.k = (const uint8_t *)p->k; a.v = (const uint8_t *)p->v; a.out = (uint8_t *)p->out;
    a.qs = p->q_stride; a.os = p->out_stride; a.ks_slot = p->k_stride; a.vs_slot = p->v_stride;
    a.cu = p->cu;
    a.window = p->window <= ATT_MAX_KEYS ? p->window : 0;
    a.c = p->scale * QT_LOG2E;
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "packed_attention: the stream's device: %s", hipGetErrorString(on.err));
    const hipError_t e = att_launch_rows<false>(a, plan, p->dtype, p->head_dim, st);
    QT_REFUSE(e != hipSuccess, "packed_attention: launch failed: %s", hipGetErrorString(e));
    return 0;
}
