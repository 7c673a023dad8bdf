// qt_pattn.hip — causal attention of several requests' new tokens: over paged caches
// (qwen_hip_op_page_attention) and over whole packed prompts (qwen_hip_op_packed_attention).
//
// o_i = sum_j p_ij v_j / sum_j p_ij,  p_ij = 2^((s_ij - m_i) c),  s_ij = q_i . k_j,  c = scale log2(e), over the
// positions j that row i sees, with the running maximum m_i and sum of one pass over the keys (all f32).
//
// Rows.  The new tokens of a request and the query heads of one kv head make its rows, row r = (token r / G, head
// r % G): heads that read the same keys share them, a decode step's heads fill a tile as a prompt's tokens do, and the
// causal edge crosses few key blocks.
//
// Products.  Scores are made transposed, S^T = K Q^T by v_mfma_f32_32x32x16: lane l supplies key row l % 32 (A) and
// query row l % 32 (B), each as 8 of the 16 dims (those of half h = l / 32), and ends with query row l % 32 and keys
// 8 (i / 4) + 4 h + i % 4 in register i.  So a lane has one query row: the softmax needs one exchange with the other
// half, scaling a row's sums is one factor a lane, and eight of its probabilities are, in place, the B operand
// of O^T = V^T P^T over 16 keys (a sum over keys in the order of the registers: key 16 s + 8 (j / 4) + 4 h + j % 4 in
// place (h, j)).  V's operand wants those 8 keys of one dim: read transposed from LDS where K and V are there (k_att_tile),
// else a lane loads NT = HD / 32 neighbouring dims of each key's row (the 32 lanes of a half a whole row) and transposes
// them in registers; dim NT m + t is row m of product t.
//
// Types.  16-bit rows over a cache of their type: one product each; the probabilities are rounded to that type for
// V's product (bf16: at most 2^-8 of each, f16: 2^-11, of either sign over the keys), and a row's sum is that of the
// rounded ones, so a key that outweighs the rest gives its value whatever its probability rounds to.  f32 rows over a bf16 cache: q and p as three bf16 planes whose sum is exact, three products.  All f32: both
// operands as planes, six products (qt_planes.h).
//
// What a row does not see never reaches it: hidden scores become -infinity before the maximum.  Their probabilities
// are 0, and 0 times an infinite or NaN v would still be NaN: where a tile ends with anything that is not
// finite, its rows are done again one by one over what each of them sees (att_serial), which also serves f32 values
// that have no planes (infinite, NaN, past bf16's range after rounding).  So are rows whose maximum times c is past
// f32's range: the 16-bit kernels' s c - m c makes every probability 0 there (a sum of 0 under a maximum shows it) or infinite.
#include "qt_ops.h"
#include "qt_planes.h"
#include <type_traits>

typedef float qt_f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 qt_f16x8 __attribute__((ext_vector_type(8)));

#define ATT_MAX_KEYS (1 << 30)              // positions of a request: their arithmetic stays in 32 bits

struct AttArgs {
    const uint8_t *q, *k, *v;
    uint8_t *out;
    long long qs, os;                       // elements between tokens
    long long ks_page, ks_head, ks_slot;    // paged: of k and v; packed: ks_slot, vs_slot between tokens, head HD apart
    long long vs_slot;
    const int *cu, *kv_len, *table;
    long long ts;
    int cols, n_pages, ps;
    int near;                               // paged: every element of k (of v) within 2^32 bytes of its first
    QtDiv div, gdiv;                        // by page_size, by G
    int B, T, nkv, G, window;
    float c;                                // scale log2(e)
    int tps;                                // > 0: launch slots a request, else slots by att_find
    int splits, chunk;                      // key ranges a tile at most, 32-key blocks in each (att_ranges)
    float *po, *pm;                         // splits > 1: sums [split][T nh][HD], and maximum, sum [split][T nh][2]
};

template <typename T> __device__ __forceinline__ qt_f32x16 att_mma(qt_u32x4 a, qt_u32x4 b, qt_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(qt_bf16x8, a), __builtin_bit_cast(qt_bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ qt_f32x16 att_mma<QtF16>(qt_u32x4 a, qt_u32x4 b, qt_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(qt_f16x8, a), __builtin_bit_cast(qt_f16x8, b), c, 0, 0, 0);
}
// c + both halves of p, in f32
template <typename T> __device__ __forceinline__ float att_add2(uint32_t p, float c) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, p), __builtin_bit_cast(b2, 0x3F803F80u), c, false);
}
template <> __device__ __forceinline__ float att_add2<QtF16>(uint32_t p, float c) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, p), __builtin_bit_cast(h2, 0x3C003C00u), c, false);
}
// sum over planes, the smallest products first
template <typename T, int NA, int NB>
__device__ __forceinline__ qt_f32x16 att_planes(const qt_u32x4 (&a)[NA], const qt_u32x4 (&b)[NB], qt_f32x16 c) {
#pragma unroll
    for (int s = NA + NB - 2; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++)
            if (s - i >= 0 && s - i < NB && s <= 2) c = att_mma<T>(a[i], b[s - i], c);
    return c;
}

__device__ __forceinline__ float att_other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// The request that a launch slot belongs to when a request begins at slot floor(first row / TR) + b, TR rows a tile:
// its ceil(rows / TR) tiles fit before the next one's, whatever the lengths, so floor(all rows / TR) + B slots are
// enough for the host, which does not know them.
// Offsets are the caller's: one out of range is brought into it, so that nothing is read or written past T.
__device__ __forceinline__ int att_cu(const AttArgs &a, int b) { return min(max(a.cu[b], 0), a.T); }
template <int TR> __device__ __forceinline__ int att_first(const AttArgs &a, int b) {
    return (int)((long long)att_cu(a, b) * a.G / TR) + b;
}
template <int TR> __device__ __forceinline__ int att_find(const AttArgs &a, int slot) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int n = a.B; n > 1;) {                         // 64 requests' first slots at a time, one of every `step`
        const int step = (n + 63) / 64;
        const bool before = lane * step < n && att_first<TR>(a, b + lane * step) <= slot;
        const int c = max((int)__popcll(__ballot(before)) - 1, 0);
        b += c * step;
        n = min(step, n - c * step);
    }
    return b;
}

// one tile's geometry, uniform over the workgroup
struct AttTile {
    int q0, rows, r0;           // first token of the request, its rows, the tile's first row
    int shift, kmax;            // a token's position is shift + its place; keys at or past kmax do not exist
    int lo, hi;                 // keys that some row of the tile may see
};
// one request's tokens and keys
struct AttReq { int q0, n, kv; };
template <bool PAGED> __device__ __forceinline__ AttReq att_req(const AttArgs &a, int b) {
    const int q0 = att_cu(a, b), n = max(att_cu(a, b + 1) - q0, 0);
    return {q0, n, PAGED ? min(max(a.kv_len[b], 0), ATT_MAX_KEYS) : n};
}
template <int TR, bool PAGED>
__device__ __forceinline__ AttTile att_tile(const AttArgs &a, AttReq q, int tile) {
    AttTile t;
    t.q0 = q.q0;
    const int n = q.n, kv = q.kv;
    t.rows = n * a.G;
    t.r0 = TR * tile;
    t.kmax = PAGED ? min(kv, a.cols * a.ps) : n;
    t.shift = kv - n;
    const int first = t.shift + qt_quot(t.r0, a.gdiv), last = t.shift + qt_quot(min(t.r0 + TR - 1, t.rows - 1), a.gdiv);
    t.lo = a.window > 0 ? max(first - a.window + 1, 0) : 0;
    t.hi = min(t.kmax, last + 1);
    return t;
}

// The tile of 128 rows that comes at `slot` when the requests are in the order of their keys, longest first (in 64s), and
// each one's tiles from its last to its first: little work is left for the end, and tiles that read the same keys run at
// the same time and find them in the L2.  How many tiles belong to requests of w keys or more is a sum over the requests (four
// a lane); a search by halves finds the w that holds the slot, a running sum the request among its equals: about half
// a us.  False: no tile.
#define ATT_SORT_B 256
template <bool PAGED> __device__ __forceinline__ bool att_longest(const AttArgs &a, int slot, int &b, int &tile, AttReq &req) {
    const int lane = threadIdx.x & 63;
    AttReq q[4];
    int n[4], w[4], top = 0;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        q[r] = {0, 0, 0};
        if (64 * r < a.B && 64 * r + lane < a.B) q[r] = att_req<PAGED>(a, 64 * r + lane);
        n[r] = (q[r].n * a.G + 127) / 128;
        w[r] = q[r].kv >> 6;
        top = max(top, w[r]);
    }
    top = wave_max_i(top);
    const auto longer = [&](int x) {                    // tiles of requests of x or more
        int c = 0;
#pragma unroll
        for (int r = 0; r < 4; r++) c += w[r] >= x ? n[r] : 0;
        return group_sum_i<64>(c);
    };
    if (longer(0) <= slot) return false;
    int lo = 0, hi = top + 1, over = 0;                 // longer(lo) > slot >= longer(hi) = over
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2, c = longer(mid);
        if (c > slot) lo = mid; else { hi = mid; over = c; }
    }
    int k = slot - over;                                // the k-th tile of the requests of lo
    b = -1;
#pragma unroll
    for (int r = 0; r < 4; r++) {
        if (b >= 0 || 64 * r >= a.B) break;
        const int upto = wave_scan_i(w[r] == lo ? n[r] : 0);
        const unsigned long long past = __ballot(upto > k);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            b = 64 * r + at;
            tile = __builtin_amdgcn_readlane(upto, at) - 1 - k;
            req = {__builtin_amdgcn_readlane(q[r].q0, at), __builtin_amdgcn_readlane(q[r].n, at), __builtin_amdgcn_readlane(q[r].kv, at)};
        }
        k -= __builtin_amdgcn_readlane(upto, 63);
    }
    return b >= 0;
}

// The ranges that a tile's blocks of keys make, equal ones: of `chunk` blocks at most where the host's bound on the
// keys holds, longer ones in as many ranges as there are where it does not.
__device__ __forceinline__ int att_ranges(const AttArgs &a, int blocks, int chunk) {
    return max(min((blocks + chunk - 1) / chunk, a.splits), 1);
}

// The table's entry for a key, -1 past the keys.  It is looked at (att_has) only where it is used: that waits for the
// load, and with it for every load before it.
__device__ __forceinline__ int att_page(const AttArgs &a, const int *table, const AttTile &t, int key) {
    int p = -1;
    if (key < t.kmax) p = table[qt_quot(key, a.div)];
    return p;
}
__device__ __forceinline__ bool att_has(const AttArgs &a, int page) { return (unsigned)page < (unsigned)a.n_pages; }
__device__ __forceinline__ long long att_slot(const AttArgs &a, int page, int key) {
    return page * a.ks_page + (key - qt_quot(key, a.div) * a.ps) * a.ks_slot;
}

// A key that does not exist takes the place of one in its block that does (`ok`, not 0 in any block that is worked on unless
// its pages are bad): places that nobody has written may hold NaN, which would send the tile to att_serial.
__device__ __forceinline__ long long att_instead(long long off, bool mine, unsigned long long ok) {
    const int from = ok ? __ffsll((unsigned long long)ok) - 1 : 0;
    const int lo = ok ? __builtin_amdgcn_readlane((int)off, from) : 0, hi = ok ? __builtin_amdgcn_readlane((int)(off >> 32), from) : 0;
    return mine ? off : (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
}

// Writes NT elements of a row's output, dim NT m.
template <typename QT, int NT> __device__ __forceinline__ void att_put(uint8_t *p, const float (&v)[NT]) {
    if constexpr (sizeof(typename QT::elem) == 4) {
        __builtin_memcpy(__builtin_assume_aligned(p, NT * 4 < 16 ? NT * 4 : 16), v, NT * 4);
    } else {
        typedef uint32_t uv __attribute__((ext_vector_type(NT / 2)));
        uv x;
#pragma unroll
        for (int t = 0; t < NT / 2; t++) x[t] = qt_round2<QT>(v[2 * t], v[2 * t + 1]);
        *reinterpret_cast<uv *>(p) = x;
    }
}

// One row over keys [k0, k1) in f32 without the matrix core; only what the row sees is read into its sums.  A wave: 64 keys
// at a time, a lane a key for the scores, dims lane + 64 e for the sums.  It ends where the row is NaN whatever follows.
template <typename QT, typename KT, int HD, bool PAGED>
__device__ __forceinline__ void att_serial(const AttArgs &a, AttTile t, const int *table, int head, int r, int k0, int k1, bool part, int split) {
    constexpr int EQ = sizeof(typename QT::elem), EK = sizeof(typename KT::elem), D = HD / 64;
    const int lane = threadIdx.x & 63, tok = qt_quot(r, a.gdiv), qh = head * a.G + r - tok * a.G, pos = t.shift + tok;
    const uint8_t *qp = a.q + ((size_t)((t.q0 + tok) * a.qs) + (size_t)qh * HD) * EQ;
    float o[D], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < D; e++) o[e] = 0.f;
    k0 = max(max(k0, a.window > 0 ? pos - a.window + 1 : 0), 0);
    k1 = min(k1, min(t.kmax, pos + 1));
    for (int j0 = k0; j0 < k1 && l == l; j0 += 64) {
        const int j = j0 + lane;
        bool see = j < k1;
        long long ko = 0, vo = 0;
        if (PAGED) {
            const int p = see ? att_page(a, table, t, j) : -1;
            see = att_has(a, p);
            if (see) ko = vo = att_slot(a, p, j) + head * a.ks_head;
        } else if (see) {
            ko = (long long)(t.q0 + j) * a.ks_slot + head * HD;
            vo = (long long)(t.q0 + j) * a.vs_slot + head * HD;
        }
        float s = -INFINITY;
        if (see) {
            s = 0.f;
            for (int d = 0; d < HD; d += 8) {
                float q[8], k[8];
                qt_load8<QT>(qp + d * EQ, q);
                qt_load8<KT>(a.k + (ko + d) * EK, k);
#pragma unroll
                for (int e = 0; e < 8; e++) s = fmaf(q[e], k[e], s);
            }
        }
        const float mn = fmaxf(m, group_max<64>(s)), mr = mn == -INFINITY ? 0.f : mn, f = qt_exp2((m - mr) * a.c);
        const float p = see ? qt_exp2((s - mr) * a.c) : 0.f;
        l = l * f + group_sum<64>(p);
#pragma unroll
        for (int e = 0; e < D; e++) o[e] *= f;
        const int lo = (int)vo, hi = (int)(vo >> 32);
        for (unsigned long long some = __ballot(see); some; some &= some - 1) {
            const int i = __ffsll(some) - 1;
            const float pi = lane_bcast(p, i);
            const long long v = ((long long)__builtin_amdgcn_readlane(hi, i) << 32) | (unsigned)__builtin_amdgcn_readlane(lo, i);
#pragma unroll
            for (int e = 0; e < D; e++) o[e] = fmaf(pi, qt_load1<KT>(a.v + (v + lane + 64 * e) * EK), o[e]);
        }
        m = mn;
    }
    const size_t at = (size_t)(t.q0 + tok) * (a.nkv * a.G) + qh;
    if (part) {
        const size_t row = (size_t)split * a.T * (a.nkv * a.G) + at;
#pragma unroll
        for (int e = 0; e < D; e++) a.po[row * HD + lane + 64 * e] = o[e];
        if (lane == 0) { a.pm[2 * row] = m; a.pm[2 * row + 1] = l; }
    } else {
        uint8_t *op = a.out + ((size_t)((t.q0 + tok) * a.os) + (size_t)qh * HD) * EQ;
#pragma unroll
        for (int e = 0; e < D; e++) qt_store1<QT>(op + (lane + 64 * e) * EQ, l == 0.f ? 0.f : o[e] / l);
    }
}

// Waits for the wave's stores: what it writes next to the same places comes after them.
__device__ __forceinline__ void att_stored() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

#define ATT_WV 4

// ---- f32 prompts ---------------------------------------------------------------------------------
// A workgroup takes 32 rows; its four waves take the 32-key blocks in turn, each with a softmax of its own, K and V
// going from memory into operand registers without LDS or barriers and split there; the waves' sums are merged through
// LDS at the end.  V is loaded when K is used up: both at once spill.  Bound by the splitting (VALU) next to the
// products: two prompts of 4000 positions 925 us, 142 TFLOP/s of f32 products (a library's f32 matrix product of 8192^3:
// 153); with V loaded ahead of the scores 1105, in 16-row tiles (k_att_one) 1377.
template <int HD>
__global__ __launch_bounds__(64 * ATT_WV) __attribute__((amdgpu_waves_per_eu(2))) void k_att_f32(AttArgs a) {
    constexpr int NT = HD / 32, NS = HD / 16;
    constexpr int OB = 32 * HD * 4;                     // one wave's sums
    __shared__ __align__(16) uint8_t sm[OB * ATT_WV];   // first the queries' planes [plane][32][HD] bf16
    __shared__ float sst[2][ATT_WV][32];
    static_assert(3 * 32 * HD * 2 <= OB * ATT_WV, "the queries' planes and the sums share the LDS");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lr = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.nkv, slot = blockIdx.x / a.nkv;
    const int b = att_find<32>(a, slot);
    const int tile = slot - att_first<32>(a, b);
    const AttTile t = att_tile<32, false>(a, att_req<false>(a, b), tile);
    if (tile < 0 || t.r0 >= t.rows) return;             // (offsets that fall give tiles before the first)
    const int r = min(t.r0 + lr, t.rows - 1), pos = qt_quot(r, a.gdiv);
    const int first = qt_quot(t.r0, a.gdiv), last = qt_quot(min(t.r0 + 31, t.rows - 1), a.gdiv);
    for (int u = tid; u < 32 * (HD / 8); u += 64 * ATT_WV) {
        const int row = u / (HD / 8), ch = u % (HD / 8), rr = min(t.r0 + row, t.rows - 1), tk = qt_quot(rr, a.gdiv);
        float v[8];
        qt_u32x4 pl[3];
        qt_load8<QtF32>(a.q + ((size_t)((t.q0 + tk) * a.qs) + (size_t)(head * a.G + rr - tk * a.G) * HD + 8 * ch) * 4, v);
        qt_planes8(v, pl);
#pragma unroll
        for (int p = 0; p < 3; p++)
            *reinterpret_cast<qt_u32x4 *>(sm + (p * 32 + row) * HD * 2 + 16 * (ch ^ (row & (HD / 8 - 1)))) = pl[p];
    }
    __syncthreads();
    const int kb0 = t.lo / 32, kb1 = t.hi > t.lo ? (t.hi + 31) / 32 : kb0;
    float m = -INFINITY, l = 0.f;                       // l: of this half's keys
    qt_f32x16 o[NT];
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.f;
    const uint8_t *kbase = a.k + (head * HD + 8 * h) * 4, *vbase = a.v + (head * HD + NT * lr) * 4;
    for (int kb = kb0 + wave; kb < kb1; kb += ATT_WV) {
        float kr[NS][8], vr[2][8][NT];
        const uint8_t *kp = kbase + (long long)(t.q0 + min(32 * kb + lr, t.kmax - 1)) * a.ks_slot * 4;
#pragma unroll
        for (int s = 0; s < NS; s++) qt_load8<QtF32>(kp + 64 * s, kr[s]);
        qt_f32x16 sc;
#pragma unroll
        for (int i = 0; i < 16; i++) sc[i] = 0.f;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            qt_u32x4 ka[3], qa[3];
            qt_planes8(kr[s], ka);
#pragma unroll
            for (int p = 0; p < 3; p++) qa[p] = qt_lds16(sm + (p * 32 + lr) * HD * 2 + 16 * ((2 * s + h) ^ (lr & (HD / 8 - 1))));
            sc = att_planes<QtBf16, 3, 3>(ka, qa, sc);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int vk = min(32 * kb + 16 * s + 8 * (j >> 2) + 4 * h + (j & 3), t.kmax - 1);
                __builtin_memcpy(vr[s][j], __builtin_assume_aligned(vbase + (long long)(t.q0 + vk) * a.vs_slot * 4, NT * 4), NT * 4);
            }
        // hidden keys; a block that every row sees whole needs no look
        if (32 * kb + 31 > first || (a.window > 0 && 32 * kb <= last - a.window)) {
            const int d = pos - 32 * kb - 4 * h, w = a.window > 0 ? d - a.window : -1000;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int j = 8 * (i >> 2) + (i & 3);
                sc[i] = j <= d && j > w ? sc[i] : -INFINITY;
            }
        }
        float bm = m;
#pragma unroll
        for (int i = 0; i < 16; i++) bm = fmaxf(bm, sc[i]);
        bm = fmaxf(bm, att_other_half(bm));
        const float mr = bm == -INFINITY ? 0.f : bm, f = qt_exp2((m - mr) * a.c);
        m = bm;
        float p[2][8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            // the difference first: the rounding of a large m c would not cancel between blocks
            p[i >> 3][i & 7] = qt_exp2((sc[i] - mr) * a.c);
            sum += p[i >> 3][i & 7];
        }
        l = l * f + sum;
#pragma unroll
        for (int d = 0; d < NT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] *= f;
#pragma unroll
        for (int s = 0; s < 2; s++) {
            qt_u32x4 pb[3];
            qt_planes8(p[s], pb);
#pragma unroll
            for (int d = 0; d < NT; d++) {
                float v[8];
                qt_u32x4 va[3];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = vr[s][j][d];
                qt_planes8(v, va);
                o[d] = att_planes<QtBf16, 3, 3>(va, pb, o[d]);
            }
        }
    }
    l += att_other_half(l);
    if (h == 0) { sst[0][wave][lr] = m; sst[1][wave][lr] = l; }
    __syncthreads();                                    // also: the queries' planes are read
    {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < ATT_WV; w++) M = fmaxf(M, sst[0][w][lr]);
        const float f = M == -INFINITY ? 0.f : qt_exp2((m - M) * a.c);
        float *os = reinterpret_cast<float *>(sm + wave * OB) + lr * HD;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int mm = 8 * (i >> 2) + 4 * h + (i & 3);
#pragma unroll
            for (int d = 0; d < NT; d++) os[NT * (mm ^ lr) + d] = o[d][i] * f;
        }
    }
    __syncthreads();
    bool bad = false;
    for (int u = tid; u < 32 * 32; u += 64 * ATT_WV) {
        const int row = u >> 5, mm = u & 31, rr = t.r0 + row;
        float M = -INFINITY, L = 0.f, v[NT];
#pragma unroll
        for (int w = 0; w < ATT_WV; w++) M = fmaxf(M, sst[0][w][row]);
#pragma unroll
        for (int d = 0; d < NT; d++) v[d] = 0.f;
        if (M != -INFINITY)
#pragma unroll
            for (int w = 0; w < ATT_WV; w++) L += sst[1][w][row] * qt_exp2((sst[0][w][row] - M) * a.c);
#pragma unroll
        for (int w = 0; w < ATT_WV; w++)
#pragma unroll
            for (int d = 0; d < NT; d++) v[d] += (reinterpret_cast<const float *>(sm + w * OB) + row * HD)[NT * (mm ^ row) + d];
        float chk = L;
#pragma unroll
        for (int d = 0; d < NT; d++) chk = fmaf(v[d], 0.f, chk);
        if (rr >= t.rows) continue;
        bad |= !(chk - chk == 0.f);
        const int rt = qt_quot(rr, a.gdiv);
        const float inv = L > 0.f ? 1.0f / L : 0.f;
#pragma unroll
        for (int d = 0; d < NT; d++) v[d] *= inv;
        att_put<QtF32, NT>(a.out + ((size_t)((t.q0 + rt) * a.os) + (size_t)(head * a.G + rr - rt * a.G) * HD + NT * mm) * 4, v);
    }
    att_stored();
    if (__syncthreads_or(bad))
        for (int row = wave; row < 32 && t.r0 + row < t.rows; row += ATT_WV)
            att_serial<QtF32, QtF32, HD, false>(a, t, nullptr, head, t.r0 + row, 32 * kb0, 32 * kb1, false, 0);
}

// ---- rows of one tile of 16 ------------------------------------------------------------------------
// The same with v_mfma_f32_16x16x32 for the rows of single tokens, and for calls whose 32-row tiles leave CUs without
// work: half the registers, so 12 waves a CU have their loads in flight.  Lane l supplies key row l % 16 of two
// 16-key tiles and query row l % 16, each as the 8 dims of group g = l / 16 of 32, and ends with query row l % 16 and keys
// 16 t + 4 g + i; the 8 probabilities of a lane are the operand of V's product in place, V's rows are loaded 8 keys by
// HD / 16 dims a lane, and dim (HD / 16) m + u is row m of product u.  The four waves take the blocks of 32 keys in
// turn, each with a softmax of its own and no barrier, and are merged through LDS; the ranges of keys by k_att_merge.
// Bound by the cache's bytes for many streams: 64 of 1000 to 8000 keys bf16 197 us, 6.0 TB/s of reads (32-row tiles 217); by
// the chain of dependent loads (lengths, table, keys) for few: 4 streams f32 11.5 us with the merge (15.6), three prompts
// of 21 to 128 f32 8.1 (15.9).
template <typename T> __device__ __forceinline__ qt_f32x4 att_mma16(qt_u32x4 a, qt_u32x4 b, qt_f32x4 c) { return qt_mfma_bf16(a, b, c); }
template <> __device__ __forceinline__ qt_f32x4 att_mma16<QtF16>(qt_u32x4 a, qt_u32x4 b, qt_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(qt_f16x8, a), __builtin_bit_cast(qt_f16x8, b), c, 0, 0, 0);
}
template <typename T, int NA, int NB>
__device__ __forceinline__ qt_f32x4 att_planes16(const qt_u32x4 (&a)[NA], const qt_u32x4 (&b)[NB], qt_f32x4 c) {
#pragma unroll
    for (int s = NA + NB - 2; s >= 0; s--)
#pragma unroll
        for (int i = 0; i < NA; i++)
            if (s - i >= 0 && s - i < NB && s <= 2) c = att_mma16<T>(a[i], b[s - i], c);
    return c;
}
// over the four groups of a query row's lanes
__device__ __forceinline__ float att_max4(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float t = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
    const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float att_sum4(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    const float t = __uint_as_float(p[0]) + __uint_as_float(p[1]);
    const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(t), __float_as_uint(t), false, false);
    return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}

// STREAM: for one workgroup, and not kept for others
template <typename V, bool STREAM> __device__ __forceinline__ V att_ld(const uint8_t *p) {
    if constexpr (STREAM) return __builtin_nontemporal_load(reinterpret_cast<const V *>(p));
    else return *reinterpret_cast<const V *>(p);
}

template <typename QT, typename KT, int HD, bool PAGED, bool STREAM>
__global__ __launch_bounds__(64 * ATT_WV) __attribute__((amdgpu_waves_per_eu(sizeof(typename KT::elem) == 4 ? 2 : 3))) void k_att_one(AttArgs a) {
    constexpr bool QF = sizeof(typename QT::elem) == 4, KF = sizeof(typename KT::elem) == 4;
    constexpr int EQ = sizeof(typename QT::elem), EK = sizeof(typename KT::elem);
    constexpr int NU = HD / 16, NS = HD / 32, NQ = QF ? 3 : 1, NK = KF ? 3 : 1;
    constexpr int OB = 16 * HD * 4;                     // one wave's sums
    __shared__ __align__(16) uint8_t sm[OB * ATT_WV];   // QF: first the queries' planes [plane][16][HD] bf16
    __shared__ float sst[2][ATT_WV][16];
    __shared__ __align__(16) long long voff[PAGED ? ATT_WV : 1][32];
    static_assert(3 * 16 * HD * 2 <= OB * ATT_WV, "the queries' planes and the sums share the LDS");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, li = lane & 15, g = lane >> 4;
    const int head = blockIdx.x % a.nkv, slot = blockIdx.x / a.nkv, split = blockIdx.y;
    const int b = a.tps > 0 ? slot / a.tps : att_find<16>(a, slot);
    int tile = a.tps > 0 ? slot % a.tps : slot - att_first<16>(a, b);
    const int *table = PAGED ? a.table + b * a.ts : nullptr;
    const AttReq req = att_req<PAGED>(a, b);
    for (;; tile += a.tps) {
    const AttTile t = att_tile<16, PAGED>(a, req, tile);
    if (tile < 0 || t.r0 >= t.rows) return;               // (offsets that fall give tiles before the first)
    const int r = min(t.r0 + li, t.rows - 1), tok = qt_quot(r, a.gdiv), qh = head * a.G + r - tok * a.G, pos = t.shift + tok;
    const int first = t.shift + qt_quot(t.r0, a.gdiv), last = t.shift + qt_quot(min(t.r0 + 15, t.rows - 1), a.gdiv);
    // the range's 32-key blocks
    const int blk0 = t.lo / 32, blk1 = t.hi > t.lo ? (t.hi + 31) / 32 : blk0;
    const int n = att_ranges(a, blk1 - blk0, a.chunk), size = (blk1 - blk0 + n - 1) / n;
    const bool part = n > 1;                            // else the first range has it all
    if (split > 0 && !part) { if (a.tps <= 0) return; continue; }
    const int kb0 = min(blk1, blk0 + split * size), kb1 = min(blk1, kb0 + size);
    // (looked up here, so that the entry and the queries come in together)
    int page = PAGED && kb0 + wave < kb1 ? att_page(a, table, t, 32 * (kb0 + wave) + (lane & 31)) : 0;
    // the queries' operands; step s: dims 32 s + 8 g ..
    qt_u32x4 qf[QF ? 1 : NS];
    if constexpr (QF) {
        for (int u = tid; u < 16 * (HD / 8); u += 64 * ATT_WV) {
            const int row = u / (HD / 8), ch = u % (HD / 8), rr = min(t.r0 + row, t.rows - 1), tk = qt_quot(rr, a.gdiv);
            float v[8];
            qt_u32x4 pl[3];
            qt_load8<QT>(a.q + ((size_t)((t.q0 + tk) * a.qs) + (size_t)(head * a.G + rr - tk * a.G) * HD + 8 * ch) * EQ, v);
            qt_planes8(v, pl);
#pragma unroll
            for (int p = 0; p < 3; p++)
                *reinterpret_cast<qt_u32x4 *>(sm + (p * 16 + row) * HD * 2 + 16 * (ch ^ (row & (HD / 8 - 1)))) = pl[p];
        }
        __syncthreads();
    } else {
        const uint8_t *qp = a.q + ((size_t)((t.q0 + tok) * a.qs) + (size_t)qh * HD + 8 * g) * EQ;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = *reinterpret_cast<const qt_u32x4 *>(qp + 32 * s * EQ);
    }
    float m = -INFINITY, l = 0.f;                       // l: of this group's keys
    const qt_f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    qt_f32x4 o[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) o[u] = zero;
    const uint8_t *kbase = a.k + (head * (PAGED ? a.ks_head : (long long)HD) + 8 * g) * EK;
    const uint8_t *vbase = a.v + (head * (PAGED ? a.ks_head : (long long)HD) + NU * li) * EK;
    for (int kb = kb0 + wave; kb < kb1; kb += ATT_WV) {
        const int key = 32 * kb + (lane & 31);
        qt_u32x4 kr[2][NS][KF ? 2 : 1];
        uint32_t vr[8][NU * EK / 4];
        uint32_t ok;                                    // keys of the block that exist
        long long koff[2];
        if constexpr (PAGED) {
            const bool has = att_has(a, page);
            ok = (uint32_t)__ballot(has);
            const long long off = att_instead(att_slot(a, page, key), has, ok);
            __builtin_amdgcn_wave_barrier();
            if (lane < 32) voff[wave][lane] = off;
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int u = 0; u < 2; u++) koff[u] = voff[wave][16 * u + li];
            page = kb + ATT_WV < kb1 ? att_page(a, table, t, key + 32 * ATT_WV) : 0;
        } else {
            ok = (uint32_t)__ballot(key < t.kmax);
#pragma unroll
            for (int u = 0; u < 2; u++) koff[u] = (long long)(t.q0 + min(32 * kb + 16 * u + li, t.kmax - 1)) * a.ks_slot;
        }
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int s = 0; s < NS; s++)
#pragma unroll
                for (int e = 0; e < (KF ? 2 : 1); e++)
                    kr[u][s][e] = att_ld<qt_u32x4, STREAM>(kbase + (koff[u] + 32 * s) * EK + 16 * e);
        const auto values = [&] {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int vk = 16 * (j >> 2) + 4 * g + (j & 3);
                const long long vo = PAGED ? voff[wave][vk] : (long long)(t.q0 + min(32 * kb + vk, t.kmax - 1)) * a.vs_slot;
                typedef uint32_t part __attribute__((ext_vector_type(NU * EK < 16 ? NU * EK / 4 : 4)));
#pragma unroll
                for (int e = 0; e < (NU * EK + 15) / 16; e++) {
                    const part x = att_ld<part, STREAM>(vbase + vo * EK + 16 * e);
                    __builtin_memcpy(&vr[j][4 * e], &x, sizeof x);
                }
            }
        };
        if constexpr (!KF) values();
        qt_f32x4 sc[2];
#pragma unroll
        for (int u = 0; u < 2; u++) {
            sc[u] = zero;
#pragma unroll
            for (int s = 0; s < NS; s++) {
                qt_u32x4 ka[NK], qa[NQ];
                if constexpr (KF) {
                    float v[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = __uint_as_float(kr[u][s][e >> 2][e & 3]);
                    qt_planes8(v, ka);
                } else {
                    ka[0] = kr[u][s][0];
                }
#pragma unroll
                for (int p = 0; p < NQ; p++)
                    if constexpr (QF) qa[p] = qt_lds16(sm + (p * 16 + li) * HD * 2 + 16 * ((4 * s + g) ^ (li & (HD / 8 - 1))));
                    else qa[p] = qf[s];
                sc[u] = att_planes16<KT, NK, NQ>(ka, qa, sc[u]);
            }
        }
        if constexpr (KF) {                             // f32 keys leave no room for the values earlier
            __builtin_amdgcn_sched_barrier(0);
            values();
        }
        if (!(ok == 0xFFFFFFFFu && 32 * kb + 31 <= first && (a.window <= 0 || 32 * kb > last - a.window))) {
            const int d = pos - 32 * kb - 4 * g, w = a.window > 0 ? d - a.window : -1000;
            const uint32_t mine = ok >> (4 * g);
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int j = 16 * u + i;
                    sc[u][i] = j <= d && j > w && (mine >> j & 1u) ? sc[u][i] : -INFINITY;
                }
        }
        float bm = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])), fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
        bm = fmaxf(m, att_max4(bm));
        const float mr = bm == -INFINITY ? 0.f : bm, mc = mr * a.c, f = qt_exp2((m - mr) * a.c);
        m = bm;
        float p[8], sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            // f32: the difference first, since the rounding of a large m c would not cancel between blocks
            p[j] = QF ? qt_exp2((sc[j >> 2][j & 3] - mr) * a.c) : qt_exp2(fmaf(sc[j >> 2][j & 3], a.c, -mc));
            if (QF) sum += p[j];
        }
        qt_u32x4 pb[NQ];
        if constexpr (QF) {
            qt_planes8(p, pb);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                pb[0][j] = qt_round2<QT>(p[2 * j], p[2 * j + 1]);
                sum = att_add2<QT>(pb[0][j], sum);
            }
        }
        l = l * f + sum;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            qt_u32x4 va[NK];
            if constexpr (KF) {
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] = __uint_as_float(vr[j][u]);
                qt_planes8(v, va);
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    va[0][j] = __builtin_amdgcn_perm(vr[2 * j + 1][u >> 1], vr[2 * j][u >> 1], u & 1 ? 0x07060302u : 0x05040100u);
            }
            o[u] = att_planes16<KT, NK, NQ>(va, pb, o[u] * f);
        }
    }
    l = att_sum4(l);
    if (g == 0) { sst[0][wave][li] = m; sst[1][wave][li] = l; }
    __syncthreads();                                    // also: the queries' planes are read
    {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < ATT_WV; w++) M = fmaxf(M, sst[0][w][li]);
        const float f = M == -INFINITY ? 0.f : qt_exp2((m - M) * a.c);
        float *os = reinterpret_cast<float *>(sm + wave * OB) + li * HD;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int u = 0; u < NU; u++) os[NU * ((4 * g + i) ^ li) + u] = o[u][i] * f;
    }
    __syncthreads();
    bool bad = false;
    {
        const int row = tid >> 4, mm = tid & 15, rr = t.r0 + row;
        float M = -INFINITY, L = 0.f, v[NU];
#pragma unroll
        for (int w = 0; w < ATT_WV; w++) M = fmaxf(M, sst[0][w][row]);
#pragma unroll
        for (int u = 0; u < NU; u++) v[u] = 0.f;
        if (M != -INFINITY)
#pragma unroll
            for (int w = 0; w < ATT_WV; w++) L += sst[1][w][row] * qt_exp2((sst[0][w][row] - M) * a.c);
#pragma unroll
        for (int w = 0; w < ATT_WV; w++)
#pragma unroll
            for (int u = 0; u < NU; u++) v[u] += (reinterpret_cast<const float *>(sm + w * OB) + row * HD)[NU * (mm ^ row) + u];
        float chk = L;
#pragma unroll
        for (int u = 0; u < NU; u++) chk = fmaf(v[u], 0.f, chk);
        if (rr < t.rows) {
            bad = !(chk - chk == 0.f) || (!QF && L == 0.f && M > -INFINITY);
            const int rt = qt_quot(rr, a.gdiv);
            const size_t tk = t.q0 + rt, hd = head * a.G + rr - rt * a.G;
            if (part) {
                const size_t prow = ((size_t)split * a.T + tk) * (a.nkv * a.G) + hd;
                if (kb0 < kb1) att_put<QtF32, NU>(reinterpret_cast<uint8_t *>(a.po + prow * HD + NU * mm), v);
                if (mm == 0) { a.pm[2 * prow] = M; a.pm[2 * prow + 1] = L; }
            } else {
                const float inv = L > 0.f ? 1.0f / L : 0.f;
                if (a.splits > 1 && mm == 0) a.pm[2 * (tk * (a.nkv * a.G) + hd) + 1] = -1.0f;
#pragma unroll
                for (int u = 0; u < NU; u++) v[u] *= inv;
                att_put<QT, NU>(a.out + (tk * a.os + hd * HD + NU * mm) * EQ, v);
            }
        }
    }
    att_stored();
    if (__syncthreads_or(bad))
        for (int row = wave; row < 16 && t.r0 + row < t.rows; row += ATT_WV)
            att_serial<QT, KT, HD, PAGED>(a, t, table, head, t.r0 + row, 32 * kb0, 32 * kb1, part, split);
    if (a.tps <= 0) return;
    __syncthreads();                                    // the next tile's planes take the LDS
    }
}

// ---- many rows -----------------------------------------------------------------------------------
// A workgroup takes 128 rows, 32 a wave, and goes through its keys 64 at a time: K and V of a block are copied from
// memory straight into LDS (no registers), two blocks deep, one barrier a block, and every wave reads both
// operands from there.  16-bit types only.  Block kb + 1's scores do not wait for block kb's softmax: K is a block ahead of
// V.  Bound by the matrix core's and the vector unit's shares together (50 and 48 % of the cycles of two prompts of 5003 and
// 8191 f16: 407 to 428 us, 881 TFLOP/s and more at the 1.7 GHz that the load leaves; LDS 25 %, no bank conflicts; 32-row tiles
// straight from memory 1031 us), by the first loads of each workgroup for short prompts (16 of 40 to 1500 bf16: 86 us, 211).
//   K, row k: 16-byte chunk c at place c ^ swk(k): the 16 lanes of a phase of a wave's read (16 rows, one chunk)
//   fall on 16 different groups of banks.  V: chunk c at place c ^ swv(k): a transposing read takes 4 rows by 64 bytes
//   a half-wave, which fall on different banks.
template <int HD> __device__ __forceinline__ int att_swk(int row) { return HD == 128 ? row & 15 : (row >> 1) & 7; }
template <int HD> __device__ __forceinline__ int att_swv(int row) { return HD == 128 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }

// 16 bytes a lane from memory to LDS at dst + 16 lane (dst uniform), as assembly: the compiler, which would take
// every later LDS read for a reader of these bytes, does not wait for them; att_wait does.  The second form reads at
// base + off, base uniform.
__device__ __forceinline__ unsigned att_lds(void *dst) { return (unsigned)(uintptr_t)(__attribute__((address_space(3))) void *)dst; }
__device__ __forceinline__ void att_copy16(const uint8_t *src, unsigned dst) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
}
__device__ __forceinline__ void att_copy16(const uint8_t *base, unsigned off, unsigned dst) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
}
__device__ __forceinline__ void att_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

template <typename T, int HD, bool PAGED>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2))) void k_att_tile(AttArgs a) {
    constexpr int NT = HD / 32, NS = HD / 16, RB = 2 * HD, CPR = RB / 16, RPC = 64 / CPR, NC = 64 / RPC / 4;
    __shared__ __align__(16) uint8_t sk[2 * 64 * RB], sv[3 * 64 * RB];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lr = lane & 31, h = lane >> 5;
    const int head = blockIdx.x % a.nkv, slot = blockIdx.x / a.nkv, split = blockIdx.y;
    int b, tile;
    AttReq req;
    if (a.B <= ATT_SORT_B) {
        if (!att_longest<PAGED>(a, slot, b, tile, req)) return;
    } else {
        b = att_find<128>(a, slot);
        tile = slot - att_first<128>(a, b);
        req = att_req<PAGED>(a, b);
    }
    b = __builtin_amdgcn_readfirstlane(b);
    tile = __builtin_amdgcn_readfirstlane(tile);
    req = {__builtin_amdgcn_readfirstlane(req.q0), __builtin_amdgcn_readfirstlane(req.n), __builtin_amdgcn_readfirstlane(req.kv)};
    const int *table = PAGED ? a.table + b * a.ts : nullptr;
    // where this lane reads a block's operands: K row lr, V rows 4 h + (lane % 16) / 4
    int ka[NS], va[NT];
#pragma unroll
    for (int s = 0; s < NS; s++) ka[s] = lr * RB + 16 * ((2 * s + h) ^ att_swk<HD>(lr));
    {
        const int i = lane & 15, row = 4 * h + (i >> 2);
#pragma unroll
        for (int d = 0; d < NT; d++)
            va[d] = row * RB + 16 * ((4 * d + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ att_swv<HD>(row)) + 8 * (i & 1);
    }
    // where this lane's copies read: row crow + i RPC of a block, and the chunk that belongs at its place
    const int crow = wave * NC * RPC + lane / CPR, cc = lane % CPR;
    const AttTile t = att_tile<128, PAGED>(a, req, tile);
    if (tile < 0 || t.r0 >= t.rows) return;               // (offsets that fall give tiles before the first)
    const int w0 = t.r0 + 32 * wave, r = min(w0 + lr, t.rows - 1), tok = qt_quot(r, a.gdiv), qh = head * a.G + r - tok * a.G, pos = t.shift + tok;
    // the wave's first and last position
    const int first = t.shift + qt_quot(min(w0, t.rows - 1), a.gdiv), last = t.shift + qt_quot(min(w0 + 31, t.rows - 1), a.gdiv);
    qt_u32x4 qf[NS];
    {
        const uint8_t *qp = a.q + ((size_t)((t.q0 + tok) * a.qs) + (size_t)qh * HD + 8 * h) * 2;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = *reinterpret_cast<const qt_u32x4 *>(qp + 32 * s);
    }
    // the range's 64-key blocks; chunk is in blocks of 32, even
    const int blk0 = t.lo / 64, blk1 = t.hi > t.lo ? (t.hi + 63) / 64 : blk0;
    const int n = att_ranges(a, blk1 - blk0, a.chunk / 2), size = (blk1 - blk0 + n - 1) / n;
    const bool part = n > 1;                            // else the first range has it all
    if (split > 0 && !part) return;
    const int kb0 = min(blk1, blk0 + split * size), kb1 = min(blk1, kb0 + size);
    float m = -INFINITY, l = 0.f;                       // m: the maximum so far, or up to 2^8 under it; l: of this half's keys
    qt_f32x16 o[NT];
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.f;
    const uint8_t *kbase = a.k + (head * (PAGED ? a.ks_head : (long long)HD) + (PAGED ? 0 : t.q0 * a.ks_slot)) * 2;
    const uint8_t *vbase = a.v + (head * (PAGED ? a.ks_head : (long long)HD) + (PAGED ? 0 : t.q0 * a.vs_slot)) * 2;
    int page = -1;                                                       // PAGED: of key 64 kb + lane, block kb the next to copy
    unsigned long long okv = ~0ull, okk = ~0ull, okn = ~0ull;            // keys that exist: of the block of V, of K, of the next K
    // block kb to a K and a V buffer
    const unsigned lk = att_lds(sk), lv = att_lds(sv);
    const auto copy = [&](int kb, unsigned kdst, unsigned vdst) {
        if constexpr (PAGED) {
            const bool has = att_has(a, page);
            okn = __ballot(has);
            const int key = 64 * kb + lane, from = okn ? __ffsll(okn) - 1 : 0;
            if (a.near) {
                const int c = qt_quot(key, a.div);
                unsigned off = 2u * ((unsigned)page * (unsigned)a.ks_page + (unsigned)(key - c * a.ps) * (unsigned)a.ks_slot);
                const unsigned other = okn ? (unsigned)__builtin_amdgcn_readlane((int)off, from) : 0u;
                off = has ? off : other;
#pragma unroll
                for (int i = 0; i < NC; i++) {
                    const int row = crow + i * RPC, to = (wave * NC + i) * RPC * RB;
                    const unsigned at = (unsigned)__shfl((int)off, row);
                    att_copy16(kbase, at + 16 * (cc ^ att_swk<HD>(row)), kdst + to);
                    att_copy16(vbase, at + 16 * (cc ^ att_swv<HD>(row)), vdst + to);
                }
            } else {
                int place = cc;
                asm volatile("" : "+v"(place));          // addresses are formed here: held over the loop they cost 20 registers
                const long long off = 2 * att_instead(att_slot(a, page, key), has, okn);
#pragma unroll
                for (int i = 0; i < NC; i++) {
                    const int row = crow + i * RPC, to = (wave * NC + i) * RPC * RB;
                    const long long at = ((long long)__shfl((int)(off >> 32), row) << 32) | (unsigned)__shfl((int)off, row);
                    att_copy16(kbase + at + 16 * (place ^ att_swk<HD>(row)), kdst + to);
                    att_copy16(vbase + at + 16 * (place ^ att_swv<HD>(row)), vdst + to);
                }
            }
            page = kb + 1 < kb1 ? att_page(a, table, t, 64 * (kb + 1) + lane) : -1;
        } else {
#pragma unroll
            for (int i = 0; i < NC; i++) {
                const int row = crow + i * RPC, to = (wave * NC + i) * RPC * RB;
                const int real = min(row, t.kmax - 1 - 64 * kb);         // rows past the sequence: its last one again
                att_copy16(kbase + 64ll * kb * a.ks_slot * 2, (unsigned)(real * (int)a.ks_slot * 2 + 16 * (cc ^ att_swk<HD>(row))), kdst + to);
                att_copy16(vbase + 64ll * kb * a.vs_slot * 2, (unsigned)(real * (int)a.vs_slot * 2 + 16 * (cc ^ att_swv<HD>(row))), vdst + to);
            }
        }
    };
    const auto scores = [&](qt_f32x16 (&sc)[2], const uint8_t *kbuf) {
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[kt][i] = 0.f;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int kt = 0; kt < 2; kt++) sc[kt] = att_mma<T>(qt_lds16(kbuf + 32 * kt * RB + ka[s]), qf[s], sc[kt]);
    };
    // block kb: its scores are in sc, K of block kb + 1 is in the other K buffer than kb's was, V in buffer vb
    int vb = 0;
    const auto step = [&](int kb, qt_f32x16 (&sc)[2], qt_f32x16 (&sn)[2], auto bufc) {
        constexpr int BUF = decltype(bufc)::value;
        // K of the next block is in, V of this one since the last step (the wave's own copies by the wait, the others' by
        // the barrier, which they pass after theirs), and every wave has left the buffers that block kb + 2 takes
        att_wait();
        __syncthreads();
        okv = okk;
        okk = okn;
        const uint8_t *vbuf = sv + vb * 64 * RB;
        vb = vb == 2 ? 0 : vb + 1;
        if (kb + 2 < kb1) copy(kb + 2, lk + BUF * 64 * RB, lv + (vb == 2 ? 0 : vb + 1) * 64 * RB);
        if (64 * kb + 63 > first || (a.window > 0 && 64 * kb <= last - a.window)) {
            const int d = pos - 64 * kb - 4 * h, w = a.window > 0 ? d - a.window : -1000;
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int j = 32 * kt + 8 * (i >> 2) + (i & 3);
                    sc[kt][i] = j <= d && j > w ? sc[kt][i] : -INFINITY;
                }
        }
        if (PAGED && okv != ~0ull) {                                     // the end of the keys, or a bad page
#pragma unroll
            for (int kt = 0; kt < 2; kt++) {
                const uint32_t w = (uint32_t)(okv >> (32 * kt)) >> (4 * h);
#pragma unroll
                for (int i = 0; i < 16; i++) sc[kt][i] = w >> (8 * (i >> 2) + (i & 3)) & 1u ? sc[kt][i] : -INFINITY;
            }
        }
        float bm = sc[0][0];
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) bm = fmaxf(bm, sc[kt][i]);
        bm = fmaxf(bm, att_other_half(bm));
        // probabilities up to 2^8 are as good as up to 1: the sums shrink only when a row's maximum has risen by more
        if (__ballot((bm - m) * a.c > 8.0f || (m == -INFINITY && bm > m))) {
            const float mn = fmaxf(m, bm), f = mn == -INFINITY ? 0.f : qt_exp2((m - mn) * a.c);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < NT; d++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[d][i] *= f;
        }
        const float mc = m == -INFINITY ? 0.f : m * a.c;
        if (kb + 1 < kb1) scores(sn, sk + (BUF ^ 1) * 64 * RB);
#pragma unroll
        for (int kt = 0; kt < 2; kt++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[kt][i] = qt_exp2(fmaf(sc[kt][i], a.c, -mc));
#pragma unroll
        for (int s = 0; s < 4; s++) {
            qt_u32x4 pb;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                pb[j] = qt_round2<T>(sc[s >> 1][8 * (s & 1) + 2 * j], sc[s >> 1][8 * (s & 1) + 2 * j + 1]);
                sum = att_add2<T>(pb[j], sum);
            }
            l += sum;
#pragma unroll
            for (int d = 0; d < NT; d++) {
                const uint16_t *vp = reinterpret_cast<const uint16_t *>(vbuf + 16 * s * RB + va[d]);
                o[d] = att_mma<T>(qt_lds_tr8x2(vp, vp + 8 * HD), pb, o[d]);
            }
        }
    };
    if (kb0 < kb1) {
        if (PAGED) page = att_page(a, table, t, 64 * kb0 + lane);
        copy(kb0, lk, lv);
        okk = okn;
        if (kb0 + 1 < kb1) copy(kb0 + 1, lk + 64 * RB, lv + 64 * RB);
        att_wait();
        __syncthreads();
        qt_f32x16 s0[2], s1[2];
        scores(s0, sk);
        for (int kb = kb0; kb < kb1; kb += 2) {
            step(kb, s0, s1, std::integral_constant<int, 0>{});
            if (kb + 1 < kb1) step(kb + 1, s1, s0, std::integral_constant<int, 1>{});
        }
    }
    // the rows' results; o[d][i] is dim 32 d + 8 (i / 4) + 4 h + i % 4
    l += att_other_half(l);
    float chk = l;
#pragma unroll
    for (int d = 0; d < NT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) chk = fmaf(o[d][i], 0.f, chk);
    const bool live = w0 + lr < t.rows;
    const size_t tk = t.q0 + tok;
    if (live) {
        if (part) {
            const size_t prow = ((size_t)split * a.T + tk) * (a.nkv * a.G) + qh;
            if (kb0 < kb1)
#pragma unroll
            for (int d = 0; d < NT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<float4 *>(a.po + prow * HD + 32 * d + 8 * i + 4 * h) =
                        make_float4(o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]);
            if (h == 0) { a.pm[2 * prow] = m; a.pm[2 * prow + 1] = l; }
        } else {
            const float inv = l > 0.f ? 1.0f / l : 0.f;
            if (a.splits > 1 && h == 0) a.pm[2 * (tk * (a.nkv * a.G) + qh) + 1] = -1.0f;
            uint8_t *op = a.out + (tk * a.os + (size_t)qh * HD + 4 * h) * 2;
#pragma unroll
            for (int d = 0; d < NT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    *reinterpret_cast<uint2 *>(op + 2 * (32 * d + 8 * i)) =
                        make_uint2(qt_round2<T>(o[d][4 * i] * inv, o[d][4 * i + 1] * inv), qt_round2<T>(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv));
        }
    }
    if (__ballot(live && (!(chk - chk == 0.f) || (l == 0.f && m > -INFINITY)))) {
        att_stored();
        for (int row = w0; row < min(w0 + 32, t.rows); row++)
            att_serial<T, T, HD, PAGED>(a, t, table, head, row, 64 * kb0, 64 * kb1, part, split);
    }
}

// A row's ranges under their common maximum: a wave a row, 4 rows a workgroup.  splits <= 64.  A range without keys (its
// sum 0) has written no sums.  Bound by the sums' bytes (3370 tokens of 16 heads, two ranges: 12 us), for few rows by
// three dependent loads (4 rows of 16 heads, 6 ranges: 3.5).
template <typename QT, int HD>
__global__ __launch_bounds__(256) void k_att_merge(AttArgs a) {
    constexpr int D = HD / 64, EQ = sizeof(typename QT::elem);
    const int nh = a.nkv * a.G, lane = threadIdx.x & 63;
    const long long at = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (long long)a.T * nh;
    if (at >= rows) return;
    const int tok = (int)(at / nh), hd = (int)(at % nh);
    float m = -INFINITY, l = 0.f;
    if (lane < a.splits) {
        m = a.pm[2 * (lane * rows + at)];
        l = a.pm[2 * (lane * rows + at) + 1];
    }
    if (tok < att_cu(a, 0) || tok >= att_cu(a, a.B)) return;      // rows of no request stay
    if (lane_bcast(l, 0) < 0.f) return;                           // the first range had all its keys and wrote it
    const float M = group_max<64>(m), f = l == 0.f ? 0.f : qt_exp2((m - M) * a.c);
    const float L = group_sum<64>(l * f);
    float o[D];
#pragma unroll
    for (int e = 0; e < D; e++) o[e] = 0.f;
    for (unsigned long long some = __ballot(l != 0.f); some;) {   // four ranges' loads at a time
        float v[4][D], fs[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int s = some ? __ffsll(some) - 1 : 0;
            fs[k] = some ? lane_bcast(f, s) : 0.f;
#pragma unroll
            for (int e = 0; e < D; e++) v[k][e] = some ? a.po[(s * rows + at) * HD + D * lane + e] : 0.f;
            some &= some - 1;
        }
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int e = 0; e < D; e++) o[e] = fmaf(fs[k], v[k][e], o[e]);
    }
    const float inv = L == 0.f ? 0.f : 1.0f / L;
#pragma unroll
    for (int e = 0; e < D; e++) qt_store1<QT>(a.out + ((size_t)tok * a.os + (size_t)hd * HD + D * lane + e) * EQ, o[e] * inv);
}

// ---- host side -------------------------------------------------------------------------------------

// The kernel, its launch slots and key ranges.  Launch slots: by request (max_q as far as known) or by rows, whichever is
// fewer.  Key ranges: enough workgroups to fill the CUs, 256 keys each at least.
enum AttKind { ATT_ONE, ATT_F32, ATT_TILE };
struct AttPlan { AttKind kind; long long slots; bool stream; };
static AttPlan att_plan(AttArgs &a, int dtype, bool paged, int max_q, int max_kv) {
    AttPlan p = {ATT_ONE, 0, false};
    a.gdiv = qt_div_of(a.G);
    a.tps = 0;
    const long long rows = (long long)a.T * a.G;
    if (dtype == QWEN_HIP_DT_F32) {
        // 32-row tiles for prompts while they give every CU work (one of 512 positions 23.7 us against 25.4 in 16-row tiles,
        // 16 of 64 16.6 against 20.4; three of 21 to 128 11.9 against 8.9)
        if (!paged && (rows / 32 + a.B) * a.nkv >= 256) p.kind = ATT_F32;
    } else if (rows >= 32ll * a.B && (paged || (rows / 128 + a.B) * a.nkv >= 96)) {
        // 128-row tiles from 32 rows a request on (64 requests of 32 tokens 42 us against 79 in 16-row tiles, 8 of 16 over
        // 3000 keys 27.3 against 27.8, 32 of 4 70 against 60); prompts, whose keys are not split, while there are tiles
        // enough (8 of 100 to 300 13.1 us against 20.3; one of 512 15.9 against 13.0, three of 21 to 128 9.2 against 8.4).
        // Those are equal requests.  The rule goes by a call's mean, so a step of single tokens and a chunk takes one kernel
        // for both (bf16, 16 over 8 heads, a chunk over 2000 keys: 64 streams of 1000 to 8000 keys and 512 tokens in 16-row tiles
        // 259 us, 198 and 33 in a call each; 32 of them and 1024 tokens in 128-row tiles 160, 110 and 49)
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
    // 171 us, 1 226, 3 190, 4 205).
    const long long wgs = p.slots * a.nkv, blocks = ((long long)max_kv + 31) / 32;
    long long n = wgs > 0 && paged ? ((p.kind == ATT_TILE ? 512 : 4096) + wgs - 1) / wgs : 1;
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

static int paged_args(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p, AttArgs &a, AttPlan &plan) {
    if (qt_check_pages("page_attention", kv)) return -1;
    QT_REFUSE(!p, "page_attention: null descriptor");
    if (check_rows("page_attention", p->dtype, p->n_heads, kv->n_kv_heads, kv->head_dim, p->B, p->T, p->window, p->scale)) return -1;
    QT_REFUSE(p->dtype == QWEN_HIP_DT_F32 ? kv->dtype != QWEN_HIP_DT_BF16 : p->dtype != kv->dtype,
              "page_attention: rows of dtype %d over a cache of dtype %d (f32 over bf16, else the cache's own)", p->dtype, kv->dtype);
    QT_REFUSE(p->max_q < 0 || p->max_kv < 0, "page_attention: max_q %d, max_kv %d", p->max_q, p->max_kv);
    QT_REFUSE(p->table_cols < 1 || (long long)p->table_cols * kv->page_size > ATT_MAX_KEYS || p->table_stride < p->table_cols,
              "page_attention: table_cols %d of stride %lld (at least 1, 2^30 positions at most)", p->table_cols, p->table_stride);
    a = AttArgs{};
    a.B = p->B; a.T = p->T; a.nkv = kv->n_kv_heads; a.G = p->n_heads / kv->n_kv_heads;
    plan = att_plan(a, p->dtype, true, p->max_q < p->T ? p->max_q : p->T, p->max_kv);
    plan.stream = plan.stream && 4ll * p->B * p->max_kv * kv->n_kv_heads * kv->head_dim > 256ll << 20;
    return 0;
}

extern "C" long long qwen_hip_op_page_attention_workspace(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p) {
    AttArgs a;
    AttPlan plan;
    if (paged_args(kv, p, a, plan)) return -1;
    return a.splits > 1 ? (long long)a.splits * a.T * p->n_heads * (kv->head_dim + 2) * 4 : 0;
}

template <typename QT, typename KT, int HD, bool PAGED>
static hipError_t att_launch(const AttArgs &a, const AttPlan &plan, hipStream_t st) {
    const dim3 grid((unsigned)(plan.slots * a.nkv), a.splits);
    hipError_t e;
    if (plan.kind == ATT_ONE && PAGED && plan.stream) e = qt_launch(k_att_one<QT, KT, HD, PAGED, PAGED>, grid, dim3(64 * ATT_WV), 0, st, a);
    else if (plan.kind == ATT_ONE) e = qt_launch(k_att_one<QT, KT, HD, PAGED, false>, grid, dim3(64 * ATT_WV), 0, st, a);
    else if constexpr (sizeof(typename QT::elem) == 2) e = qt_launch(k_att_tile<QT, HD, PAGED>, grid, dim3(256), 0, st, a);
    else e = qt_launch(k_att_f32<HD>, grid, dim3(64 * ATT_WV), 0, st, a);
    if (e == hipSuccess && a.splits > 1) {
        const long long rows = (long long)a.T * a.nkv * a.G;
        e = qt_launch(k_att_merge<QT, HD>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
    }
    return e;
}

extern "C" int qwen_hip_op_page_attention(const qwen_hip_kv_pages_t *kv, const qwen_hip_page_attn_t *p, void *stream) {
    AttArgs a;
    AttPlan plan;
    if (paged_args(kv, p, a, plan)) return -1;
    if (p->B == 0 || p->T == 0) return 0;
    QT_REFUSE(!p->q || !p->out || !p->cu_q || !p->kv_len || !p->table, "page_attention: null pointer");
    QT_REFUSE(p->out == p->q, "page_attention: out must not be q");
    const int A = 16 / qt_dt_size(p->dtype);
    QT_REFUSE(qt_off16(p->q) || qt_off16(p->out) || qt_off16(p->workspace), "page_attention: pointers have to be aligned to 16 bytes");
    QT_REFUSE(p->q_stride % A || p->q_stride < 0 || p->out_stride % A || p->out_stride < (long long)p->n_heads * kv->head_dim,
              "page_attention: strides %lld, %lld (multiples of 16 bytes, out's at least a token's)", p->q_stride, p->out_stride);
    const long long need = a.splits > 1 ? (long long)a.splits * a.T * p->n_heads * (kv->head_dim + 2) * 4 : 0;
    QT_REFUSE(need > 0 && (!p->workspace || p->workspace_bytes < need), "page_attention: a workspace of %lld bytes is needed, %lld given",
              need, p->workspace ? p->workspace_bytes : 0ll);
    QT_REFUSE(plan.slots * a.nkv > 0xFFFFFFll, "page_attention: too many tiles for one launch");
    const long long E = qt_dt_size(p->dtype), row = (long long)p->n_heads * kv->head_dim * E;
    QT_REFUSE(qt_rows_meet(p->out, p->out_stride * E, row, p->q, p->q_stride * E, row, p->T), "page_attention: out overlaps q");
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "page_attention: the stream's device: %s", hipGetErrorString(on.err));
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
    hipError_t e;
    if (p->dtype == QWEN_HIP_DT_F32)
        e = kv->head_dim == 128 ? att_launch<QtF32, QtBf16, 128, true>(a, plan, st) : att_launch<QtF32, QtBf16, 64, true>(a, plan, st);
    else if (p->dtype == QWEN_HIP_DT_BF16)
        e = kv->head_dim == 128 ? att_launch<QtBf16, QtBf16, 128, true>(a, plan, st) : att_launch<QtBf16, QtBf16, 64, true>(a, plan, st);
    else
        e = kv->head_dim == 128 ? att_launch<QtF16, QtF16, 128, true>(a, plan, st) : att_launch<QtF16, QtF16, 64, true>(a, plan, st);
    QT_REFUSE(e != hipSuccess, "page_attention: launch failed: %s", hipGetErrorString(e));
    return 0;
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
    const AttPlan plan = att_plan(a, p->dtype, false, 0, 0);
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
    hipError_t e;
    if (p->dtype == QWEN_HIP_DT_F32)
        e = p->head_dim == 128 ? att_launch<QtF32, QtF32, 128, false>(a, plan, st) : att_launch<QtF32, QtF32, 64, false>(a, plan, st);
    else if (p->dtype == QWEN_HIP_DT_BF16)
        e = p->head_dim == 128 ? att_launch<QtBf16, QtBf16, 128, false>(a, plan, st) : att_launch<QtBf16, QtBf16, 64, false>(a, plan, st);
    else
        e = p->head_dim == 128 ? att_launch<QtF16, QtF16, 128, false>(a, plan, st) : att_launch<QtF16, QtF16, 64, false>(a, plan, st);
    QT_REFUSE(e != hipSuccess, "packed_attention: launch failed: %s", hipGetErrorString(e));
    return 0;
}
