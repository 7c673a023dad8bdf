// qt_tree.hip — trees of drafted tokens: a step's positions and masks (qwen_hip_op_tree_plan), verification against the
// target's probabilities (qwen_hip_op_tree_verify), and what is kept of the step (qwen_hip_op_tree_commit).
#include "qt_ops.h"
#include <type_traits>

#define TREE_MAX_LEN (1 << 30)

// A request's tokens: offsets are the caller's, one out of range is brought into it.
struct TreeReq { int q0, n; };
__device__ __forceinline__ TreeReq tree_req(const int *cu, int b, int T) {
    const int q0 = min(max(cu[b], 0), T);
    return {q0, max(min(max(cu[b + 1], 0), T) - q0, 0)};
}

// ---- positions and masks ---------------------------------------------------------------------------
// A workgroup a request.  A token walks up through its parents, held in LDS: they have smaller indices, so the words of its mask
// come from the highest down and each is stored once; `window` steps up and further its ancestors are counted only.  Bound by the launch (8 requests of 5 to 16 tokens and 512 of 1 to 61 both about 6 us a pass, the
// kernel 2.8 and 4.5).
struct TreePlanArgs {
    const int *parent, *cu, *kv;
    int *pos;
    uint32_t *mask;
    long long ms;
    int T, words, window;
};

__global__ __launch_bounds__(256) void k_tree_plan(TreePlanArgs a) {
    __shared__ int up[1024];
    const int b = blockIdx.x, nt = blockDim.x;
    const TreeReq r = tree_req(a.cu, b, a.T);
    const int first = min(max(a.kv[b], 0), TREE_MAX_LEN) - r.n;
    if (r.n > 32 * a.words) {
        for (int i = threadIdx.x; i < r.n; i += nt) a.pos[r.q0 + i] = first + i;
        return;
    }
    for (int i = threadIdx.x; i < r.n; i += nt) {
        const int p = a.parent[r.q0 + i];
        up[i] = p >= 0 && p < i ? p : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < r.n; i += nt) {
        uint32_t *m = a.mask + (r.q0 + i) * a.ms;
        int w = i >> 5, depth = 0;
        for (int z = a.words - 1; z > w; z--) m[z] = 0u;
        uint32_t bits = 1u << (i & 31);
        for (int j = up[i]; j >= 0; j = up[j]) {
            depth++;
            for (; w > j >> 5; w--) { m[w] = bits; bits = 0u; }
            if (depth < a.window) bits |= 1u << (j & 31);
        }
        for (; w >= 0; w--) { m[w] = bits; bits = 0u; }
        a.pos[r.q0 + i] = first + depth;
    }
}

extern "C" int qwen_hip_op_tree_plan(const qwen_hip_tree_plan_t *p, void *stream) {
    QT_REFUSE(!p, "tree_plan: null descriptor");
    QT_REFUSE(p->B < 0 || p->B > 65535, "tree_plan: B %d out of range (0..65535)", p->B);
    QT_REFUSE(p->T < 0 || p->T > 1 << 26, "tree_plan: T %d out of range (0..2^26)", p->T);
    QT_REFUSE(p->mask_words < 1 || p->mask_words > 32 || p->mask_stride < p->mask_words,
              "tree_plan: mask_words %d of stride %lld (1..32, the stride at least as many)", p->mask_words, p->mask_stride);
    QT_REFUSE(p->window < 0, "tree_plan: window %d is negative", p->window);
    if (p->B == 0 || p->T == 0) return 0;
    QT_REFUSE(!p->parent || !p->cu_q || !p->kv_len || !p->pos || !p->mask, "tree_plan: null pointer");
    const long long T = p->T, B = p->B;
    const QtMem out[] = {{p->pos, 4 * T, "pos", nullptr}, {p->mask, 4 * ((T - 1) * p->mask_stride + p->mask_words), "mask", nullptr}};
    const QtMem in[] = {{p->parent, 4 * T, 0, 0}, {p->cu_q, 4 * (B + 1), 0, 0}, {p->kv_len, 4 * B, 0, 0}};
    const QtMem *const bad = qt_meets(out, 2, in, 3);
    QT_REFUSE(bad, "tree_plan: %s overlaps what is read or written beside it", bad->name);
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "tree_plan: the stream's device: %s", hipGetErrorString(on.err));
    const TreePlanArgs a = {p->parent, p->cu_q, p->kv_len, p->pos, p->mask, p->mask_stride, p->T, p->mask_words, p->window > 0 ? p->window : 1024};      // (no token has as many above it)
    const hipError_t e = qt_launch(k_tree_plan, dim3(p->B), dim3(p->mask_words > 4 ? 256 : p->mask_words > 2 ? 128 : 64), 0, st, a);
    QT_REFUSE(e != hipSuccess, "tree_plan: launch failed: %s", hipGetErrorString(e));
    return 0;
}

// ---- verification ----------------------------------------------------------------------------------
// From the current token, w = p's row and z = 1; child c of token x is kept where u q(x) z < w(x), else w <- max(w / z - q, 0),
// z <- sum w.  After rejections w is max(A p - B q, 0) with two numbers: A, B -> A / z, B / z + 1 (a token whose w
// has become 0 stays at 0).  So the walk needs each token's p and q at its parent's row, gathered once for 64 tokens, and a pass over the
// vocabulary only where a sum is asked for: by a further child after a rejection, and by the next token at the end.
// The pass sums tiles of 1024 entries, two a wave; the next token's tile is found in the tiles' sums, the token by a scan of its tile.
// All in f64: an f32 sum over a vocabulary would move the border between two tokens by more than some tokens have.
//
// Large vocabularies: launches of a wave for two tiles, the first of which walks to the first sum (every workgroup for itself: a few
// dependent loads), the others from the sum before to the next where there is one; then a launch of a workgroup a request, which goes on
// from there, makes further sums itself, and picks.  64 trees of 5 to 13 tokens over 128 003 bf16: 25 to 29 us, of which the rows' bytes are 6.7 (all sums but
// the first in the launch that picks 44, but the first two 36; one workgroup a request for everything past the first sum, without tiles a wave, 96);
// bound by sums that wait for each other.  6 chains over 2048 f32, one launch: 6.9, a chain of five dependent loads.
#define VF_TILE 1024
#define VF_MAX_V (1 << 20)
#define VF_MANY 2                   // tiles of a wave at a time, their loads in flight together
#define VF_WAVES 16                 // of the workgroup that picks
#define VF_SUM_WAVES 4

struct VerifyState { double A, B, z; int cur, last, kept, ask, buf, pad; };   // ask: z is the sum that is to be made; buf: which sums are w's
struct VerifyArgs {
    const uint8_t *p, *q;
    long long ps, qs;
    const int *tok, *parent, *cu;
    const float *u, *r;
    int *path, *out, *n_path;
    VerifyState *state;             // [2][B]
    double *sums;                   // [2][B][tiles]
    int B, T, V, tiles, round;      // round: launches of sums before this one
};

template <typename TY> __device__ __forceinline__ double vf_at(const uint8_t *row, long long i) {
    const float x = qt_load1<TY>(row + i * (long long)sizeof(typename TY::elem));
    return x > 0.f ? (double)x : 0.0;
}

// lane `l`'s value (l uniform)
__device__ __forceinline__ double vf_lane(double v, int l) {
    const long long u = __builtin_bit_cast(long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((int)u, l), hi = __builtin_amdgcn_readlane((int)(u >> 32), l);
    return __builtin_bit_cast(double, (long long)((unsigned long long)hi << 32 | lo));
}

// A wave: goes on from s to the next sum that is asked for (s.ask = 1) or to the last kept token (0).  `put`: writes what is kept.
template <typename TY, bool DRAFT>
__device__ __forceinline__ void vf_walk(const VerifyArgs &a, TreeReq r, VerifyState &s, bool put) {
    constexpr int E = sizeof(typename TY::elem);
    const int lane = threadIdx.x & 63;
    for (int base = (s.last + 1) & ~63; base < r.n; base += 64) {
        const int i = base + lane;
        const bool real = i < r.n && i > s.last;
        int up = -2, x = -1;
        float u = 0.f;
        double px = 0.0, qx = 1.0;
        if (real) {
            up = a.parent[r.q0 + i];
            x = a.tok[r.q0 + i];
            u = a.u[r.q0 + i];
            if (up < 0 || up >= i || x < 0 || x >= a.V) up = -2;       // no one's child
            else {
                px = vf_at<TY>(a.p + (r.q0 + up) * a.ps * E, x);
                if (DRAFT) qx = vf_at<TY>(a.q + (r.q0 + up) * a.qs * E, x);
            }
        }
        for (;;) {
            const unsigned long long kids = __ballot(up == s.cur && i > s.last);
            if (!kids) break;
            const int c = __ffsll(kids) - 1, id = base + c, cx = __builtin_amdgcn_readlane(x, c);
            if (s.ask) return;                                          // (after a rejection, and only if another child comes)
            const double cp = vf_lane(px, c), cq = vf_lane(qx, c);
            const float cu = lane_bcast(u, c);
            double w;
            if (DRAFT) {
                w = fmax(s.A * cp - s.B * cq, 0.0);
            } else {                                                    // 0 where a sibling before it had the same token
                w = cp;
                bool again = __ballot(up == s.cur && i < id && x == cx) != 0;
                for (int j = s.cur + 1 + lane; j < base; j += 64)
                    again |= __ballot(a.parent[r.q0 + j] == s.cur && a.tok[r.q0 + j] == cx) != 0;
                if (__ballot(again)) w = 0.0;
            }
            if (cu < 0.f || (double)cu * cq * s.z < w) {
                if (put && lane == 0) {
                    a.out[r.q0 + s.kept - 1] = cx;
                    a.path[r.q0 + s.kept] = id;
                }
                s.kept++;
                s.cur = id;
                s.A = 1.0; s.B = 0.0; s.z = 1.0;
            } else if (!DRAFT) {
                s.z = fmax(s.z - w, 0.0);
                s.B = 1.0;                                              // some siblings' tokens are out
            } else if (s.z > 0.0) {
                s.A /= s.z;
                s.B = s.B / s.z + 1.0;
                s.ask = 1;
            }
            s.last = id;
        }
        if (base + 63 > s.last) s.last = min(base + 63, r.n - 1);
    }
    s.ask = 0;
}

// w of 8 entries of p and q: max(A p - B q, 0), or p where no rejected sibling has that token (`gone`: a bit for each)
template <bool DRAFT>
__device__ __forceinline__ void vf_weigh(const VerifyState &s, const float (&x)[8], const float (&y)[8], uint32_t gone, double (&w)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const double px = x[e] > 0.f ? (double)x[e] : 0.0;
        if (DRAFT) w[e] = fmax(s.A * px - s.B * (y[e] > 0.f ? (double)y[e] : 0.0), 0.0);
        else w[e] = gone >> e & 1u ? 0.0 : px;
    }
}
__device__ __forceinline__ double vf_add(const double (&w)[8]) { return ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])); }
// Entries v .. v + 7 of a row.  A lane whose eight pass the row's end loads the row's last eight instead, `skip` of which come before v: those
// are 0, and so is everything past the end.
template <typename TY, bool DRAFT> struct VfEight {
    static constexpr int E = sizeof(typename TY::elem), NW = E / 2;
    qt_w4 x[NW], y[DRAFT ? NW : 1];
    __device__ __forceinline__ static int base(const VerifyArgs &a, int v) { return min(v, max(a.V - 8, 0)); }
    __device__ __forceinline__ void load(const VerifyArgs &a, const uint8_t *p, const uint8_t *q, int v) {
        const long long at = (long long)base(a, v) * E;
#pragma unroll
        for (int i = 0; i < NW; i++) {
            x[i] = qt_load16<E>(p + at + 16 * i);
            if (DRAFT) y[i] = qt_load16<E>(q + at + 16 * i);
        }
    }
    // of a row that has no eight
    __device__ __forceinline__ void load_few(const VerifyArgs &a, const uint8_t *p, const uint8_t *q) {
        typename TY::elem ex[8] = {}, ey[8] = {};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if (e < a.V) ex[e] = reinterpret_cast<const typename TY::elem *>(p)[e];
            if (DRAFT && e < a.V) ey[e] = reinterpret_cast<const typename TY::elem *>(q)[e];
        }
        __builtin_memcpy(x, ex, sizeof ex);
        if (DRAFT) __builtin_memcpy(y, ey, sizeof ey);
    }
    template <int N> __device__ __forceinline__ static void load_all(VfEight (&x)[N], const VerifyArgs &a, const uint8_t *p, const uint8_t *q, int v0) {
        if (a.V < 8) {
#pragma unroll
            for (int k = 0; k < N; k++) x[k].load_few(a, p, q);
        } else {
#pragma unroll
            for (int k = 0; k < N; k++) x[k].load(a, p, q, v0 + 512 * k);
        }
    }
    // their w; bits: those of the tile's tokens that rejected siblings have, the tile beginning at v0
    __device__ __forceinline__ void weigh(const VerifyArgs &a, const VerifyState &s, const uint32_t *bits, int v0, int v, double (&w)[8]) const {
        float fx[8], fy[8] = {};
        qt_widen8<TY>(x, fx);
        if constexpr (DRAFT) qt_widen8<TY>(y, fy);
        const int skip = v - base(a, v), at = v - v0;
        uint32_t gone = 0;
        if (!DRAFT && s.B != 0.0) {
            gone = bits[at >> 5] >> (at & 31) & 0xFFu;                 // at: a multiple of 8
            gone = skip < 8 ? gone << skip : 0u;
        }
        if (skip > 0) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e < skip) fx[e] = 0.f;
        }
        vf_weigh<DRAFT>(s, fx, fy, gone, w);
    }
    // the entry that w[e] is of
    __device__ __forceinline__ static int entry(const VerifyArgs &a, int v, int e) { return base(a, v) + e; }
};

__device__ __forceinline__ double vf_wave_sum(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
__device__ __forceinline__ double vf_wave_scan(double v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double y = __shfl_up(v, o, 64);
        if (lane >= o) v += y;
    }
    return v;
}

// A wave: marks a tile's tokens that rejected siblings have (certain drafts only).
template <bool DRAFT>
__device__ __forceinline__ void vf_marks(const VerifyArgs &a, TreeReq r, const VerifyState &s, int tile, uint32_t *bits) {
    if (DRAFT || s.B == 0.0) return;
    const int lane = threadIdx.x & 63;
    __threadfence_block();                              // the words are the wave's own: its stores and atomics in their order
    for (int i = lane; i < VF_TILE / 32; i += 64) bits[i] = 0u;
    __threadfence_block();
    for (int i = s.cur + 1 + lane; i < r.n; i += 64)
        if (a.parent[r.q0 + i] == s.cur) {
            const int x = a.tok[r.q0 + i], t = x - tile * VF_TILE;
            if (x >= 0 && t >= 0 && t < VF_TILE) atomicOr(&bits[t >> 5], 1u << (t & 31));
        }
    __threadfence_block();
}

// A wave: the sums of N tiles from the first on, in every lane; a lane takes 8 entries of every 512, all loads in flight together.
#define VF_PARTS (VF_TILE / 512)
template <typename TY, bool DRAFT, int N>
__device__ __forceinline__ void vf_tiles(const VerifyArgs &a, TreeReq r, const VerifyState &s, int first, uint32_t *bits, double (&sum)[N]) {
    constexpr int E = sizeof(typename TY::elem);
    const int lane = threadIdx.x & 63;
    const uint8_t *p = a.p + (r.q0 + s.cur) * a.ps * E, *q = DRAFT ? a.q + (r.q0 + s.cur) * a.qs * E : nullptr;
    VfEight<TY, DRAFT> x[N * VF_PARTS];
    const int v0 = first * VF_TILE + 8 * lane;
    VfEight<TY, DRAFT>::load_all(x, a, p, q, v0);
#pragma unroll
    for (int t = 0; t < N; t++) {
        vf_marks<DRAFT>(a, r, s, first + t, bits);
        double y = 0.0;
#pragma unroll
        for (int k = 0; k < VF_PARTS; k++) {
            double w[8];
            x[VF_PARTS * t + k].weigh(a, s, bits, (first + t) * VF_TILE, v0 + 512 * (VF_PARTS * t + k), w);
            y += vf_add(w);
        }
        sum[t] = vf_wave_sum(y);
    }
}
// A wave: the sum of the tiles' sums.
template <typename P> __device__ __forceinline__ double vf_total(P sums, int tiles) {
    const int lane = threadIdx.x & 63, per = (tiles + 63) / 64, t1 = min((lane + 1) * per, tiles);
    double x = 0.0;
    for (int t = lane * per; t < t1; t++) x += sums[t];
    return vf_wave_sum(x);
}
__device__ __forceinline__ bool vf_same(const VerifyState &x, const VerifyState &y) { return x.A == y.A && x.B == y.B && x.cur == y.cur; }

template <typename TY, bool DRAFT>
__global__ __launch_bounds__(64 * VF_SUM_WAVES) void k_tree_sums(VerifyArgs a) {
    __shared__ VerifyState s;
    __shared__ uint32_t bits[VF_SUM_WAVES][VF_TILE / 32];
    __shared__ int more;
    const int b = blockIdx.y, wave = threadIdx.x >> 6, tile = (blockIdx.x * VF_SUM_WAVES + wave) * VF_MANY, now = a.round & 1;
    const bool first = blockIdx.x == 0;                 // writes what the request's workgroups all find
    const TreeReq r = tree_req(a.cu, b, a.T);
    if (r.n == 0) return;
    if (wave == 0) {
        VerifyState w = {1.0, 0.0, 1.0, 0, 0, 1, 0, 0, 0};
        bool make = true;
        if (a.round > 0) {
            w = a.state[(size_t)(now ^ 1) * a.B + b];
            make = w.ask;
            if (make) {
                const VerifyState before = w;
                w.z = vf_total(a.sums + ((size_t)w.buf * a.B + b) * a.tiles, a.tiles);
                w.ask = 0;
                vf_walk<TY, DRAFT>(a, r, w, first);
                make = !vf_same(w, before);
            }
        } else {
            vf_walk<TY, DRAFT>(a, r, w, first);
        }
        if (make) w.buf = now;
        if (threadIdx.x == 0) {
            s = w;
            more = make;
            if (first) a.state[(size_t)now * a.B + b] = w;
        }
    }
    __syncthreads();
    if (!more || tile >= a.tiles) return;
    const VerifyState mine = s;
    double sum[VF_MANY];
    vf_tiles<TY, DRAFT, VF_MANY>(a, r, mine, tile, bits[wave], sum);
#pragma unroll
    for (int t = 0; t < VF_MANY; t++)
        if (tile + t < a.tiles && (threadIdx.x & 63) == t) a.sums[((size_t)now * a.B + b) * a.tiles + tile + t] = sum[t];
}

template <typename TY, bool DRAFT>
__global__ __launch_bounds__(64 * VF_WAVES) void k_tree_pick(VerifyArgs a) {
    __shared__ VerifyState s;
    __shared__ uint32_t bits[VF_WAVES][VF_TILE / 32];
    __shared__ double sums[VF_MAX_V / VF_TILE];
    __shared__ int state_s;                             // 0: the sums are to be made, 1: they are, 2: and no more are asked for
    __shared__ double total_s;
    constexpr int E = sizeof(typename TY::elem);
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const TreeReq r = tree_req(a.cu, b, a.T);
    if (r.n == 0) {
        if (threadIdx.x == 0) a.n_path[b] = 0;
        return;
    }
    if (wave == 0) {
        VerifyState w = {1.0, 0.0, 1.0, 0, 0, 1, 0, 0, 0};
        if (a.round > 0) w = a.state[(size_t)((a.round - 1) & 1) * a.B + b];
        else vf_walk<TY, DRAFT>(a, r, w, true);
        if (lane == 0) { s = w; state_s = a.round > 0; }
    }
    __syncthreads();
    if (a.round > 0) {
        const double *from = a.sums + ((size_t)s.buf * a.B + b) * a.tiles;
        for (int t = threadIdx.x; t < a.tiles; t += blockDim.x) sums[t] = from[t];
    }
    for (bool again = false;;) {                        // a sum for each rejected child at most, and one more
        const bool none = state_s == 0;
        __syncthreads();
        if (none) {
            const VerifyState mine = s;
            const auto make = [&](auto n) {             // n tiles at a time
                constexpr int N = decltype(n)::value;
                for (int t = wave * N; t < a.tiles; t += waves * N) {
                    double sum[N];
                    vf_tiles<TY, DRAFT, N>(a, r, mine, t, bits[wave], sum);
#pragma unroll
                    for (int u = 0; u < N; u++)
                        if (t + u < a.tiles && lane == u) sums[t + u] = sum[u];
                }
            };
            if (a.tiles <= waves) make(std::integral_constant<int, 1>{});
            else make(std::integral_constant<int, VF_MANY>{});
            __syncthreads();
        }
        if (wave == 0) {
            VerifyState w = s;
            const double z = vf_total(sums, a.tiles);
            int next = 2;
            if (s.ask) {
                w.z = z;
                w.ask = 0;
                vf_walk<TY, DRAFT>(a, r, w, true);
                next = !vf_same(w, s) ? 0 : w.ask ? 1 : 2;
            }
            if (next == 2 && !(z > 0.0) && !again) {    // nothing is left: p's row as it is
                again = true;
                w.A = 1.0; w.B = 0.0;
                next = 0;
            }
            if (lane == 0) { s = w; state_s = next; total_s = z; }
        }
        __syncthreads();
        if (state_s == 2) break;
    }
    if (wave == 0) {
        // the first tile whose sum takes the running sum past the goal, or else the last one that is not 0 (sums that rounding
        // leaves just under it); then the first of its entries in the same way
        const double goal = (double)a.r[b] * total_s;
        const int per = (a.tiles + 63) / 64, t0 = min(lane * per, a.tiles), t1 = min(t0 + per, a.tiles);
        double mine = 0.0;
        for (int t = t0; t < t1; t++) mine += sums[t];
        const double upto = vf_wave_scan(mine), lower = __shfl_up(upto, 1, 64);
        double x = lane ? lower : 0.0;
        int tile = -1, some = -1;
        double x_tile = 0.0, x_some = 0.0;
        for (int t = t0; t < t1; t++) {
            const double y = sums[t];
            if (y > 0.0) { some = t; x_some = x; }
            if (tile < 0 && y > 0.0 && x + y > goal) { tile = t; x_tile = x; }
            x += y;
        }
        int token = -1;
        unsigned long long who = __ballot(tile >= 0);
        int from = who ? __ffsll(who) - 1 : -1;
        if (!who && (who = __ballot(some >= 0))) { from = 63 - __clzll((long long)who); tile = some; x_tile = x_some; }
        if (from >= 0) {
            tile = __builtin_amdgcn_readlane(tile, from);
            double before = vf_lane(x_tile, from);
            const VerifyState w = s;
            const uint8_t *p = a.p + (r.q0 + w.cur) * a.ps * E, *q = DRAFT ? a.q + (r.q0 + w.cur) * a.qs * E : nullptr;
            vf_marks<DRAFT>(a, r, w, tile, bits[0]);
            double e8[VF_PARTS][8];
            VfEight<TY, DRAFT> x8[VF_PARTS];
            const int v0 = tile * VF_TILE + 8 * lane;
            VfEight<TY, DRAFT>::load_all(x8, a, p, q, v0);
#pragma unroll
            for (int k = 0; k < VF_PARTS; k++) x8[k].weigh(a, w, bits[0], tile * VF_TILE, v0 + 512 * k, e8[k]);
            int found = -1, any = -1;                   // the wave's
#pragma unroll
            for (int k = 0; k < VF_PARTS; k++) {
                const double scan = vf_wave_scan(vf_add(e8[k])), below = __shfl_up(scan, 1, 64);
                double y = before + (lane ? below : 0.0);
                int f = -1, last = -1;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    y += e8[k][e];
                    if (e8[k][e] > 0.0) {
                        last = x8[k].entry(a, v0 + 512 * k, e);
                        if (f < 0 && y > goal) f = last;
                    }
                }
                const unsigned long long fs = __ballot(f >= 0), ls = __ballot(last >= 0);
                if (found < 0 && fs) found = __builtin_amdgcn_readlane(f, __ffsll(fs) - 1);
                if (ls) any = __builtin_amdgcn_readlane(last, 63 - __clzll((long long)ls));
                before += vf_lane(scan, 63);
            }
            token = found >= 0 ? found : any;
        }
        if (lane == 0) {
            a.path[r.q0] = 0;
            a.out[r.q0 + s.kept - 1] = token;
            a.n_path[b] = s.kept;
        }
    }
    for (int k = s.kept + threadIdx.x; k < r.n; k += blockDim.x) a.path[r.q0 + k] = a.out[r.q0 + k] = -1;
}

static int verify_args(const qwen_hip_tree_verify_t *p, VerifyArgs &a) {
    QT_REFUSE(!p, "tree_verify: null descriptor");
    QT_REFUSE(!qt_dt_size(p->dtype), "tree_verify: dtype %d (f32, bf16 or f16)", p->dtype);
    QT_REFUSE(p->B < 0 || p->B > 65535, "tree_verify: B %d out of range (0..65535)", p->B);
    QT_REFUSE(p->T < 0 || p->T > 1 << 26, "tree_verify: T %d out of range (0..2^26)", p->T);
    QT_REFUSE(p->V < 1 || p->V > VF_MAX_V, "tree_verify: V %d out of range (1..2^20)", p->V);
    QT_REFUSE(p->max_children < 0, "tree_verify: max_children %d is negative", p->max_children);
    a = VerifyArgs{};
    a.B = p->B; a.T = p->T; a.V = p->V;
    a.tiles = (p->V + VF_TILE - 1) / VF_TILE;
    return 0;
}
static long long verify_bytes(const VerifyArgs &a) { return 2ll * a.B * (sizeof(VerifyState) + 8ll * a.tiles); }

extern "C" long long qwen_hip_op_tree_verify_workspace(const qwen_hip_tree_verify_t *p) {
    VerifyArgs a;
    if (verify_args(p, a)) return -1;
    return verify_bytes(a);
}

// Launches of sums before the one that picks.  Up to 48 tiles that one makes them as fast (40 000 entries bf16, 4 and 64 requests: chains 11.8 and 12.7
// us, trees 17.3 and 22.1; 50 000: chains 13.5 and 14.5 against 17.2 and 18.6 in four launches, trees 20.6 and 24.5 against 19.1 and 22.3).
static int verify_rounds(const VerifyArgs &a, bool draft, int max_children) {
    if (a.tiles <= 48) return 0;
    return draft && max_children != 1 ? 3 : 1;
}
static int vf_waves(int tiles) { return tiles < VF_WAVES ? tiles : VF_WAVES; }
template <typename TY, bool DRAFT> static hipError_t verify_launch(VerifyArgs a, int rounds, hipStream_t st) {
    hipError_t e = hipSuccess;
    for (; a.round < rounds && e == hipSuccess; a.round++)
        e = qt_launch(k_tree_sums<TY, DRAFT>, dim3((a.tiles + VF_SUM_WAVES * VF_MANY - 1) / (VF_SUM_WAVES * VF_MANY), a.B), dim3(64 * VF_SUM_WAVES), 0, st, a);
    if (e == hipSuccess) e = qt_launch(k_tree_pick<TY, DRAFT>, dim3(a.B), dim3(64 * vf_waves(a.tiles)), 0, st, a);
    return e;
}

extern "C" int qwen_hip_op_tree_verify(const qwen_hip_tree_verify_t *p, void *stream) {
    VerifyArgs a;
    if (verify_args(p, a)) return -1;
    if (p->B == 0) return 0;
    QT_REFUSE(!p->cu_q || !p->n_path || !p->r || (p->T > 0 && (!p->p || !p->tok || !p->parent || !p->u || !p->path || !p->out_tok)),
              "tree_verify: null pointer");
    const int E = qt_dt_size(p->dtype);
    QT_REFUSE((uintptr_t)p->p % E || (uintptr_t)p->q % E, "tree_verify: p and q have to be aligned to their elements");
    QT_REFUSE(p->p_stride < p->V || (p->q && p->q_stride < p->V), "tree_verify: strides %lld, %lld under %d entries", p->p_stride, p->q_stride, p->V);
    const long long need = verify_bytes(a);
    QT_REFUSE(!p->workspace || p->workspace_bytes < need, "tree_verify: a workspace of %lld bytes is needed, %lld given", need,
              p->workspace ? p->workspace_bytes : 0ll);
    QT_REFUSE(qt_off16(p->workspace), "tree_verify: the workspace has to be aligned to 16 bytes");
    const long long T = p->T, B = p->B;
    const QtMem out[] = {{p->path, 4 * T, "path", nullptr}, {p->out_tok, 4 * T, "out_tok", nullptr}, {p->n_path, 4 * B, "n_path", nullptr},
                         {p->workspace, need, "workspace", nullptr}};
    const QtMem in[] = {{p->tok, 4 * T, 0, 0}, {p->parent, 4 * T, 0, 0}, {p->u, 4 * T, 0, 0}, {p->cu_q, 4 * (B + 1), 0, 0}, {p->r, 4 * B, 0, 0},
                        {p->p, E * ((T - 1) * p->p_stride + p->V), 0, 0}, {p->q, E * ((T - 1) * p->q_stride + p->V), 0, 0}};
    const QtMem *const bad = qt_meets(out, 4, in, 7);
    QT_REFUSE(bad, "tree_verify: %s overlaps what is read or written beside it", bad->name);
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "tree_verify: the stream's device: %s", hipGetErrorString(on.err));
    a.p = (const uint8_t *)p->p; a.q = (const uint8_t *)p->q;
    a.ps = p->p_stride; a.qs = p->q_stride;
    a.tok = p->tok; a.parent = p->parent; a.cu = p->cu_q; a.u = p->u; a.r = p->r;
    a.path = p->path; a.out = p->out_tok; a.n_path = p->n_path;
    a.state = (VerifyState *)p->workspace;
    a.sums = (double *)(a.state + 2ll * p->B);
    const int rounds = verify_rounds(a, p->q != nullptr, p->max_children);
#define VERIFY(TY) (p->q ? verify_launch<TY, true>(a, rounds, st) : verify_launch<TY, false>(a, rounds, st))
    const hipError_t e = p->dtype == QWEN_HIP_DT_F32 ? VERIFY(QtF32) : p->dtype == QWEN_HIP_DT_BF16 ? VERIFY(QtBf16) : VERIFY(QtF16);
#undef VERIFY
    QT_REFUSE(e != hipSuccess, "tree_verify: launch failed: %s", hipGetErrorString(e));
    return 0;
}

// ---- what is kept ----------------------------------------------------------------------------------
// Row path[k] goes to place k.  Since path[k] >= k, a place that has been written is no later row's source: a thread that takes 16
// bytes of a head's rows, or a head's scales, through all moves in the order of k, eight loads before their stores, reads every source before it
// is overwritten, and no two threads share bytes.  A workgroup takes a request's rows in one layer.  Lengths and pages: one workgroup.
// Moves done twice are not moves done once, so a commit that cannot be moves nothing.  While that is CM_LOOK looks in all, each workgroup looks at all requests
// first (commit_stands), and the lengths' workgroup is one more of the launch; past it, and where lengths or the count are replaced in place, the lengths'
// launch is before the moves', which go by its status (bf16, 2 heads of 64, one launch and two: 300 requests of 8 layers 8.0 and 9.6 us, 1024 of one 7.5
// and 9.8, 512 of 8 11.8 and 11.1, 300 of 28 18.5 and 14.5; without looking 512 of 8 7.2).
// Bound by a chain of dependent loads (lengths, path, table, rows): 8 requests, one layer of bf16 6.7 us a pass, the kernel 4.6; 64 requests,
// 28 layers of codes 15.2 (without the look at all requests 13.9), the rows' 42 to 49 MB being 10.
#define CM_T 256
#define CM_MAX_B 2048
#define CM_LOOK (1 << 20)
struct CommitArgs {
    const int *path, *n_path, *cu, *kv, *table, *n_free;
    long long ts;
    int *kv_out, *free_pages, *n_free_out, *status;
    uint8_t *k, *v, *ks, *vs;                           // codes and strides in bytes
    long long layer, page, head, slot, s_layer, s_page, s_head, s_slot;
    int B, T, cols, ps, n_pages, layers, nkv, row;      // row: bytes of a head's row
    int moves, lengths;                                 // this launch moves rows; makes lengths and pages
    int made;                                           // lengths and status are there: kv_out is of after the moves
    int count;                                          // the call makes them: its moves look at the free list's count, too
    QtDiv div;
};

__device__ __forceinline__ int commit_kept(const CommitArgs &a, int b, int n) { return min(max(a.n_path[b], 0), n); }
// whether a request's lengths are ones that a table can hold
__device__ __forceinline__ bool commit_fits(const CommitArgs &a, int kv, int n) { return kv >= n && (long long)kv <= (long long)a.cols * a.ps; }
__device__ __forceinline__ int commit_pages(const CommitArgs &a, int len) { return qt_quot(len, a.div) + (len % a.ps != 0); }

// The pages that a request gives back; `bad` where its lengths cannot be.
__device__ __forceinline__ unsigned commit_back(const CommitArgs &a, int b, bool &bad) {
    const int n = tree_req(a.cu, b, a.T).n, kv = a.kv[b], kept = commit_kept(a, b, n);
    if (commit_fits(a, kv, n)) return commit_pages(a, kv) - commit_pages(a, kv - n + kept);
    bad = true;
    return 0;
}
// A workgroup: whether the call is one that can be, by what commit_lengths refuses.
__device__ __forceinline__ bool commit_stands(const CommitArgs &a) {
    __shared__ unsigned long long wsum[CM_T / 64];
    bool bad = false;
    if (!a.count) {                                     // rows only: lengths alone
        for (int b = threadIdx.x; b < a.B; b += CM_T) bad |= !commit_fits(a, a.kv[b], tree_req(a.cu, b, a.T).n);
        return !__syncthreads_or(bad);
    }
    const int n_free = a.n_free[0];
    unsigned long long mine = 0;                        // 2048 requests of 2^30 pages at most
    bad = n_free < 0 || n_free > a.n_pages;
    for (int b = threadIdx.x; b < a.B; b += CM_T) mine += commit_back(a, b, bad);
#pragma unroll
    for (int o = 32; o; o >>= 1) mine += __shfl_xor(mine, o, 64);
    if ((threadIdx.x & 63) == 0) wsum[threadIdx.x >> 6] = mine;
    bad = __syncthreads_or(bad);
    unsigned long long all = max(n_free, 0);
#pragma unroll
    for (int w = 0; w < CM_T / 64; w++) all += wsum[w];
    return !bad && all <= (unsigned long long)a.n_pages;
}

// A piece of every row through n moves.
template <typename V> __device__ __forceinline__ void commit_piece(uint8_t *base, int n, const long long *from, const long long *to) {
    for (int j = 0; j < n; j += 8) {
        V x[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (j + e < n) x[e] = *reinterpret_cast<const V *>(base + from[j + e]);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (j + e < n) *reinterpret_cast<V *>(base + to[j + e]) = x[e];
    }
}

__device__ __forceinline__ void commit_move(const CommitArgs &a, int b, int layer) {
    __shared__ long long from[2][CM_T], to[2][CM_T];    // of codes, of scales
    __shared__ int moves_s[CM_T / 64];
    const TreeReq r = tree_req(a.cu, b, a.T);
    const int keep = commit_kept(a, b, r.n), kv = a.made ? a.kv_out[b] + r.n - keep : a.kv[b], lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (a.made ? a.status[0] != 0 : !commit_stands(a)) return;
    const int *table = a.table + b * a.ts;
    for (int k0 = 0; k0 < keep; k0 += CM_T) {
        const int k = k0 + threadIdx.x;
        int pgs = -1, pgd = -1, os = 0, od = 0;
        if (k < keep) {
            const int src = a.path[r.q0 + k];
            if (src > k && src < r.n) {
                const int ps = kv - r.n + src, pd = kv - r.n + k, cs = qt_quot(ps, a.div), cd = qt_quot(pd, a.div);
                pgs = table[cs];
                pgd = table[cd];
                os = ps - cs * a.ps;
                od = pd - cd * a.ps;
            }
        }
        const bool moves = (unsigned)pgs < (unsigned)a.n_pages && (unsigned)pgd < (unsigned)a.n_pages;
        const unsigned long long some = __ballot(moves);
        __syncthreads();                                // the last rounds' list is read
        if (lane == 0) moves_s[wave] = __popcll(some);
        __syncthreads();
        int at = __popcll(some & ((1ull << lane) - 1)), n = 0;
#pragma unroll
        for (int w = 0; w < CM_T / 64; w++) {
            if (w < wave) at += moves_s[w];
            n += moves_s[w];
        }
        if (moves) {
            from[0][at] = pgs * a.page + os * a.slot;
            to[0][at] = pgd * a.page + od * a.slot;
            from[1][at] = pgs * a.s_page + os * a.s_slot;
            to[1][at] = pgd * a.s_page + od * a.s_slot;
        }
        __syncthreads();
        const int chunks = a.row / 16, rows = a.nkv * chunks, pieces = 2 * rows + (a.ks ? 2 * a.nkv : 0);
        for (int i = threadIdx.x; i < pieces; i += CM_T) {
            if (i < 2 * rows) {
                const int j = i >= rows ? i - rows : i;
                commit_piece<qt_w4>((i >= rows ? a.v : a.k) + layer * a.layer + j / chunks * a.head + 16 * (j % chunks), n, from[0], to[0]);
            } else {
                const int j = i - 2 * rows;
                commit_piece<uint8_t>((j >= a.nkv ? a.vs + (j - a.nkv) * a.s_head : a.ks + j * a.s_head) + layer * a.s_layer, n, from[1], to[1]);
            }
        }
    }
}

__device__ __forceinline__ void commit_lengths(const CommitArgs &a) {
    __shared__ unsigned long long wsum[CM_T / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n_free = a.n_free[0];
    const int per = (a.B + CM_T - 1) / CM_T, b0 = min((int)threadIdx.x * per, a.B), b1 = min(b0 + per, a.B);
    unsigned long long mine = 0;
    bool bad = n_free < 0 || n_free > a.n_pages;
    for (int b = b0; b < b1; b++) mine += commit_back(a, b, bad);
    unsigned long long upto = mine;                     // 2048 requests of 2^30 pages at most
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long y = __shfl_up(upto, o, 64);
        if (lane >= o) upto += y;
    }
    if (lane == 63) wsum[wave] = upto;
    bad = __syncthreads_or(bad);
    unsigned long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < CM_T / 64; w++) {
        if (w < wave) before += wsum[w];
        all += wsum[w];
    }
    bad |= (unsigned long long)max(n_free, 0) + all > (unsigned long long)a.n_pages;
    if (!bad) {
        int at = n_free + (int)(before + upto - mine);
        for (int b = b0; b < b1; b++) {
            const int n = tree_req(a.cu, b, a.T).n, kv = a.kv[b], len = kv - n + commit_kept(a, b, n);
            for (int c = commit_pages(a, len); c < commit_pages(a, kv); c++) a.free_pages[at++] = a.table[b * a.ts + c];
            a.kv_out[b] = len;
        }
    } else if (a.kv_out != a.kv) {
        for (int b = b0; b < b1; b++) a.kv_out[b] = a.kv[b];
    }
    if (threadIdx.x == 0) {
        a.n_free_out[0] = bad ? n_free : n_free + (int)all;
        a.status[0] = bad ? QWEN_HIP_PLAN_INVALID : 0;
    }
}

__global__ __launch_bounds__(CM_T) void k_tree_commit(CommitArgs a) {
    if (a.moves) {
        const int b = blockIdx.x % a.B, layer = blockIdx.x / a.B;
        if (layer < a.layers) { commit_move(a, b, layer); return; }
    }
    commit_lengths(a);
}

extern "C" int qwen_hip_op_tree_commit(const qwen_hip_kv_pages_t *kv, const qwen_hip_tree_commit_t *p, void *stream) {
    if (qt_check_pages("tree_commit", kv)) return -1;
    QT_REFUSE(!p, "tree_commit: null descriptor");
    QT_REFUSE(p->B < 0 || p->B > CM_MAX_B, "tree_commit: B %d out of range (0..%d)", p->B, CM_MAX_B);
    QT_REFUSE(p->T < 0 || p->T > 1 << 26, "tree_commit: T %d out of range (0..2^26)", p->T);
    QT_REFUSE(p->n_layers < 0 || (long long)p->n_layers * p->B > 0xFFFFFEll, "tree_commit: %d layers of %d requests (2^24 - 2 at most)", p->n_layers, p->B);
    QT_REFUSE(p->table_cols < 1 || (long long)p->table_cols * kv->page_size > TREE_MAX_LEN || p->table_stride < p->table_cols,
              "tree_commit: table_cols %d of stride %lld (at least 1, 2^30 positions at most)", p->table_cols, p->table_stride);
    if (p->B == 0) return 0;
    QT_REFUSE(!p->n_path || !p->cu_q || !p->kv_len || !p->table || (p->T > 0 && !p->path), "tree_commit: null pointer");
    QT_REFUSE(p->kv_len_out && (!p->free_pages || !p->n_free || !p->n_free_out || !p->status), "tree_commit: null pointer (lengths need the free list and status)");
    const bool codes = kv->dtype == QWEN_HIP_DT_E4M3;
    const int E = qt_kv_size(kv->dtype);
    if (p->n_layers > 0 && qt_check_pages_apart("tree_commit", kv, p->n_layers, p->layer_stride, p->scale_layer_stride)) return -1;
    QT_REFUSE(p->n_layers > 1 && p->layer_stride % (16 / E), "tree_commit: layer_stride %lld (a multiple of 16 bytes)", p->layer_stride);
    if (p->kv_len_out) {
        const long long T = p->T, B = p->B;
        const QtMem out[] = {{p->kv_len_out, 4 * B, "kv_len_out", p->kv_len}, {p->n_free_out, 4, "n_free_out", p->n_free}, {p->status, 4, "status", nullptr},
                             {p->free_pages, 4ll * kv->n_pages, "free_pages", nullptr}};
        const QtMem in[] = {{p->path, 4 * T, 0, 0}, {p->n_path, 4 * B, 0, 0}, {p->cu_q, 4 * (B + 1), 0, 0}, {p->kv_len, 4 * B, 0, 0}, {p->n_free, 4, 0, 0},
                            {p->table, 4 * ((B - 1) * p->table_stride + p->table_cols), 0, 0}};
        const QtMem *const bad = qt_meets(out, 4, in, 6);
        QT_REFUSE(bad, "tree_commit: %s overlaps what is read or written beside it", bad->name);
    }
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "tree_commit: the stream's device: %s", hipGetErrorString(on.err));
    CommitArgs a = {};
    a.path = p->path; a.n_path = p->n_path; a.cu = p->cu_q; a.kv = p->kv_len; a.table = p->table; a.n_free = p->n_free;
    a.ts = p->table_stride;
    a.kv_out = p->kv_len_out; a.free_pages = p->free_pages; a.n_free_out = p->n_free_out; a.status = p->status;
    a.k = (uint8_t *)kv->k; a.v = (uint8_t *)kv->v;
    a.layer = p->layer_stride * E; a.page = kv->page_stride * E; a.head = kv->head_stride * E; a.slot = kv->slot_stride * E;
    if (codes) {
        a.ks = kv->k_scale; a.vs = kv->v_scale;
        a.s_layer = p->scale_layer_stride; a.s_page = kv->scale_page_stride; a.s_head = kv->scale_head_stride; a.s_slot = kv->scale_slot_stride;
    }
    a.B = p->B; a.T = p->T; a.cols = p->table_cols; a.ps = kv->page_size; a.n_pages = kv->n_pages; a.layers = p->n_layers;
    a.nkv = kv->n_kv_heads; a.row = kv->head_dim * E;
    a.div = qt_div_of(kv->page_size);
    const bool in_place = p->kv_len_out == p->kv_len || p->n_free_out == p->n_free;
    const bool moves = p->n_layers > 0 && p->T > 0, first = p->kv_len_out && moves && (in_place || (long long)p->n_layers * p->B * p->B > CM_LOOK);     // lengths in a launch before the moves'
    a.moves = moves && !first;
    a.lengths = a.count = p->kv_len_out != nullptr;
    const unsigned wgs = (unsigned)(moves ? p->n_layers * p->B : 0);
    hipError_t e = hipSuccess;
    if (a.moves || a.lengths) e = qt_launch(k_tree_commit, dim3((a.moves ? wgs : 0) + (a.lengths ? 1 : 0)), dim3(CM_T), 0, st, a);
    if (e == hipSuccess && first) {
        a.moves = a.made = 1;
        a.lengths = 0;
        e = qt_launch(k_tree_commit, dim3(wgs), dim3(CM_T), 0, st, a);
    }
    QT_REFUSE(e != hipSuccess, "tree_commit: launch failed: %s", hipGetErrorString(e));
    return 0;
}
