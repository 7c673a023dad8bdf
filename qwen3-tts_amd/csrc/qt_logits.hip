// qt_logits.hip — the rules on a batch's logits before sampling (qwen_hip_op_logit_rules): repetition,
// presence and frequency penalties, token biases, an allowed-token bit mask.
//
// A workgroup of RULES_T threads takes 16 RULES_T neighbouring tokens of one row, loaded at once.  Few of them are in the row's history or
// its biases: those are marked in LDS, then counted there (integer atomics: the order does not matter; of a token's
// bias entries the largest index wins), and a thread goes through the marked ones of its own before it stores.  So a row's
// history is read once a workgroup, from the L2, and no counts of V tokens a row are held in memory, cleared or read back.
// A token has one word, its count in the lower 16 bits and its last bias entry in the upper, so that all threads of a CU have one
// in LDS.
// Bound by the chain of offsets, history, marks and counts before the first store next to the logits' bytes: 64 rows of
// 128 003 bf16, histories of up to 4000, 50 biases, a mask 11.5 us, 3.0 TB/s (a copy of the logits alone 5.9); 6 rows of 2048
// f32 6.3, the launch.
#include "qt_ops.h"


struct RulesArgs {
    const uint8_t *x;
    uint8_t *out;
    long long xs, os, ms;
    const int *hist, *hoff, *npr;
    const float *rep, *pres, *freq;
    const int *btok;
    const float *bval;
    const int *boff;
    const uint32_t *mask;
    int V, hcap, bcap, each;
};

// Row b's part of a list of `cap` entries.  Offsets are the caller's: one out of range is brought into it, and entries are
// counted from the part's begin, unsigned, so that no sum of an index and a step passes 2^32.
struct ListPart { int at; unsigned n; };
__device__ __forceinline__ ListPart list_part(const int *off, int b, int cap) {
    const int at = min(max(off[b], 0), cap), end = min(max(off[b + 1], at), cap);
    return {at, (unsigned)(end - at)};
}

// BIAS: with bias lists.  EACH: the penalty once for every entry.  Rows may begin anywhere that their elements can: 16-byte
// accesses at 2- or 4-byte alignment are one instruction on this GPU.
template <typename T, bool BIAS, bool EACH, int RULES_T>
__global__ __launch_bounds__(RULES_T) void k_logit_rules(RulesArgs a) {
    constexpr int E = sizeof(typename T::elem), NV = 2, RULES_CH = 8 * NV * RULES_T;
    constexpr int RULES_HELD = 4096 / RULES_T;          // history entries a thread keeps between marking and counting
    __shared__ unsigned bits[RULES_CH / 32], seen[RULES_CH / 32], word[RULES_CH], times[EACH ? RULES_CH : 1];
    __shared__ float value[BIAS ? RULES_T : 1];         // of the first bias entries
    const int tid = threadIdx.x, b = blockIdx.y, v0 = blockIdx.x * RULES_CH, n = min(RULES_CH, a.V - v0);
    const bool counts = a.rep || a.pres || a.freq;
    const uint8_t *xr = a.x + ((size_t)b * a.xs + v0) * E;
    uint8_t *yr = a.out + ((size_t)b * a.os + v0) * E;
    const uint32_t *mr = a.mask ? a.mask + (size_t)b * a.ms + v0 / 32 : nullptr;
    const ListPart h = counts ? list_part(a.hoff, b, a.hcap) : ListPart{0, 0u};
    const ListPart e = BIAS ? list_part(a.boff, b, a.bcap) : ListPart{0, 0u};
    const int *hist = a.hist + h.at, *btok = a.btok + e.at;
    const float *bval = a.bval + e.at;
    const unsigned hn = h.n, en = min(e.n, 65534u);
    const float rep = a.rep ? a.rep[b] : 1.f, pres = a.pres ? a.pres[b] : 0.f, freq = a.freq ? a.freq[b] : 0.f;
    const unsigned prompt = counts && a.npr ? max(a.npr[b], 0) : 0;
    const bool full = hn > 65535;                       // counts may reach the word's lower half
    unsigned held[RULES_HELD], held_bias = ~0u;
#pragma unroll
    for (int k = 0; k < RULES_HELD; k++) {
        const unsigned i = tid + k * RULES_T;
        held[k] = i < hn ? (unsigned)hist[i] - (unsigned)v0 : ~0u;
    }
    if (BIAS && (unsigned)tid < en) {
        held_bias = (unsigned)btok[tid] - (unsigned)v0;
        value[tid] = bval[tid];
    }
    // a thread's tokens: 8 at 8 tid + 8 RULES_T v, as they are in memory; after the lists, whose marks need not wait for them
    qt_w4 raw[NV][E / 2];
    uint32_t allow[NV];
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int i = 8 * (tid + RULES_T * v);
        allow[v] = mr && i < n ? mr[i >> 5] >> (i & 31) : 0xFFu;
        if (i + 8 <= n)
#pragma unroll
            for (int e = 0; e < E / 2; e++) raw[v][e] = qt_load16<E>(xr + (size_t)i * E + 16 * e);
    }
    if (tid < RULES_CH / 32) bits[tid] = seen[tid] = 0;
    __syncthreads();
    const auto mark = [&](unsigned t, bool hist) {
        if (t >= (unsigned)n) return;
        word[t] = 0;                                    // the same from every thread
        if (EACH) times[t] = 0;
        atomicOr(hist ? &seen[t >> 5] : &bits[t >> 5], 1u << (t & 31));
    };
    const auto count = [&](unsigned t, unsigned i) {
        if (t >= (unsigned)n) return;
        if (EACH) atomicAdd(&times[t], 1u);
        if (i < prompt) return;
        if (!full) {
            atomicAdd(&word[t], 1u);
        } else {                                        // up to 65535
            unsigned was = word[t], now;
            while ((was & 0xFFFFu) != 0xFFFFu && (now = atomicCAS(&word[t], was, was + 1u)) != was) was = now;
        }
    };
    // entry i of the biases, before any count: the largest word is the last entry's
    const auto bias = [&](unsigned t, unsigned i) {
        if (t < (unsigned)n) atomicMax(&word[t], (i + 1u) << 16);
    };
#pragma unroll
    for (int k = 0; k < RULES_HELD; k++) mark(held[k], true);
    for (unsigned i = tid + RULES_HELD * RULES_T; i < hn; i += RULES_T) mark((unsigned)hist[i] - (unsigned)v0, true);
    if (BIAS) {
        mark(held_bias, false);
        for (unsigned i = tid + RULES_T; i < en; i += RULES_T) mark((unsigned)btok[i] - (unsigned)v0, false);
        __syncthreads();
        bias(held_bias, tid);
        for (unsigned i = tid + RULES_T; i < en; i += RULES_T) bias((unsigned)btok[i] - (unsigned)v0, i);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < RULES_HELD; k++) count(held[k], tid + k * RULES_T);
    for (unsigned i = tid + RULES_HELD * RULES_T; i < hn; i += RULES_T) count((unsigned)hist[i] - (unsigned)v0, i);
    __syncthreads();
    const auto rules = [&](float y, int t) {
        if (a.rep && (seen[t >> 5] >> (t & 31) & 1u)) {
            unsigned k = EACH ? times[t] : 1u;
            float was;
            do { was = y; y = y > 0.f ? y / rep : y * rep; } while (--k && y != was);   // until nothing changes any more
        }
        const unsigned w = word[t], o = w & 0xFFFFu, last = w >> 16;
        if (o) {
            if (a.freq) y -= (float)o * freq;
            if (a.pres) y -= pres;
        }
        if (BIAS && last) y += last <= RULES_T ? value[last - 1] : bval[last - 1];
        return y;
    };
#pragma unroll
    for (int v = 0; v < NV; v++) {
        const int i = 8 * (tid + RULES_T * v);
        if (i >= n) continue;
        unsigned todo = (seen[i >> 5] | bits[i >> 5]) >> (i & 31) & allow[v] & 0xFFu;
        if (i + 8 <= n) {
            float x[8];
            qt_widen8<T>(raw[v], x);
            while (todo) {
                const int e = __builtin_ctz(todo);
                todo &= todo - 1;
                float y = x[0];
#pragma unroll
                for (int k = 1; k < 8; k++) y = k == e ? x[k] : y;
                y = rules(y, i + e);
#pragma unroll
                for (int k = 0; k < 8; k++) x[k] = k == e ? y : x[k];
            }
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = allow[v] >> e & 1u ? x[e] : -INFINITY;
            qt_store8<T, E>(yr + (size_t)i * E, x);
        } else {
            for (int e = 0; i + e < n; e++) {
                float y = qt_load1<T>(xr + (size_t)(i + e) * E);
                if (todo >> e & 1u) y = rules(y, i + e);
                qt_store1<T>(yr + (size_t)(i + e) * E, allow[v] >> e & 1u ? y : -INFINITY);
            }
        }
    }
}

extern "C" int qwen_hip_op_logit_rules(const qwen_hip_logit_rules_t *p, void *stream) {
    QT_REFUSE(!p, "logit_rules: null descriptor");
    const int E = qt_dt_size(p->dtype);
    QT_REFUSE(!E, "logit_rules: dtype %d (f32, bf16 or f16)", p->dtype);
    QT_REFUSE(p->B < 0 || p->B > 65535 || p->V < 1 || p->V > (1 << 30), "logit_rules: %d rows of %d (0..65535, 1..2^30)", p->B, p->V);
    if (p->B == 0) return 0;
    QT_REFUSE(!p->logits || !p->out, "logit_rules: null logits or out");
    QT_REFUSE(p->logits_stride < p->V || p->out_stride < p->V, "logit_rules: strides %lld, %lld under V %d", p->logits_stride,
              p->out_stride, p->V);
    QT_REFUSE(p->logits == p->out && p->logits_stride != p->out_stride, "logit_rules: in place with two strides");
    const bool counts = p->rep || p->presence || p->frequency;
    QT_REFUSE(counts && (!p->hist_off || p->hist_cap < 0 || (!p->hist && p->hist_cap > 0)), "logit_rules: penalties need a history");
    QT_REFUSE(p->bias_tok && (!p->bias_val || !p->bias_off || p->bias_cap < 0), "logit_rules: biases need values and offsets");
    QT_REFUSE(p->mask && p->mask_stride < (p->V + 31) / 32, "logit_rules: mask_stride %lld under %d words", p->mask_stride, (p->V + 31) / 32);
    QT_REFUSE(((uintptr_t)p->logits | (uintptr_t)p->out) % E, "logit_rules: logits and out have to be aligned to their elements");
    QT_REFUSE(p->logits != p->out && qt_rows_meet(p->out, p->out_stride * E, (long long)p->V * E, p->logits, p->logits_stride * E,
                                                  (long long)p->V * E, p->B),
              "logit_rules: out overlaps logits (it may be them)");
    const hipStream_t st = qt_stream(stream);
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "logit_rules: the stream's device: %s", hipGetErrorString(on.err));
    const RulesArgs a = {(const uint8_t *)p->logits, (uint8_t *)p->out, p->logits_stride, p->out_stride, p->mask_stride, p->hist,
                         p->hist_off, p->n_prompt, p->rep, p->presence, p->frequency, p->bias_tok, p->bias_val, p->bias_off,
                         p->mask, p->V, p->hist_cap, p->bias_cap, p->rep_each};
    // A row's history is read by each of its workgroups, so large vocabularies take large ones (64 rows of 128003 with histories
    // of up to 4000: 11.5 us with 1024 threads, 12.4 with 512, 18.9 with 256); up to two small ones take those (6 rows
    // of 2048: 6.1 us against 6.4).
    const int threads = p->V > 8192 ? 1024 : 256;
    const dim3 grid((p->V + 16 * threads - 1) / (16 * threads), p->B);
#define RULES3(T, BIAS, EACH) (threads == 1024 ? k_logit_rules<T, BIAS, EACH, 1024> : k_logit_rules<T, BIAS, EACH, 256>)
#define RULES2(T, BIAS) (p->rep_each ? RULES3(T, BIAS, true) : RULES3(T, BIAS, false))
#define RULES(T) (p->bias_tok ? RULES2(T, true) : RULES2(T, false))
    void (*const kernel)(RulesArgs) = p->dtype == QWEN_HIP_DT_F32    ? RULES(QtF32)
                                      : p->dtype == QWEN_HIP_DT_BF16 ? RULES(QtBf16)
                                                                     : RULES(QtF16);
#undef RULES
#undef RULES2
#undef RULES3
    const hipError_t e = qt_launch(kernel, grid, dim3(threads), 0, st, a);
    QT_REFUSE(e != hipSuccess, "logit_rules: launch failed: %s", hipGetErrorString(e));
    return 0;
}
