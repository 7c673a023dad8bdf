// qt_logits.hip — the rules on a batch's logits before sampling (qwen_hip_op_logit_rules): repetition,
// presence and frequency penalties, token biases, an allowed-token bit mask.
//
// A workgroup takes RULES_CH neighbouring tokens of one row.  It counts the row's history entries that fall on them in
// LDS (integer atomics: the order does not matter), finds each token's last bias entry there the same way (the
// largest index wins), then streams its logits once.  So a row's history is read once a workgroup, from the L2,
// and no counts of V tokens a row are held in global memory, cleared or read back.
// Bound by the logits' bytes for a large vocabulary, by the latency of offsets, history and logits for a small one.
#include "qt_ops.h"

#define RULES_T 256
#define RULES_CH 4096

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

// BIAS: with bias lists.  Rows may begin anywhere that their elements can: 16-byte accesses at 2- or 4-byte
// alignment are one instruction on this GPU.
template <typename T, bool BIAS>
__global__ __launch_bounds__(RULES_T) void k_logit_rules(RulesArgs a) {
    constexpr int E = sizeof(typename T::elem);
    __shared__ __align__(16) unsigned seen[RULES_CH], said[RULES_CH];
    __shared__ __align__(16) int last[BIAS ? RULES_CH : 4];
    const int tid = threadIdx.x, b = blockIdx.y, v0 = blockIdx.x * RULES_CH, n = min(RULES_CH, a.V - v0);
    const bool counts = a.rep || a.pres || a.freq;
    if (counts || BIAS) {
        for (int i = tid; i < RULES_CH; i += RULES_T) {
            seen[i] = 0; said[i] = 0;
            if (BIAS) last[i] = -1;
        }
        __syncthreads();
        if (counts) {
            const int h0 = max(a.hoff[b], 0), h1 = min(a.hoff[b + 1], a.hcap);
            const long long h2 = a.npr ? (long long)h0 + max(a.npr[b], 0) : h0;
            for (int i = h0 + tid; i < h1; i += RULES_T) {
                const unsigned t = (unsigned)a.hist[i] - (unsigned)v0;
                if (t >= (unsigned)n) continue;
                atomicAdd(&seen[t], 1u);
                if (i >= h2) atomicAdd(&said[t], 1u);
            }
        }
        if (BIAS) {
            const int e0 = max(a.boff[b], 0), e1 = min(a.boff[b + 1], a.bcap);
            for (int i = e0 + tid; i < e1; i += RULES_T) {
                const unsigned t = (unsigned)a.btok[i] - (unsigned)v0;
                if (t < (unsigned)n) atomicMax(&last[t], i);
            }
        }
        __syncthreads();
    }
    const float rep = a.rep ? a.rep[b] : 1.f, pres = a.pres ? a.pres[b] : 0.f, freq = a.freq ? a.freq[b] : 0.f;
    const uint8_t *xr = a.x + (size_t)b * a.xs * E;
    uint8_t *yr = a.out + (size_t)b * a.os * E;
    const uint32_t *mr = a.mask ? a.mask + (size_t)b * a.ms : nullptr;
    const auto rules = [&](float x, int i, uint32_t allowed) {
        if (counts) {
            const unsigned c = seen[i], o = said[i];
            if (c && a.rep) {
                // once, or once for every entry until nothing changes any more
                float was;
                unsigned k = a.each ? c : 1u;
                do { was = x; x = x > 0.f ? x / rep : x * rep; } while (--k && x != was);
            }
            if (o) {
                if (a.freq) x -= (float)o * freq;
                if (a.pres) x -= pres;
            }
        }
        if (BIAS) {
            const int e = last[i];
            if (e >= 0) x += a.bval[e];
        }
        return allowed & 1u ? x : -INFINITY;
    };
    for (int i = 8 * tid; i < n; i += 8 * RULES_T) {
        const int t = v0 + i;
        const uint32_t bits = mr ? mr[t >> 5] >> (t & 31) : 0xFFu;
        if (i + 8 <= n) {
            float x[8];
            qt_load8<T, E>(xr + (size_t)t * E, x);
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = rules(x[e], i + e, bits >> e);
            qt_store8<T, E>(yr + (size_t)t * E, x);
        } else {
            for (int e = 0; i + e < n; e++)
                qt_store1<T>(yr + (size_t)(t + e) * E, rules(qt_load1<T>(xr + (size_t)(t + e) * E), i + e, bits >> e));
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
    hipStream_t st = (hipStream_t)stream;
    QtOnDevice on(st);
    QT_REFUSE(on.err != hipSuccess, "logit_rules: the stream's device: %s", hipGetErrorString(on.err));
    const RulesArgs a = {(const uint8_t *)p->logits, (uint8_t *)p->out, p->logits_stride, p->out_stride, p->mask_stride, p->hist,
                         p->hist_off, p->n_prompt, p->rep, p->presence, p->frequency, p->bias_tok, p->bias_val, p->bias_off,
                         p->mask, p->V, p->hist_cap, p->bias_cap, p->rep_each};
    const dim3 grid((p->V + RULES_CH - 1) / RULES_CH, p->B);
#define RULES(T) do { \
        if (p->bias_tok) hipLaunchKernelGGL((k_logit_rules<T, true>), grid, dim3(RULES_T), 0, st, a); \
        else hipLaunchKernelGGL((k_logit_rules<T, false>), grid, dim3(RULES_T), 0, st, a); } while (0)
    if (p->dtype == QWEN_HIP_DT_F32) RULES(QtF32);
    else if (p->dtype == QWEN_HIP_DT_BF16) RULES(QtBf16);
    else RULES(QtF16);
#undef RULES
    const hipError_t e = hipGetLastError();
    QT_REFUSE(e != hipSuccess, "logit_rules: launch failed: %s", hipGetErrorString(e));
    return 0;
}
