// qt_ops.h — what the operators of paged, batched serving share: element types, rounding, the
// division by a page size, and the host side of a call (the stream's device, argument checks).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qt_device.h"
#include "qwen_tts_hip.h"

extern "C" void qt_seterr(const char *fmt, ...) __attribute__((format(printf, 1, 2)));   // qwen_hip_last_error's text

// Element types, as template arguments.  Every load widens to f32, every store rounds once to the
// nearest, ties to even (bf16 off by at most 2^-8 of the value, f16 by 2^-11).
struct QtF32 { typedef float elem; };
struct QtBf16 { typedef uint16_t elem; };
struct QtF16 { typedef uint16_t elem; };
struct QtE4m3 { typedef uint8_t elem; };    // codes of a quantised cache, whose rows have a scale beside them

template <typename T> __device__ __forceinline__ uint32_t qt_round2(float a, float b);
template <> __device__ __forceinline__ uint32_t qt_round2<QtBf16>(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{a, b}), b2));
}
template <> __device__ __forceinline__ uint32_t qt_round2<QtF16>(float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, (h2{(_Float16)a, (_Float16)b}));
}
template <typename T> __device__ __forceinline__ float qt_lo(uint32_t u);
template <typename T> __device__ __forceinline__ float qt_hi(uint32_t u);
template <> __device__ __forceinline__ float qt_lo<QtBf16>(uint32_t u) { return __uint_as_float(u << 16); }
template <> __device__ __forceinline__ float qt_hi<QtBf16>(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }
template <> __device__ __forceinline__ float qt_lo<QtF16>(uint32_t u) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(u & 0xFFFFu));
}
template <> __device__ __forceinline__ float qt_hi<QtF16>(uint32_t u) {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> 16));
}

// 8 consecutive elements; p needs `A` bytes of alignment
typedef uint32_t qt_w4 __attribute__((ext_vector_type(4)));
template <int A> __device__ __forceinline__ qt_w4 qt_load16(const void *p) {
    qt_w4 a;
    __builtin_memcpy(&a, __builtin_assume_aligned(p, A), 16);
    return a;
}
template <int A> __device__ __forceinline__ void qt_store16(void *p, qt_w4 a) { __builtin_memcpy(__builtin_assume_aligned(p, A), &a, 16); }
template <typename T, int N> __device__ __forceinline__ void qt_widen8(const qt_w4 (&w)[N], float (&v)[8]) {
    if constexpr (N == 2) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = __uint_as_float(w[i >> 2][i & 3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) { v[2 * i] = qt_lo<T>(w[0][i]); v[2 * i + 1] = qt_hi<T>(w[0][i]); }
    }
}
template <typename T, int A = 16> __device__ __forceinline__ void qt_load8(const void *p, float (&v)[8]) {
    static_assert(sizeof(typename T::elem) >= 2, "codes: qt_widen_e4m3");
    qt_w4 w[sizeof(typename T::elem) / 2];
#pragma unroll
    for (unsigned e = 0; e < sizeof(typename T::elem) / 2; e++) w[e] = qt_load16<A>((const uint8_t *)p + 16 * e);
    qt_widen8<T>(w, v);
}
template <typename T, int A = 16> __device__ __forceinline__ void qt_store8(void *p, const float (&v)[8]) {
    uint8_t *b = (uint8_t *)p;
    qt_w4 x, y;
    if constexpr (sizeof(typename T::elem) == 4) {
#pragma unroll
        for (int i = 0; i < 4; i++) { x[i] = __float_as_uint(v[i]); y[i] = __float_as_uint(v[4 + i]); }
        qt_store16<A>(b, x);
        qt_store16<A>(b + 16, y);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = qt_round2<T>(v[2 * i], v[2 * i + 1]);
        qt_store16<A>(b, x);
    }
}
// 8 codes as the numbers they stand for, and 8 numbers of at most 448 as the nearest codes, ties to even
__device__ __forceinline__ void qt_widen_e4m3(uint32_t lo, uint32_t hi, float (&v)[8]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)lo, true);
    const f2 c = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)hi, true);
    v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1]; v[4] = c[0]; v[5] = c[1]; v[6] = d[0]; v[7] = d[1];
}
__device__ __forceinline__ uint2 qt_codes_e4m3(const float (&v)[8]) {
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false), hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4], v[5], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], lo, true);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6], v[7], hi, true);
    return make_uint2((unsigned)lo, (unsigned)hi);
}
// The byte of a row whose largest magnitude has the bits m: 2^e is enough for 448 2^e = 1.75 2^(e + 8) where e is m's exponent
// less 8, and one more past a fraction of 1.75, which then carries.  Magnitudes of 2^127 and more, infinities and NaN, whose bits
// order after them: 255.
#define QT_SCALE_MIN 63u        // 2^-64
#define QT_SCALE_MAX 246u       // of 448 2^119, the largest code under 2^127
__device__ __forceinline__ uint32_t qt_scale_byte(uint32_t m) {
    if (m >= 0x7F000000u) return 255u;
    const uint32_t e = (m + 0x1FFFFFu) >> 23;
    return e < QT_SCALE_MIN + 8u ? QT_SCALE_MIN : e - 8u;
}
// a byte as its row is read: NaN past the largest that is written
__device__ __forceinline__ float qt_scale_of(uint32_t byte) {
    return byte > QT_SCALE_MAX ? __uint_as_float(0x7FC00000u) : __uint_as_float(max(byte, QT_SCALE_MIN) << 23);
}

template <typename T> __device__ __forceinline__ float qt_load1(const void *p) {
    if constexpr (sizeof(typename T::elem) == 4) return *reinterpret_cast<const float *>(p);
    else if constexpr (sizeof(typename T::elem) == 1) return __builtin_amdgcn_cvt_f32_fp8(*reinterpret_cast<const uint8_t *>(p), 0);
    else return qt_lo<T>(*reinterpret_cast<const uint16_t *>(p));
}
template <typename T> __device__ __forceinline__ void qt_store1(void *p, float v) {
    if constexpr (sizeof(typename T::elem) == 4) *reinterpret_cast<float *>(p) = v;
    else *reinterpret_cast<uint16_t *>(p) = (uint16_t)qt_round2<T>(v, 0.f);
}

// n / d for 0 <= n < 2^31 by one product: m = ceil(2^(31 + l) / d) with l = ceil(log2 d), so m d exceeds 2^(31 + l)
// by less than d <= 2^l, and n times that excess stays under 2^(31 + l).
struct QtDiv { uint32_t m, l; };
static inline QtDiv qt_div_of(int d) {
    uint32_t l = 0;
    while ((1u << l) < (uint32_t)d) l++;
    return {(uint32_t)(((1ull << (31 + l)) + (uint32_t)d - 1) / (uint32_t)d), l};
}
__device__ __forceinline__ int qt_quot(int n, QtDiv d) { return (int)(__umulhi(2u * (uint32_t)n, d.m) >> d.l); }

// Over a wave's 64 lanes by DPP: the largest of non-negative v, in every lane; the running sum up to each lane.
template <int CTRL, int ROWS> __device__ __forceinline__ int qt_dpp0(int v) {        // 0 from lanes that there are not
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ int wave_scan_i(int v) {
    v += qt_dpp0<0x111, 0xf>(v);                         // lanes 1, 2, 4, 8 before, in rows of 16
    v += qt_dpp0<0x112, 0xf>(v);
    v += qt_dpp0<0x114, 0xf>(v);
    v += qt_dpp0<0x118, 0xf>(v);
    v += qt_dpp0<DPP_BCAST15, 0xa>(v);
    return v + qt_dpp0<DPP_BCAST31, 0xc>(v);
}
__device__ __forceinline__ int wave_max_i(int v) {
    v = max(v, qt_dpp0<0x111, 0xf>(v));
    v = max(v, qt_dpp0<0x112, 0xf>(v));
    v = max(v, qt_dpp0<0x114, 0xf>(v));
    v = max(v, qt_dpp0<0x118, 0xf>(v));
    v = max(v, qt_dpp0<DPP_BCAST15, 0xa>(v));
    v = max(v, qt_dpp0<DPP_BCAST31, 0xc>(v));
    return __builtin_amdgcn_readlane(v, 63);
}

// ---- host side ----

// hipStreamLegacy is another name of the null stream, and one that not every runtime's hipStreamGetDevice takes.
static inline hipStream_t qt_stream(void *stream) { return (hipStream_t)stream == hipStreamLegacy ? nullptr : (hipStream_t)stream; }

// Makes the stream's device the current one while a call launches (kernels are looked up for the
// current device), and the caller's current again afterwards.
struct QtOnDevice {
    int cur = -1, dev = -1;
    hipError_t err = hipSuccess;
    explicit QtOnDevice(hipStream_t st) {
        if (!st) return;                                   // the null stream is the current device's
        err = hipStreamGetDevice(st, &dev);
        if (err == hipSuccess) err = hipGetDevice(&cur);
        if (err == hipSuccess && cur != dev) err = hipSetDevice(dev);
    }
    ~QtOnDevice() {
        if (cur >= 0 && dev >= 0 && cur != dev) (void)hipSetDevice(cur);
    }
    QtOnDevice(const QtOnDevice &) = delete;
    QtOnDevice &operator=(const QtOnDevice &) = delete;
};

// Launches a kernel.  The status is this launch's own: the thread's last error may be one that an earlier call left, and
// stays the caller's to read.
template <typename Args>
static inline hipError_t qt_launch(void (*kernel)(Args), dim3 grid, dim3 block, size_t lds, hipStream_t st, Args args) {
    void *p[] = {&args};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, p, lds, st);
    if (e != hipSuccess) (void)hipGetLastError();
    return e;
}

#define QT_REFUSE(cond, ...) do { if (cond) { qt_seterr(__VA_ARGS__); return -1; } } while (0)

static inline int qt_dt_size(int dt) { return dt == QWEN_HIP_DT_F32 ? 4 : dt == QWEN_HIP_DT_BF16 || dt == QWEN_HIP_DT_F16 ? 2 : 0; }
// Whether n rows of aw bytes, as apart (at least aw), share memory with n rows of bw bytes, bs apart (0: one row).  Row i of
// one meets row i + d of the other where a - b + d as lies between -aw and bw: the first d past the lower end decides.  Rows of two
// strides count as sharing memory where their ranges do.
static inline bool qt_rows_meet(const void *a, long long as, long long aw, const void *b, long long bs, long long bw, long long n) {
    const long long D = (long long)((intptr_t)a - (intptr_t)b);
    if (D >= (n - 1) * bs + bw || -D >= (n - 1) * as + aw) return false;
    if (n == 1 || (bs != as && bs != 0)) return true;
    const long long x = -aw - D;                                      // the first d with d as > x
    long long d = (x >= 0 ? x / as : -((-x + as - 1) / as)) + 1;
    if (d < (bs ? 1 - n : 0)) d = bs ? 1 - n : 0;
    return d < n && D + d * as < bw;
}
// Whether one of the outputs shares memory with another one or with an input.  `same`: an output that may be that input itself.
struct QtMem { const void *p; long long bytes; const char *name; const void *same; };
static inline const QtMem *qt_meets(const QtMem *out, int n_out, const QtMem *in, int n_in) {
    const auto meet = [](const QtMem &a, const QtMem &b) {
        const intptr_t x = (intptr_t)a.p, y = (intptr_t)b.p;
        return a.p && b.p && a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
    };
    for (int i = 0; i < n_out; i++) {
        for (int j = i + 1; j < n_out; j++)
            if (meet(out[i], out[j])) return &out[i];
        for (int j = 0; j < n_in; j++)
            if (meet(out[i], in[j]) && !(out[i].p == in[j].p && out[i].same == in[j].p)) return &out[i];
    }
    return nullptr;
}
static inline bool qt_off16(const void *p) { return ((uintptr_t)p & 15) != 0; }

// bytes of a cache's element
static inline int qt_kv_size(int dt) { return dt == QWEN_HIP_DT_E4M3 ? 1 : 2; }

// the cache's descriptor; `who` names the call
static inline int qt_check_pages(const char *who, const qwen_hip_kv_pages_t *kv) {
    QT_REFUSE(!kv, "%s: null cache descriptor", who);
    QT_REFUSE(!kv->k || !kv->v, "%s: null cache pointer", who);
    const bool codes = kv->dtype == QWEN_HIP_DT_E4M3;
    QT_REFUSE(kv->dtype != QWEN_HIP_DT_BF16 && kv->dtype != QWEN_HIP_DT_F16 && !codes, "%s: cache dtype %d (bf16, f16 or e4m3)", who, kv->dtype);
    QT_REFUSE(kv->head_dim != 64 && kv->head_dim != 128, "%s: head_dim %d (64 or 128)", who, kv->head_dim);
    QT_REFUSE(kv->n_kv_heads < 1 || kv->n_kv_heads > 65535, "%s: n_kv_heads %d out of range (1..65535)", who, kv->n_kv_heads);
    QT_REFUSE(kv->n_pages < 1 || kv->page_size < 1 || (long long)kv->n_pages * kv->page_size > 0x7FFFFFFFll,
              "%s: %d pages of %d (both at least 1, 2^31 - 1 slots at most)", who, kv->n_pages, kv->page_size);
    QT_REFUSE(qt_off16(kv->k) || qt_off16(kv->v), "%s: cache pointers have to be aligned to 16 bytes", who);
    const int A = 16 / qt_kv_size(kv->dtype);
    QT_REFUSE(kv->page_stride % A || kv->head_stride % A || kv->slot_stride % A || kv->page_stride < 0 || kv->head_stride < 0 ||
                  kv->slot_stride < 0,
              "%s: cache strides %lld, %lld, %lld (multiples of %d elements, not negative)", who, kv->page_stride,
              kv->head_stride, kv->slot_stride, A);
    QT_REFUSE((kv->n_pages > 1 && kv->page_stride < kv->head_dim) || (kv->n_kv_heads > 1 && kv->head_stride < kv->head_dim) ||
                  (kv->page_size > 1 && kv->slot_stride < kv->head_dim),
              "%s: cache strides %lld, %lld, %lld under head_dim %d: rows would overlap", who, kv->page_stride, kv->head_stride,
              kv->slot_stride, kv->head_dim);
    if (!codes) return 0;
    QT_REFUSE(!kv->k_scale || !kv->v_scale, "%s: null scale pointer", who);
    QT_REFUSE(kv->scale_page_stride < 0 || kv->scale_head_stride < 0 || kv->scale_slot_stride < 0,
              "%s: scale strides %lld, %lld, %lld are negative", who, kv->scale_page_stride, kv->scale_head_stride, kv->scale_slot_stride);
    return 0;
}

// A cache that is written: every place's row is memory of its own, in k and in v.  The strides nest (each is at least the extent of all
// smaller ones), as they do in any order of pages, heads and places; so a row of v meets one of k only where their distance
// is, stride by stride from the largest, the multiple below or above what is left of it, and less than a row at the end.
struct QtDim { __int128 stride, count; };
static inline bool qt_dims_meet(const QtDim *d, int n, __int128 left, int row) {
    if (n == 0) return left < row && -left < row;
    const __int128 s = d[n - 1].stride, c = left / s - (left % s < 0);
    return (c < d[n - 1].count && -c < d[n - 1].count && qt_dims_meet(d, n - 1, left - c * s, row)) ||
           (c + 1 < d[n - 1].count && -(c + 1) < d[n - 1].count && qt_dims_meet(d, n - 1, left - (c + 1) * s, row));
}
// Whether one of the stretches `bw` wide meets one of those `aw` wide, the first of which is `left` before theirs: two of them are left + sum t_i stride_i
// apart, lo_i <= t_i <= hi_i, the largest stride last.  Those that reach over many strides count as meeting.
struct QtRange { __int128 stride, lo, hi; };
static inline bool qt_stretches_meet(const QtRange *d, int n, __int128 left, __int128 aw, __int128 bw) {
    if (n == 0) return left < aw && -left < bw;
    const __int128 s = d[n - 1].stride;
    __int128 least = 0, most = 0;                                     // what the smaller strides add
    for (int i = 0; i < n - 1; i++) { least += d[i].lo * d[i].stride; most += d[i].hi * d[i].stride; }
    const auto down = [s](__int128 x) { return x / s - (x % s < 0); };
    __int128 t = down(-bw - left - most) + 1, end = -down(-(aw - left - least)) - 1;
    if (t < d[n - 1].lo) t = d[n - 1].lo;
    if (end > d[n - 1].hi) end = d[n - 1].hi;
    if (end - t > 8) return true;
    for (; t <= end; t++)
        if (qt_stretches_meet(d, n - 1, left + t * s, aw, bw)) return true;
    return false;
}
// rows of `row` units (at k, and `between` units further at v); the strides in units
static inline int qt_check_rows_apart(const char *who, const char *what, const qwen_hip_kv_pages_t *kv, long long page, long long head, long long slot,
                                      int row, __int128 between, int layers, long long layer) {
    QtDim all[4] = {{page, kv->n_pages}, {head, kv->n_kv_heads}, {slot, kv->page_size}, {layer, layers}}, d[4];
    int n = 0;
    __int128 extent = row;
    for (int i = 0; i < 4; i++) {
        if (all[i].count == 1) continue;
        int at = n++;
        for (; at > 0 && d[at - 1].stride > all[i].stride; at--) d[at] = d[at - 1];
        d[at] = all[i];
    }
    for (int i = 0; i < n; i++) {
        QT_REFUSE(d[i].stride < extent, "%s: %s strides %lld, %lld, %lld: rows of different places%s overlap", who, what, page, head, slot, layers > 1 ? " or layers" : "");
        extent += (d[i].count - 1) * d[i].stride;
    }
    QT_REFUSE(qt_dims_meet(d, n, between, row), "%s: %s: rows of k and v overlap", who, what);
    return 0;
}
static inline int qt_check_pages_apart(const char *who, const qwen_hip_kv_pages_t *kv, int layers = 1, long long layer = 0, long long scale_layer = 0) {
    const int E = qt_kv_size(kv->dtype);
    if (qt_check_rows_apart(who, "cache", kv, kv->page_stride, kv->head_stride, kv->slot_stride, kv->head_dim,
                            ((intptr_t)kv->v - (intptr_t)kv->k) / E, layers, layer))     // both aligned to 16
        return -1;
    if (kv->dtype != QWEN_HIP_DT_E4M3) return 0;
    if (qt_check_rows_apart(who, "scale", kv, kv->scale_page_stride, kv->scale_head_stride, kv->scale_slot_stride, 1,
                            (__int128)((intptr_t)kv->v_scale - (intptr_t)kv->k_scale), layers, scale_layer))
        return -1;
    // A page's codes and a page's scales, each as one stretch, and all pages' as one more where they are of two strides
    __int128 cw = (__int128)(kv->n_kv_heads - 1) * kv->head_stride + (__int128)(kv->page_size - 1) * kv->slot_stride + kv->head_dim;
    __int128 sw = (__int128)(kv->n_kv_heads - 1) * kv->scale_head_stride + (__int128)(kv->page_size - 1) * kv->scale_slot_stride + 1;
    const __int128 pages = kv->n_pages - 1, more = layers - 1;
    QtRange d[3];
    int n = 0;
    if (pages && kv->page_stride == kv->scale_page_stride) {
        d[n++] = {kv->page_stride, -pages, pages};
    } else {
        cw += pages * kv->page_stride;
        sw += pages * kv->scale_page_stride;
    }
    if (more && layer == scale_layer) {
        d[n++] = {layer, -more, more};
    } else if (more) {
        d[n++] = {layer, -more, 0};
        d[n++] = {scale_layer, 0, more};
    }
    for (int i = 1; i < n; i++)
        for (int k = i; k > 0 && d[k - 1].stride > d[k].stride; k--) { const QtRange x = d[k]; d[k] = d[k - 1]; d[k - 1] = x; }
    for (const void *c : {kv->k, kv->v})
        for (const uint8_t *s : {kv->k_scale, kv->v_scale})
            QT_REFUSE(qt_stretches_meet(d, n, (intptr_t)s - (intptr_t)c, cw, sw), "%s: scales lie among the codes of a page", who);
    return 0;
}
