// The global norm of a list of gradients, and the list scaled down to a largest norm:
//     norm = sqrt(sum_i sum g_i^2),   out_i = g_i * clip / max(norm, clip)
//
// Bound by memory: the sums read every gradient once, the scaling reads and writes it once more; nothing can be written
// before the last gradient has been read.  Two launches for a list of up to 128 tensors of any types:
//   square_kernel  every workgroup walks the 32 KB chunks of the list (the list itself -- pointers, lengths, types, first
//                  chunks -- travels in the kernel's arguments, so a call copies nothing to the device and can be
//                  captured) and leaves one partial sum.  Squares are summed in 64 bits: a fp32 gradient of 1e25 or of
//                  1e-25 has a square that fp32 does not hold, and the conversion hides behind the loads.
//   scale_kernel   every workgroup adds up the partial sums in the same order (so all of them get the same bits, and so
//                  does the next call), then scales.  It walks the list from its END: the last 200 MB or so that the first
//                  launch read are still in the memory-side cache.  Out of place it copies even where nothing is clipped;
//                  in place it then returns at once.  Lists beyond that cache are read and written past it (503 MB of
//                  bf16: 280 -> 248 us); shorter ones stay in it for the optimizer that reads them next.
// 503 MB: sums 86 us (5.9 TB/s), scaling 161 us (6.2 TB/s).  1024 workgroups: what the registers let reside at once (2048
// ran in two rounds, 115 us).
// Longer lists: one launch of each kernel per 128 tensors, with norm_kernel between.
// A norm that is not finite makes every output NaN, so that a step with such gradients cannot pass unseen.
#include <stdlib.h>

#include "dense_common.h"

using namespace dense;

namespace {

constexpr int kList = 128, kChunk = 32768, kBlocks = 1024;
constexpr long kStream = 8192;                         // chunks (256 MB) that the memory-side cache holds
typedef unsigned u4 __attribute__((ext_vector_type(4)));

struct List {
    const void *p[kList];
    void *out[kList];
    long n[kList];
    int first[kList + 1];         // chunk at which a tensor starts; [count] = chunks in all
    unsigned char type[kList];
    int count;
};
static_assert(sizeof(List) < 3900, "kernel arguments end at 4 KB");

inline __host__ __device__ int per_chunk(int type) { return type == kF32 ? kChunk / 4 : kChunk / 2; }

// Sum over the 256 threads, in a fixed order, for all of them.
__device__ __forceinline__ double block_sum(double v) {
    __shared__ double part[4];
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

template <class T>
__device__ __forceinline__ double sum_squares(const T *p, long n) {      // one chunk: n <= kChunk / sizeof(T)
    constexpr int V = 16 / sizeof(T);
    struct alignas(16) Pack { T x[V]; };
    double s = 0.0;
    const int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    if (head && (int)threadIdx.x < head && threadIdx.x < n) {
        const double g = to_f32<T>(p[threadIdx.x]);
        s = g * g;
    }
    if (n <= head) return s;
    const Pack *q = (const Pack *)(p + head);
    const int packs = (int)((n - head) / V);
    if (packs == kChunk / 16) {                                          // a whole chunk: all of its loads at once
        Pack v[kChunk / 16 / 256];
#pragma unroll
        for (int i = 0; i < kChunk / 16 / 256; ++i) v[i] = q[threadIdx.x + 256 * i];
#pragma unroll
        for (int i = 0; i < kChunk / 16 / 256; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const double g = to_f32<T>(v[i].x[j]);
                s = fma(g, g, s);
            }
        return s;
    }
    for (int i = threadIdx.x; i < packs; i += 256) {
        const Pack v = q[i];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const double g = to_f32<T>(v.x[j]);
            s = fma(g, g, s);
        }
    }
    const int done = head + packs * V;
    if (done + (int)threadIdx.x < n) {
        const double g = to_f32<T>(p[done + threadIdx.x]);
        s = fma(g, g, s);
    }
    return s;
}

__global__ __launch_bounds__(256) void square_kernel(List L, double *partial) {
    const int total = L.first[L.count];
    double s = 0.0;
    int t = 0;
    for (int c = blockIdx.x; c < total; c += gridDim.x) {
        while (c >= L.first[t + 1]) ++t;
        const int type = L.type[t], per = per_chunk(type);
        const long at = (long)(c - L.first[t]) * per, left = L.n[t] - at, n = left < per ? left : per;
        if (type == kF32) s += sum_squares((const float *)L.p[t] + at, n);
        else if (type == kBF16) s += sum_squares((const bf16_t *)L.p[t] + at, n);
        else s += sum_squares((const f16_t *)L.p[t] + at, n);
    }
    s = block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__device__ __forceinline__ float norm_of(const double *partial, int count) {
    double s = 0.0;
    for (int i = threadIdx.x; i < count; i += 256) s += partial[i];
    return (float)sqrt(block_sum(s));
}

__global__ __launch_bounds__(256) void norm_kernel(const double *partial, int count, float *norm) {
    const float v = norm_of(partial, count);
    if (threadIdx.x == 0) *norm = v;
}

// What a gradient is multiplied by: `by`, after a power of two where the factor is below 2^-100.  There one fp32 number would have
// lost bits, or been 0, while the products are ordinary numbers (1e36 clipped to 1e-9).
struct Factor {
    float first, by;
};
template <class T>
__device__ __forceinline__ T scaled(T g, Factor f) { return from_f32<T>(to_f32<T>(g) * f.first * f.by); }

template <class T, bool STREAM>
__device__ __forceinline__ void scale_chunk(const T *p, T *o, long n, Factor f) {
    constexpr int V = 16 / sizeof(T);
    struct alignas(16) Pack { T x[V]; };
    if ((((uintptr_t)p ^ (uintptr_t)o) & 15) != 0) {                     // source and result differ in alignment
        for (long i = threadIdx.x; i < n; i += 256) o[i] = scaled<T>(p[i], f);
        return;
    }
    const int head = (int)((16 - ((uintptr_t)p & 15)) & 15) / (int)sizeof(T);
    if ((int)threadIdx.x < head && threadIdx.x < n) o[threadIdx.x] = scaled<T>(p[threadIdx.x], f);
    if (n <= head) return;
    const Pack *q = (const Pack *)(p + head);
    Pack *w = (Pack *)(o + head);
    const int packs = (int)((n - head) / V);
    if (packs == kChunk / 16) {
        Pack v[kChunk / 16 / 256];
#pragma unroll
        for (int i = 0; i < kChunk / 16 / 256; ++i) {
            if constexpr (STREAM) v[i] = __builtin_bit_cast(Pack, __builtin_nontemporal_load((const u4 *)q + threadIdx.x + 256 * i));
            else v[i] = q[threadIdx.x + 256 * i];
        }
#pragma unroll
        for (int i = 0; i < kChunk / 16 / 256; ++i) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[i].x[j] = scaled<T>(v[i].x[j], f);
            if constexpr (STREAM) __builtin_nontemporal_store(__builtin_bit_cast(u4, v[i]), (u4 *)w + threadIdx.x + 256 * i);
            else w[threadIdx.x + 256 * i] = v[i];
        }
        return;
    }
    for (int i = threadIdx.x; i < packs; i += 256) {
        Pack v = q[i];
#pragma unroll
        for (int j = 0; j < V; ++j) v.x[j] = scaled<T>(v.x[j], f);
        w[i] = v;
    }
    const int done = head + packs * V;
    if (done + (int)threadIdx.x < n) o[done + threadIdx.x] = scaled<T>(p[done + threadIdx.x], f);
}

// partial null: the norm is read from `given`.  norm_out may be null.
template <bool STREAM>
__global__ __launch_bounds__(256) void scale_kernel(List L, const double *partial, int count, const float *given, float clip,
                                                    float *norm_out) {
    const float norm = partial ? norm_of(partial, count) : *given;
    if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
    // a norm that is NaN, infinite or (given) negative scales by NaN
    const bool ok = norm >= 0.0f && norm <= 3.402823466e38f;
    double exact = !ok ? __builtin_nan("") : norm > clip ? (double)clip / (double)norm : 1.0;
    Factor f{1.0f, 0.0f};
    if (exact < 0x1p-100) {                            // down to 2^-277: half of the exponent first, as far as fp32 goes
        const int half = ilogb(exact) / 2;
        f.first = ldexpf(1.0f, half > -126 ? half : -126);
        exact /= f.first;
    }
    f.by = (float)exact;
    const int total = L.first[L.count];
    int t = L.count - 1;
    for (int c = total - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
        while (c < L.first[t]) --t;
        if (f.by == 1.0f && L.out[t] == L.p[t]) continue;
        const int type = L.type[t], per = per_chunk(type);
        const long at = (long)(c - L.first[t]) * per, left = L.n[t] - at, n = left < per ? left : per;
        if (type == kF32) scale_chunk<float, STREAM>((const float *)L.p[t] + at, (float *)L.out[t] + at, n, f);
        else if (type == kBF16) scale_chunk<bf16_t, STREAM>((const bf16_t *)L.p[t] + at, (bf16_t *)L.out[t] + at, n, f);
        else scale_chunk<f16_t, STREAM>((const f16_t *)L.p[t] + at, (f16_t *)L.out[t] + at, n, f);
    }
}

// The next up to kList tensors with elements, from index `at` on; returns the index behind them, or -1 where the lengths
// do not fit (chunk numbers are 32-bit).
int fill(List &L, int at, int count, const void *const *p, void *const *out, const long *n, const int *type) {
    L.count = 0;
    long chunks = 0;
    for (; at < count && L.count < kList; ++at) {
        if (n[at] == 0) continue;
        const int i = L.count++;
        L.p[i] = p[at];
        L.out[i] = out ? out[at] : nullptr;
        L.n[i] = n[at];
        L.type[i] = (unsigned char)type[at];
        L.first[i] = (int)chunks;
        chunks += (n[at] + per_chunk(type[at]) - 1) / per_chunk(type[at]);
        if (chunks > 0x7ffffff0L - kBlocks) return -1;
    }
    L.first[L.count] = (int)chunks;
    return at;
}
inline int blocks_of(const List &L) {
    const int c = L.first[L.count];
    return c < kBlocks ? c : kBlocks;
}

bool list_ok(int count, const void *const *p, void *const *out, bool wants_out, const long *n, const int *type) {
    if (count < 0 || (count && (!p || !n || !type || (wants_out && !out)))) return false;
    for (int i = 0; i < count; ++i) {
        if (n[i] < 0 || type[i] < kF32 || type[i] > kF16) return false;
        const uintptr_t mask = type[i] == kF32 ? 3 : 1;
        if (n[i] && (!p[i] || ((uintptr_t)p[i] & mask) || (wants_out && (!out[i] || ((uintptr_t)out[i] & mask))))) return false;
    }
    return true;
}
// Bytes of a tensor that is written.
struct Span {
    uintptr_t lo, hi;
};
int by_start(const void *a, const void *b) {
    const uintptr_t x = ((const Span *)a)->lo, y = ((const Span *)b)->lo;
    return x < y ? -1 : x > y;
}
bool meets(const Span *w, int count, Span r) {         // w: disjoint, in order
    int lo = 0, hi = count;                            // the first that starts at or behind r's end
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (w[mid].lo < r.hi) lo = mid + 1;
        else hi = mid;
    }
    return lo > 0 && w[lo - 1].hi > r.lo;
}
// Workgroups read and write in no order: results may not overlap one another, nor anything that is read but their own
// gradient, which they may only share whole.
int check_overlap(int count, const void *const *p, void *const *out, const long *n, const int *type, const float *use_norm) {
    if (count == 0) return SA_OK;
    Span *w = (Span *)malloc(sizeof(Span) * count);
    if (!w) return SA_ERR_INVALID;
    int used = 0;
    auto span = [&](const void *q, int i) { return Span{(uintptr_t)q, (uintptr_t)q + n[i] * (type[i] == kF32 ? 4 : 2)}; };
    for (int i = 0; i < count; ++i)
        if (n[i]) w[used++] = span(out[i], i);
    qsort(w, used, sizeof(Span), by_start);
    bool bad = false;
    for (int i = 1; i < used; ++i) bad = bad || w[i].lo < w[i - 1].hi;
    for (int i = 0; i < count && !bad; ++i)
        if (n[i] && out[i] != p[i]) bad = meets(w, used, span(p[i], i));
    if (!bad && use_norm) bad = meets(w, used, Span{(uintptr_t)use_norm, (uintptr_t)use_norm + 4});
    free(w);
    return bad ? SA_ERR_INVALID : SA_OK;
}
inline unsigned long ws_need(int count) { return (unsigned long)((count + kList - 1) / kList) * kBlocks * sizeof(double); }

// The partial sums of the whole list; *used = how many, *lists = launches made.
int square(int count, const void *const *p, const long *n, const int *type, double *partial, int *used, int *lists, List &L,
           hipStream_t s) {
    *used = *lists = 0;
    for (int at = 0; at < count;) {
        at = fill(L, at, count, p, nullptr, n, type);
        if (at < 0) return SA_ERR_UNSUPPORTED;
        if (L.count == 0) break;
        const int g = blocks_of(L);
        hipLaunchKernelGGL(square_kernel, dim3(g), dim3(256), 0, s, L, partial + *used);
        SA_CHECK_LAUNCH();
        *used += g;
        ++*lists;
    }
    return SA_OK;
}

}  // namespace

extern "C" int sa_global_norm_ws(int count, unsigned long *bytes) {
    if (count < 0 || !bytes) return SA_ERR_INVALID;
    *bytes = ws_need(count);
    return SA_OK;
}

extern "C" int sa_global_norm(int count, const void *const *p, const long *n, const int *type, float *norm, void *ws,
                              unsigned long ws_bytes, void *stream) {
    if (!list_ok(count, p, nullptr, false, n, type) || !norm || ws_bytes < ws_need(count) || (count && !ws)) return SA_ERR_INVALID;
    hipStream_t s = (hipStream_t)stream;
    List L;
    int used, lists;
    const int rc = square(count, p, n, type, (double *)ws, &used, &lists, L, s);
    if (rc) return rc;
    hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(256), 0, s, (const double *)ws, used, norm);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

extern "C" int sa_clip_by_global_norm(int count, const void *const *p, void *const *out, const long *n, const int *type,
                                      float clip, const float *use_norm, float *norm, void *ws, unsigned long ws_bytes,
                                      void *stream) {
    if (!list_ok(count, p, out, true, n, type) || !(clip > 0.0f)) return SA_ERR_INVALID;
    if (check_overlap(count, p, out, n, type, use_norm) != SA_OK) return SA_ERR_INVALID;
    hipStream_t s = (hipStream_t)stream;
    List L;
    int used = 0, lists = 0;
    if (!use_norm) {
        if (!norm || ws_bytes < ws_need(count) || (count && !ws)) return SA_ERR_INVALID;
        const int rc = square(count, p, n, type, (double *)ws, &used, &lists, L, s);
        if (rc) return rc;
        if (lists != 1) {
            hipLaunchKernelGGL(norm_kernel, dim3(1), dim3(256), 0, s, (const double *)ws, used, norm);
            SA_CHECK_LAUNCH();
        }
    }
    const bool direct = !use_norm && lists == 1;
    long bytes = 0;
    for (int i = 0; i < count; ++i) bytes += n[i] * (type[i] == kF32 ? 4 : 2);
    const bool stream_it = bytes > kStream * kChunk;
    for (int at = 0; at < count;) {
        at = fill(L, at, count, p, out, n, type);
        if (at < 0) return SA_ERR_UNSUPPORTED;
        if (L.count == 0) break;
        hipLaunchKernelGGL(stream_it ? scale_kernel<true> : scale_kernel<false>, dim3(blocks_of(L)), dim3(256), 0, s, L,
                           direct ? (const double *)ws : nullptr, used, use_norm ? use_norm : norm, clip, direct ? norm : nullptr);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}
