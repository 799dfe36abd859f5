// Shared by the dense layer's kernels (dense.hip): element types, activations and their slopes, the
// epilogue that every product ends in, and the description of one product.
//
//   forward          Z = X W + b,  Y = act(Z) + R                        X [rows,cin], W [cin,cout], R [rows,cout]
//   backward         dZ = G act'(Z),  dX = dZ W^T,  dW = X^T dZ,  db = column sums of dZ
//
// All three products are D(m,n) = sum_k A(m,k) B(n,k); what differs is which index of an operand is contiguous:
//   forward  A = X  (k contiguous)   B = W   (n contiguous)
//   dX       A = dZ (k contiguous)   B = W   (k contiguous)
//   dW       A = X  (m contiguous)   B = dZ  (n contiguous)
#pragma once
#include "sa_common.h"

namespace dense {

enum Type { kF32 = 0, kBF16 = 1, kF16 = 2 };
enum Act { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4, kPlanes = 5 };      // kPlanes: see Product::zact
constexpr int kRoundSlopes = 16;      // added to a gradient's activation: a 16-bit dZ is rounded instead of going in two planes

typedef float f4 __attribute__((ext_vector_type(4)));
typedef short s8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// 16-bit elements travel as bit patterns in tags of their own, so that a template knows which it has
struct bf16_t { unsigned short u; };
struct f16_t { unsigned short u; };

template <class T> __device__ __forceinline__ float to_f32(T v);
template <> __device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f32<bf16_t>(bf16_t v) { return __uint_as_float((unsigned)v.u << 16); }
template <> __device__ __forceinline__ float to_f32<f16_t>(f16_t v) { return (float)__builtin_bit_cast(_Float16, v.u); }
// round to nearest even; overflow to infinity, NaN stays NaN
template <class T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ bf16_t from_f32<bf16_t>(float v) {
    return bf16_t{__builtin_bit_cast(unsigned short, (__bf16)v)};
}
template <> __device__ __forceinline__ f16_t from_f32<f16_t>(float v) {
    return f16_t{__builtin_bit_cast(unsigned short, (_Float16)v)};
}

// ---- activations -------------------------------------------------------------------------------------------------
// In fp32 whatever the type, with the hardware's exp2 and reciprocal (an ulp each): the epilogue of a 128 x 128 tile with the
// library's erfc took 35 us where its products take 15.  exp may overflow to infinity, which gives the right 0.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * 1.4426950408889634f); }
__device__ __forceinline__ float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }
constexpr float kGeluC = 1.5957691216057308f;        // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

// The normal distribution's lower tail at -|z|, and exp(-z^2 / 2).  erfc(x) exp(x^2) / t is smooth in t = 1 / (1 + 0.3 x); the
// polynomial is a least-squares fit of it, reweighted towards equal errors over 0 <= x <= 9.6 (2e-8 relative).  No
// cancellation: the tail is relatively exact to a few ulps of its exponent.
__device__ __forceinline__ float normal_tail(float z, float &bell) {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.3f * 0.70710678118654752f, fabsf(z), 1.0f));
    float q = -0.129458237f;
    q = fmaf(q, t, 0.485223401f);
    q = fmaf(q, t, -0.511512505f);
    q = fmaf(q, t, 0.546755526f);
    q = fmaf(q, t, -0.0939086903f);
    q = fmaf(q, t, 0.214569621f);
    q = fmaf(q, t, 0.148443406f);
    q = fmaf(q, t, 0.170698284f);
    q = fmaf(q, t, 0.169189176f);
    bell = __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
    return 0.5f * bell * t * q;
}

template <int ACT>
__device__ __forceinline__ float activate(float z) {
    if constexpr (ACT == kRelu) return z > 0.0f ? z : (z != z ? z : 0.0f);              // NaN passes through
    if constexpr (ACT == kGelu) {
        float bell;
        const float tail = normal_tail(z, bell);
        return z * (z >= 0.0f ? 1.0f - tail : tail);
    }
    if constexpr (ACT == kGeluTanh) return z * logistic(kGeluC * (z + kGeluA * z * z * z));     // 0.5 (1 + tanh u) = logistic(2 u)
    if constexpr (ACT == kSilu) return z * logistic(z);
    return z;
}
// f(std::integral_constant-like tag of the activation): one branch for a whole row instead of one per element
template <int V> struct Tag { static constexpr int value = V; };
template <class F>
__device__ __forceinline__ void with_activation(int act, F &&f) {
    switch (act) {
        case kRelu: return f(Tag<kRelu>{});
        case kGelu: return f(Tag<kGelu>{});
        case kGeluTanh: return f(Tag<kGeluTanh>{});
        case kSilu: return f(Tag<kSilu>{});
        default: return f(Tag<kNone>{});
    }
}
// g act'(z).  ReLU selects: what a closed unit receives, infinities among it, does not come through.  An infinite z has the slope
// 0 or 1 (a fp16 z is kept as an infinity from 65520 on, where the forward pass had a finite one): past |z| = 14, 12 or 110 the
// integral or the logistic is 0 or 1 to every bit, and the product beside it, in which z may be infinite and the other factor
// 0, is left out.
template <int ACT>
__device__ __forceinline__ float times_slope(float g, float z) {
    if constexpr (ACT == kRelu) return z > 0.0f ? g : (z != z ? z : 0.0f);
    if constexpr (ACT == kGelu) {
        float bell;
        const float tail = normal_tail(z, bell), p = z >= 0.0f ? 1.0f - tail : tail;
        return g * (fabsf(z) > 14.0f ? p : fmaf(z * 0.39894228040143268f, bell, p));
    }
    if constexpr (ACT == kGeluTanh) {
        const float s = logistic(kGeluC * (z + kGeluA * z * z * z));
        return g * (fabsf(z) > 12.0f ? s : s + z * s * (1.0f - s) * kGeluC * (1.0f + 3.0f * kGeluA * z * z));
    }
    if constexpr (ACT == kSilu) {
        const float s = logistic(z);
        return g * (fabsf(z) > 110.0f ? s : s + z * s * (1.0f - s));
    }
    return g;
}

// dZ = G act'(Z) as an operand of 16-bit matrix instructions.  One rounding of it to the layer's type would add its own half step to
// that of each result (an error 1.4 times as large), so it goes in two planes: what truncation leaves, and the rest, rounded -- to
// 2^-16 of a bf16 dZ, 2^-22 of a fp16 one.  fp16's second plane is 2048 times the rest, or dZ below 2^-13 would have none (so it
// reaches down to 2^-35).  Truncated, both planes have one sign, and neither is 0 unless dZ or its first plane is (an exact dZ's
// second plane is the smallest number): an infinite weight gives an infinity, not NaN.  ReLU's dZ is G itself or 0: one plane.
template <class T> struct Low;
template <> struct Low<bf16_t> { static constexpr float scale = 1.0f; static constexpr int inf = 0x7f80; };
template <> struct Low<f16_t> { static constexpr float scale = 2048.0f; static constexpr int inf = 0x7c00; };
template <class T> __device__ __forceinline__ T truncated(float v);
template <> __device__ __forceinline__ bf16_t truncated<bf16_t>(float v) { return bf16_t{(unsigned short)(__float_as_uint(v) >> 16)}; }
template <> __device__ __forceinline__ f16_t truncated<f16_t>(float v) {
    return f16_t{(unsigned short)__builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(v, 0.0f))};
}
template <class T>
__device__ __forceinline__ void split_slope(float d, T &high, T &low) {
    high = truncated<T>(d);
    unsigned short l = from_f32<T>((d - to_f32<T>(high)) * Low<T>::scale).u;
    // nothing left, or infinity less itself
    if ((unsigned short)((l & 0x7fff) - 1) >= Low<T>::inf) l = high.u & 0x7fff ? (high.u & 0x8000) | 1 : 0;
    low.u = l;
}

// ---- epilogue ----------------------------------------------------------------------------------------------------
struct Epilogue {
    void *y;              // [M,N] rows of ldy elements
    long ldy;
    void *pre;            // Z in y's type, or null
    long ldp;
    const void *bias;     // [N], or null
    int bias_f32;         // bias is fp32 (else y's type)
    const void *res;      // [M,N] rows of ldr elements, or null
    long ldr;
    int act;
};

// N neighbours of any alignment: the hardware takes wide accesses at every address of whole elements
template <class T, int N> struct Pack { T x[N]; };
template <class T, int N>
__device__ __forceinline__ Pack<T, N> load_pack(const T *p) {
    Pack<T, N> v;
    __builtin_memcpy(&v, p, sizeof v);
    return v;
}
template <class T, int N>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, N> &v) { __builtin_memcpy(p, &v, sizeof v); }

// W columns from n0 on of the bias, 0 where there is none
template <class T, int W>
__device__ __forceinline__ void load_bias(const Epilogue &e, long n0, long N, float *b) {
#pragma unroll
    for (int i = 0; i < W; ++i) b[i] = 0.0f;
    if (!e.bias) return;
    if (n0 + W <= N) {
        if (e.bias_f32) {
            const auto v = load_pack<float, W>((const float *)e.bias + n0);
#pragma unroll
            for (int i = 0; i < W; ++i) b[i] = v.x[i];
        } else {
            const auto v = load_pack<T, W>((const T *)e.bias + n0);
#pragma unroll
            for (int i = 0; i < W; ++i) b[i] = to_f32<T>(v.x[i]);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < W; ++i)
        if (n0 + i < N) b[i] = e.bias_f32 ? ((const float *)e.bias)[n0 + i] : to_f32<T>(((const T *)e.bias)[n0 + i]);
}

// W columns from n0 on of row m of the residual (zeros behind the last column), asked for ahead of finish()
template <class T, int W>
__device__ __forceinline__ Pack<T, W> load_residual(const Epilogue &e, long m, long n0, long N) {
    Pack<T, W> p;
    const T *from = (const T *)e.res + m * e.ldr + n0;
    if (n0 + W <= N) return load_pack<T, W>(from);
#pragma unroll
    for (int i = 0; i < W; ++i) p.x[i] = n0 + i < N ? from[i] : T{};
    return p;
}

template <class T, int W>
__device__ __forceinline__ void store_row(T *to, const float *z, long n0, long N) {
    Pack<T, W> p;
#pragma unroll
    for (int i = 0; i < W; ++i) p.x[i] = from_f32<T>(z[i]);
    if (n0 + W <= N) {
        store_pack<T, W>(to, p);
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (n0 + i < N) to[i] = p.x[i];
    }
}

// W consecutive columns n0 .. n0 + W of row m: v = the sums in fp32, b = the bias, r = the residual's columns where there is
// one.  Each output is rounded once, from fp32.
template <class T, int W>
__device__ __forceinline__ void finish(const Epilogue &e, long m, long n0, long N, const float *v, const float *b, const Pack<T, W> &r) {
    float z[W];
#pragma unroll
    for (int i = 0; i < W; ++i) z[i] = v[i] + b[i];
    if (e.pre) store_row<T, W>((T *)e.pre + m * e.ldp + n0, z, n0, N);
    with_activation(e.act, [&](auto act) {
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] = activate<decltype(act)::value>(z[i]);
    });
    if (e.res) {
#pragma unroll
        for (int i = 0; i < W; ++i) z[i] += to_f32<T>(r.x[i]);
    }
    store_row<T, W>((T *)e.y + m * e.ldy + n0, z, n0, N);
}

// ---- one product -------------------------------------------------------------------------------------------------
struct Product {
    const void *a, *b;
    long lda, ldb;        // elements between neighbours of the index that is not contiguous
    long M, N, K;
    int vec_a, vec_b;     // 16-byte aligned base and rows
    int splits;           // the k range is cut into this many pieces, each summed by a workgroup of its own
    long kchunk;          // k indices (tiles: steps) of one piece
    int passes;           // tiles: 1; 6 for fp32 operands in three bf16 planes each; 2 for a dZ in two (the second plane first)
    long plane_a, plane_b;   // elements between planes
    float *part;          // splits > 1: [splits][M][Np] partial sums, Np = N rounded up to a multiple of 4
    Epilogue e;
    int alone;            // small products: a block for each wave of a workgroup
    unsigned first;       // small products: the first block, or group of `alone` blocks, of this launch
    // small backward products
    const void *z;        // operand G becomes G act'(z), or null
    long ldz;
    int vec_z;
    int zact;             // the activation; kPlanes: G and z are the two planes of dZ
    int two;              // 16-bit types: dZ in two planes, formed or read
    void *colsum;         // dW: sums of B over k, or null
    int col_f32;
    float *colpart;       // splits > 1: [splits][N]
};
__host__ __device__ inline long round_up(long v, long m) { return (v + m - 1) / m * m; }

}  // namespace dense
