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
enum Act { kNone = 0, kRelu = 1, kGelu = 2, kGeluTanh = 3, kSilu = 4 };

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
// fp32 throughout, with the library's exp / erfc (about an ulp).  gelu is written with erfc because 1 + erf cancels for
// negative arguments.  Logistic forms divide by 1 + exp(-x): exp may overflow to infinity, which gives the right 0.
__device__ __forceinline__ float logistic(float x) { return 1.0f / (1.0f + expf(-x)); }
constexpr float kGeluC = 1.5957691216057308f;        // 2 sqrt(2 / pi)
constexpr float kGeluA = 0.044715f;

__device__ __forceinline__ float activate(float z, int act) {
    switch (act) {
        case kRelu: return z > 0.0f ? z : (z != z ? z : 0.0f);                  // NaN passes through
        case kGelu: return 0.5f * z * erfcf(z * -0.70710678118654752f);
        case kGeluTanh: return z / (1.0f + expf(-kGeluC * (z + kGeluA * z * z * z)));   // 0.5 (1 + tanh u) = logistic(2 u)
        case kSilu: return z / (1.0f + expf(-z));
        default: return z;
    }
}
// (ReLU's is a selection, made by the caller)
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case kGelu: return fmaf(z * 0.39894228040143268f, expf(-0.5f * z * z), 0.5f * erfcf(z * -0.70710678118654752f));
        case kGeluTanh: {
            const float s = logistic(kGeluC * (z + kGeluA * z * z * z));
            // past |z| = 12 the logistic is 0 or 1 to every bit and the product below would be 0 times infinity
            return fabsf(z) > 12.0f ? s : s + z * s * (1.0f - s) * kGeluC * (1.0f + 3.0f * kGeluA * z * z);
        }
        case kSilu: {
            const float s = logistic(z);
            return s + z * s * (1.0f - s);
        }
        default: return 1.0f;
    }
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
    int vec;              // y, pre, res: 16-byte aligned bases and rows, N a multiple of 8
};

// W columns from n0 on of the bias, 0 where there is none
template <class T, int W>
__device__ __forceinline__ void load_bias(const Epilogue &e, long n0, long N, float *b) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
        b[i] = 0.0f;
        if (e.bias && n0 + i < N) b[i] = e.bias_f32 ? ((const float *)e.bias)[n0 + i] : to_f32<T>(((const T *)e.bias)[n0 + i]);
    }
}

// W consecutive columns n0 .. n0 + W of row m: v = the sums in fp32, b = the bias.  Each output is rounded once, from fp32.
template <class T, int W>
__device__ __forceinline__ void finish(const Epilogue &e, long m, long n0, long N, const float *v, const float *b) {
    static_assert(W % 4 == 0, "whole groups of four columns");
    constexpr int G = sizeof(T) == 4 ? 4 : (W % 8 == 0 ? 8 : 4);      // columns of one 8- or 16-byte access
    struct alignas(sizeof(T) * G) Pack { T x[G]; };
    if (e.vec) {
#pragma unroll
        for (int g = 0; g < W; g += G) {
            const long n = n0 + g;
            if (n >= N) return;
            float z[G];
            Pack p;
#pragma unroll
            for (int i = 0; i < G; ++i) z[i] = v[g + i] + b[g + i];
            if (e.pre) {
#pragma unroll
                for (int i = 0; i < G; ++i) p.x[i] = from_f32<T>(z[i]);
                *(Pack *)((T *)e.pre + m * e.ldp + n) = p;
            }
#pragma unroll
            for (int i = 0; i < G; ++i) z[i] = activate(z[i], e.act);
            if (e.res) {
                const Pack r = *(const Pack *)((const T *)e.res + m * e.ldr + n);
#pragma unroll
                for (int i = 0; i < G; ++i) z[i] += to_f32<T>(r.x[i]);
            }
#pragma unroll
            for (int i = 0; i < G; ++i) p.x[i] = from_f32<T>(z[i]);
            *(Pack *)((T *)e.y + m * e.ldy + n) = p;
        }
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const long n = n0 + i;
            if (n >= N) return;
            float z = v[i] + b[i];
            if (e.pre) ((T *)e.pre)[m * e.ldp + n] = from_f32<T>(z);
            z = activate(z, e.act);
            if (e.res) z += to_f32<T>(((const T *)e.res)[m * e.ldr + n]);
            ((T *)e.y)[m * e.ldy + n] = from_f32<T>(z);
        }
    }
}

// ---- one product -------------------------------------------------------------------------------------------------
struct Product {
    const void *a, *b;
    long lda, ldb;        // elements between neighbours of the index that is not contiguous
    long M, N, K;
    int vec_a, vec_b;     // 16-byte aligned base and rows
    int splits;           // the k range is cut into this many pieces, each summed by a workgroup of its own
    long kchunk;          // k indices (tiles: steps) of one piece
    int passes;           // tiles: 1, or 6 for fp32 operands in three bf16 planes each
    long plane_a, plane_b;   // elements between planes
    float *part;          // splits > 1: [splits][M][Np] partial sums, Np = N rounded up to a multiple of 4
    Epilogue e;
};
__host__ __device__ inline long round_up(long v, long m) { return (v + m - 1) / m * m; }

}  // namespace dense
