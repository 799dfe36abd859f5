// The dense layer on plain weights: y = act(x W + b) + residual in fp32, bf16 or fp16, and its gradient
// (dense_common.h has the formulas).  This file: the product kernel that takes any size, stride and alignment, the
// pass in front of a backward product (dZ = G act'(Z) and its column sums), the join of split sums, and the C ABI.
//
// product_kernel: a workgroup of four waves owns a 64 x 64 tile of D and walks k in steps of 32.  Both operands go through
// registers into LDS in [row][k] order whatever their layout in memory -- one step ahead of the products, so the loads of
// a step fly while the last one is multiplied -- and come back as 16-byte fragments (rows padded to 80 / 144 bytes: eight
// neighbouring rows start in eight different bank groups).  16-bit types run on v_mfma_f32_16x16x32, fp32 on
// v_mfma_f32_16x16x4 (exact products, fp32 sums); a lane of the fp32 form reads four k values at once and gives them to
// four MFMAs, which permutes k inside a step the same way on both sides.  The n index sits on the MFMA's row side, so that
// a lane ends with four consecutive columns of one output row.
// Few tiles: the k range is cut into pieces (Product::splits), whose fp32 sums meet in join_kernel in piece order.
#include "dense_common.h"

using namespace dense;

namespace {

constexpr int kT = 64, kStep = 32;                     // tile edge, k indices per step

template <class T> struct Tile;
template <> struct Tile<float> { static constexpr int ld = 36; };
template <> struct Tile<bf16_t> { static constexpr int ld = 40; };
template <> struct Tile<f16_t> { static constexpr int ld = 40; };

template <class T> struct alignas(16) Eight { T x[8]; };

// Eight neighbours in memory: elements (row, k .. k + 8) of an operand with k contiguous, or (row .. row + 8, k) of one
// with rows contiguous; zeros outside [0, rows) x [0, kend).
template <class T, bool ROWS>
__device__ __forceinline__ Eight<T> fetch(const T *p, long ld, int vec, long row, long rows, long k, long kend) {
    Eight<T> v;
    const long fast = ROWS ? row : k, nfast = ROWS ? rows : kend;
    const bool in = ROWS ? k < kend : row < rows;
    const T *q = p + (ROWS ? k * ld + row : row * ld + k);
    if (vec && in && fast + 8 <= nfast) {
        v = *(const Eight<T> *)q;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.x[i] = (in && fast + i < nfast) ? q[i] : T{};
    }
    return v;
}

template <class T, bool ROWS>
__device__ __forceinline__ void stage(T *lds, int t, const Eight<T> &v) {
    constexpr int ld = Tile<T>::ld;
    if (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; ++i) lds[((t & 7) * 8 + i) * ld + (t >> 3)] = v.x[i];
    } else {
        *(Eight<T> *)(lds + (t >> 2) * ld + (t & 3) * 8) = v;
    }
}

template <class T>
__device__ __forceinline__ f4 mfma_step(const T *a, const T *b, f4 c);   // a, b: fragment start of this lane's row
template <>
__device__ __forceinline__ f4 mfma_step<bf16_t>(const bf16_t *a, const bf16_t *b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*(const b8 *)a, *(const b8 *)b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f4 mfma_step<f16_t>(const f16_t *a, const f16_t *b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(*(const h8 *)a, *(const h8 *)b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f4 mfma_step<float>(const float *a, const float *b, f4 c) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {                      // k = 16 s + 4 (lane / 16) + j
        const f4 x = *(const f4 *)(a + 16 * s), y = *(const f4 *)(b + 16 * s);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], y[j], c, 0, 0, 0);
    }
    return c;
}

template <class T, bool TA, bool TB>
__global__ __launch_bounds__(256) void product_kernel(Product P) {
    __shared__ T sa[kT * Tile<T>::ld], sb[kT * Tile<T>::ld];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const long tn = (P.N + kT - 1) / kT;
    const long tile = blockIdx.x, m0 = tile / tn * kT, n0 = tile % tn * kT;
    const long k0 = (long)blockIdx.y * P.kchunk, kend = k0 + P.kchunk < P.K ? k0 + P.kchunk : P.K;
    const T *A = (const T *)P.a, *B = (const T *)P.b;
    const long ra = m0 + (TA ? (t & 7) * 8 : t >> 2), rb = n0 + (TB ? (t & 7) * 8 : t >> 2);
    const int ka = TA ? t >> 3 : (t & 3) * 8, kb = TB ? t >> 3 : (t & 3) * 8;
    const int wm = (wave & 1) * 32, wn = (wave >> 1) * 32;
    // this lane's k offset inside a fragment: eight 16-bit values or one float4
    const int frag = (lane & 15) * Tile<T>::ld + (lane >> 4) * (sizeof(T) == 4 ? 4 : 8);
    f4 acc[2][2] = {};
    Eight<T> va{}, vb{};
    if (k0 < kend) {
        va = fetch<T, TA>(A, P.lda, P.vec_a, ra, P.M, k0 + ka, kend);
        vb = fetch<T, TB>(B, P.ldb, P.vec_b, rb, P.N, k0 + kb, kend);
    }
    for (long k = k0; k < kend; k += kStep) {
        stage<T, TA>(sa, t, va);
        stage<T, TB>(sb, t, vb);
        __syncthreads();
        if (k + kStep < kend) {
            va = fetch<T, TA>(A, P.lda, P.vec_a, ra, P.M, k + kStep + ka, kend);
            vb = fetch<T, TB>(B, P.ldb, P.vec_b, rb, P.N, k + kStep + kb, kend);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                acc[j][i] = mfma_step<T>(sb + (wn + 16 * j) * Tile<T>::ld + frag, sa + (wm + 16 * i) * Tile<T>::ld + frag,
                                         acc[j][i]);
        __syncthreads();
    }
    const long Np = round_up(P.N, 4);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const long n = n0 + wn + 16 * j + (lane >> 4) * 4;
        if (n >= P.N) continue;
        float b[4];
        if (P.splits == 1) load_bias<T, 4>(P.e, n, P.N, b);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const long m = m0 + wm + 16 * i + (lane & 15);
            if (m >= P.M) continue;
            const float v[4] = {acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]};
            if (P.splits > 1) *(f4 *)(P.part + ((long)blockIdx.y * P.M + m) * Np + n) = acc[j][i];
            else finish<T, 4>(P.e, m, n, P.N, v, b);
        }
    }
}

// The pieces of a split k range, summed in piece order, then the epilogue.
template <class T>
__global__ __launch_bounds__(256) void join_kernel(Product P) {
    const long Np = round_up(P.N, 4), per = Np / 4, total = P.M * per, plane = P.M * Np;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long m = i / per, n = (i - m * per) * 4;
        const float *p = P.part + m * Np + n;
        f4 s = *(const f4 *)p;
        for (int z = 1; z < P.splits; ++z) s += *(const f4 *)(p + z * plane);
        float b[4];
        load_bias<T, 4>(P.e, n, P.N, b);
        const float v[4] = {s[0], s[1], s[2], s[3]};
        finish<T, 4>(P.e, m, n, P.N, v, b);
    }
}

// ---- in front of a backward product: dZ = G act'(Z), and the column sums of dZ ------------------------------------------
// A thread owns eight columns of every eighth row of its block's strip; the eight row lanes of a block meet in LDS, the
// strips in sum_strips_kernel, both in a fixed order.  dZ is rounded to the layer's type, since the products read it as an
// operand of the same MFMAs as X and W (the sums for the bias are taken before the rounding).
struct Slope {
    const void *g, *z;    // z null: no activation
    long ldg, ldz;
    int vec;              // g and z: 16-byte aligned bases and rows
    int act;
    long rows;
    int cols;
    void *dz;             // [rows][ldd] in the layer's type, ldd = cols rounded up to 8, zeros behind the last column; null: sums only
    long ldd;
    float *sums;          // [strips][cols], or null
    long strip;           // rows of a block
};

template <class T>
__global__ __launch_bounds__(256) void slope_kernel(Slope S) {
    __shared__ float part[8][256 + 4];
    const int c0 = blockIdx.x * 256 + (threadIdx.x & 31) * 8, rl = threadIdx.x >> 5;
    const long r0 = (long)blockIdx.y * S.strip, r1 = r0 + S.strip < S.rows ? r0 + S.strip : S.rows;
    float sum[8] = {};
    if (c0 < S.cols) {
        for (long r = r0 + rl; r < r1; r += 8) {
            const Eight<T> g = fetch<T, false>((const T *)S.g, S.ldg, S.vec, r, S.rows, c0, S.cols);
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) d[i] = to_f32<T>(g.x[i]);
            if (S.z) {
                const Eight<T> z = fetch<T, false>((const T *)S.z, S.ldz, S.vec, r, S.rows, c0, S.cols);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float zi = to_f32<T>(z.x[i]);
                    // ReLU selects: what a closed unit receives, infinities among it, does not come through
                    if (S.act == kRelu) d[i] = zi > 0.0f ? d[i] : (zi != zi ? zi : 0.0f);
                    else d[i] = c0 + i < S.cols ? d[i] * act_slope(zi, S.act) : 0.0f;
                }
            }
            if (S.dz) {
                Eight<T> o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o.x[i] = from_f32<T>(d[i]);
                *(Eight<T> *)((T *)S.dz + r * S.ldd + c0) = o;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum[i] += d[i];
        }
    }
    if (!S.sums) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) part[rl][(threadIdx.x & 31) * 8 + i] = sum[i];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c < S.cols) {
        float s = part[0][threadIdx.x];
        for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
        S.sums[(long)blockIdx.y * S.cols + c] = s;
    }
}

template <class T>
__global__ __launch_bounds__(256) void sum_strips_kernel(const float *sums, int strips, int cols, T *out) {
    __shared__ float part[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), q = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < cols)
        for (int i = q; i < strips; i += 4) s += sums[(long)i * cols + c];
    part[q][threadIdx.x & 63] = s;
    __syncthreads();
    if (q == 0 && c < cols) out[c] = from_f32<T>((part[0][c & 63] + part[1][c & 63]) + (part[2][c & 63] + part[3][c & 63]));
}

// ---- host ----------------------------------------------------------------------------------------------------------
inline long esize(int type) { return type == kF32 ? 4 : 2; }
inline bool aligned(const void *p, long ld, int type) { return ((uintptr_t)p & 15) == 0 && (ld * esize(type)) % 16 == 0; }

// Pieces of the k range: enough workgroups for two per CU, at least 128 k indices each.
inline void split(Product &P) {
    const long tiles = ((P.M + kT - 1) / kT) * ((P.N + kT - 1) / kT);
    long s = (512 + tiles - 1) / tiles;
    const long most = P.K / 128;
    if (s > most) s = most;
    if (s < 1) s = 1;
    P.kchunk = round_up((P.K + s - 1) / s, kStep);
    if (P.kchunk < kStep) P.kchunk = kStep;
    P.splits = (int)((P.K + P.kchunk - 1) / P.kchunk);
    if (P.splits < 1) P.splits = 1;
}
inline unsigned long part_bytes(const Product &P) {
    return P.splits > 1 ? (unsigned long)P.splits * P.M * round_up(P.N, 4) * 4 : 0;
}

template <class T, bool TA, bool TB>
int launch(const Product &P, hipStream_t s) {
    const long tiles = ((P.M + kT - 1) / kT) * ((P.N + kT - 1) / kT);
    if (tiles > 0x7fffffffL) return SA_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((product_kernel<T, TA, TB>), dim3((unsigned)tiles, P.splits), dim3(256), 0, s, P);
    SA_CHECK_LAUNCH();
    if (P.splits > 1) {
        const long blocks = (P.M * (round_up(P.N, 4) / 4) + 255) / 256;
        hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, s, P);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}
template <bool TA, bool TB>
int launch(int type, const Product &P, hipStream_t s) {
    if (type == kF32) return launch<float, TA, TB>(P, s);
    if (type == kBF16) return launch<bf16_t, TA, TB>(P, s);
    return launch<f16_t, TA, TB>(P, s);
}

inline bool sizes_ok(int type, long rows, int cin, int cout) {
    return type >= kF32 && type <= kF16 && rows >= 0 && cin >= 0 && cout >= 0;
}

// Scratch of a call, piece by piece at 256-byte steps.  With base null only the size is counted.
struct Scratch {
    char *base;
    unsigned long used = 0;
    void *take(unsigned long bytes) {
        if (bytes == 0) return nullptr;
        void *p = base ? base + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        return p;
    }
};

Product forward_product(long rows, int cin, int cout) {
    Product P{};
    P.M = rows; P.N = cout; P.K = cin;
    split(P);
    return P;
}

struct Backward {
    Product dx, dw;
    Slope slope;
    int strips;
};
constexpr int kWantX = 1, kWantW = 2, kWantB = 4;

void plan_backward(Backward &b, Scratch &ws, int type, long rows, int cin, int cout, int act, int want) {
    b = Backward{};
    Slope &S = b.slope;
    S.rows = rows; S.cols = cout; S.act = act;
    S.strip = 64 * ((rows + 64 * 512 - 1) / (64 * 512));
    if (S.strip < 64) S.strip = 64;
    b.strips = (int)((rows + S.strip - 1) / S.strip);
    S.ldd = round_up(cout, 8);
    if (act != kNone && (want & (kWantX | kWantW))) S.dz = ws.take((unsigned long)rows * S.ldd * esize(type));
    if (want & kWantB) S.sums = (float *)ws.take((unsigned long)b.strips * cout * 4);
    if (want & kWantX) {
        b.dx.M = rows; b.dx.N = cin; b.dx.K = cout;
        split(b.dx);
        b.dx.part = (float *)ws.take(part_bytes(b.dx));
    }
    if (want & kWantW) {
        b.dw.M = cin; b.dw.N = cout; b.dw.K = rows;
        split(b.dw);
        b.dw.part = (float *)ws.take(part_bytes(b.dw));
    }
}

template <class T>
int launch_slope(const Backward &b, void *db, int db_f32, hipStream_t s) {
    const Slope &S = b.slope;
    if (S.rows > 0 && (S.dz || S.sums)) {
        hipLaunchKernelGGL((slope_kernel<T>), dim3((S.cols + 255) / 256, b.strips), dim3(256), 0, s, S);
        SA_CHECK_LAUNCH();
    }
    if (db) {
        if (db_f32)
            hipLaunchKernelGGL((sum_strips_kernel<float>), dim3((S.cols + 63) / 64), dim3(256), 0, s, S.sums, b.strips, S.cols,
                               (float *)db);
        else
            hipLaunchKernelGGL((sum_strips_kernel<T>), dim3((S.cols + 63) / 64), dim3(256), 0, s, S.sums, b.strips, S.cols, (T *)db);
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

}  // namespace

extern "C" int sa_dense_forward_ws(int dtype, long rows, int cin, int cout, int flags, unsigned long *bytes) {
    (void)flags;
    if (!bytes || !sizes_ok(dtype, rows, cin, cout)) return SA_ERR_INVALID;
    *bytes = rows && cout ? part_bytes(forward_product(rows, cin, cout)) : 0;
    return SA_OK;
}

extern "C" int sa_dense_forward(int dtype, long rows, int cin, int cout, const void *x, long ldx, const void *w, long ldw,
                                const void *bias, int bias_f32, const void *res, long ldr, int act, void *y, void *pre,
                                void *ws, unsigned long ws_bytes, void *stream) {
    if (!sizes_ok(dtype, rows, cin, cout) || act < kNone || act > kSilu) return SA_ERR_INVALID;
    if (rows == 0 || cout == 0) return SA_OK;
    if (!y || (cin && (!x || !w)) || ldx < cin || ldw < cout || (res && ldr < cout)) return SA_ERR_INVALID;
    Product P = forward_product(rows, cin, cout);
    P.a = x; P.lda = ldx; P.vec_a = aligned(x, ldx, dtype);
    P.b = w; P.ldb = ldw; P.vec_b = aligned(w, ldw, dtype);
    if (part_bytes(P) > ws_bytes || (part_bytes(P) && !ws)) return SA_ERR_INVALID;
    P.part = (float *)ws;
    P.e = Epilogue{y, cout, pre, cout, bias, bias_f32, res, ldr, act, 0};
    P.e.vec = cout % 8 == 0 && aligned(y, cout, dtype) && (!pre || aligned(pre, cout, dtype)) && (!res || aligned(res, ldr, dtype));
    return launch<false, true>(dtype, P, (hipStream_t)stream);
}

extern "C" int sa_dense_backward_ws(int dtype, long rows, int cin, int cout, int act, int want, int flags, unsigned long *bytes) {
    (void)flags;
    if (!bytes || !sizes_ok(dtype, rows, cin, cout) || act < kNone || act > kSilu || want < 0 || want > 7) return SA_ERR_INVALID;
    Backward b;
    Scratch s{nullptr};
    plan_backward(b, s, dtype, rows, cin, cout, act, want);
    *bytes = s.used;
    return SA_OK;
}

extern "C" int sa_dense_backward(int dtype, long rows, int cin, int cout, const void *x, long ldx, const void *w, long ldw,
                                 const void *g, long ldg, const void *z, long ldz, int act, void *dx, void *dw, void *db,
                                 int db_f32, void *ws, unsigned long ws_bytes, void *stream) {
    if (!sizes_ok(dtype, rows, cin, cout) || act < kNone || act > kSilu) return SA_ERR_INVALID;
    const int want = (dx && rows && cin ? kWantX : 0) | (dw && cin && cout ? kWantW : 0) | (db && cout ? kWantB : 0);
    if (!want) return SA_OK;
    if (rows && cout && (!g || ldg < cout || (act != kNone && (!z || ldz < cout)))) return SA_ERR_INVALID;
    if ((want & kWantX) && cout && (!w || ldw < cout)) return SA_ERR_INVALID;
    if ((want & kWantW) && rows && (!x || ldx < cin)) return SA_ERR_INVALID;
    Backward b;
    Scratch s{(char *)ws};
    plan_backward(b, s, dtype, rows, cin, cout, act, want);
    if (s.used > ws_bytes || (s.used && !ws)) return SA_ERR_INVALID;
    Slope &S = b.slope;
    S.g = g; S.ldg = ldg;
    S.z = act == kNone ? nullptr : z; S.ldz = ldz;
    S.vec = aligned(g, ldg, dtype) && (!S.z || aligned(z, ldz, dtype));
    hipStream_t st = (hipStream_t)stream;
    int rc = dtype == kF32 ? launch_slope<float>(b, want & kWantB ? db : nullptr, db_f32, st)
             : dtype == kBF16 ? launch_slope<bf16_t>(b, want & kWantB ? db : nullptr, db_f32, st)
                              : launch_slope<f16_t>(b, want & kWantB ? db : nullptr, db_f32, st);
    if (rc) return rc;
    const void *dz = S.dz ? S.dz : g;
    const long ldd = S.dz ? S.ldd : ldg;
    const int vec_dz = aligned(dz, ldd, dtype);
    if (want & kWantX) {
        Product &P = b.dx;
        P.a = dz; P.lda = ldd; P.vec_a = vec_dz;
        P.b = w; P.ldb = ldw; P.vec_b = aligned(w, ldw, dtype);
        P.e = Epilogue{dx, cin, nullptr, 0, nullptr, 0, nullptr, 0, kNone, cin % 8 == 0 && aligned(dx, cin, dtype)};
        if ((rc = launch<false, false>(dtype, P, st))) return rc;
    }
    if (want & kWantW) {
        Product &P = b.dw;
        P.a = x; P.lda = ldx; P.vec_a = aligned(x, ldx, dtype);
        P.b = dz; P.ldb = ldd; P.vec_b = vec_dz;
        P.e = Epilogue{dw, cout, nullptr, 0, nullptr, 0, nullptr, 0, kNone, cout % 8 == 0 && aligned(dw, cout, dtype)};
        if ((rc = launch<true, true>(dtype, P, st))) return rc;
    }
    return SA_OK;
}
