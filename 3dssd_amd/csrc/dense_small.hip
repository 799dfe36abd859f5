// The products of the dense layer that are too small for tiles in LDS, and those of a few rows (one token, a handful of
// proposals), where every weight is used once and the layer costs what reading W costs.  Any size, stride and alignment.
//
// A workgroup owns a small block of D and all of k (or one of P.splits pieces).  Its waves take turns at steps of 32 k:
// each loads its operands from memory straight into MFMA fragments, several steps ahead, and multiplies the block by itself;
// the waves' sums meet in LDS once, at the end.  No LDS and no barrier on the way, so a call costs little more than one
// round trip to memory, and one launch where the k range is not split.
//   bf16, fp16: v_mfma_f32_16x16x32, eight k values of a row per lane.  fp32: v_mfma_f32_16x16x4 (exact products, fp32
//   sums), one k value per lane; the eight that a lane holds go to eight MFMAs, permuting k the same way on both sides.
//   k contiguous in memory: a lane's eight values of a row are one or two loads; N blocks of 16 rows.
//   rows contiguous: a lane reads N neighbouring rows (2 to 16 bytes) at each of its eight k, and MFMA t of a step takes row
//   t of them: which rows of the block the MFMA's 16 stand for is free, so turning the lane's 8 x N block is a few byte
//   permutations between its own registers.
// The n index is on the MFMA's row side: a lane holds four rows r of it at one m.
//
// A small layer's backward pass is one launch: dX's and dW's workgroups side by side, dZ = G act'(Z) formed in registers by
// whoever loads G and Z, and the bias gradient summed (before dZ is rounded) by the dW workgroups of the first rows.
#include "dense_common.h"
#include "dense_products.h"

using namespace dense;

namespace {

constexpr unsigned kOutside = 0x80000000u;             // past every buffer's range: the load gives zeros

template <int B> struct Bytes;
template <> struct Bytes<2> { typedef unsigned short t; };
template <> struct Bytes<4> { typedef unsigned t; };
template <> struct Bytes<8> { typedef unsigned t __attribute__((ext_vector_type(2))); };
template <> struct Bytes<16> { typedef unsigned t __attribute__((ext_vector_type(4))); };

template <int B>
__device__ __forceinline__ typename Bytes<B>::t load(__amdgpu_buffer_rsrc_t r, unsigned off) {
    if constexpr (B == 2) return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
    else if constexpr (B == 4) return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
    else if constexpr (B == 8) return __builtin_bit_cast(typename Bytes<8>::t, __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0));
    else return __builtin_bit_cast(typename Bytes<16>::t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer(const char *p) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, (short)0, 0x7fffffff, 0x00020000);
}

// Elements t of a lane's words
template <class T, class W>
__device__ __forceinline__ float element(W v, int t) {
    if constexpr (sizeof(T) == 4) {
        if constexpr (sizeof(W) == 4) return __uint_as_float(v);
        else return __uint_as_float(v[t]);
    } else {
        unsigned w;
        if constexpr (sizeof(W) <= 4) w = v;
        else w = v[t / 2];
        return to_f32<T>(T{(unsigned short)(t & 1 ? w >> 16 : w)});
    }
}

// One operand of a wave's block: N blocks of 16 rows.
template <class T, bool ROWS, int N> struct Side;

template <class T, int N>
struct Side<T, false, N> {                             // k contiguous
    static constexpr int E = sizeof(T);
    typedef typename Bytes<16>::t u4;
    struct Regs { u4 v[N][E / 2]; };
    unsigned off[N];
    int g8;
    __device__ __forceinline__ void init(int lane, long ld, long rows_left) {
        g8 = 8 * (lane >> 4);
#pragma unroll
        for (int t = 0; t < N; ++t) {
            const int row = 16 * t + (lane & 15);
            off[t] = row < rows_left ? (unsigned)((row * ld + g8) * E) : kOutside;
        }
    }
    // left: valid k of this step, up to 32; vec: 16-byte aligned base and rows
    __device__ __forceinline__ void fetch(Regs &r, const char *base, int left, bool vec) const {
        const auto b = buffer(base);
#pragma unroll
        for (int t = 0; t < N; ++t) {
            if (vec && (left & 7) == 0) {
#pragma unroll
                for (int h = 0; h < E / 2; ++h) r.v[t][h] = load<16>(b, g8 < left ? off[t] + 16 * h : kOutside);
            } else {
#pragma unroll
                for (int h = 0; h < E / 2; ++h) r.v[t][h] = u4{0, 0, 0, 0};
                if (off[t] != kOutside && g8 + 8 <= left) {
                    __builtin_memcpy(r.v[t], base + off[t], 8 * E);    // (buffers want aligned 16 bytes, pointers do not)
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const unsigned e = load<E>(b, g8 + j < left ? off[t] + j * E : kOutside);
                        if constexpr (E == 4) r.v[t][j / 4][j % 4] = e;
                        else r.v[t][0][j / 2] |= j & 1 ? e << 16 : e;
                    }
                }
            }
        }
    }
    static __device__ __forceinline__ float at(const Regs &r, int t, int j) {
        if constexpr (E == 4) return __uint_as_float(r.v[t][j / 4][j % 4]);
        else return element<T>(r.v[t][0], j);
    }
    static __device__ __forceinline__ s8 fragment(const Regs &r, int t) { return __builtin_bit_cast(s8, r.v[t][0]); }
    static __device__ __forceinline__ int row(int t, int i) { return 16 * t + i; }
};

template <class T, int N>
struct Side<T, true, N> {                              // rows contiguous
    static constexpr int E = sizeof(T), B = E * N;
    typedef typename Bytes<B>::t word_t;
    struct Regs { word_t v[8]; };
    unsigned off, step;
    int g8, left_rows;
    __device__ __forceinline__ void init(int lane, long ld, long rows_left) {
        g8 = 8 * (lane >> 4);
        const int row = N * (lane & 15);
        left_rows = rows_left < row ? 0 : rows_left - row > N ? N : (int)(rows_left - row);
        off = left_rows > 0 ? (unsigned)((g8 * ld + row) * E) : kOutside;
        step = (unsigned)(ld * E);
    }
    // vec: pieces of N rows are aligned and there are no parts of them
    __device__ __forceinline__ void fetch(Regs &r, const char *base, int left, bool vec) const {
        const auto b = buffer(base);
        if (N == 1 || vec || N > 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) r.v[j] = load<B>(b, g8 + j < left ? off + j * step : kOutside);
        } else if constexpr (N == 2) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const unsigned lo = load<E>(b, g8 + j < left ? off + j * step : kOutside);
                const unsigned hi = load<E>(b, g8 + j < left && left_rows > 1 ? off + j * step + E : kOutside);
                if constexpr (E == 2) r.v[j] = lo | hi << 16;
                else r.v[j] = word_t{lo, hi};
            }
        }
    }
    static __device__ __forceinline__ unsigned word(const word_t &v, int i) {
        if constexpr (B <= 4) return v;
        else return v[i];
    }
    static __device__ __forceinline__ float at(const Regs &r, int t, int j) { return element<T>(r.v[j], t); }
    static __device__ __forceinline__ s8 fragment(const Regs &r, int t) {
        typename Bytes<16>::t o;
#pragma unroll
        for (int i = 0; i < 4; ++i)                    // the halves t of k 2 i and 2 i + 1
            o[i] = __builtin_amdgcn_perm(word(r.v[2 * i + 1], t / 2), word(r.v[2 * i], t / 2), t & 1 ? 0x07060302 : 0x05040100);
        return __builtin_bit_cast(s8, o);
    }
    static __device__ __forceinline__ int row(int t, int i) { return N * i + t; }
};

// What a step's products take of a side: fragments of 16-bit values, or eight fp32 values per block
template <class T, int N> struct Operand {
    s8 f[N];
    __device__ __forceinline__ void set(int t, const float *v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[t][j] = (short)from_f32<T>(v[j]).u;
    }
    __device__ __forceinline__ void set(int t, const float *v, Operand &low) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            T high, rest;
            split_slope<T>(v[j], high, rest);
            f[t][j] = (short)high.u;
            low.f[t][j] = (short)rest.u;
        }
    }
};
template <int N> struct Operand<float, N> {
    float f[N][8];
    __device__ __forceinline__ void set(int t, const float *v) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[t][j] = v[j];
    }
};
template <class T, bool ROWS, int N>
__device__ __forceinline__ void take(Operand<T, N> &o, const typename Side<T, ROWS, N>::Regs &r) {
#pragma unroll
    for (int t = 0; t < N; ++t) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) o.f[t][j] = Side<T, ROWS, N>::at(r, t, j);
        } else {
            o.f[t] = Side<T, ROWS, N>::fragment(r, t);
        }
    }
}
// dZ = G act'(Z) in place of G, as an operand of the products: in 16-bit types in two planes (LOW; or g and z are those planes
// already) or rounded; sums += the values as they were, if wanted
template <class T, bool ROWS, int N, bool LOW>
__device__ __forceinline__ void take_slope(Operand<T, N> &o, Operand<T, N> &low, const typename Side<T, ROWS, N>::Regs &g,
                                           const typename Side<T, ROWS, N>::Regs &z, int act, bool summed, float *sums) {
    if constexpr (LOW)
        if (act == kPlanes) {
            take<T, ROWS, N>(o, g);
            take<T, ROWS, N>(low, z);
            return;
        }
#pragma unroll
    for (int t = 0; t < N; ++t) {
        float d[8];
        with_activation(act, [&](auto a) __attribute__((always_inline)) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                d[j] = times_slope<decltype(a)::value>(Side<T, ROWS, N>::at(g, t, j), Side<T, ROWS, N>::at(z, t, j));
        });
        if constexpr (LOW) o.set(t, d, low);
        else o.set(t, d);
        if (summed)
#pragma unroll
            for (int j = 0; j < 8; ++j) sums[t] += d[j];
    }
}

template <class T, int NA, int NB>
__device__ __forceinline__ void multiply(f4 (&acc)[NB][NA], const Operand<T, NA> &a, const Operand<T, NB> &b) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int y = 0; y < NB; ++y)
#pragma unroll
                for (int x = 0; x < NA; ++x) acc[y][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(b.f[y][j], a.f[x][j], acc[y][x], 0, 0, 0);
    } else {
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int x = 0; x < NA; ++x) {
                if constexpr (__is_same(T, bf16_t))
                    acc[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, b.f[y]), __builtin_bit_cast(b8, a.f[x]),
                                                                        acc[y][x], 0, 0, 0);
                else
                    acc[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, b.f[y]), __builtin_bit_cast(h8, a.f[x]),
                                                                       acc[y][x], 0, 0, 0);
            }
    }
}

// The form for up to four steps: there are many such workgroups (a few channels of many points), each no more than a
// round trip to memory, so what counts is how many a CU holds: five, with 96 registers.  bf16 16384 x 64 x 256: 20 us with
// two steps ahead (128 registers), 13.6 us with one; fp32 23 and 18.7.  (64 registers spill: 15.6 and 26.)
constexpr bool few_steps(int na, int nb, int nw) { return na == 2 && nb == 2 && nw == 4; }

constexpr int kSums = 64 * 256;                        // floats of LDS for the waves' sums

// The waves of a block wait for each other; one alone needs its own LDS accesses in order only (and has no partners: the other
// waves of its workgroup may be done).
template <int NW>
__device__ __forceinline__ void meet() {
    if constexpr (NW > 1) {
        __syncthreads();
    } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
}

// Block `pos` of a product, k piece `piece`, by NW neighbouring waves, with `sums` for them alone; the workgroup's other waves do
// the same with blocks of their own, or beyond the last.  Z: A (ZSIDE 0) or B (ZSIDE 1) is G, and the product takes
// G act'(Z) with Z = P.z in G's place (rows of P.ldz), with LOW in two planes.
template <class T, bool TA, bool TB, int NA, int NB, int NW, int ZSIDE, bool LOW = false>
__device__ __forceinline__ void block_product(const Product &P, unsigned pos, int piece, float *sums) {
    constexpr int E = sizeof(T), kM = 16 * NA, kN = 16 * NB;
    // steps in flight, by the registers of one; four waves of a 32 x 32 block have one step each
    constexpr int kSlot = 2 * E * (NA + NB + (ZSIDE == 0 ? NA : ZSIDE == 1 ? NB : 0));
    constexpr int kAhead = few_steps(NA, NB, NW) || LOW ? 1 : kSlot <= 16 ? 4 : kSlot <= 32 ? 2 : 1;
    static_assert(NW * kM * kN <= kSums, "the waves' sums");
    const int thread = threadIdx.x % (NW * 64), lane = thread & 63, wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    const unsigned nb = (unsigned)((P.N + kN - 1) / kN);
    const long m0 = (long)(pos / nb) * kM, n0 = (long)(pos % nb) * kN;
    const long k0 = (long)piece * P.kchunk, kend = k0 + P.kchunk < P.K ? k0 + P.kchunk : P.K;
    const char *A = (const char *)P.a + (TA ? m0 + k0 * P.lda : m0 * P.lda + k0) * E;
    const char *B = (const char *)P.b + (TB ? n0 + k0 * P.ldb : n0 * P.ldb + k0) * E;
    const long stepa = (TA ? P.lda : 1) * 32 * E, stepb = (TB ? P.ldb : 1) * 32 * E;
    constexpr bool TZ = ZSIDE == 1 ? TB : TA;
    constexpr int NZ = ZSIDE == 1 ? NB : NA;
    const long z0 = ZSIDE == 1 ? n0 : m0;
    const char *Z = (const char *)P.z + (TZ ? z0 + k0 * P.ldz : z0 * P.ldz + k0) * E;
    const long stepz = (TZ ? P.ldz : 1) * 32 * E;
    typedef Side<T, TA, NA> SA;
    typedef Side<T, TB, NB> SB;
    typedef Side<T, TZ, NZ> SZ;
    SA a;
    SB b;
    SZ z;
    a.init(lane, P.lda, P.M - m0);
    b.init(lane, P.ldb, P.N - n0);
    if (ZSIDE >= 0) z.init(lane, P.ldz, (ZSIDE == 1 ? P.N : P.M) - z0);

    f4 acc[NB][NA] = {};
    constexpr bool kApart = LOW && __is_same(T, f16_t);        // fp16's second plane has a scale
    f4 apart[kApart ? NB : 1][kApart ? NA : 1] = {};
    float column[NB] = {};                             // sums of B's rows over k (the bias gradient), where wanted
    const bool summed = P.colsum && m0 == 0;
    typename SA::Regs ra[kAhead];
    typename SB::Regs rb[kAhead];
    typename SZ::Regs rz[ZSIDE >= 0 ? kAhead : 1];
    const long steps = m0 < P.M ? (kend - k0 + 31) / 32 : 0;
    auto fetch = [&](int slot, long s) {
        const long l = kend - k0 - s * 32;
        const int left = l < 32 ? (int)l : 32;
        a.fetch(ra[slot], A + s * stepa, left, P.vec_a);
        b.fetch(rb[slot], B + s * stepb, left, P.vec_b);
        if constexpr (ZSIDE >= 0) z.fetch(rz[slot], Z + s * stepz, left, P.vec_z);
    };
    auto products = [&](int slot) {
        Operand<T, NA> oa, la;
        Operand<T, NB> ob, lb;
        if constexpr (ZSIDE == 0) take_slope<T, TA, NA, LOW>(oa, la, ra[slot], rz[slot], P.zact, false, nullptr);
        else take<T, TA, NA>(oa, ra[slot]);
        if constexpr (ZSIDE == 1) {
            take_slope<T, TB, NB, LOW>(ob, lb, rb[slot], rz[slot], P.zact, summed, column);
        } else {
            take<T, TB, NB>(ob, rb[slot]);
            if (summed)
#pragma unroll
                for (int t = 0; t < NB; ++t)
#pragma unroll
                    for (int j = 0; j < 8; ++j) column[t] += SB::at(rb[slot], t, j);
        }
        if constexpr (LOW) {
            const Operand<T, NA> &xa = ZSIDE == 0 ? la : oa;
            const Operand<T, NB> &xb = ZSIDE == 1 ? lb : ob;
            if constexpr (kApart) multiply<T, NA, NB>(apart, xa, xb);
            else multiply<T, NA, NB>(acc, xa, xb);
        }
        multiply<T, NA, NB>(acc, oa, ob);
    };
    long s = wave;
#pragma unroll
    for (int h = 0; h < kAhead; ++h)
        if (s + h * NW < steps) fetch(h, s + h * NW);
    for (; s < steps; s += kAhead * NW) {
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
            if (s + h * NW < steps) products(h);
            if (s + (h + kAhead) * NW < steps) fetch(h, s + (h + kAhead) * NW);
        }
    }

    if constexpr (kApart)
#pragma unroll
        for (int x = 0; x < NA; ++x)
#pragma unroll
            for (int y = 0; y < NB; ++y) acc[y][x] += apart[y][x] * (1.0f / Low<T>::scale);
#pragma unroll
    for (int x = 0; x < NA; ++x)
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sums[(wave * kM + SA::row(x, lane & 15)) * kN + SB::row(y, 4 * (lane >> 4) + r)] = acc[y][x][r];
    meet<NW>();
    const long Np = round_up(P.N, 4);
    const int used = steps < NW ? (int)steps : NW;     // the others' sums are zero
#pragma unroll 1
    for (int q = thread; q < kM * kN / 4; q += NW * 64) {
        const int lm = q / (kN / 4), ln = q % (kN / 4) * 4;
        const long m = m0 + lm, n = n0 + ln;
        if (m >= P.M || n >= P.N) continue;
        float bias[4];
        Pack<T, 4> r{};
        if (P.splits == 1) {
            load_bias<T, 4>(P.e, n, P.N, bias);
            if (P.e.res) r = load_residual<T, 4>(P.e, m, n, P.N);
        }
        f4 v = *(const f4 *)(sums + lm * kN + ln);
#pragma unroll 4
        for (int w = 1; w < used; ++w) v += *(const f4 *)(sums + (w * kM + lm) * kN + ln);
        if (P.splits > 1) {
            *(f4 *)(P.part + ((long)piece * P.M + m) * Np + n) = v;
        } else {
            const float o[4] = {v[0], v[1], v[2], v[3]};
            finish<T, 4>(P.e, m, n, P.N, o, bias, r);
        }
    }
    if (summed) {                                      // four k groups of NW waves for each column
        meet<NW>();
#pragma unroll
        for (int t = 0; t < NB; ++t) sums[(wave * 4 + (lane >> 4)) * kN + SB::row(t, lane & 15)] = column[t];
        meet<NW>();
        const long n = n0 + thread;
        if (thread < kN && n < P.N) {
            float v = 0.0f;
#pragma unroll 8
            for (int w = 0; w < 4 * NW; ++w) v += sums[w * kN + thread];
            if (P.splits > 1) P.colpart[(long)piece * P.N + n] = v;
            else if (P.col_f32) ((float *)P.colsum)[n] = v;
            else ((T *)P.colsum)[n] = from_f32<T>(v);
        }
    }
}

// neighbouring blocks of n on one XCD: they share the rows of A, and with pieces below 16 bytes the lines of B
__device__ __forceinline__ unsigned on_xcd(unsigned b, unsigned blocks) {
    const unsigned q8 = blocks >> 3, r8 = blocks & 7, xcd = b & 7;
    return xcd * q8 + (xcd < r8 ? xcd : r8) + (b >> 3);
}

template <class T, bool TA, bool TB, int NA, int NB, int NW>
__global__ __launch_bounds__(NW * 64, few_steps(NA, NB, NW) ? 5 : NW / 4) void small_kernel(Product P) {
    __shared__ __attribute__((aligned(16))) float sums[NW * 256 * NA * NB];
    block_product<T, TA, TB, NA, NB, NW, -1>(P, P.first + on_xcd(blockIdx.x, gridDim.x), blockIdx.y, sums);
}

// A workgroup's share of a product: block `group`, or with P.alone (ALONE: which may be set) a block for each of its waves.
template <class T, bool TA, bool TB, int WT, int NW, int ZSIDE, bool ALONE, bool LOW = false>
__device__ __forceinline__ void group_product(const Product &P, unsigned group, int piece, float *sums) {
    if (!ALONE || !P.alone) {
        block_product<T, TA, TB, WT, WT, NW, ZSIDE, LOW>(P, group, piece, sums);
    } else {
        const unsigned mine = threadIdx.x >> 6;
        block_product<T, TA, TB, WT, WT, 1, ZSIDE, LOW>(P, group * NW + mine, piece, sums + mine * (256 * WT * WT));
    }
}

// dX and dW of a layer in one launch: the workgroups from x0 to x1 are dX's (all blocks of a piece, then the next piece), the
// others, in front of those or behind, dW's.  dW's blocks have WT x WT MFMA tiles.  128 registers: two workgroups of eight
// waves per CU.  Z: 0 without slopes, 1 with, 2 with, in two planes.
template <class T, int Z, int WT, int NW, bool ALONE>
__global__ __launch_bounds__(NW * 64, 4) void small_backward_kernel(Product X, Product W, unsigned x0, unsigned x1) {
    __shared__ __attribute__((aligned(16))) float sums[NW * 1024];
    if (blockIdx.x < x0 || blockIdx.x >= x1) {
        const unsigned b = blockIdx.x < x0 ? blockIdx.x : blockIdx.x - x1, groups = (gridDim.x - (x1 - x0)) / W.splits;
        group_product<T, true, true, WT, NW, Z ? 1 : -1, ALONE, Z == 2>(W, W.first + on_xcd(b % groups, groups), b / groups, sums);
    } else {
        const unsigned b = blockIdx.x - x0, groups = (x1 - x0) / X.splits;
        group_product<T, false, false, 2, NW, Z ? 0 : -1, ALONE, Z == 2>(X, X.first + on_xcd(b % groups, groups), b / groups, sums);
    }
}

inline long blocks_of(const Product &P, long m, long n) { return ((P.M + m - 1) / m) * ((P.N + n - 1) / n); }

// A grid ends at 2^32 work items -- beyond, it is cut off without an error -- and a narrow layer of 2^27 rows has more: then the
// blocks go in several launches.  (A k range is only split where there are fewer blocks than CUs.)
inline long most(long threads) { return (1L << 31) / threads; }
template <class F>
int in_launches(long blocks, long threads, F &&one) {
    if (blocks > 0x7fffffffL) return SA_ERR_UNSUPPORTED;
    for (long at = 0; at < blocks; at += most(threads)) {
        one((unsigned)at, (unsigned)(blocks - at < most(threads) ? blocks - at : most(threads)));
        SA_CHECK_LAUNCH();
    }
    return SA_OK;
}

// four blocks of 32 x 32 for as many waves
template <class T>
__global__ __launch_bounds__(256, 4) void small_alone_kernel(Product P) {
    __shared__ __attribute__((aligned(16))) float sums[4 * 1024];
    group_product<T, false, true, 2, 4, -1, true>(P, P.first + on_xcd(blockIdx.x, gridDim.x), blockIdx.y, sums);
}
template <class T>
int launch_alone(Product P, hipStream_t s) {
    P.alone = 1;
    return in_launches((blocks_of(P, 32, 32) + 3) / 4, 256, [&](unsigned first, unsigned groups) {
        P.first = first;
        hipLaunchKernelGGL((small_alone_kernel<T>), dim3(groups, P.splits), dim3(256), 0, s, P);
    });
}

template <class T, bool TA, bool TB, int NA, int NB, int NW>
int launch(Product P, hipStream_t s) {
    return in_launches(blocks_of(P, 16 * NA, 16 * NB), NW * 64, [&](unsigned first, unsigned blocks) {
        P.first = first;
        hipLaunchKernelGGL((small_kernel<T, TA, TB, NA, NB, NW>), dim3(blocks, P.splits), dim3(NW * 64), 0, s, P);
    });
}

// pieces of c rows of an operand with rows contiguous: aligned, and no parts of them
inline bool whole(const void *p, long ld, long rows, long c, long e) {
    return ((uintptr_t)p % (c * e)) == 0 && ld % c == 0 && rows % c == 0;
}

template <class T>
int launch_forward(Product P, hipStream_t s) {
    constexpr long E = sizeof(T);
    auto can = [&](long c) { return whole(P.b, P.ldb, P.N, c, E) && P.N * P.splits >= 128 * 16 * c; };
    if (P.M > 32 || (P.M > 16 && !can(4))) {
        // blocks of 32 x 32; four waves suffice for four steps
        P.vec_b = whole(P.b, P.ldb, P.N, 2, E);
        if (P.kchunk <= (E == 4 ? 32 : 64) && blocks_of(P, 32, 32) >= 2048) return launch_alone<T>(P, s);
        return P.kchunk <= 128 ? launch<T, false, true, 2, 2, 4>(P, s) : launch<T, false, true, 2, 2, 16>(P, s);
    }
    // few rows: as many columns per lane as the alignment allows and as still leave 128 workgroups
    P.vec_b = 1;
    if (P.M > 16) {
        if constexpr (E == 2)
            if (can(8)) return launch<T, false, true, 2, 8, 4>(P, s);
        return launch<T, false, true, 2, 4, 8>(P, s);
    }
    if constexpr (E == 2)
        if (can(8)) return launch<T, false, true, 1, 8, 8>(P, s);
    if (can(4)) return launch<T, false, true, 1, 4, 16>(P, s);
    if (whole(P.b, P.ldb, P.N, 2, E) && (E == 2 || P.N * P.splits >= 128 * 32)) return launch<T, false, true, 1, 2, 16>(P, s);
    return launch<T, false, true, 1, 1, 16>(P, s);
}

// nx, nw: blocks of a piece
template <class T, int Z, int WT, int NW>
int launch_backward(Product X, Product W, long nx, long nw, hipStream_t s) {
    // One wave's steps are few where a layer is narrow on one side, and the product on that side all output: fp32 6 x 3217 x
    // 16023, whose dW is 200 MB of sums of six terms, takes 190 us instead of 412.  (With a few workgroups only, the waves
    // share the work of a block as elsewhere.  No rule looks at the other product: the order of a sum does not depend on it.)
    auto groups = [](Product &P, long blocks) {
        P.alone = P.kchunk <= 64 && blocks * P.splits >= 2048;
        return (P.alone ? (blocks + NW - 1) / NW : blocks) * P.splits;
    };
    const long gx = groups(X, nx), gw = groups(W, nw), x0 = X.kchunk > W.kchunk ? 0 : gw;      // the longer ones first
    const dim3 block(NW * 64);
    auto launch = [&](unsigned blocks, unsigned x0, unsigned x1) {
        if (X.alone || W.alone) hipLaunchKernelGGL((small_backward_kernel<T, Z, WT, NW, true>), dim3(blocks), block, 0, s, X, W, x0, x1);
        else hipLaunchKernelGGL((small_backward_kernel<T, Z, WT, NW, false>), dim3(blocks), block, 0, s, X, W, x0, x1);
    };
    if (gx + gw <= most(NW * 64)) {
        launch((unsigned)(gx + gw), (unsigned)x0, (unsigned)(x0 + gx));
        SA_CHECK_LAUNCH();
        return SA_OK;
    }
    const int rc = in_launches(gx, NW * 64, [&](unsigned first, unsigned blocks) {
        X.first = first;
        launch(blocks, 0, blocks);
    });
    return rc ? rc : in_launches(gw, NW * 64, [&](unsigned first, unsigned blocks) {
        W.first = first;
        launch(blocks, 0, 0);
    });
}
template <class T, int WT>
int launch_backward(const Product &X, Product W, long nx, hipStream_t s) {
    constexpr long E = sizeof(T);
    long nw = 0;
    if (W.a || W.colsum || W.e.y) {
        W.vec_a = whole(W.a, W.lda, W.M, WT, E);
        W.vec_b = whole(W.b, W.ldb, W.N, WT, E);
        W.vec_z = W.z && whole(W.z, W.ldz, W.N, WT, E);
        nw = blocks_of(W, 16 * WT, 16 * WT);
    }
    const bool shorter = (nx == 0 || X.kchunk <= 128) && (nw == 0 || W.kchunk <= 128);
    if constexpr (E == 2)
        if (X.two || W.two) return shorter ? launch_backward<T, 2, WT, 4>(X, W, nx, nw, s) : launch_backward<T, 2, WT, 8>(X, W, nx, nw, s);
    if (X.z || W.z) return shorter ? launch_backward<T, 1, WT, 4>(X, W, nx, nw, s) : launch_backward<T, 1, WT, 8>(X, W, nx, nw, s);
    return shorter ? launch_backward<T, 0, WT, 4>(X, W, nx, nw, s) : launch_backward<T, 0, WT, 8>(X, W, nx, nw, s);
}
template <class T>
int launch_backward(const Product *px, const Product *pw, hipStream_t s) {
    Product X{}, W{};
    X.splits = W.splits = 1;
    if (px) X = *px;
    if (pw) W = *pw;
    const long nx = px ? blocks_of(X, 32, 32) : 0;
    // fp32 products take a CU long (16 x 16 x 4 per MFMA of 32 cycles): smaller blocks where there are few
    if constexpr (sizeof(T) == 4)
        if (blocks_of(W, 32, 32) * W.splits < 256) return launch_backward<T, 1>(X, W, nx, s);
    return launch_backward<T, 2>(X, W, nx, s);
}

}  // namespace

int dense::launch_small_forward(int type, const Product &P, hipStream_t s) {
    return type == kF32 ? launch_forward<float>(P, s) : type == kBF16 ? launch_forward<bf16_t>(P, s) : launch_forward<f16_t>(P, s);
}
int dense::launch_small_backward(int type, const Product *x, const Product *w, hipStream_t s) {
    return type == kF32 ? launch_backward<float>(x, w, s) : type == kBF16 ? launch_backward<bf16_t>(x, w, s)
                                                                         : launch_backward<f16_t>(x, w, s);
}
