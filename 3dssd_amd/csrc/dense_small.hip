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
#include "dense_common.h"
#include "dense_tile.h"

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
    __device__ __forceinline__ void fetch(Regs &r, const char *base, int left, bool vec) const {
        const auto b = buffer(base);
#pragma unroll
        for (int t = 0; t < N; ++t) {
            if (vec && (left & 7) == 0) {              // (left: valid k of this step, up to 32)
#pragma unroll
                for (int h = 0; h < E / 2; ++h) r.v[t][h] = load<16>(b, g8 < left ? off[t] + 16 * h : kOutside);
            } else {
#pragma unroll
                for (int h = 0; h < E / 2; ++h) r.v[t][h] = u4{0, 0, 0, 0};
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const unsigned e = load<E>(b, g8 + j < left ? off[t] + j * E : kOutside);
                    if constexpr (E == 4) r.v[t][j / 4][j % 4] = e;
                    else r.v[t][0][j / 2] |= j & 1 ? e << 16 : e;
                }
            }
        }
    }
    static __device__ __forceinline__ s8 fragment(const Regs &r, int t) { return __builtin_bit_cast(s8, r.v[t][0]); }
    static __device__ __forceinline__ float value(const Regs &r, int t, int j) { return __uint_as_float(r.v[t][j / 4 * (E / 4)][j % 4]); }
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
    static __device__ __forceinline__ s8 fragment(const Regs &r, int t) {
        typename Bytes<16>::t o;
#pragma unroll
        for (int i = 0; i < 4; ++i)                    // the halves t of k 2 i and 2 i + 1
            o[i] = __builtin_amdgcn_perm(word(r.v[2 * i + 1], t / 2), word(r.v[2 * i], t / 2), t & 1 ? 0x07060302 : 0x05040100);
        return __builtin_bit_cast(s8, o);
    }
    static __device__ __forceinline__ float value(const Regs &r, int t, int j) { return __uint_as_float(word(r.v[j], t)); }
    static __device__ __forceinline__ int row(int t, int i) { return N * i + t; }
};

template <class T, bool TA, bool TB, int NA, int NB, int NW>
__global__ __launch_bounds__(NW * 64, NW / 4) void small_kernel(Product P) {
    constexpr int E = sizeof(T), kM = 16 * NA, kN = 16 * NB, kAhead = E * (NA + NB) <= 8 ? 4 : 2;
    static_assert(NA * NB * NW <= 64, "the waves' sums: 64 KB");
    __shared__ __attribute__((aligned(16))) float sums[NW * kM * kN];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // neighbouring blocks of n on one XCD: they share the rows of A, and with pieces below 16 bytes the lines of B
    const unsigned q8 = gridDim.x >> 3, r8 = gridDim.x & 7, xcd = blockIdx.x & 7;
    const unsigned pos = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3), nb = (unsigned)((P.N + kN - 1) / kN);
    const long m0 = (long)(pos / nb) * kM, n0 = (long)(pos % nb) * kN;
    const long k0 = (long)blockIdx.y * P.kchunk, kend = k0 + P.kchunk < P.K ? k0 + P.kchunk : P.K;
    const char *A = (const char *)P.a + (TA ? m0 + k0 * P.lda : m0 * P.lda + k0) * E;
    const char *B = (const char *)P.b + (TB ? n0 + k0 * P.ldb : n0 * P.ldb + k0) * E;
    const long stepa = (TA ? P.lda : 1) * 32 * E, stepb = (TB ? P.ldb : 1) * 32 * E;
    typedef Side<T, TA, NA> SA;
    typedef Side<T, TB, NB> SB;
    SA a;
    SB b;
    a.init(lane, P.lda, P.M - m0);
    b.init(lane, P.ldb, P.N - n0);

    f4 acc[NB][NA] = {};
    typename SA::Regs ra[kAhead];
    typename SB::Regs rb[kAhead];
    const long steps = (kend - k0 + 31) / 32;
    auto fetch = [&](int slot, long s) {
        const long l = kend - k0 - s * 32;
        const int left = l < 32 ? (int)l : 32;
        a.fetch(ra[slot], A + s * stepa, left, P.vec_a);
        b.fetch(rb[slot], B + s * stepb, left, P.vec_b);
    };
    auto multiply = [&](int slot) {
        if constexpr (E == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int y = 0; y < NB; ++y)
#pragma unroll
                    for (int x = 0; x < NA; ++x)
                        acc[y][x] = __builtin_amdgcn_mfma_f32_16x16x4f32(SB::value(rb[slot], y, j), SA::value(ra[slot], x, j),
                                                                         acc[y][x], 0, 0, 0);
        } else {
            s8 fa[NA];
#pragma unroll
            for (int x = 0; x < NA; ++x) fa[x] = SA::fragment(ra[slot], x);
#pragma unroll
            for (int y = 0; y < NB; ++y) {
                const s8 fb = SB::fragment(rb[slot], y);
#pragma unroll
                for (int x = 0; x < NA; ++x) {
                    if constexpr (__is_same(T, bf16_t))
                        acc[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, fb), __builtin_bit_cast(b8, fa[x]),
                                                                            acc[y][x], 0, 0, 0);
                    else
                        acc[y][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, fb), __builtin_bit_cast(h8, fa[x]),
                                                                           acc[y][x], 0, 0, 0);
                }
            }
        }
    };
    long s = wave;
#pragma unroll
    for (int h = 0; h < kAhead; ++h)
        if (s + h * NW < steps) fetch(h, s + h * NW);
    for (; s < steps; s += kAhead * NW) {
#pragma unroll
        for (int h = 0; h < kAhead; ++h) {
            if (s + h * NW < steps) multiply(h);
            if (s + (h + kAhead) * NW < steps) fetch(h, s + (h + kAhead) * NW);
        }
    }

#pragma unroll
    for (int x = 0; x < NA; ++x)
#pragma unroll
        for (int y = 0; y < NB; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sums[(wave * kM + SA::row(x, lane & 15)) * kN + SB::row(y, 4 * (lane >> 4) + r)] = acc[y][x][r];
    __syncthreads();
    const long Np = round_up(P.N, 4);
#pragma unroll 1
    for (int q = threadIdx.x; q < kM * kN / 4; q += NW * 64) {
        const int lm = q / (kN / 4), ln = q % (kN / 4) * 4;
        const long m = m0 + lm, n = n0 + ln;
        if (m >= P.M || n >= P.N) continue;
        f4 v = *(const f4 *)(sums + lm * kN + ln);
#pragma unroll
        for (int w = 1; w < NW; ++w) v += *(const f4 *)(sums + (w * kM + lm) * kN + ln);
        if (P.splits > 1) {
            *(f4 *)(P.part + ((long)blockIdx.y * P.M + m) * Np + n) = v;
        } else {
            float bias[4];
            load_bias<T, 4>(P.e, n, P.N, bias);
            const float o[4] = {v[0], v[1], v[2], v[3]};
            finish<T, 4>(P.e, m, n, P.N, o, bias);
        }
    }
}

template <class T, bool TA, bool TB, int NA, int NB, int NW>
int launch(const Product &P, hipStream_t s) {
    const long blocks = ((P.M + 16 * NA - 1) / (16 * NA)) * ((P.N + 16 * NB - 1) / (16 * NB));
    if (blocks > 0x7fffffffL) return SA_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((small_kernel<T, TA, TB, NA, NB, NW>), dim3((unsigned)blocks, P.splits), dim3(NW * 64), 0, s, P);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

// pieces of c rows of an operand with rows contiguous: aligned, and no parts of them
inline bool whole(const void *p, long ld, long rows, long c, long e) {
    return ((uintptr_t)p % (c * e)) == 0 && ld % c == 0 && rows % c == 0;
}

template <class T>
int launch(bool ta, bool tb, Product P, hipStream_t s) {
    constexpr long E = sizeof(T);
    if (P.M > 16 || ta || !tb) {
        // blocks of 32 x 32; four waves suffice for four steps
        const bool shorter = P.kchunk <= 128;
        if (ta) P.vec_a = whole(P.a, P.lda, P.M, 2, E);
        if (tb) P.vec_b = whole(P.b, P.ldb, P.N, 2, E);
        if (ta) return shorter ? launch<T, true, true, 2, 2, 4>(P, s) : launch<T, true, true, 2, 2, 16>(P, s);
        if (!tb) return shorter ? launch<T, false, false, 2, 2, 4>(P, s) : launch<T, false, false, 2, 2, 16>(P, s);
        if (P.M > 32 || !whole(P.b, P.ldb, P.N, 4, E) || P.N * P.splits < 128 * 64)
            return shorter ? launch<T, false, true, 2, 2, 4>(P, s) : launch<T, false, true, 2, 2, 16>(P, s);
    }
    // few rows: as many columns per lane as the alignment allows and as still leave 128 workgroups
    auto can = [&](long c) { return whole(P.b, P.ldb, P.N, c, E) && P.N * P.splits >= 128 * 16 * c; };
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

}  // namespace

int dense::launch_small(int type, bool ta, bool tb, const Product &P, hipStream_t s) {
    return type == kF32 ? launch<float>(ta, tb, P, s) : type == kBF16 ? launch<bf16_t>(ta, tb, P, s) : launch<f16_t>(ta, tb, P, s);
}
