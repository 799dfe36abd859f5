// The large products of the dense layer: operands of 16-bit elements with 16-byte aligned rows (others are brought into
// that form first, dense.hip).  D(m,n) = sum_k A(m,k) B(n,k), tiles of BM x BN per workgroup, k in steps of 64.
//
// Both operands go from memory straight into LDS (buffer loads with an LDS destination, 16 bytes per lane, whole 128-byte
// lines of a row).  A lane outside the operand gets an offset beyond the buffer's range, which fills its 16 bytes with zeros:
// no edge of m, n or k needs code of its own, and nothing outside the operand is read.
//   k contiguous      LDS rows of 64 k (128 bytes), whose 16-byte pieces are permuted by the row, for ds_read_b128.
//   m / n contiguous  LDS rows of one k, whose 32-byte slots are permuted by k, for ds_read_b64_tr_b16, which transposes
//                     4 k x 16 rows between the lanes.
// Either way a fragment read touches every bank once.  The permutation costs nothing: a lane of the load picks which 16
// bytes it fetches, the LDS side stays linear.
//
// A step is two halves of 32 k.  While a wave multiplies the fragments of one half it reads those of the next and sends off
// loads, one such operation between two MFMAs.  LDS holds three steps of A and two of B (160 KB at 256 x 256): the first
// half of step t loads A of step t + 2, into the buffer that step t - 1 has left; the second loads B of step t + 2, into that
// of step t, which no wave reads any more.  One barrier per step, between the halves, orders both, and the loads have one to
// two steps of products to arrive in.
#include "dense_common.h"
#include "dense_products.h"

using namespace dense;

namespace {

constexpr int kBK = 64;
constexpr unsigned kOutside = 0x80000000u;             // past every buffer's range

typedef __attribute__((address_space(3))) char *lds_ptr;
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 *lds_s4;

template <class MT> __device__ __forceinline__ f4 mfma(s8 a, s8 b, f4 c);
template <> __device__ __forceinline__ f4 mfma<bf16_t>(s8 a, s8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f4 mfma<f16_t>(s8 a, s8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// 16 bytes per lane from buffer r + off to LDS `to` + 16 lane.  Written as assembly because the compiler, which knows the
// builtin's loads by the LDS they write, waits for all of them in front of the next read of any LDS -- the other buffer's
// included -- and the loads would never fly under the products.  Nothing comes back in registers; the kernel waits for
// vmcnt itself, in front of the barrier that publishes the buffer.  (Nothing else in the kernel uses m0.)
__device__ __forceinline__ void lds_load(u4 r, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r), "s"(to) : "memory");
}

__device__ __forceinline__ u4 buffer(const char *p) {
    return u4{(unsigned)(uintptr_t)p, (unsigned)((uintptr_t)p >> 32) & 0xffff, 0x7fffffffu, 0x00020000u};
}
// s_waitcnt's code for vmcnt(n) lgkmcnt(0)
constexpr int wait_code(int n) { return (n & 15) | (n >> 4) << 14 | 0x70; }

// Permutation of the 32-byte slots of row k: half a wave of ds_read_b64_tr_b16 reads rows 8 g .. + 4 of two neighbouring g,
// which have to lie in eight different slots (mod 8: 256 bytes, all banks once)
__device__ __forceinline__ int slot_of(int k) { return (k & 3) | ((k >> 3) & 1) << 2; }

// Permutation of the 16-byte pieces of a row of 64 k
__device__ __forceinline__ int piece_of(int row) { return row & 7; }

// One operand's way into LDS: a tile of R rows x 64 k by W waves.
template <int R, int W, bool ROWS>
struct Loader {
    static constexpr int kLoads = R * kBK * 2 / 1024 / W;      // 1024-byte loads per wave
    static constexpr int kPieces = R / 8;                      // 16-byte pieces of one k (ROWS)
    unsigned off[kLoads];
    int k[kLoads];                                             // k of the lane's piece inside a step
    __device__ __forceinline__ void init(int wave, int lane, long ld, long rows_left) {
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
            const int j = wave * kLoads + q;                   // which kilobyte of the tile
            if (ROWS) {
                const int b = j * 1024 + lane * 16;
                const int kk = b / (R * 2), p = (b >> 4) & (kPieces - 1);
                const int piece = p ^ (2 * slot_of(kk));
                k[q] = kk;
                off[q] = piece * 8 < rows_left ? (unsigned)(kk * ld * 2 + piece * 16) : kOutside;
            } else {
                const int row = j * 8 + (lane >> 3), piece = (lane & 7) ^ piece_of(row);
                k[q] = piece * 8;
                off[q] = row < rows_left ? (unsigned)(row * ld * 2 + piece * 16) : kOutside;
            }
        }
    }
    // Load q of this wave.  r: the tile's first row at this step's first k; k_left: valid k indices from there (none: all
    // lanes get zeros)
    __device__ __forceinline__ void load(u4 r, int k_left, unsigned lds, int wave, int q) const {
        lds_load(r, k[q] < k_left ? off[q] : kOutside, lds + (wave * kLoads + q) * 1024);
    }
};

// Fragments of a wave: F blocks of 16 rows from row `first` on, 32 k each (half s of the step)
template <int R, int F, bool ROWS>
struct Reader {
    int at[ROWS ? F : 2];
    __device__ __forceinline__ void init(int first, int lane) {
        const int i = lane & 15, g = lane >> 4;
        if (ROWS) {
            const int kk = 8 * g + (i >> 2);
#pragma unroll
            for (int f = 0; f < F; ++f) at[f] = kk * R * 2 + (((first / 16 + f) ^ slot_of(kk)) * 32) + (i & 3) * 8;
        } else {
            at[0] = (first + i) * 128 + ((g ^ piece_of(i)) * 16);
            at[1] = at[0] ^ 64;
        }
    }
    __device__ __forceinline__ s8 read(const char *lds, int f, int s) const {
        if (ROWS) {                                            // (k + 4 has the same permutation)
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + at[f] + s * 64 * R));
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + at[f] + s * 64 * R + 4 * R * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return *(const s8 *)(lds + at[s] + f * 2048);
    }
};

// Planes of a fp32 operand (dense.hip): which plane of A meets which of B, the smallest terms first
__device__ constexpr int kPlaneA[6] = {2, 0, 1, 1, 0, 0}, kPlaneB[6] = {0, 2, 1, 0, 1, 0};

template <int BM, int BN, int WM, int WN, class MT, class OT, bool TA, bool TB>
__global__ __launch_bounds__(WM *WN * 64, BM == 256 ? WM * WN / 4 : 2) void tile_kernel(Product P) {
    constexpr int W = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, kA = BM * kBK * 2, kB = BN * kBK * 2;
    static_assert(FN % 4 == 0 && FM % 4 == 0 && W * 16384 <= 3 * kA + 2 * kB, "the epilogue takes 64 x 64 of a wave at a time");
    __shared__ __attribute__((aligned(1024))) char lds[3 * kA + 2 * kB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // tiles in groups of eight tile rows, each XCD a contiguous run of them: neighbours share operands in one L2
    const unsigned tm = (unsigned)((P.M + BM - 1) / BM), tn = (unsigned)((P.N + BN - 1) / BN), total = tm * tn;
    const unsigned q8 = total >> 3, r8 = total & 7, xcd = blockIdx.x & 7;
    const unsigned pos = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
    const unsigned group = pos / (8 * tn), in = pos - group * 8 * tn, rows = tm - group * 8 < 8 ? tm - group * 8 : 8;
    const long m0 = (long)(group * 8 + in % rows) * BM, n0 = (long)(in / rows) * BN;

    Loader<BM, W, TA> la;
    Loader<BN, W, TB> lb;
    la.init(wave, lane, P.lda, P.M - m0);
    lb.init(wave, lane, P.ldb, P.N - n0);
    Reader<BM, FM, TA> ra;
    Reader<BN, FN, TB> rb;
    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    ra.init(wm, lane);
    rb.init(wn, lane);

    const long per = (P.K + kBK - 1) / kBK;            // steps of one pass over k
    const long first = (long)blockIdx.y * P.kchunk, all = per * P.passes;
    const int steps = (int)((first + P.kchunk < all ? first + P.kchunk : all) - first);
    const char *A0 = (const char *)P.a + (TA ? m0 : m0 * P.lda) * 2, *B0 = (const char *)P.b + (TB ? n0 : n0 * P.ldb) * 2;
    const long stepa = (TA ? P.lda : 1) * kBK * 2, stepb = (TB ? P.ldb : 1) * kBK * 2;

    // the step whose loads go out: its buffers, valid k, places in LDS
    int pass = (int)(first / per), ahead = 0;
    long kstep = first - pass * per;
    const unsigned base = (unsigned)(uintptr_t)(lds_ptr)lds;
    unsigned to_a = base, to_b = base + 3 * kA;
    u4 ra_, rb_;
    int left = 0;
    auto next = [&]() {
        const char *a = A0 + kstep * stepa, *b = B0 + kstep * stepb;
        if (P.passes > 1 && pass < 6) {
            a += kPlaneA[pass] * P.plane_a * 2;
            b += kPlaneB[pass] * P.plane_b * 2;
        }
        ra_ = buffer(a);
        rb_ = buffer(b);
        const long k_left = P.K - kstep * kBK;
        left = ahead >= steps ? 0 : k_left < kBK ? (int)k_left : kBK;
        ++ahead;
        if (++kstep == per) kstep = 0, ++pass;
    };
    constexpr int LA = Loader<BM, W, TA>::kLoads, LB = Loader<BN, W, TB>::kLoads;
    auto load_a = [&](int q) {
        la.load(ra_, left, to_a, wave, q);
        if (q == LA - 1) to_a = to_a == base + 2 * kA ? base : to_a + kA;
    };
    auto load_b = [&](int q) {
        lb.load(rb_, left, to_b, wave, q);
        if (q == LB - 1) to_b = base + 3 * kA + kB - (to_b - base - 3 * kA);
    };

    // Half a step: the products of the fragments in `use`, and between them the reads of the next half's fragments and the
    // loads, one operation every kEvery products.
    constexpr int kOps = FM + FN + (LA > LB ? LA : LB), kEvery = FM * FN / kOps;
    static_assert(kEvery >= 1, "an operation per product at most");
    struct Fragments { s8 a[FM], b[FN]; };
    f4 acc[FN][FM] = {};
    Fragments f0, f1;
    auto read = [&](Fragments &f, const char *a, const char *b, int s, int op) {
        if (op < FN) f.b[op] = rb.read(b, op, s);
        else f.a[op - FN] = ra.read(a, op - FN, s);
    };
    auto half = [&](Fragments &use, Fragments &get, const char *a, const char *b, int s, auto &&load, int loads) {
#pragma unroll
        for (int x = 0; x < FM * FN; ++x) {
            const int j = x / FM, i = x % FM;
            acc[j][i] = mfma<MT>(use.b[j], use.a[i], acc[j][i]);
            if (x % kEvery == 0) {
                const int op = x / kEvery;
                if (op < FM + FN) read(get, a, b, s, op);
                else if (op < FM + FN + loads) load(op - FM - FN);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int i = 0; i < 2; ++i) {                      // steps 0 and 1
        next();
#pragma unroll
        for (int q = 0; q < LA; ++q) load_a(q);
#pragma unroll
        for (int q = 0; q < LB; ++q) load_b(q);
    }
    // loads return in order: with those of step 1 outstanding, step 0's have arrived
    __builtin_amdgcn_s_waitcnt(wait_code(LA + LB));
    __builtin_amdgcn_s_barrier();
    const char *a0 = lds, *b0 = lds + 3 * kA;          // this step's buffers
#pragma unroll
    for (int op = 0; op < FM + FN; ++op) read(f0, a0, b0, 0, op);
    for (int step = 0; step < steps; ++step) {
        next();
        half(f0, f1, a0, b0, 1, load_a, LA);
        // step + 1 has arrived (this wave's part; the barrier makes it everyone's), and everyone has read all of this step
        __builtin_amdgcn_s_waitcnt(wait_code(LA));
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        a0 = a0 == lds + 2 * kA ? lds : a0 + kA;
        b0 = lds + 3 * kA + kB - (b0 - lds - 3 * kA);
        half(f1, f0, a0, b0, 0, load_b, LB);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                // the zeros of the steps past the end have arrived too

    // The sums leave through LDS, 64 x 64 of a wave at a time (16 KB of its own): the epilogue's code then exists once, and
    // eight lanes write 128 neighbouring bytes (16-bit) of a row.  16-byte pieces of a row are permuted by ^ row & 15.
    const long Np = round_up(P.N, 4);
    char *mine = lds + wave * 16384;
    __syncthreads();
#pragma unroll 1
    for (int h = 0; h < FM * FN / 16; ++h) {
#pragma unroll
        for (int hh = 0; hh < FM * FN / 16; ++hh)
            if (hh == h) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int row = 16 * i + (lane & 15), piece = (4 * j + (lane >> 4)) ^ (lane & 15);
                        *(f4 *)(mine + row * 256 + piece * 16) = acc[4 * (hh / (FM / 4)) + j][4 * (hh % (FM / 4)) + i];
                    }
            }
        const long n = n0 + wn + 64 * (h / (FM / 4)) + (lane & 7) * 8, mh = m0 + wm + 64 * (h % (FM / 4));
        float bias[8];
        load_bias<OT, 8>(P.e, n, P.N, bias);           // (none in a product whose sums are joined later)
#pragma unroll 1
        for (int q = 0; q < 8; ++q) {
            const int row = q * 8 + (lane >> 3), piece = (lane & 7) * 2;
            const f4 lo = *(const f4 *)(mine + row * 256 + ((piece ^ (row & 15)) * 16));
            const f4 hi = *(const f4 *)(mine + row * 256 + (((piece + 1) ^ (row & 15)) * 16));
            const long m = mh + row;
            if (m >= P.M || n >= P.N) continue;
            if (P.splits > 1) {
                float *p = P.part + ((long)blockIdx.y * P.M + m) * Np + n;
                *(f4 *)p = lo;
                if (n + 4 < P.N) *(f4 *)(p + 4) = hi;
            } else {
                const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                finish<OT, 8>(P.e, m, n, P.N, v, bias);
            }
        }
    }
}

template <int BM, int BN, int WM, int WN, class MT, class OT>
int launch(bool ta, bool tb, const Product &P, hipStream_t s) {
    const long tiles = ((P.M + BM - 1) / BM) * ((P.N + BN - 1) / BN);
    if (tiles > 0x3fffffffL) return SA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)tiles, P.splits), block(WM * WN * 64);
    if (ta) hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, true, true>), grid, block, 0, s, P);
    else if (tb) hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, false, true>), grid, block, 0, s, P);
    else hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, false, false>), grid, block, 0, s, P);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

template <class MT, class OT>
int launch(int edge, bool ta, bool tb, const Product &P, hipStream_t s) {
    if (edge == 256) return launch<256, 256, 2, 4, MT, OT>(ta, tb, P, s);
    return launch<128, 128, 2, 2, MT, OT>(ta, tb, P, s);
}

}  // namespace

int dense::launch_tiles(int edge, int type, int out_type, bool ta, bool tb, const Product &P, hipStream_t s) {
    if (out_type == kF32) return launch<bf16_t, float>(edge, ta, tb, P, s);
    if (type == kBF16) return launch<bf16_t, bf16_t>(edge, ta, tb, P, s);
    return launch<f16_t, f16_t>(edge, ta, tb, P, s);
}
