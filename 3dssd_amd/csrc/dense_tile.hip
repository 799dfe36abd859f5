// The large products of the dense layer: operands of 16-bit elements with 16-byte aligned rows (others are brought into
// that form first, dense.hip).  D(m,n) = sum_k A(m,k) B(n,k), tiles of BM x BN per workgroup, k in steps of 64.
//
// Both operands go from memory straight into LDS (buffer loads with an LDS destination, 16 bytes per lane, whole 128-byte
// lines of a row).  A step's buffer ends with the operand, and what lies behind its last row reads as zeros; nothing outside
// the operand is read.  Past the last k both sides have to be zero: the buffer's end sees to it where rows run along m or n,
// an offset beyond the buffer where they run along k.  Past the last m or n anything may be read (of the same operand): it
// only reaches sums that are not stored.
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
//
// The grid is what the chip holds at once; a workgroup walks over its tiles (and pieces of k) as one sequence of steps.  The
// loads run on into the next tile while a tile's sums leave, so only the first tile waits for memory.  The sums go through
// LDS 16 rows at a time, in the part of the one free buffer of A that the same wave will load into next: nothing to wait for.
#include "dense_common.h"
#include "dense_products.h"

using namespace dense;

namespace {

constexpr int kBK = 64;
constexpr unsigned kOutside = 0x80000000u;             // past every buffer's range

typedef __attribute__((address_space(3))) char *lds_ptr;
typedef unsigned u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 *lds_s4;
typedef __attribute__((address_space(3))) s8 *lds_s8;
typedef __attribute__((address_space(3))) f4 *lds_f4;

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

__device__ __forceinline__ u4 buffer(const char *p, unsigned bytes) {
    return u4{(unsigned)(uintptr_t)p, (unsigned)((uintptr_t)p >> 32) & 0xffff, bytes, 0x00020000u};
}
// s_waitcnt's code for vmcnt(n) lgkmcnt(0)
constexpr int wait_code(int n) { return (n & 15) | (n >> 4) << 14 | 0x70; }

// Permutation of the 32-byte slots of row k: half a wave of ds_read_b64_tr_b16 reads rows 8 g .. + 4 of two neighbouring g,
// which have to lie in eight different slots (mod 8: 256 bytes, all banks once)
__device__ __forceinline__ int slot_of(int k) { return (k & 3) | ((k >> 3) & 1) << 2; }

// Permutation of the 16-byte pieces of a row of 64 k
__device__ __forceinline__ int piece_of(int row) { return row & 7; }

// One operand's way into LDS: a tile of R rows x 64 k by W waves, kLoads loads of 1024 bytes each.  Load q of wave w fills
// kilobyte q W + w: kStep rows (or k) lie between the loads of a wave, which leaves its permutation alone, so that one offset
// per lane serves them all and the buffer moves instead.
template <int R, int W, bool ROWS>
struct Loader {
    static constexpr int kLoads = R * kBK * 2 / 1024 / W, kStep = W * (ROWS ? 512 / R : 8);
    static_assert(kStep % 16 == 0, "the permutations use four bits");
    unsigned off;
    int key;                                                   // k of the lane's piece (k contiguous)
    __device__ __forceinline__ void init(int wave, int lane, long ld) {
        int outer, piece;
        if (ROWS) {
            outer = (wave * 1024 + lane * 16) / (R * 2);
            piece = (lane & (R / 8 - 1)) ^ (2 * slot_of(outer));
        } else {
            outer = wave * 8 + (lane >> 3);
            piece = (lane & 7) ^ piece_of(outer);
        }
        key = piece * 8;
        off = (unsigned)(outer * ld * 2 + piece * 16);
    }
    // The bytes of a step's buffer: k and rows of it are there
    static __device__ __forceinline__ unsigned bytes(long ld, int rows, int k) {
        const int outer = ROWS ? k : rows, inner = ROWS ? rows : k;
        return (unsigned)((outer - 1) * ld * 2 + ((inner * 2 + 15) & ~15));
    }
    // Load q; inc: the bytes of kStep rows (or k)
    __device__ __forceinline__ void load(u4 &r, unsigned inc, int k, unsigned lds, int wave, int q) const {
        lds_load(r, ROWS || key < k ? off : kOutside, lds + (q * W + wave) * 1024);
        if (q + 1 < kLoads) {
            const uint64_t p = ((uint64_t)r[1] << 32 | r[0]) + inc;
            r[0] = (unsigned)p;
            r[1] = (unsigned)(p >> 32);
            const int rest = (int)r[2] - (int)inc;             // (signed, for the scalar unit: both are below 2^31)
            r[2] = rest > 0 ? rest : 0;
        }
    }
};

// Fragments of a wave: blocks of 16 rows from row `first` on (a multiple of 64), 32 k each (half s of the step).  One address
// per wave: what a block, or a half, changes in it are bits that nothing else uses, flipped at the read.
template <int R, bool ROWS>
struct Reader {
    unsigned at;
    __device__ __forceinline__ void init(int first, int lane) {
        const int i = lane & 15, g = lane >> 4, kk = 8 * g + (i >> 2);
        at = ROWS ? kk * R * 2 + (((first / 16) ^ slot_of(kk)) * 32) + (i & 3) * 8 : (first + i) * 128 + ((g ^ piece_of(i)) * 16);
    }
    __device__ __forceinline__ s8 read(unsigned lds, int f, int s) const {
        if (ROWS) {                                            // (k + 4 has the same permutation)
            const unsigned p = ((lds + at) ^ (f * 32)) + s * 64 * R;
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)p);
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(p + 4 * R * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return *(lds_s8)(uintptr_t)(((lds + at) ^ (s * 64)) + f * 2048);
    }
};

// Planes of a fp32 operand (dense.hip): which plane of A meets which of B, the smallest terms first
__device__ constexpr int kPlaneA[6] = {2, 0, 1, 1, 0, 0}, kPlaneB[6] = {0, 2, 1, 0, 1, 0};

// f(Tag<i>): a register array's element by a number known at run time, without the array going to memory for it
template <int I, int N, class F>
__device__ __forceinline__ void pick(int i, F &&f) {
    if constexpr (I + 1 < N) {
        if (i == I) f(Tag<I>{});
        else pick<I + 1, N>(i, f);
    } else {
        f(Tag<I>{});
    }
}

// The kernel's argument, read anew: kept in scalar registers through the main loop its fields would not fit.
__device__ __forceinline__ const Product &arguments() {
    auto p = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const Product *)(__attribute__((address_space(4))) const Product *)p;
}

template <int BM, int BN, int WM, int WN, class MT, class OT, bool TA, bool TB>
__global__ __launch_bounds__(WM *WN * 64, 2) void tile_kernel(Product P) {
    constexpr int W = WM * WN, FM = BM / WM / 16, FN = BN / WN / 16, kA = BM * kBK * 2, kB = BN * kBK * 2;
    static_assert(FN == 4 && kA == W * 4096, "the epilogue takes 16 x 64 of a wave at a time, in the wave's share of a buffer");
    __shared__ __attribute__((aligned(1024))) char lds[3 * kA + 2 * kB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Items: the tiles of every piece of k.  Each XCD has a contiguous run of them, its workgroups take turns; tiles go in
    // groups of eight tile rows, so that neighbours share operands in one L2.
    const unsigned items = (unsigned)(((P.M + BM - 1) / BM) * ((P.N + BN - 1) / BN)) * P.splits;
    const unsigned xcd = blockIdx.x & 7, q8 = items >> 3, r8 = items & 7;
    const unsigned stride = (gridDim.x + 7 - xcd) >> 3, end = (xcd + 1) * q8 + (xcd + 1 < r8 ? xcd + 1 : r8);
    unsigned item = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);
    struct Place {
        long m0, n0;
        int first, steps, piece;
    };
    auto place = [](const Product &P, unsigned it) {
        const unsigned tm = (unsigned)((P.M + BM - 1) / BM), tn = (unsigned)((P.N + BN - 1) / BN), tiles = tm * tn;
        const unsigned piece = it / tiles, pos = it - piece * tiles;
        const unsigned group = pos / (8 * tn), in = pos - group * 8 * tn, rows = tm - group * 8 < 8 ? tm - group * 8 : 8;
        const int all = (int)((P.K + kBK - 1) / kBK) * P.passes, first = (int)(piece * P.kchunk), left = all - first;
        return Place{(long)(group * 8 + in % rows) * BM, (long)(in / rows) * BN, first, left < P.kchunk ? left : (int)P.kchunk, (int)piece};
    };

    Loader<BM, W, TA> la;
    Loader<BN, W, TB> lb;
    la.init(wave, lane, P.lda);
    lb.init(wave, lane, P.ldb);
    Reader<BM, TA> ra;
    Reader<BN, TB> rb;
    const int wm = wave % WM * (BM / WM), wn = wave / WM * (BN / WN);
    ra.init(wm, lane);
    rb.init(wn, lane);

    // The step whose loads go out: what is left of its item, its operands there, and its buffers and places in LDS.  A pass
    // over k is `per` steps, the last of k_tail; full and tail are the bytes of the operands' buffers in either.
    const int per = (int)((P.K + kBK - 1) / kBK), k_tail = (int)(P.K - (long)(per - 1) * kBK);
    const int step_a = (int)(TA ? P.lda : 1) * kBK * 2, step_b = (int)(TB ? P.ldb : 1) * kBK * 2;
    const unsigned inc_a = (unsigned)P.lda * 2 * la.kStep, inc_b = (unsigned)P.ldb * 2 * lb.kStep;
    unsigned load_item = item;
    int load_left = 0, pass = 0, kstep = 0, kk = 0;
    unsigned full_a = 0, full_b = 0, tail_a = 0, tail_b = 0;
    const char *at_a = nullptr, *at_b = nullptr;
    u4 buf_a, buf_b;
    const unsigned base = (unsigned)(uintptr_t)(lds_ptr)lds;
    unsigned to_a = base, to_b = base + 3 * kA;
    auto start_pass = [&]() {                              // a rare one: the product's description is read again
        const Product &R = arguments();
        const Place p = place(R, load_item - stride);
        at_a = (const char *)R.a + ((TA ? p.m0 : p.m0 * R.lda) + (R.passes > 1 ? kPlaneA[pass] * R.plane_a : 0)) * 2 + (long)kstep * step_a;
        at_b = (const char *)R.b + ((TB ? p.n0 : p.n0 * R.ldb) + (R.passes > 1 ? kPlaneB[pass] * R.plane_b : 0)) * 2 + (long)kstep * step_b;
    };
    auto next = [&]() {
        if (load_left == 0 && load_item < end) {
            const Product &R = arguments();
            const Place p = place(R, load_item);
            load_item += stride;
            load_left = p.steps;
            pass = p.first / per;
            kstep = p.first - pass * per;
            const int rows_a = R.M - p.m0 < BM ? (int)(R.M - p.m0) : BM, rows_b = R.N - p.n0 < BN ? (int)(R.N - p.n0) : BN;
            full_a = la.bytes(R.lda, rows_a, kBK);
            full_b = lb.bytes(R.ldb, rows_b, kBK);
            tail_a = la.bytes(R.lda, rows_a, k_tail);
            tail_b = lb.bytes(R.ldb, rows_b, k_tail);
            start_pass();
        }
        const bool some = load_left != 0, last = kstep == per - 1;     // past the last item: zeros, from nowhere
        kk = last ? k_tail : kBK;
        buf_a = buffer(at_a, some ? last ? tail_a : full_a : 0);
        buf_b = buffer(at_b, some ? last ? tail_b : full_b : 0);
        if (some) {
            --load_left;
            ++kstep;
            at_a += step_a;
            at_b += step_b;
            if (last && load_left) {
                kstep = 0;
                ++pass;
                start_pass();
            }
        }
    };
    constexpr int LA = Loader<BM, W, TA>::kLoads, LB = Loader<BN, W, TB>::kLoads;
    auto load_a = [&](int q) {
        la.load(buf_a, inc_a, kk, to_a, wave, q);
        if (q == LA - 1) to_a = to_a == base + 2 * kA ? base : to_a + kA;
    };
    auto load_b = [&](int q) {
        lb.load(buf_b, inc_b, kk, to_b, wave, q);
        if (q == LB - 1) to_b = base + 3 * kA + kB - (to_b - base - 3 * kA);
    };

    // Half a step: the products of the fragments in `use`, and between them the reads of the next half's fragments and the
    // loads, one operation every kEvery products.
    constexpr int kOps = FM + FN + (LA > LB ? LA : LB), kEvery = FM * FN / kOps;
    static_assert(kEvery >= 1, "an operation per product at most");
    struct Fragments { s8 a[FM], b[FN]; };
    f4 acc[FN][FM];
    Fragments f0, f1;
    auto read = [&](Fragments &f, unsigned a, unsigned b, int s, int op) {
        if (op < FN) f.b[op] = rb.read(b, op, s);
        else f.a[op - FN] = ra.read(a, op - FN, s);
    };
    auto half = [&](Fragments &use, Fragments &get, unsigned a, unsigned b, int s, auto &&load, int loads) {
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
    unsigned a0 = base, b0 = base + 3 * kA;            // this step's buffers
    for (; item < end; item += stride) {
        const int steps = place(arguments(), item).steps;
        // (the last half before read these too; kept from there they would take 48 registers through the end of the tile)
#pragma unroll
        for (int op = 0; op < FM + FN; ++op) read(f0, a0, b0, 0, op);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[j][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int step = 0; step < steps; ++step) {
            next();
            half(f0, f1, a0, b0, 1, load_a, LA);
            // step + 1 has arrived (this wave's part; the barrier makes it everyone's), and everyone has read all of this one
            __builtin_amdgcn_s_waitcnt(wait_code(LA));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            a0 = a0 == base + 2 * kA ? base : a0 + kA;
            b0 = base + 3 * kA + kB - (b0 - base - 3 * kA);
            half(f1, f0, a0, b0, 0, load_b, LB);
        }

        // The sums: 16 rows of the wave's 64 columns at a time, through 4 KB of LDS (16-byte pieces of a row permuted by ^ row),
        // so that eight lanes write 128 neighbouring bytes (16-bit) of a row.
        const Product &R = arguments();
        int l = lane;                                  // (computed from anew: kept, its offsets would take main loop registers)
        asm volatile("" : "+v"(l));
        const Place p = place(R, item);
        const long n = p.n0 + wn + (l & 7) * 8, mw = p.m0 + wm + (l >> 3), N = R.N, M = R.M;
        const unsigned mine = to_a + wave * 1024;      // kilobytes wave, W + wave, ..: four rows each
        const unsigned put = mine + ((l & 15) >> 2) * (W * 1024) + (l & 3) * 256, take = mine + (l >> 5) * (W * 1024) + ((l >> 3) & 3) * 256;
        auto leave = [&](int i) __attribute__((always_inline)) {       // blocks i of the wave's columns into LDS
            pick<0, FM>(i, [&](auto block) __attribute__((always_inline)) {
                constexpr int b = decltype(block)::value;
                const unsigned g = l >> 4, x = l & 15;
                f4 v[4] = {acc[0][b], acc[1][b], acc[2][b], acc[3][b]};
                // (branches that only differ in where they read the array from would be made one, and the array memory)
                asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]));
#pragma unroll
                for (int j = 0; j < 4; ++j) *(lds_f4)(uintptr_t)(put + (((4 * j + g) ^ x) * 16)) = v[j];
            });
        };
        auto row = [&](int q, float *v) __attribute__((always_inline)) {              // columns n .. n + 8 of row 8 q + l / 8 of them
            const int r = 8 * q + (l >> 3), piece = (l & 7) * 2;
            const f4 lo = *(lds_f4)(uintptr_t)(take + q * 2 * (W * 1024) + ((piece ^ r) * 16));
            const f4 hi = *(lds_f4)(uintptr_t)(take + q * 2 * (W * 1024) + (((piece + 1) ^ r) * 16));
#pragma unroll
            for (int c = 0; c < 4; ++c) v[c] = lo[c], v[4 + c] = hi[c];
        };
        if (R.splits > 1) {
            const long Np = round_up(N, 4);
            float *to = R.part + ((long)p.piece * M + mw) * Np + n;
#pragma unroll 1
            for (int i = 0; i < FM; ++i) {
                leave(i);
#pragma unroll
                for (int q = 0; q < 2; ++q, to += 8 * Np) {
                    float v[8];
                    row(q, v);
                    if (mw + 16 * i + 8 * q < M) {
                        if (n < N) *(f4 *)to = f4{v[0], v[1], v[2], v[3]};
                        if (n + 4 < N) *(f4 *)(to + 4) = f4{v[4], v[5], v[6], v[7]};
                    }
                }
            }
        } else if (p.n0 + BN <= N) {
            // whole columns: no lane looks at the edge, and the activation is chosen once
            const Epilogue &E = R.e;
            const long ldy = E.ldy, ldp = E.ldp, ldr = E.ldr;
            OT *to = (OT *)E.y + mw * ldy + n, *pre = (OT *)E.pre + mw * ldp + n;
            const OT *res = (const OT *)E.res + mw * ldr + n;
            const bool has_pre = E.pre, has_res = E.res;
            float bias[8];
            load_bias<OT, 8>(E, n, N, bias);
            Pack<OT, 8> r[2] = {};
            auto ask = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                for (int q = 0; q < 2; ++q, res += 8 * ldr)
                    if (mw + 16 * i + 8 * q < M) r[q] = load_pack<OT, 8>(res);
            };
            if (has_res) ask(0);
            with_activation(E.act, [&](auto act) __attribute__((always_inline)) {
#pragma unroll 1
                for (int i = 0; i < FM; ++i) {
                    leave(i);
                    const Pack<OT, 8> now[2] = {r[0], r[1]};
                    if (has_res && i + 1 < FM) ask(i + 1);
#pragma unroll
                    for (int q = 0; q < 2; ++q, to += 8 * ldy, pre += 8 * ldp) {
                        float z[8];
                        row(q, z);
                        if (mw + 16 * i + 8 * q >= M) continue;
                        Pack<OT, 8> o;
#pragma unroll
                        for (int c = 0; c < 8; ++c) z[c] += bias[c];
                        if (has_pre) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) o.x[c] = from_f32<OT>(z[c]);
                            store_pack<OT, 8>(pre, o);
                        }
#pragma unroll
                        for (int c = 0; c < 8; ++c) z[c] = activate<decltype(act)::value>(z[c]);
                        if (has_res) {
#pragma unroll
                            for (int c = 0; c < 8; ++c) z[c] += to_f32<OT>(now[q].x[c]);
                        }
#pragma unroll
                        for (int c = 0; c < 8; ++c) o.x[c] = from_f32<OT>(z[c]);
                        store_pack<OT, 8>(to, o);
                    }
                }
            });
        } else {
            float bias[8];
            load_bias<OT, 8>(R.e, n, N, bias);
#pragma unroll 1
            for (int i = 0; i < FM; ++i) {
                leave(i);
#pragma unroll 1
                for (int q = 0; q < 2; ++q) {
                    const long m = mw + 16 * i + 8 * q;
                    float v[8];
                    row(q, v);
                    if (m >= M || n >= N) continue;
                    Pack<OT, 8> r{};
                    if (R.e.res) r = load_residual<OT, 8>(R.e, m, n, N);
                    finish<OT, 8>(R.e, m, n, N, v, bias, r);
                }
            }
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                // the zeros of the steps past the end have arrived too
}

template <int BM, int BN, int WM, int WN, class MT, class OT>
int launch(bool ta, bool tb, const Product &P, int slots, hipStream_t s) {
    const long items = ((P.M + BM - 1) / BM) * ((P.N + BN - 1) / BN) * P.splits;
    if (items > 0x3fffffffL) return SA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(items < slots ? items : slots)), block(WM * WN * 64);
    if (ta) hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, true, true>), grid, block, 0, s, P);
    else if (tb) hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, false, true>), grid, block, 0, s, P);
    else hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, false, false>), grid, block, 0, s, P);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

template <class MT, class OT>
int launch(int shape, bool ta, bool tb, const Product &P, hipStream_t s) {
    if (shape == kTile256) return launch<256, 256, 2, 4, MT, OT>(ta, tb, P, 256, s);
    if (shape == kTile256x128) return launch<256, 128, 4, 2, MT, OT>(ta, tb, P, 256, s);
    return launch<128, 128, 2, 2, MT, OT>(ta, tb, P, 512, s);
}

}  // namespace

int dense::launch_tiles(int shape, int type, int out_type, bool ta, bool tb, const Product &P, hipStream_t s) {
    if (out_type == kF32) return launch<bf16_t, float>(shape, ta, tb, P, s);
    if (type == kBF16) return launch<bf16_t, bf16_t>(shape, ta, tb, P, s);
    return launch<f16_t, f16_t>(shape, ta, tb, P, s);
}
