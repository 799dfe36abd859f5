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
#include "dense_lds.h"
#include "dense_products.h"

using namespace dense;

namespace {

constexpr int kBK = 64;

// Planes of a fp32 operand (dense.hip): which plane of A meets which of B, the smallest terms first
__device__ constexpr int kPlaneA[6] = {2, 0, 1, 1, 0, 0}, kPlaneB[6] = {0, 2, 1, 0, 1, 0};
// Of two passes the first has the second plane of dZ; the other operand has one plane (and 0 elements to the next)
__device__ __forceinline__ int plane_of(const int (&table)[6], int pass, int passes) { return passes == 2 ? 1 - pass : table[pass]; }

// CARRY: two passes of fp16, of which the first's operand has a scale.  (In a kernel of its own: the tile's end spills for it, and one
// pass of 4096^3 took 250 us in both gradients instead of 235.)
template <int BM, int BN, int WM, int WN, class MT, class OT, bool TA, bool TB, bool CARRY = false>
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

    Loader<BM, W, TA, kBK> la;
    Loader<BN, W, TB, kBK> lb;
    la.init(wave, lane, P.lda);
    lb.init(wave, lane, P.ldb);
    Reader<BM, TA, kBK> ra;
    Reader<BN, TB, kBK> rb;
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
        const Place p = place<BM, BN, kBK>(R, load_item - stride);
        at_a = (const char *)R.a + ((TA ? p.m0 : p.m0 * R.lda) + (R.passes > 1 ? plane_of(kPlaneA, pass, R.passes) * R.plane_a : 0)) * 2 + (long)kstep * step_a;
        at_b = (const char *)R.b + ((TB ? p.n0 : p.n0 * R.ldb) + (R.passes > 1 ? plane_of(kPlaneB, pass, R.passes) * R.plane_b : 0)) * 2 + (long)kstep * step_b;
    };
    auto next = [&]() {
        if (load_left == 0 && load_item < end) {
            const Product &R = arguments();
            const Place p = place<BM, BN, kBK>(R, load_item);
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
    constexpr int LA = Loader<BM, W, TA, kBK>::kLoads, LB = Loader<BN, W, TB, kBK>::kLoads;
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
        const Place whole = place<BM, BN, kBK>(arguments(), item);
        // fp16's second plane of dZ has a scale: what its pass, the first of two, has summed loses it before the next
        int run = whole.steps, rest = 0;
        if constexpr (CARRY) {
            run = per - whole.first < 0 ? 0 : per - whole.first < run ? per - whole.first : run;
            rest = whole.steps - run;
        }
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[j][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int part = 0;; ++part) {
            // (the last half before read these too; kept from there they would take 48 registers through the end of the tile)
#pragma unroll
            for (int op = 0; op < FM + FN; ++op) read(f0, a0, b0, 0, op);
            for (int step = 0; step < run; ++step) {
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
            if (!CARRY || part == 1) break;
#pragma unroll
            for (int j = 0; j < FN; ++j)
#pragma unroll
                for (int i = 0; i < FM; ++i) acc[j][i] *= 1.0f / Low<f16_t>::scale;
            run = rest;
        }

        leave_tile<BM, BN, kBK, W, OT>(acc, item, wm, wn, wave, lane, to_a);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                // the zeros of the steps past the end have arrived too
}

template <int BM, int BN, int WM, int WN, class MT, class OT>
int launch(bool ta, bool tb, const Product &P, int slots, hipStream_t s) {
    const long items = ((P.M + BM - 1) / BM) * ((P.N + BN - 1) / BN) * P.splits;
    if (items > 0x3fffffffL) return SA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(items < slots ? items : slots)), block(WM * WN * 64);
    auto go = [&](auto carry) {
        constexpr bool C = decltype(carry)::value;
        if (ta) hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, true, true, C>), grid, block, 0, s, P);
        else if (tb) hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, false, true>), grid, block, 0, s, P);
        else hipLaunchKernelGGL((tile_kernel<BM, BN, WM, WN, MT, OT, false, false, C>), grid, block, 0, s, P);
    };
    if (__is_same(MT, f16_t) && P.passes == 2) go(Tag<__is_same(MT, f16_t)>{});
    else go(Tag<0>{});
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
