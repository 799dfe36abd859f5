// Large fp32 products on bf16 matrix instructions: D(m,n) = sum_k A(m,k) B(n,k) with A in fp32 (k contiguous) and B as three
// bf16 planes (dense.hip).  A's values are cut into their three planes x = h + m + l in registers, and the six products
// l h, h l, m m, m h, h m, h h of every pair go into one fp32 sum: 24 bits of each factor, at 6 / 16 of the cost of fp32
// matrix instructions.
//
// Against running the tile kernel six times over planes of both (dense_tile.hip): A is read once as 4 bytes instead of six
// times as 2, and no pass in front has to write 6 bytes for each of its values; a fragment of B serves two or three products
// while it is in registers, so LDS gives 28 KB per 32 k and wave instead of 72.  32768 x 1536 x 512: XX us instead of 326.
//
// 256 x 256 tiles, eight waves of 128 x 64, steps of 32 k in two buffers (A 32 KB, B 3 x 16 KB), one barrier per step.  A wave
// holds B's twelve fragments of the step and walks over its eight blocks of A: 24 MFMAs for each, and between them the
// splitting of the next block, one third of a pair at a time, and the loads of the next step.
#include "dense_common.h"
#include "dense_lds.h"
#include "dense_products.h"

using namespace dense;

namespace {

constexpr int kEdge = 256, kK = 32, W = 8, FM = 8, FN = 4, kA = kEdge * kK * 4, kB = kEdge * kK * 2;

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef unsigned w4 __attribute__((ext_vector_type(4)));

// Eight values of a row on their way into planes
struct Splitting {
    float x[8];
    w4 plane[3];
    // Third `part` (plane h, m or l) of values 2 p and 2 p + 1: the plane is the rounded rest, the new rest what that leaves
    // (exactly).  What would round past bf16's largest value is held at it; the planes below have the rest.
    __device__ __forceinline__ void cut(int p, int part) {
        float a = x[2 * p], b = x[2 * p + 1];
        if (part == 0) {
            a = __builtin_amdgcn_fmed3f(a, -3.3895314e38f, 3.3895314e38f);
            b = __builtin_amdgcn_fmed3f(b, -3.3895314e38f, 3.3895314e38f);
        }
        const unsigned v = __builtin_bit_cast(unsigned, __builtin_convertvector((f2{a, b}), b2));
        plane[part][p] = v;
        if (part < 2) {
            x[2 * p] -= __uint_as_float(v << 16);
            x[2 * p + 1] -= __uint_as_float(v & 0xffff0000u);
        }
    }
    // After the last part: an infinity becomes (+-1, 0, +-infinity), as in dense.hip.  So far it is (largest, infinity, NaN),
    // and its last rest, like a NaN's and no other's, is NaN.
    __device__ __forceinline__ void infinities() {
        bool some = false;
#pragma unroll
        for (int p = 0; p < 4; ++p) some |= __builtin_isunordered(x[2 * p], x[2 * p + 1]);
        if (__builtin_expect(__ballot(some) != 0, 0)) {
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int at = 0; at < 32; at += 16) {
                    const unsigned m = plane[1][p] >> at & 0xffff, sign = m & 0x8000, mask = 0xffffu << at;
                    if ((m & 0x7fff) != 0x7f80) continue;
                    plane[0][p] = (plane[0][p] & ~mask) | (sign | 0x3f80) << at;
                    plane[1][p] &= ~mask;
                    plane[2][p] = (plane[2][p] & ~mask) | (sign | 0x7f80) << at;
                }
        }
    }
};

template <bool TB>
__global__ __launch_bounds__(W * 64, 2) void split_kernel(Product P) {
    __shared__ __attribute__((aligned(1024))) char lds[2 * kA + 6 * kB];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned items = (unsigned)(((P.M + kEdge - 1) / kEdge) * ((P.N + kEdge - 1) / kEdge)) * P.splits;
    const unsigned xcd = blockIdx.x & 7, q8 = items >> 3, r8 = items & 7;
    const unsigned stride = (gridDim.x + 7 - xcd) >> 3, end = (xcd + 1) * q8 + (xcd + 1 < r8 ? xcd + 1 : r8);
    unsigned item = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);

    // A's values go into LDS as pairs of 16-bit elements: the same 128-byte rows as 64 k of those
    Loader<kEdge, W, false, 64> la;
    Loader<kEdge, W, TB, kK> lb;
    la.init(wave, lane, P.lda * 2);
    lb.init(wave, lane, P.ldb);
    Reader<kEdge, TB, kK> rb;
    const int wm = wave % 2 * 128, wn = wave / 2 * 64;
    rb.init(wn, lane);
    // block f of the wave's rows: values 8 (lane / 16) .. + 8 of row lane & 15, two 16-byte pieces
    const unsigned ra = (wm + (lane & 15)) * 128 + (((lane >> 4) * 2) ^ piece_of<64>(lane & 15)) * 16;

    const int per = (int)((P.K + kK - 1) / kK), k_tail = (int)(P.K - (long)(per - 1) * kK);
    const int step_b = (int)(TB ? P.ldb : 1) * kK * 2;
    const unsigned inc_a = (unsigned)P.lda * 4 * la.kStep, inc_b = (unsigned)P.ldb * 2 * lb.kStep;
    const long plane = P.plane_b * 2;
    unsigned load_item = item;
    int load_left = 0, kstep = 0, kk = 0;
    unsigned full_a = 0, full_b = 0, tail_a = 0, tail_b = 0, bytes_b = 0;
    const char *at_a = nullptr, *at_b = nullptr, *plane_at = nullptr;
    u4 buf_a, buf_b;
    const unsigned base = (unsigned)(uintptr_t)(lds_ptr)lds;
    unsigned to = 0;                                   // which buffers the loads go to
    auto next = [&]() {
        if (load_left == 0 && load_item < end) {
            const Product &R = arguments();
            const Place p = place<kEdge, kEdge, kK>(R, load_item);
            load_item += stride;
            load_left = p.steps;
            kstep = p.first;
            const int rows_a = R.M - p.m0 < kEdge ? (int)(R.M - p.m0) : kEdge, rows_b = R.N - p.n0 < kEdge ? (int)(R.N - p.n0) : kEdge;
            full_a = la.bytes(R.lda * 2, rows_a, 2 * kK);
            tail_a = la.bytes(R.lda * 2, rows_a, 2 * k_tail);
            full_b = lb.bytes(R.ldb, rows_b, kK);
            tail_b = lb.bytes(R.ldb, rows_b, k_tail);
            at_a = (const char *)R.a + (p.m0 * R.lda + (long)kstep * kK) * 4;
            at_b = (const char *)R.b + (TB ? p.n0 : p.n0 * R.ldb) * 2 + (long)kstep * step_b;
        }
        const bool some = load_left != 0, last = kstep == per - 1;     // past the last item: zeros, from nowhere
        kk = last ? k_tail : kK;
        buf_a = buffer(at_a, some ? last ? tail_a : full_a : 0);
        bytes_b = some ? last ? tail_b : full_b : 0;
        plane_at = at_b;
        if (some) {
            --load_left;
            ++kstep;
            at_a += 4 * kK;
            at_b += step_b;
        }
    };
    constexpr int LA = la.kLoads, LB = lb.kLoads, kLoads = LA + 3 * LB;
    auto load = [&](int q) {                           // load q of the step
        if (q < LA) {
            la.load(buf_a, inc_a, 2 * kk, base + to * kA, wave, q);
        } else {
            const int p = (q - LA) / LB, w = (q - LA) % LB;
            if (w == 0) {
                buf_b = buffer(plane_at, bytes_b);
                plane_at += plane;
            }
            lb.load(buf_b, inc_b, kk, base + 2 * kA + to * 3 * kB + p * kB, wave, w);
        }
        if (q == kLoads - 1) to ^= 1;
    };

    next();
#pragma unroll
    for (int q = 0; q < kLoads; ++q) load(q);
    unsigned cur = 0;
    f4 acc[FN][FM];
    for (; item < end; item += stride) {
        const int steps = place<kEdge, kEdge, kK>(arguments(), item).steps;
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[j][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int step = 0; step < steps; ++step) {
            // this step has arrived, and every wave has left the other buffers
            __builtin_amdgcn_s_waitcnt(wait_code(0));
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            next();
            const unsigned a0 = base + cur * kA + ra, b0 = base + 2 * kA + cur * 3 * kB;
            cur ^= 1;
            auto fetch = [&](Splitting &s, int f) __attribute__((always_inline)) {
                const f4 lo = *(lds_f4)(uintptr_t)(a0 + f * 2048), hi = *(lds_f4)(uintptr_t)((a0 ^ 16) + f * 2048);
#pragma unroll
                for (int c = 0; c < 4; ++c) s.x[c] = lo[c], s.x[4 + c] = hi[c];
            };
            Splitting now, then;
            fetch(now, 0);
            s8 fb[3][FN];
#pragma unroll
            for (int p = 0; p < 3; ++p)
#pragma unroll
                for (int j = 0; j < FN; ++j) fb[p][j] = rb.read(b0 + p * kB, j, 0);
            fetch(then, 1);
#pragma unroll
            for (int p = 0; p < 12; ++p) now.cut(p % 4, p / 4);
            now.infinities();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
                Splitting after;
#pragma unroll
                for (int x = 0; x < 24; ++x) {
                    constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
                    const int j = x % 4, t = x / 4;
                    acc[j][i] = mfma<bf16_t>(fb[pb[t]][j], __builtin_bit_cast(s8, now.plane[pa[t]]), acc[j][i]);
                    const int op = i * 24 + x;
                    if (x == 0 && i + 2 < FM) fetch(after, i + 2);
                    if (x % 2 == 1 && i + 1 < FM) then.cut(x / 2 % 4, x / 8);
                    if (op % 4 == 2 && op / 4 < kLoads) load(op / 4);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (i + 1 < FM) then.infinities();
                now = then;
                then = after;
            }
        }
        // every wave has left A's buffer of the last step: the sums may go through it
        __builtin_amdgcn_s_waitcnt(0xc07f);            // (lgkmcnt(0): the next step's loads stay in flight)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        leave_tile<kEdge, kEdge, kK, W, float>(acc, item, wm, wn, wave, lane, base + (cur ^ 1) * kA);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                // the zeros of the step past the end have arrived too
}

}  // namespace

int dense::launch_split(bool tb, const Product &P, hipStream_t s) {
    const long items = ((P.M + kEdge - 1) / kEdge) * ((P.N + kEdge - 1) / kEdge) * P.splits;
    if (items > 0x3fffffffL) return SA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(items < 256 ? items : 256));
    if (tb) hipLaunchKernelGGL(split_kernel<true>, grid, dim3(W * 64), 0, s, P);
    else hipLaunchKernelGGL(split_kernel<false>, grid, dim3(W * 64), 0, s, P);
    SA_CHECK_LAUNCH();
    return SA_OK;
}
