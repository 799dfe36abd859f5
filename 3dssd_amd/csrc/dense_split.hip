// Large fp32 layers on bf16 matrix instructions: D(m,n) = sum_k A(m,k) B(k,n) with A in fp32 (k contiguous) and B as three
// bf16 planes (dense.hip).  A's values become three planes x = h + m + l on their way, and the six products l h, m m, m h,
// h l, h m, h h of every pair go into one fp32 sum: 24 bits of each factor (of one below 2^-110 those from
// 2^-134 on), at 6 / 16 of the cost of fp32 matrix instructions.
//
// Against the tile kernel run six times over planes of both (dense_tile.hip): A is read once, as 4 bytes instead of six times
// 2; no pass in front has to write 6 bytes for each of its values; and a fragment serves two or three products while it is in
// registers, so LDS gives 36 KB per 32 k and wave instead of 72.  32768 x 1536 x 512: 223 us instead of 326 (fp32 matrix
// instructions of a library: 362), 1.4 PFLOP/s of bf16 products, which is what large bf16 products reach on this chip.  With
// little k to a tile, or few rows, the planes cost less than this kernel's single shape of tile: dense.hip compares.
//
// 256 x 256 tiles, eight waves of 128 x 64, steps of 32 k.  A wave holds B's twelve fragments of the step and walks over its
// eight blocks of A (0 to 7 below), 24 MFMAs for each.  Between them, one operation after a MFMA:
//   block 0     reads the thread's 16 values of the next step's A (two pieces of eight k) into registers;
//   block 1     sends off the loads of the next step's B -- into the same 48 KB of LDS, since every wave has its fragments;
//   blocks 4, 5 cut the values into planes, and write them into A's other 48 KB;
//   block 7     reads the first fragments of the next step, each plane into the registers of one that is done with.
// So each value is cut once per workgroup: with every wave cutting what it reads, four times as often, the same product took
// 248 us.  One barrier after block 0 (B's LDS may be written), one after block 6 (the next step is complete).
// Bound by the matrix instructions at the clock that their power leaves (2.0 GHz, 66 % of the cycles busy).
#include "dense_common.h"
#include "dense_lds.h"
#include "dense_products.h"

using namespace dense;

namespace {

constexpr int kEdge = 256, kK = 32, W = 8, FM = 8, FN = 4, kPlane = kEdge * kK * 2;

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef unsigned w4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) w4 *lds_w4;

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
    // After the last part: an infinity becomes (+-1, 0, +-infinity), and a value of up to 2^-134 (+-2^-133, -+2^-133, 0), as in
    // dense.hip.  So far the former is (largest, infinity, NaN), and its last rest is NaN, like a NaN's; the latter is three
    // zeros, and its last rest, itself, is below the normal range, like those of values below 2^-109.
    __device__ __forceinline__ void far_ends() {
        bool some = false;
#pragma unroll
        for (int p = 0; p < 8; ++p) some |= __builtin_amdgcn_classf(x[p], 0x93);           // NaN, subnormal
        if (__builtin_expect(__ballot(some) != 0, 0)) {
#pragma unroll
            for (int p = 0; p < 4; ++p)
#pragma unroll
                for (int at = 0; at < 32; at += 16) {
                    const unsigned m = plane[1][p] >> at & 0xffff, mask = 0xffffu << at;
                    const float rest = x[2 * p + at / 16];
                    if ((m & 0x7fff) == 0x7f80) {
                        const unsigned sign = m & 0x8000;
                        plane[0][p] = (plane[0][p] & ~mask) | (sign | 0x3f80) << at;
                        plane[1][p] &= ~mask;
                        plane[2][p] = (plane[2][p] & ~mask) | (sign | 0x7f80) << at;
                    } else if ((plane[0][p] >> at & 0x7fff) == 0 && rest != 0.0f) {
                        const unsigned sign = __float_as_uint(rest) >> 16 & 0x8000;
                        plane[0][p] = (plane[0][p] & ~mask) | (sign | 1) << at;
                        plane[1][p] = (plane[1][p] & ~mask) | ((sign ^ 0x8000) | 1) << at;
                    }
                }
        }
    }
};

template <bool TA>
__global__ __launch_bounds__(W * 64, 2) void split_kernel(Product P) {
    __shared__ __attribute__((aligned(1024))) char lds[9 * kPlane];    // A's planes of two steps, B's of one
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // items: as in the tile kernel
    const unsigned items = (unsigned)(((P.M + kEdge - 1) / kEdge) * ((P.N + kEdge - 1) / kEdge)) * P.splits;
    const unsigned xcd = blockIdx.x & 7, q8 = items >> 3, r8 = items & 7;
    const unsigned stride = (gridDim.x + 7 - xcd) >> 3, end = (xcd + 1) * q8 + (xcd + 1 < r8 ? xcd + 1 : r8);
    unsigned item = xcd * q8 + (xcd < r8 ? xcd : r8) + (blockIdx.x >> 3);

    Loader<kEdge, W, true, kK> lb;
    lb.init(wave, lane, P.ldb);
    Reader<kEdge, TA, kK> ra;
    Reader<kEdge, true, kK> rb;
    const int wm = wave % 2 * 128, wn = wave / 2 * 64;
    ra.init(wm, lane);
    rb.init(wn, lane);
    // A's values on their way: pieces of eight along k (m with TA), number g 512 + thread; 4 (32) neighbours have one row (k)
    const int outer = threadIdx.x / (TA ? 32 : 4), piece = threadIdx.x % (TA ? 32 : 4), key = piece * 8;
    const unsigned off = (unsigned)(outer * P.lda + key) * 4;
    const unsigned put = TA ? outer * 512 + (piece ^ 2 * slot_of(outer)) * 16 : outer * 64 + (piece ^ piece_of<kK>(outer)) * 16;

    const int per = (int)((P.K + kK - 1) / kK), k_tail = (int)(P.K - (long)(per - 1) * kK);
    const int step_a = (int)(TA ? P.lda : 1) * kK * 4, step_b = (int)P.ldb * kK * 2;
    const unsigned inc_a = (unsigned)P.lda * 4 * (TA ? 16 : 128), inc_b = (unsigned)P.ldb * 2 * lb.kStep;
    const long plane = P.plane_b * 2;
    unsigned load_item = item;
    int load_left = 0, kstep = 0, kk = 0;
    unsigned full_a = 0, full_b = 0, tail_a = 0, tail_b = 0, bytes_a = 0, bytes_b = 0;
    const char *next_a = nullptr, *next_b = nullptr, *at_a = nullptr, *at_b = nullptr;
    u4 buf_b;
    const unsigned base = (unsigned)(uintptr_t)(lds_ptr)lds, to_b = base + 6 * kPlane;
    auto next = [&]() {                                // the step whose loads go out
        if (load_left == 0 && load_item < end) {
            const Product &R = arguments();
            const Place p = place<kEdge, kEdge, kK>(R, load_item);
            load_item += stride;
            load_left = p.steps;
            kstep = p.first;
            const int rows_a = R.M - p.m0 < kEdge ? (int)(R.M - p.m0) : kEdge, rows_b = R.N - p.n0 < kEdge ? (int)(R.N - p.n0) : kEdge;
            auto bytes = [&](int k) { return (unsigned)(((TA ? k - 1 : rows_a - 1) * R.lda + (TA ? rows_a : k) + 3) & ~3L) * 4; };
            full_a = bytes(kK);
            tail_a = bytes(k_tail);
            full_b = lb.bytes(R.ldb, rows_b, kK);
            tail_b = lb.bytes(R.ldb, rows_b, k_tail);
            next_a = (const char *)R.a + (TA ? p.m0 : p.m0 * R.lda) * 4 + (long)kstep * step_a;
            next_b = (const char *)R.b + p.n0 * 2 + (long)kstep * step_b;
        }
        const bool some = load_left != 0, last = kstep == per - 1;     // past the last item: zeros, from nowhere
        kk = last ? k_tail : kK;
        bytes_a = some ? last ? tail_a : full_a : 0;
        bytes_b = some ? last ? tail_b : full_b : 0;
        at_a = next_a;
        at_b = next_b;
        if (some) {
            --load_left;
            ++kstep;
            next_a += step_a;
            next_b += step_b;
        }
    };
    Splitting s[2];
    auto load_a = [&](int g) __attribute__((always_inline)) {          // piece g of the thread
        const int rest = (int)bytes_a - (int)(g * inc_a);
        const auto r = __builtin_amdgcn_make_buffer_rsrc((void *)(at_a + g * (long)inc_a), 0, rest > 0 ? rest : 0, 0x00020000);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const u4 v = __builtin_amdgcn_raw_buffer_load_b128(r, TA || key + 4 * h < kk ? off + 16 * h : kOutside, 0, 0);
#pragma unroll
            for (int c = 0; c < 4; ++c) s[g].x[4 * h + c] = __uint_as_float(v[c]);
        }
    };
    auto keep_a = [&](int g, unsigned to) __attribute__((always_inline)) {
        s[g].far_ends();
#pragma unroll
        for (int p = 0; p < 3; ++p) *(lds_w4)(uintptr_t)(to + p * kPlane + g * (kPlane / 2) + put) = s[g].plane[p];
    };
    constexpr int LB = lb.kLoads;
    auto load_b = [&](int q) __attribute__((always_inline)) {
        if (q % LB == 0) {
            buf_b = buffer(at_b, bytes_b);
            at_b += plane;
        }
        lb.load(buf_b, inc_b, kk, to_b + q / LB * kPlane, wave, q % LB);
    };

    next();
#pragma unroll
    for (int q = 0; q < 3 * LB; ++q) load_b(q);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        load_a(g);
#pragma unroll
        for (int p = 0; p < 12; ++p) s[g].cut(p % 4, p / 4);
        keep_a(g, base);
    }
    __builtin_amdgcn_s_waitcnt(wait_code(0));
    __builtin_amdgcn_s_barrier();
    unsigned cur = 0;                                  // A's planes of the step
    f4 acc[FN][FM];
    s8 f0[2], f1, f2, fb[3][FN];                       // planes of A's block, of the next one too, and of all of B's
    for (; item < end; item += stride) {
        const int steps = place<kEdge, kEdge, kK>(arguments(), item).steps;
        // (what the last step read ahead is not kept through the end of a tile)
        f2 = ra.read(base + (cur * 3 + 2) * kPlane, 0, 0);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[0][j] = rb.read(to_b, j, 0);
        f1 = ra.read(base + (cur * 3 + 1) * kPlane, 0, 0);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[1][j] = rb.read(to_b + kPlane, j, 0);
        f0[0] = ra.read(base + cur * 3 * kPlane, 0, 0);
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int i = 0; i < FM; ++i) acc[j][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        for (int step = 0; step < steps; ++step) {
            next();
            const unsigned a0 = base + cur * 3 * kPlane;
            cur ^= 1;
            const unsigned a1 = base + cur * 3 * kPlane;
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < FM; ++i) {
#pragma unroll
                for (int x = 0; x < 24; ++x) {
                    // The six products, in an order that is done early with A's third and second plane, and in the last block
                    // with B's first and second: their registers take what comes next.
                    constexpr int pa[2][6] = {{2, 1, 1, 0, 0, 0}, {2, 1, 0, 1, 0, 0}}, pb[2][6] = {{0, 1, 0, 2, 1, 0}, {0, 0, 0, 1, 1, 2}};
                    const int j = x % 4, t = x / 4, op = (i - 4) * 24 + x, last = i == FM - 1;
                    const int p = pa[last][t];
                    acc[j][i] = mfma<bf16_t>(fb[pb[last][t]][j], p == 0 ? f0[i & 1] : p == 1 ? f1 : f2, acc[j][i]);
                    const unsigned an = i + 1 < FM ? a0 : a1;
                    if (x == 4) f2 = ra.read(an + 2 * kPlane, (i + 1) % FM, 0);
                    if (x == 16) f1 = ra.read(an + kPlane, (i + 1) % FM, 0);
                    if (x == 18) f0[(i + 1) & 1] = ra.read(an, (i + 1) % FM, 0);
                    if (i == 0 && x < 4) fb[2][j] = rb.read(to_b + 2 * kPlane, j, 0);
                    if (last && x >= 12 && x < 16) fb[0][j] = rb.read(to_b, j, 0);
                    if (last && x >= 20) fb[1][j] = rb.read(to_b + kPlane, j, 0);
                    if (i == 0 && (x == 5 || x == 7)) load_a(x / 7);
                    if (i == 1 && x % 4 == 3) load_b(x / 4);
                    if (op >= 0 && op < 48 && op % 2 == 1) s[op / 24].cut(op % 24 / 2 % 4, op % 24 / 8);
                    if (op == 24 || op == 48) keep_a(op / 24 - 1, a1);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (i == 0) {                          // everyone has B's fragments: its next step may come
                    __builtin_amdgcn_s_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (i == FM - 2) {                     // the next step is there, and everyone has read all of A's this one
                    __builtin_amdgcn_s_waitcnt(wait_code(0));
                    __builtin_amdgcn_s_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        // through the planes of the last step's A, which all waves have read, and none writes before all are past block 0
        leave_tile<kEdge, kEdge, kK, W, float>(acc, item, wm, wn, wave, lane, base + (cur ^ 1) * 3 * kPlane);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                // the zeros of the step past the end have arrived too
}

}  // namespace

int dense::launch_split(bool ta, const Product &P, hipStream_t s) {
    const long items = ((P.M + kEdge - 1) / kEdge) * ((P.N + kEdge - 1) / kEdge) * P.splits;
    if (items > 0x3fffffffL) return SA_ERR_UNSUPPORTED;
    const dim3 grid((unsigned)(items < 256 ? items : 256));
    if (ta) hipLaunchKernelGGL(split_kernel<true>, grid, dim3(W * 64), 0, s, P);
    else hipLaunchKernelGGL(split_kernel<false>, grid, dim3(W * 64), 0, s, P);
    SA_CHECK_LAUNCH();
    return SA_OK;
}
