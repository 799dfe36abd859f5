// Device code that the large products' kernels share: the way of a tile into LDS and out of it, and the way of the sums from
// the registers to the result.
#pragma once
#include "dense_common.h"

namespace dense {

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
// vmcnt itself, in front of the barrier that publishes the buffer.
__device__ __forceinline__ void lds_load(u4 r, unsigned off, unsigned to) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r), "s"(to) : "memory", "m0");
}

__device__ __forceinline__ u4 buffer(const char *p, unsigned bytes) {
    return u4{(unsigned)(uintptr_t)p, (unsigned)((uintptr_t)p >> 32) & 0xffff, bytes, 0x00020000u};
}
// s_waitcnt's code for vmcnt(n) lgkmcnt(0)
constexpr int wait_code(int n) { return (n & 15) | (n >> 4) << 14 | 0x70; }

// Permutation of the 32-byte slots of row k: half a wave of ds_read_b64_tr_b16 reads rows 8 g .. + 4 of two neighbouring g,
// which have to lie in eight different slots (mod 8: 256 bytes, all banks once)
__device__ __forceinline__ int slot_of(int k) { return (k & 3) | ((k >> 3) & 1) << 2; }

// Permutation of the 16-byte pieces of a row of 64 or 32 k
template <int BK>
__device__ __forceinline__ int piece_of(int row) { return BK == 64 ? row & 7 : (row >> 1) & 3; }

// One operand's way into LDS: a tile of R rows x BK k by W waves, kLoads loads of 1024 bytes each.  Load q of wave w fills
// kilobyte q W + w: kStep rows (or k) lie between the loads of a wave, which leaves its permutation alone, so that one offset
// per lane serves them all and the buffer moves instead.
template <int R, int W, bool ROWS, int BK>
struct Loader {
    static constexpr int kLoads = R * BK * 2 / 1024 / W, kStep = W * (ROWS ? 512 / R : 512 / BK);
    static_assert(kStep % 16 == 0, "the permutations use four bits");
    unsigned off;
    int key;                                                   // k of the lane's piece (k contiguous)
    __device__ __forceinline__ void init(int wave, int lane, long ld) {
        int outer, piece;
        if (ROWS) {
            outer = (wave * 1024 + lane * 16) / (R * 2);
            piece = (lane & (R / 8 - 1)) ^ (2 * slot_of(outer));
        } else {
            outer = (wave * 64 + lane) / (BK / 8);
            piece = (lane & (BK / 8 - 1)) ^ piece_of<BK>(outer);
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
template <int R, bool ROWS, int BK>
struct Reader {
    unsigned at;
    __device__ __forceinline__ void init(int first, int lane) {
        const int i = lane & 15, g = lane >> 4, kk = 8 * g + (i >> 2);
        at = ROWS ? kk * R * 2 + (((first / 16) ^ slot_of(kk)) * 32) + (i & 3) * 8 : (first + i) * BK * 2 + ((g ^ piece_of<BK>(i)) * 16);
    }
    __device__ __forceinline__ s8 read(unsigned lds, int f, int s) const {
        if (ROWS) {                                            // (k + 4 has the same permutation)
            const unsigned p = ((lds + at) ^ (f * 32)) + s * 64 * R;
            const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)p);
            const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(uintptr_t)(p + 4 * R * 2));
            return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        }
        return *(lds_s8)(uintptr_t)(((lds + at) ^ (s * 64)) + f * 32 * BK);
    }
};

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

struct Place {
    long m0, n0;
    int first, steps, piece;
};
// Item `it` of a product: tiles of BM x BN in groups of eight tile rows, so that neighbours share operands in one L2, all of
// them for each piece of k; first and steps count steps of BK k over all passes.
template <int BM, int BN, int BK>
__device__ __forceinline__ Place place(const Product &P, unsigned it) {
    const unsigned tm = (unsigned)((P.M + BM - 1) / BM), tn = (unsigned)((P.N + BN - 1) / BN), tiles = tm * tn;
    const unsigned piece = it / tiles, pos = it - piece * tiles;
    const unsigned group = pos / (8 * tn), in = pos - group * 8 * tn, rows = tm - group * 8 < 8 ? tm - group * 8 : 8;
    const int all = (int)((P.K + BK - 1) / BK) * P.passes, first = (int)(piece * P.kchunk), left = all - first;
    return Place{(long)(group * 8 + in % rows) * BM, (long)(in / rows) * BN, first, left < P.kchunk ? left : (int)P.kchunk, (int)piece};
}

// The sums of a tile's wave (its FM x 4 blocks of 16 x 16 from wm, wn on) to the result.  They go 16 rows of its 64 columns at
// a time through 4 KB of LDS (16-byte pieces of a row permuted by ^ row), so that eight lanes write 128 neighbouring bytes
// (16-bit) of a row.  region: a buffer whose kilobytes wave, W + wave, .. are free for the wave.
template <int BM, int BN, int BK, int W, class OT, int FM, int FN>
__device__ __forceinline__ void leave_tile(f4 (&acc)[FN][FM], unsigned item, int wm, int wn, int wave, int lane, unsigned region) {
    static_assert(FN == 4, "64 columns");
    const Product &R = arguments();
    int l = lane;                                  // (computed from anew: kept, its offsets would take main loop registers)
    asm volatile("" : "+v"(l));
    const Place p = place<BM, BN, BK>(R, item);
    const long n = p.n0 + wn + (l & 7) * 8, mw = p.m0 + wm + (l >> 3), N = R.N, M = R.M;
    const unsigned mine = region + wave * 1024;      // kilobytes wave, W + wave, ..: four rows each
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

}  // namespace dense
