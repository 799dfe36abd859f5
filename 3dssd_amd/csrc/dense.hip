// The dense layer on plain weights: y = act(x W + b) + residual in fp32, bf16 or fp16, and its gradient
// (dense_common.h has the formulas).  This file: the pass in front of the products that need one, the join of split sums,
// the choice of kernel, and the C ABI.  The products are in dense_tile.hip and dense_split.hip (large) and dense_small.hip.
#include "dense_common.h"
#include "dense_products.h"

#include <initializer_list>

using namespace dense;

namespace {

template <class T> using Eight = Pack<T, 8>;

// Columns c .. c + 8 of a row; zeros behind the last column.
template <class T, bool WHOLE>
__device__ __forceinline__ Eight<T> fetch(const T *row, int c, int cols) {
    if constexpr (WHOLE) return load_pack<T, 8>(row + c);
    Eight<T> v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v.x[i] = c + i < cols ? row[c + i] : T{};
    return v;
}

// The pieces of a split k range, summed in a fixed order, then the epilogue.  G groups of threads share the pieces of the same
// sums where there are many pieces and few sums (128 x 256 sums of 228 pieces: 7.5 us with 8 groups, 14 with one).
template <class T, int G>
__global__ __launch_bounds__(256) void join_kernel(Product P) {
    constexpr int kOwn = 256 / G;
    __shared__ f4 part[G][kOwn];
    const int own = threadIdx.x % kOwn, group = threadIdx.x / kOwn;
    const long Np = round_up(P.N, 4), per = Np / 4, total = P.M * per, plane = P.M * Np;
    for (long i0 = (long)blockIdx.x * kOwn; i0 < total; i0 += (long)gridDim.x * kOwn) {
        const long i = i0 + own, m = i / per, n = (i - m * per) * 4;
        const float *p = P.part + (long)group * plane + m * Np + n;
        f4 s{0.0f, 0.0f, 0.0f, 0.0f};
        if (i < total) {
            if (group < P.splits) s = *(const f4 *)p;
#pragma unroll 8
            for (int z = group + G; z < P.splits; z += G) s += *(const f4 *)(p + (z - group) * plane);
        }
        if constexpr (G > 1) {
            __syncthreads();
            part[group][own] = s;
            __syncthreads();
#pragma unroll
            for (int g = 1; g < G; ++g) s += part[g][own];
        }
        if (group != 0 || i >= total) continue;
        float b[4];
        load_bias<T, 4>(P.e, n, P.N, b);
        const float v[4] = {s[0], s[1], s[2], s[3]};
        Pack<T, 4> r{};
        if (P.e.res) r = load_residual<T, 4>(P.e, m, n, P.N);
        finish<T, 4>(P.e, m, n, P.N, v, b, r);
    }
}

// ---- operands in front of a product ---------------------------------------------------------------------------------
// One pass over a stored matrix [rows][cols], any stride and alignment, that writes what the products read:
//   dZ = G act'(Z), where there is a Z (ReLU selects: what a closed unit receives, infinities among it, does not come
//   through), and the column sums of dZ, taken before any rounding;
//   a copy in the layer's type with 16-byte aligned rows, zeros behind the last column up to a multiple of 8 -- for the
//   tile kernel, whose loads are 16 bytes wide.  A 16-bit layer's dZ goes in two planes (dense_common.h), or, where the caller
//   asks for it, rounded to the layer's type: it is an operand of the same MFMAs as X and W;
//   or, of a fp32 matrix, three bf16 planes x = h + m + l, each the rounded rest of the one before: 27 bits, so nothing of
//   x's 24 is lost, and the six products h h, h m, m h, m m, h l, l h of two such operands leave out terms below 2^-24 of
//   the product -- fp32's own rounding -- at 6 / 16 of the cost of fp32 MFMAs.  bf16 ends where fp32's normal range does, with
//   steps of 2^-133: a x below 2^-110 is held to 2^-134, not to 2^-24 of itself.
// A thread owns eight columns; a block's threads take 256 columns of eight rows at a time, or of wide matrices 2048 of one
// (4 KB runs of 16-bit elements).  The row lanes of a block meet in LDS, the strips in
// sum_strips_kernel, in a fixed order.  Bound by memory: each element is read and written once.
struct Job {
    const void *g, *z;    // z null: no activation
    long ldg, ldz;
    int act;
    long rows;
    int cols;
    void *dst;            // [rows][ldd], or null: sums only
    long ldd;             // copied_ld(cols)
    long plane;           // elements between planes (fp32: three, else two); 0: one copy in the layer's type
    float *sums;          // [strips][cols], or null
    long strip;           // rows of a block
    int wide;             // 2048 columns of a row at a time
};
struct Jobs {
    Job j[3];
    long first[4];        // blocks of the jobs
};

// x finite and too large for bf16 rounds to its largest value (the planes below hold the rest).  An infinity is
// (+-1, 0, +-infinity): the last plane only meets the other factor's first, which has its sign and is 0 only if the factor
// is; in the first plane it would meet rests that are 0 or of the other sign, and the sum would be NaN.  For that a x of up to
// 2^-134, which bf16 rounds to 0, has a step (2^-133) in its first plane that the second takes back.
__device__ __forceinline__ void three_planes(float x, unsigned short (&o)[3]) {
    float r = x;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        unsigned short h = from_f32<bf16_t>(r).u;
        if ((h & 0x7fff) == 0x7f80) h -= 1;
        o[i] = h;
        r -= __uint_as_float((unsigned)h << 16);
    }
    const unsigned short sign = x < 0.0f ? 0x8000 : 0;
    if (fabsf(x) == __builtin_inff()) {
        o[0] = sign | 0x3f80;
        o[1] = 0;
        o[2] = sign | 0x7f80;
    }
    if ((o[0] & 0x7fff) == 0 && x != 0.0f) {
        o[0] = sign | 1;
        o[1] = (sign ^ 0x8000) | 1;
    }
}

template <class T>
__global__ __launch_bounds__(256) void prepare_kernel(Jobs J) {
    __shared__ float part[8][256 + 4];
    const int which = blockIdx.x >= J.first[2] ? 2 : blockIdx.x >= J.first[1] ? 1 : 0;
    const Job S = J.j[which];
    const long blk = blockIdx.x - J.first[which];
    const int span = S.wide ? 2048 : 256, lanes = S.wide ? 1 : 8;      // columns and rows that a block takes at a time
    const int cb = (S.cols + span - 1) / span, bx = (int)(blk % cb);
    const long by = blk / cb;
    const int c0 = bx * span + (S.wide ? threadIdx.x : threadIdx.x & 31) * 8, rl = S.wide ? 0 : threadIdx.x >> 5;
    const long r0 = by * S.strip, r1 = r0 + S.strip < S.rows ? r0 + S.strip : S.rows;
    float sum[8] = {};
    constexpr int kRows = 4;                           // rows in flight per thread
    // whole: all of the thread's columns are there.  (A branch per load instead lets the compiler share its first elements with
    // the partial case and cut the 16-byte load to pieces.)
    auto walk = [&](auto act, auto whole) __attribute__((always_inline)) {
        constexpr int A = decltype(act)::value;
        constexpr bool kWhole = decltype(whole)::value;
        for (long r = r0 + rl; r < r1 && c0 < S.cols; r += lanes * kRows) {
            Eight<T> g[kRows], z[kRows];
#pragma unroll
            for (int u = 0; u < kRows; ++u)
                if (r + lanes * u < r1) {
                    g[u] = fetch<T, kWhole>((const T *)S.g + (r + lanes * u) * S.ldg, c0, S.cols);
                    if (A != kNone) z[u] = fetch<T, kWhole>((const T *)S.z + (r + lanes * u) * S.ldz, c0, S.cols);
                }
#pragma unroll
            for (int u = 0; u < kRows; ++u) {
                if (r + lanes * u >= r1) break;
                float d[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = to_f32<T>(g[u].x[i]);
                if (A != kNone) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) d[i] = times_slope<A>(d[i], to_f32<T>(z[u].x[i]));
                }
                if (S.dst) {
                    const long at = (r + lanes * u) * S.ldd + c0;
                    if (sizeof(T) == 4 && S.plane) {
                        Eight<bf16_t> o[3];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            unsigned short h[3];
                            three_planes(d[i], h);
#pragma unroll
                            for (int p = 0; p < 3; ++p) o[p].x[i].u = h[p];
                        }
#pragma unroll
                        for (int p = 0; p < 3; ++p) store_pack<bf16_t, 8>((bf16_t *)S.dst + p * S.plane + at, o[p]);
                    } else if (sizeof(T) == 2 && S.plane) {
                        if constexpr (sizeof(T) == 2) {
                            Eight<T> o[2];
#pragma unroll
                            for (int i = 0; i < 8; ++i) split_slope<T>(d[i], o[0].x[i], o[1].x[i]);
#pragma unroll
                            for (int p = 0; p < 2; ++p) store_pack<T, 8>((T *)S.dst + p * S.plane + at, o[p]);
                        }
                    } else {
                        Eight<T> o;
#pragma unroll
                        for (int i = 0; i < 8; ++i) o.x[i] = from_f32<T>(d[i]);
                        store_pack<T, 8>((T *)S.dst + at, o);
                    }
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += d[i];
            }
        }
    };
    with_activation(S.z ? S.act : kNone, [&](auto act) __attribute__((always_inline)) {
        if (c0 + 8 <= S.cols) walk(act, Tag<1>{});
        else walk(act, Tag<0>{});
    });
    if (!S.sums) return;
    if (S.wide) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (c0 + i < S.cols) S.sums[by * S.cols + c0 + i] = sum[i];
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[rl][(threadIdx.x & 31) * 8 + i] = sum[i];
    __syncthreads();
    const int c = bx * 256 + threadIdx.x;
    if (c < S.cols) {
        float s = part[0][threadIdx.x];
        for (int i = 1; i < 8; ++i) s += part[i][threadIdx.x];
        S.sums[by * S.cols + c] = s;
    }
}

template <class T>
__global__ __launch_bounds__(1024) void sum_strips_kernel(const float *sums, int strips, int cols, T *out) {
    __shared__ float part[16][64];
    const int own = threadIdx.x & 63, c = blockIdx.x * 64 + own, q = threadIdx.x >> 6;
    float s = 0.0f;
    if (c < cols) {
#pragma unroll 8
        for (int i = q; i < strips; i += 16) s += sums[(long)i * cols + c];
    }
    part[q][own] = s;
    for (int half = 8; half >= 1; half /= 2) {
        __syncthreads();
        if (q < half) part[q][own] += part[q + half][own];
    }
    if (q == 0 && c < cols) out[c] = from_f32<T>(part[0][own]);
}

// ---- host ----------------------------------------------------------------------------------------------------------
inline long esize(int type) { return type == kF32 ? 4 : 2; }
inline bool aligned(const void *p, long ld, int type) { return ((uintptr_t)p & 15) == 0 && (ld * esize(type)) % 16 == 0 && ld * esize(type) < 2 * kMaxTileLd; }
// Whole elements: the buffer loads of the small products would round such an address down
inline bool whole(int type, std::initializer_list<const void *> ps) {
    for (const void *p : ps)
        if ((uintptr_t)p & (esize(type) - 1)) return false;
    return true;
}
inline bool scratch_ok(const void *ws, unsigned long used, unsigned long bytes) {
    return used == 0 || (ws && ((uintptr_t)ws & 255) == 0 && used <= bytes);
}
inline bool sizes_ok(int type, long rows, int cin, int cout) {
    return type >= kF32 && type <= kF16 && rows >= 0 && cin >= 0 && cout >= 0 && cin < kMaxLd && cout < kMaxLd;
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

// A stored matrix: an operand of one or two products.
struct Matrix {
    const void *p;
    long ld, rows;
    int cols;
    bool vec;             // 16-byte aligned base and rows, less than 4 MB apart
    long plane = 0;
};

// The tile kernel's loads are 16 bytes of 16-bit elements
inline bool tile_operand(int type, const Matrix &m) { return type != kF32 && m.vec && m.cols % 8 == 0; }

// Does a layer of this size go to the tile kernel?  The small kernel's time against the tiles' (us): fp32 1024 x 512 x 512
// 14 / 26, 1024^3 42 / 36; bf16 1024 x 512 x 512 11 / 11, 1024 x 1024 x 512 12 / 14, 1024^3 22 / 15; where the operands have to
// be copied first 701^3 18 / 19, 1023^3 54 / 25; gradients 1024^3 fp32 64 / 69, bf16 35 / 37, 701^3 32 / 36.  Few rows are no
// work for a tile of 128, least of all where a fp32 W has to be split first (64 x 4096 x 4096 30 / 74).
inline bool wants_tiles(int type, long rows, int cin, int cout, bool copies, bool backward) {
    // (backward: two products, for which the small kernel needs one launch and no copies)
    const double least = backward ? (copies && type != kF32 ? 7e8 : 1.3e9) : type == kF32 ? 9e8 : copies ? 4e8 : 6e8;
    return rows > (type == kF32 ? 128 : 32) && cin > 32 && cout > 32 && (double)rows * cin * cout >= least && cin < kMaxTileLd &&
           cout < kMaxTileLd;
}
// Rows of a copy begin on a line of the caches, so that a step's 128 bytes of one are not on two: the tile kernel takes
// 30.4 us instead of 32.9 for 5003 x 771 x 1283.  (Behind the zeros up to a multiple of 8 nothing is written, and nothing is read that matters.)
inline long copied_ld(long cols) { return round_up(cols, 64); }

// Makes the copy (or planes) of m that the products read, as one of J's jobs
void add_job(Jobs &J, int &n, Job j) {
    J.j[n] = j;
    const int span = j.wide ? 2048 : 256;
    J.first[n + 1] = J.first[n] + (long)((j.cols + span - 1) / span) * ((j.rows + j.strip - 1) / j.strip);
    ++n;
}
// Whether a block takes 2048 columns at a time, and its rows: a thousand blocks or more where the matrix has them, and no more
// strips than 512.
void shape_job(Job &j) {
    j.wide = j.cols >= 2048 && (j.cols % 2048 == 0 || j.cols >= 8192);
    const int span = j.wide ? 2048 : 256, lanes = j.wide ? 1 : 8;
    long s = j.rows * ((j.cols + span - 1) / span) / 1024;
    if (!j.wide && s > 63) s = 63;
    if (s < j.rows / 512) s = j.rows / 512;
    j.strip = round_up(s + 1, lanes);
}
void copy_for_tiles(Jobs &J, int &n, Scratch &ws, int type, Matrix &m, bool planes = true) {
    Job j{};
    j.g = m.p; j.ldg = m.ld; j.rows = m.rows; j.cols = m.cols;
    j.ldd = copied_ld(m.cols);
    j.plane = type == kF32 && planes ? m.rows * j.ldd : 0;
    j.dst = ws.take((unsigned long)m.rows * j.ldd * (j.plane ? 6 : esize(type)));
    shape_job(j);
    m = Matrix{j.dst, j.ldd, m.rows, m.cols, true, j.plane};
    add_job(J, n, j);
}
int launch_jobs(int type, Jobs &J, int n, hipStream_t s) {
    if (n == 0 || J.first[n] == 0) return SA_OK;
    if (J.first[n] > 0x7fffffffL) return SA_ERR_UNSUPPORTED;
    const unsigned blocks = (unsigned)J.first[n];
    for (int i = n; i < 3; ++i) J.first[i] = J.first[i + 1] = 0x7fffffffL + 1;
    if (type == kF32) hipLaunchKernelGGL((prepare_kernel<float>), dim3(blocks), dim3(256), 0, s, J);
    else if (type == kBF16) hipLaunchKernelGGL((prepare_kernel<bf16_t>), dim3(blocks), dim3(256), 0, s, J);
    else hipLaunchKernelGGL((prepare_kernel<f16_t>), dim3(blocks), dim3(256), 0, s, J);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

// A product, its kernel and its k pieces.
struct Plan {
    Product P;
    bool ta, tb;
    int shape;            // of the tiles; kNoTile: a small product
};
enum Kind { kSmall, kTiles, kSplit };
// Chooses shape and pieces; returns the time to expect (ns; tiles only).
double plan(Plan &L, int type, Kind kind, bool ta, bool tb, long M, long N, long K, bool two = false) {
    Product &P = L.P;
    L.ta = ta; L.tb = tb;
    P.M = M; P.N = N; P.K = K;
    P.two = two;
    P.passes = kind != kTiles ? 1 : type == kF32 ? 6 : two ? 2 : 1;
    auto count = [&](long m, long n) { return ((M + m - 1) / m) * ((N + n - 1) / n); };
    const long unit = kind == kTiles ? 64 : 32, steps = (K + unit - 1) / unit * P.passes;
    long pieces = 1;
    double best = 0;
    if (kind != kSmall) {
        // The shape and the number of pieces with the least time (ns): rounds over the chip's slots, each of the piece's steps
        // and a tile's end -- a step takes longer the more of the chip works (alone / full: measured on bf16, kSplit256 on fp32,
        // products of 1024^3 to 8192^3) -- and the join of the pieces: a launch, and the partial sums out and in at 8 TB/s.
        static const struct { int shape, m, n, slots; double alone, full, end; } kShapes[] = {
            {kTile256, 256, 256, 256, 1050, 1430, 8500}, {kTile256x128, 256, 128, 256, 690, 840, 5500},
            {kTile128, 128, 128, 512, 400, 890, 5000}, {kSplit256, 256, 256, 256, 2700, 4150, 8500}};
        for (const auto &t : kShapes) {
            if ((t.shape == kSplit256) != (kind == kSplit)) continue;
            const long c = count(t.m, t.n);
            for (long s = 1; s == 1 || (s <= 256 && s * 4 <= steps); s += 1 + s / 16) {
                const long per = (steps + s - 1) / s, items = c * s, rounds = items / t.slots, rest = items % t.slots;
                double time = rounds * (per * t.full + t.end);
                if (rest) time += per * (t.alone + (t.full - t.alone) * rest / t.slots) + t.end;
                if (s > 1) time += 4000 + s * (double)M * N / 1000;
                if (best == 0 || time < best) {
                    best = time;
                    L.shape = t.shape;
                    pieces = s;
                }
                if (items >= 2 * t.slots) break;
            }
        }
    } else {
        // blocks of 32 x 32 up to one per CU, in pieces long enough to be worth the join's launch
        L.shape = kNoTile;
        const long least = M <= 32 ? 128 : 64;
        pieces = 256 / count(32, 32);
        if (pieces > steps / least) pieces = steps / least;
        if (pieces < 1) pieces = 1;
    }
    long per = (steps + pieces - 1) / pieces;
    if (per < 1) per = 1;
    P.splits = (int)((steps + per - 1) / per);
    if (P.splits < 1) P.splits = 1;
    P.kchunk = kind == kSmall ? per * 32 : per;
    return best;
}
// The operands, and room for the pieces' sums
void place(Plan &L, Scratch &ws, const Matrix &a, const Matrix &b) {
    Product &P = L.P;
    P.a = a.p; P.lda = a.ld; P.vec_a = a.vec; P.plane_a = a.plane;
    P.b = b.p; P.ldb = b.ld; P.vec_b = b.vec; P.plane_b = b.plane;
    P.part = P.splits > 1 ? (float *)ws.take((unsigned long)P.splits * P.M * round_up(P.N, 4) * 4) : nullptr;
}

template <int G>
int launch_join(int type, const Product &P, hipStream_t s) {
    const long n = (P.M * (round_up(P.N, 4) / 4) + 256 / G - 1) / (256 / G);
    const dim3 blocks((unsigned)(n < 8192 ? n : 8192));
    if (type == kF32) hipLaunchKernelGGL((join_kernel<float, G>), blocks, dim3(256), 0, s, P);
    else if (type == kBF16) hipLaunchKernelGGL((join_kernel<bf16_t, G>), blocks, dim3(256), 0, s, P);
    else hipLaunchKernelGGL((join_kernel<f16_t, G>), blocks, dim3(256), 0, s, P);
    SA_CHECK_LAUNCH();
    return SA_OK;
}
int launch_join(int type, const Product &P, hipStream_t s) {
    if (P.splits == 1) return SA_OK;
    return P.splits >= 32 && P.M * P.N <= 1L << 17 ? launch_join<8>(type, P, s) : launch_join<1>(type, P, s);
}
int launch_tile_plan(int type, const Plan &L, hipStream_t s) {
    const int rc = L.shape == kSplit256 ? launch_split(L.ta, L.P, s)
                                        : launch_tiles(L.shape, type == kF16 ? kF16 : kBF16, type, L.ta, L.tb, L.P, s);
    return rc ? rc : launch_join(type, L.P, s);
}
int launch_sums(int type, const float *sums, int strips, int cols, void *out, int out_f32, hipStream_t s) {
    const dim3 grid((cols + 63) / 64);
    if (out_f32 || type == kF32) hipLaunchKernelGGL((sum_strips_kernel<float>), grid, dim3(1024), 0, s, sums, strips, cols, (float *)out);
    else if (type == kBF16) hipLaunchKernelGGL((sum_strips_kernel<bf16_t>), grid, dim3(1024), 0, s, sums, strips, cols, (bf16_t *)out);
    else hipLaunchKernelGGL((sum_strips_kernel<f16_t>), grid, dim3(1024), 0, s, sums, strips, cols, (f16_t *)out);
    SA_CHECK_LAUNCH();
    return SA_OK;
}

// Takes x (A of a large fp32 product planned on tiles, which would take `time`) as it is, or copied once for its alignment,
// where that beats its planes: 10 bytes an element, at 4.5 TB/s.
inline bool split_operand(const Matrix &x) { return x.vec && x.cols % 4 == 0; }
bool prefer_split(Plan &L, double time, const Matrix &x, bool ta) {
    const double elements = (double)x.rows * x.cols;
    Plan split{};
    const double other = plan(split, kF32, kSplit, ta, true, L.P.M, L.P.N, L.P.K) + (split_operand(x) ? 0 : 8) * elements / 4500;
    if (!(split_operand(x) || copied_ld(x.cols) < kMaxTileLd / 2) || other >= time + 10 * elements / 4500) return false;
    L = split;
    return true;
}
void copy_for_split(Jobs &J, int &n, Scratch &ws, Matrix &x) {
    if (!split_operand(x)) copy_for_tiles(J, n, ws, kF32, x, false);
}

struct Forward {
    Jobs jobs;
    int njobs;
    Plan plan;
};
void plan_forward(Forward &f, Scratch &ws, int type, long rows, int cin, int cout, Matrix x, Matrix w) {
    f = Forward{};
    const bool tiles = wants_tiles(type, rows, cin, cout, !tile_operand(type, x) || !tile_operand(type, w), false);
    const double time = plan(f.plan, type, tiles ? kTiles : kSmall, false, true, rows, cout, cin);
    const bool split = tiles && type == kF32 && prefer_split(f.plan, time, x, false);
    if (split) copy_for_split(f.jobs, f.njobs, ws, x);
    if (tiles) {
        if (!split && !tile_operand(type, x)) copy_for_tiles(f.jobs, f.njobs, ws, type, x);
        if (!tile_operand(type, w)) copy_for_tiles(f.jobs, f.njobs, ws, type, w);
    }
    place(f.plan, ws, x, w);
}

struct Backward {
    Jobs jobs;
    int njobs;
    bool tiles;
    Plan dx, dw;
    float *sums;          // the bias gradient's partial sums: of the jobs' strips, or of dW's pieces
    int strips;
    bool bias_in_dw;
};
constexpr int kWantX = 1, kWantW = 2, kWantB = 4;
// Those of the wanted gradients that have elements (a plan counts their blocks)
inline int wanted(bool x, bool w, bool b, long rows, int cin, int cout) {
    return (x && rows && cin ? kWantX : 0) | (w && cin && cout ? kWantW : 0) | (b && cout ? kWantB : 0);
}
// Whether each small block forms the dZ it reads, or a pass in front does: every block forms it anew, but the pass costs a launch and
// a round trip to memory.  Formed / with the pass, us: ReLU (a select) fp32 2048 x 128 x 256 12.8 / 19.4, 128 x 4096 x 1024 63 / 59,
// 16384 x 32 x 2048 82 / 142; GELU fp32 2048 x 128 x 256 16.3 / 19.7, 2048 x 256 x 256 26.4 / 25.9, 2048 x 512 x 256 40 / 35; rounded
// bf16 512 x 128 x 256 10.1 / 12.0, 2048 x 128 x 256 23 / 17, 64 x 2048 x 2048 48 / 28.  In two planes the slopes of a wave's steps of k
// weigh more: bf16 GELU 512 x 128 x 256 10.5 / 12.9, 768 x 384 x 384 14.5 / 17.1, 640^3 30 / 26, 4 x 1024 x 4096 50 / 25,
// 4096 x 16 x 256 47 / 27.
bool slopes_formed(int type, long rows, int cin, int cout, int act, bool two) {
    const double products = (double)rows * cin * cout;
    if (!two) return products <= (act <= kRelu ? 1L << 30 : 1L << 26);
    if (products > 1L << 27 || products == 0) return products == 0;
    Plan x{}, w{};
    plan(x, type, kSmall, false, false, rows, cin, cout);
    plan(w, type, kSmall, true, true, cin, cout, rows);
    return x.P.kchunk <= 768 && w.P.kchunk <= 768;
}

void plan_backward(Backward &b, Scratch &ws, int type, long rows, int cin, int cout, Matrix x, Matrix w, Matrix g, Matrix z,
                   int act, bool two, int want) {
    b = Backward{};
    b.tiles = wants_tiles(type, rows, cin, cout, !tile_operand(type, x) || !tile_operand(type, w), true);
    const bool products = want & (kWantX | kWantW);
    const bool formed = !b.tiles && slopes_formed(type, rows, cin, cout, act, two);
    Job j{};
    j.g = g.p; j.ldg = g.ld; j.z = act == kNone ? nullptr : z.p; j.ldz = z.ld; j.act = act;
    j.rows = rows; j.cols = cout; j.ldd = copied_ld(cout);
    shape_job(j);
    Matrix d = g;
    const bool copy = products && (b.tiles ? act != kNone || !tile_operand(type, g) : act != kNone && !formed);
    if (copy) {
        const int planes = type != kF32 ? 1 + two : b.tiles ? 3 : 1;
        j.dst = ws.take((unsigned long)rows * j.ldd * (planes > 1 ? 2 * planes : esize(type)));
        j.plane = planes > 1 ? rows * j.ldd : 0;
        d = Matrix{j.dst, j.ldd, rows, cout, true, j.plane};
    }
    b.bias_in_dw = (want & kWantB) && (want & kWantW) && !b.tiles && !copy;
    if ((want & kWantB) && !b.bias_in_dw) {
        b.strips = (int)((rows + j.strip - 1) / j.strip);
        j.sums = b.sums = (float *)ws.take((unsigned long)b.strips * cout * 4);
    }
    if (rows && cout && (copy || j.sums)) add_job(b.jobs, b.njobs, j);
    const Kind kind = b.tiles ? kTiles : kSmall;
    if (want & kWantW) {
        const double time = plan(b.dw, type, kind, true, true, cin, cout, rows, two);
        if (b.tiles && type == kF32 && prefer_split(b.dw, time, x, true)) copy_for_split(b.jobs, b.njobs, ws, x);
        else if (b.tiles && !tile_operand(type, x)) copy_for_tiles(b.jobs, b.njobs, ws, type, x);
    }
    if (b.tiles && (want & kWantX) && !tile_operand(type, w)) copy_for_tiles(b.jobs, b.njobs, ws, type, w);
    if (want & kWantX) {
        plan(b.dx, type, kind, false, false, rows, cin, cout, two);
        place(b.dx, ws, d, w);
    }
    if (want & kWantW) place(b.dw, ws, x, d);
    if (act != kNone && !copy) {
        for (Product *P : {&b.dx.P, &b.dw.P}) {
            P->z = z.p; P->ldz = z.ld; P->vec_z = z.vec; P->zact = act;
        }
    } else if (two && !b.tiles) {
        for (Product *P : {&b.dx.P, &b.dw.P}) {
            P->z = (const char *)d.p + d.plane * 2; P->ldz = d.ld; P->vec_z = 1; P->zact = kPlanes;
        }
    }
    if (b.bias_in_dw && b.dw.P.splits > 1) {
        b.strips = b.dw.P.splits;
        b.sums = (float *)ws.take((unsigned long)b.strips * cout * 4);
    }
}

}  // namespace

extern "C" int sa_dense_forward_ws(int dtype, long rows, int cin, int cout, int flags, unsigned long *bytes) {
    if (!bytes || !sizes_ok(dtype, rows, cin, cout)) return SA_ERR_INVALID;
    *bytes = 0;
    if (rows == 0 || cout == 0) return SA_OK;
    Forward f;
    Scratch s{nullptr};
    plan_forward(f, s, dtype, rows, cin, cout, Matrix{nullptr, cin, rows, cin, (flags & 1) != 0},
                 Matrix{nullptr, cout, cin, cout, (flags & 2) != 0});
    *bytes = s.used;
    return SA_OK;
}

extern "C" int sa_dense_forward(int dtype, long rows, int cin, int cout, const void *x, long ldx, const void *w, long ldw,
                                const void *bias, int bias_f32, const void *res, long ldr, int act, void *y, void *pre,
                                void *ws, unsigned long ws_bytes, void *stream) {
    if (!sizes_ok(dtype, rows, cin, cout) || act < kNone || act > kSilu) return SA_ERR_INVALID;
    if (rows == 0 || cout == 0) return SA_OK;
    if (!y || (cin && (!x || !w)) || ldx < cin || ldw < cout || (res && ldr < cout)) return SA_ERR_INVALID;
    if (!whole(dtype, {x, w, res, y, pre}) || !whole(bias_f32 ? kF32 : dtype, {bias})) return SA_ERR_INVALID;
    if (ldx >= kMaxLd || ldw >= kMaxLd) return SA_ERR_UNSUPPORTED;
    Forward f;
    Scratch s{(char *)ws};
    plan_forward(f, s, dtype, rows, cin, cout, Matrix{x, ldx, rows, cin, aligned(x, ldx, dtype)},
                 Matrix{w, ldw, cin, cout, aligned(w, ldw, dtype)});
    if (!scratch_ok(ws, s.used, ws_bytes)) return SA_ERR_INVALID;
    Epilogue &e = f.plan.P.e;
    e = Epilogue{y, cout, pre, cout, bias, bias_f32, res, ldr, act};
    const int rc = launch_jobs(dtype, f.jobs, f.njobs, (hipStream_t)stream);
    if (rc) return rc;
    if (f.plan.shape != kNoTile) return launch_tile_plan(dtype, f.plan, (hipStream_t)stream);
    const int rs = launch_small_forward(dtype, f.plan.P, (hipStream_t)stream);
    return rs ? rs : launch_join(dtype, f.plan.P, (hipStream_t)stream);
}

// An activation, with kRoundSlopes added or without, and whether dZ goes in two planes
inline bool take_act(int type, int given, int &act, bool &two) {
    act = given & ~kRoundSlopes;
    two = type != kF32 && act > kRelu && !(given & kRoundSlopes);
    return act >= kNone && act <= kSilu;
}

extern "C" int sa_dense_backward_ws(int dtype, long rows, int cin, int cout, int activation, int want, int flags, unsigned long *bytes) {
    int act;
    bool two;
    if (!bytes || !sizes_ok(dtype, rows, cin, cout) || !take_act(dtype, activation, act, two) || want < 0 || want > 7) return SA_ERR_INVALID;
    *bytes = 0;
    want = wanted(want & kWantX, want & kWantW, want & kWantB, rows, cin, cout);
    if (!want) return SA_OK;
    Backward b;
    Scratch s{nullptr};
    plan_backward(b, s, dtype, rows, cin, cout, Matrix{nullptr, cin, rows, cin, (flags & 1) != 0},
                  Matrix{nullptr, cout, cin, cout, (flags & 2) != 0}, Matrix{nullptr, cout, rows, cout, (flags & 4) != 0},
                  Matrix{nullptr, cout, rows, cout, true}, act, two, want);
    *bytes = s.used;
    return SA_OK;
}

extern "C" int sa_dense_backward(int dtype, long rows, int cin, int cout, const void *x, long ldx, const void *w, long ldw,
                                 const void *g, long ldg, const void *z, long ldz, int activation, void *dx, void *dw, void *db,
                                 int db_f32, void *ws, unsigned long ws_bytes, void *stream) {
    int act;
    bool two;
    if (!sizes_ok(dtype, rows, cin, cout) || !take_act(dtype, activation, act, two)) return SA_ERR_INVALID;
    const int want = wanted(dx, dw, db, rows, cin, cout);
    if (!want) return SA_OK;
    if (rows && cout && (!g || ldg < cout || (act != kNone && (!z || ldz < cout)))) return SA_ERR_INVALID;
    if ((want & kWantX) && cout && (!w || ldw < cout)) return SA_ERR_INVALID;
    if ((want & kWantW) && rows && (!x || ldx < cin)) return SA_ERR_INVALID;
    if (!whole(dtype, {x, w, g, act == kNone ? nullptr : z, dx, dw}) || !whole(db_f32 ? kF32 : dtype, {db})) return SA_ERR_INVALID;
    if (((want & kWantX) && ldw >= kMaxLd) || ((want & kWantW) && ldx >= kMaxLd) || ldg >= kMaxLd ||
        (act != kNone && ldz >= kMaxLd))
        return SA_ERR_UNSUPPORTED;
    Backward b;
    Scratch s{(char *)ws};
    plan_backward(b, s, dtype, rows, cin, cout, Matrix{x, ldx, rows, cin, aligned(x, ldx, dtype)},
                  Matrix{w, ldw, cin, cout, aligned(w, ldw, dtype)}, Matrix{g, ldg, rows, cout, aligned(g, ldg, dtype)},
                  Matrix{z, ldz, rows, cout, aligned(z, ldz, dtype)}, act, two, want);
    if (!scratch_ok(ws, s.used, ws_bytes)) return SA_ERR_INVALID;
    hipStream_t st = (hipStream_t)stream;
    int rc = launch_jobs(dtype, b.jobs, b.njobs, st);
    if (rc) return rc;
    if ((want & kWantB) && !b.bias_in_dw && (rc = launch_sums(dtype, b.sums, b.strips, cout, db, db_f32, st))) return rc;
    b.dx.P.e = Epilogue{dx, cin, nullptr, 0, nullptr, 0, nullptr, 0, kNone};
    b.dw.P.e = Epilogue{dw, cout, nullptr, 0, nullptr, 0, nullptr, 0, kNone};
    if (b.tiles) {
        if ((want & kWantX) && (rc = launch_tile_plan(dtype, b.dx, st))) return rc;
        return want & kWantW ? launch_tile_plan(dtype, b.dw, st) : SA_OK;
    }
    if (!(want & (kWantX | kWantW))) return SA_OK;
    if (b.bias_in_dw) {
        b.dw.P.colsum = db;
        b.dw.P.col_f32 = db_f32;
        b.dw.P.colpart = b.sums;
    }
    rc = launch_small_backward(dtype, want & kWantX ? &b.dx.P : nullptr, want & kWantW ? &b.dw.P : nullptr, st);
    if (rc) return rc;
    if ((want & kWantX) && (rc = launch_join(dtype, b.dx.P, st))) return rc;
    if ((want & kWantW) && (rc = launch_join(dtype, b.dw.P, st))) return rc;
    return b.bias_in_dw && b.dw.P.splits > 1 ? launch_sums(dtype, b.sums, b.strips, cout, db, db_f32, st) : SA_OK;
}
