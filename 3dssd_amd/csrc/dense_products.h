// Interface between dense.hip and the kernels for large (dense_tile.hip, dense_split.hip) and small products (dense_small.hip).
#pragma once
#include "dense_common.h"

namespace dense {
// Byte offsets inside a block are 31-bit: fewer than this many elements between neighbours of an operand's outer index for
// the 256 rows of a tile, and for the 32 of a small block (and no row is longer).
constexpr long kMaxTileLd = 1L << 21, kMaxLd = 1L << 24;

// D = A B^T on tiles of the given shape, of 16-bit operands with 16-byte aligned bases and rows, and whole 16-byte
// pieces along the contiguous index.  type: kBF16 / kF16 of the operands; out_type: that, or kF32.  P.kchunk counts steps of
// 64 k over all passes.  ta and not tb does not occur.
enum TileShape { kNoTile = 0, kTile256 = 1, kTile256x128 = 2, kTile128 = 3, kSplit256 = 4 };
int launch_tiles(int shape, int type, int out_type, bool ta, bool tb, const Product &P, hipStream_t s);

// A in fp32 (k, or with ta m, contiguous; 16-byte aligned base and rows, fewer than kMaxTileLd / 2 elements apart; along the
// contiguous index a multiple of 4, or zeros behind it up to one), B as three bf16 planes (n contiguous, like the tiles'
// operands), to fp32, on tiles of 256 x 256; P.passes is 1 and P.kchunk counts steps of 32 k.
int launch_split(bool ta, const Product &P, hipStream_t s);

// Any forward product (A k-contiguous, B n-contiguous); P.kchunk counts k indices (a multiple of 32).
int launch_small_forward(int type, const Product &P, hipStream_t s);
// dX (A = G or dZ and B = W, both k-contiguous) and dW (A = X, B = G or dZ, both with rows contiguous) in one launch; either
// may be null.  With P.z set the operand G becomes G act'(Z), with P.two in two planes; dW's colsum is the bias gradient.
int launch_small_backward(int type, const Product *dx, const Product *dw, hipStream_t s);
}  // namespace dense
