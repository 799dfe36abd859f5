// Interface between dense.hip and dense_tile.hip.
#pragma once
#include "dense_common.h"

namespace dense {
// D = A B^T on tiles of edge x edge (128 or 256) of 16-bit operands with 16-byte aligned bases and rows, whole 16-byte
// pieces along the contiguous index, and fewer than kMaxLd elements between neighbours of the other index (offsets inside
// a tile are 31-bit).  type: kBF16 / kF16 of the operands; out_type: that, or kF32.  P.kchunk counts steps of 64 k over all
// passes.  ta and not tb does not occur.
constexpr long kMaxLd = 1L << 21;
int launch_tiles(int edge, int type, int out_type, bool ta, bool tb, const Product &P, hipStream_t s);
}  // namespace dense
