// Where the products of linear_e4m3_backward.hip read their operands: plain arithmetic, for the host as well.
#pragma once
#include "common.h"

namespace phonlp {

// dZ as the products read it: dY itself, or its pieces in the workspace.
struct BwOperand {
    const uint8_t *at;
    long pitch, width, plane;  // bytes: from row to row, of a row that may be read, from piece to piece
};
// Without a mask and with whole steps, bf16 gradients are their own single piece.
inline bool bw_direct(const void *dy, int type, long lddy, const void *bits, int M, int N) {
    return type == PHONLP_BF16 && !bits && M % 32 == 0 && N % 32 == 0 && lddy % 8 == 0 && lddy < (1 << 22) && !((uintptr_t)dy & 15);
}
inline BwOperand bw_dz(bool direct, const void *dy, long lddy, const uint8_t *planes, int N, int Mp, int Np) {
    if (direct) return {(const uint8_t *)dy, lddy * 2, N * 2L, 0};
    return {planes, Np * 2L, Np * 2L, (long)Mp * Np * 2};
}

// Of a tile in LDS whose reduction runs down its rows, [32 r][columns]: chunk c (16 bytes) of row r at slot c ^ turn(r); a transposing
// read takes 4 rows x 32 bytes per 16 lanes, and those of 32 lanes (rows 8 apart) lie in all 64 banks.
__host__ __device__ inline int turn(int r) { return ((r & 3) << 2) | ((r >> 3 & 1) << 1); }

// The byte offset from a tile's first element, for one lane, of its part of kilobyte u of a [32 r][ROW / 2 columns] tile.  `left`: bytes
// of a row from the tile's first column on; columns behind them read its last ones.
template <int ROW>
__host__ __device__ inline uint32_t tr_offset(int u, int lane, long pitch, long left) {
    constexpr int LANES = ROW / 16;
    const int r = u * (64 / LANES) + lane / LANES;
    const long c = ((lane % LANES) ^ turn(r)) * 16L, last = left - 16;
    return (uint32_t)r * (uint32_t)pitch + (uint32_t)(c < last ? c : last);
}

}  // namespace phonlp
