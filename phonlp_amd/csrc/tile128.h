// What the kernels on 128-byte rows share (linear_e4m3.hip: 128 codes a row, linear_e4m3_backward.hip: 64 bf16 a row): tiles of
// [rows][128 bytes] brought to LDS by the LDS-DMA path, and the order in which tiles are handed to workgroups.
//
// LDS image of a tile: row r at r * 128, its 16-byte chunk c at slot c ^ (r & 7).  The eight lanes that an LDS read of 16 bytes
// per lane serves at a time hold eight consecutive rows and the same chunk: eight different slots, no bank conflict.
#pragma once
#include "common.h"

namespace phonlp {

#ifdef __HIPCC__
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// 64 lanes x 16 bytes from `base + off` (off per lane) to 1024 consecutive bytes at `lds` (wave-uniform).
__device__ __forceinline__ void dma16(const uint8_t *base, uint32_t off, uint8_t *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(base + off),
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}
// All of this wave's loads are done, LDS-DMA among them, and every wave is here.
__device__ __forceinline__ void dma_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
}

// The 16-byte chunk c of row r of a tile image.
__device__ __forceinline__ i32x4 tile_chunk(const uint8_t *tile, int r, int c) {
    return *reinterpret_cast<const i32x4 *>(tile + r * 128 + ((c ^ (r & 7)) << 4));
}
#endif

// The tile of workgroup `bid` out of num_m x num_n.  Workgroups go to the eight XCDs in turn and each XCD has its own L2: every XCD
// gets a contiguous share of the tile order, and the order runs through groups of `gm` row tiles, column by column, so that the
// workgroups that run together on one XCD share operand rows.  Returns false for the surplus workgroups of the rounded-up grid.
__device__ __forceinline__ bool tile_of(int bid, int num_m, int num_n, int gm, int *tm, int *tn) {
    const int total = num_m * num_n, share = (total + 7) / 8;
    const int id = (bid & 7) * share + (bid >> 3);
    if ((bid >> 3) >= share || id >= total) return false;
    const int per_group = gm * num_n, g = id / per_group, in = id - g * per_group;
    const int rows = min(gm, num_m - g * gm);
    *tm = g * gm + in % rows;
    *tn = in / rows;
    return true;
}
inline int tile_grid(int num_m, int num_n) { return (num_m * num_n + 7) / 8 * 8; }

}  // namespace phonlp
