// What the matrix kernels of linear_e4m3.hip and linear_e4m3_backward.hip share: loads into LDS past the registers, waits that
// count them, and the order in which output tiles are handed to workgroups.
#pragma once
#include "common.h"

namespace phonlp {

#ifdef __HIPCC__
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Byte offset of a pointer into LDS: the low half of its flat address.
__device__ __forceinline__ uint32_t lds_offset(const uint8_t *p) { return (uint32_t)(uintptr_t)p; }

// 64 lanes x 16 bytes from `base + off` (base wave-uniform, off per lane) to 1024 consecutive bytes of LDS (wave-uniform).  Inline
// asm, as the waits are: the compiler cannot tell the buffers of a ring apart and would let every LDS read wait for every load.
__device__ __forceinline__ void dma16(const uint8_t *base, uint32_t off, const uint8_t *lds) {
    const uint32_t at = lds_offset(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(off), "s"(base)
                 : "memory", "m0");
}
// The same with four bytes per lane, of the lanes in `mask` alone.  For waves whose lanes are all active: exec is -1 afterwards (a
// branch around the load would end the basic block, and the compiler moves matrix instructions across block ends).
__device__ __forceinline__ void dma4(const uint8_t *base, uint32_t off, const uint8_t *lds, unsigned long long mask) {
    const uint32_t at = lds_offset(lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_mov_b64 exec, %3\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2\n\ts_mov_b64 exec, -1" ::"s"(
                     __builtin_amdgcn_readfirstlane(at)),
                 "v"(off), "s"(base), "s"(mask)
                 : "memory", "m0");
}
// At most N of this wave's loads are still on their way (they arrive in order); then every wave is here, its LDS reads done.
template <int N>
__device__ __forceinline__ void dma_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    lds_barrier();
}
template <int N>
__device__ __forceinline__ void dma_wait() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
#endif

// The tile and the range of the reduction of workgroup `bid`, out of num_m x num_n tiles and `splits` ranges.  Workgroups go to the
// eight XCDs in turn and each XCD has its own L2: every XCD gets a contiguous share of the order, which runs range by range, in a
// range through groups of `gm` row tiles, in a group column by column, so that the workgroups that run together on one XCD share
// operand rows.  Returns false for the surplus workgroups of the rounded-up grid.
__device__ __forceinline__ bool tile_of(int bid, int num_m, int num_n, int splits, int gm, int *tm, int *tn, int *split) {
    const int tiles = num_m * num_n, total = tiles * splits, share = (total + 7) / 8;
    int id = (bid & 7) * share + (bid >> 3);
    if ((bid >> 3) >= share || id >= total) return false;
    *split = id / tiles;
    id -= *split * tiles;
    const int per_group = gm * num_n, g = id / per_group, in = id - g * per_group;
    const int rows = min(gm, num_m - g * gm);
    *tm = g * gm + in % rows;
    *tn = in / rows;
    return true;
}
inline int tile_grid(int num_m, int num_n, int splits) { return (num_m * num_n * splits + 7) / 8 * 8; }

}  // namespace phonlp
