// Dense layer on e4m3 images (e4m3.h):  Y[m][n] = act(sum_k X^[m][k] W^[n][k] + bias[n]),  X^ / W^ the values of the images.
//
// Two matrix pipes.  The 8-bit one, v_mfma_scale_f32_32x32x64_f8f6f4, multiplies 64 codes of 32 rows of each operand at twice the
// bf16 rate (4.65 against 1.87 PFLOP/s in a loop of nothing else) and applies one E8M0 exponent per row and 32 codes, so the blocks'
// powers of two go in as they are.  It adds eight products at a time, each cut off 13 bits below the largest of the eight
// (measured: 2^16 + 2^2 loses the small one, products of different eights are added in fp32): enough where the sum is then rounded to
// 8 or 11 bits, too coarse for an fp32 result.  fp32 results take the bf16 pipe, v_mfma_f32_32x32x16_bf16, whose sums are fp32
// throughout: the values of an image are exact in bf16, converted with their scale from the codes as those leave LDS
// (v_cvt_scalef32_pk_bf16_fp8, two codes each).
// Both operands are K-contiguous and an instruction's K order is free (A and B share it).
#include "e4m3.h"
#include "tile128.h"

namespace phonlp {

struct E4m3Args {
    const uint8_t *x, *xe, *w, *we;
    const float *bias;
    void *y;
    uint32_t *bits;
    int M, N, Kp, KB4, num_m, num_n, relu, words;
};

// LDS image of a tile: row r (128 codes) at r * 128, its 16-byte chunk c at slot c ^ ((r >> 1) & 7): sixteen rows' chunks c lie in
// sixteen different slots of the 64 banks.
__device__ __forceinline__ i32x4 tile_chunk(const uint8_t *tile, int r, int c) {
    return *reinterpret_cast<const i32x4 *>(tile + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
}

// Bias, ReLU, the rounding to T, and the row's bits: acc register r of a lane holds row (r & 3) + 8 (r >> 2) + 4 (lane >> 5),
// column lane & 31 of a 32 x 32 sub-tile, so one ballot is a 32-column word of two rows.
template <class T>
__device__ __forceinline__ void e4m3_store(const E4m3Args &a, const f32x16 &acc, int m0, int n0, int lane) {
    const int n = n0 + (lane & 31), half = lane >> 5;
    const bool in = n < a.N;
    const float b = in && a.bias ? a.bias[n] : 0.f;
    T *y = (T *)a.y;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int m = m0 + (r & 3) + 8 * (r >> 2) + 4 * half;
        float v = acc[r] + b;
        if (a.relu) v = v < 0.f ? 0.f : v;  // keeps NaN
        if (a.bits) {
            const unsigned long long up = __ballot(in && v > 0.f);
            if ((lane & 31) == 0 && m < a.M && n0 < a.N) a.bits[(long)m * a.words + (n0 >> 5)] = (uint32_t)(half ? up >> 32 : up);
        }
        if (in && m < a.M) y[(long)m * a.N + n] = (T)v;
    }
}

// Sixteen codes times their block's scale -> the bf16 operands of two matrix instructions.
__device__ __forceinline__ void widen(const i32x4 &c, float scale, bf16x8 (&v)[2]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const bf16x2 lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[q], scale, false);
        const bf16x2 hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c[q], scale, true);
        v[q >> 1][(q & 1) * 4 + 0] = lo[0];
        v[q >> 1][(q & 1) * 4 + 1] = lo[1];
        v[q >> 1][(q & 1) * 4 + 2] = hi[0];
        v[q >> 1][(q & 1) * 4 + 3] = hi[1];
    }
}
__device__ __forceinline__ float scale_of(int exponents) { return __int_as_float((exponents & 0xFF) << 23); }  // e + 127 >= 1

// TM x TN tile, WM x WN waves, k blocks of 128 double-buffered in LDS.
template <int TM, int TN, int WM, int WN, class T>
__global__ __launch_bounds__(WM *WN * 64) void linear_e4m3_kernel(E4m3Args a) {
    constexpr int NW = WM * WN, RA = TM / WM / 32, RB = TN / WN / 32, LOADS = (TM + TN) / 8 / NW;
    extern __shared__ uint8_t lds[];  // [2][TM + TN][128]
    int tm, tn, split;
    if (!tile_of(blockIdx.x, a.num_m, a.num_n, 1, 8, &tm, &tn, &split)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    const int wm = wave / WN, wn = wave % WN;
    const int m0 = tm * TM, n0 = tn * TN;
    const uint8_t *xb = a.x + (long)m0 * a.Kp, *wb = a.w + (long)n0 * a.Kp;

    uint32_t off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {  // rows behind the matrix read its last row: their products are not stored
        const int r = (wave + i * NW) * 8 + (lane >> 3);
        const int row = r < TM ? min(r, a.M - 1 - m0) : min(r - TM, a.N - 1 - n0);
        off[i] = (uint32_t)row * (uint32_t)a.Kp + (((lane & 7) ^ ((r >> 1) & 7)) << 4);
    }
    auto load = [&](int kb, int buf) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r8 = wave + i * NW;
            dma16((r8 * 8 < TM ? xb : wb) + kb * 128, off[i], lds + buf * (TM + TN) * 128 + r8 * 1024);
        }
    };
    const uint8_t *xe[RA], *we[RB];
#pragma unroll
    for (int i = 0; i < RA; ++i) xe[i] = a.xe + (long)min(m0 + (wm * RA + i) * 32 + l32, a.M - 1) * a.KB4;
#pragma unroll
    for (int j = 0; j < RB; ++j) we[j] = a.we + (long)min(n0 + (wn * RB + j) * 32 + l32, a.N - 1) * a.KB4;

    f32x16 acc[RA][RB];
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    int sx[RA], sw[RB];
    const int nkb = a.Kp / 128;
    load(0, 0);
    for (int kb = 0; kb < nkb; ++kb) {
        if ((kb & 3) == 0) {  // four blocks' exponents are one dword; the instruction takes the lowest byte
#pragma unroll
            for (int i = 0; i < RA; ++i) sx[i] = *reinterpret_cast<const int *>(xe[i] + kb);
#pragma unroll
            for (int j = 0; j < RB; ++j) sw[j] = *reinterpret_cast<const int *>(we[j] + kb);
        }
        dma_wait_barrier<0>();  // block kb has landed; everybody is done with the other buffer
        if (kb + 1 < nkb) load(kb + 1, (kb + 1) & 1);
        const uint8_t *A = lds + (kb & 1) * (TM + TN) * 128, *B = A + TM * 128;
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                i32x8 fa[RA], fb[RB];
#pragma unroll
                for (int i = 0; i < RA; ++i) {
                    const int r = (wm * RA + i) * 32 + l32, c = s * 4 + half * 2;
                    const i32x4 lo = tile_chunk(A, r, c), hi = tile_chunk(A, r, c + 1);
                    fa[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
#pragma unroll
                for (int j = 0; j < RB; ++j) {
                    const int r = (wn * RB + j) * 32 + l32, c = s * 4 + half * 2;
                    const i32x4 lo = tile_chunk(B, r, c), hi = tile_chunk(B, r, c + 1);
                    fb[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                }
#pragma unroll
                for (int i = 0; i < RA; ++i)
#pragma unroll
                    for (int j = 0; j < RB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fa[i], fb[j], acc[i][j], 0, 0, 0, sx[i], 0, sw[j]);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                bf16x8 fa[RA][2], fb[RB][2];
#pragma unroll
                for (int i = 0; i < RA; ++i) widen(tile_chunk(A, (wm * RA + i) * 32 + l32, s * 2 + half), scale_of(sx[i]), fa[i]);
#pragma unroll
                for (int j = 0; j < RB; ++j) widen(tile_chunk(B, (wn * RB + j) * 32 + l32, s * 2 + half), scale_of(sw[j]), fb[j]);
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < RA; ++i)
#pragma unroll
                        for (int j = 0; j < RB; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i][q], fb[j][q], acc[i][j], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < RA; ++i) sx[i] = (unsigned)sx[i] >> 8;
#pragma unroll
        for (int j = 0; j < RB; ++j) sw[j] = (unsigned)sw[j] >> 8;
    }
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) e4m3_store<T>(a, acc[i][j], m0 + (wm * RA + i) * 32, n0 + (wn * RB + j) * 32, lane);
}

template <int TM, int TN, int WM, int WN, class T>
static int launch_tile(E4m3Args a, hipStream_t st) {
    static PerDeviceOnce once;
    int dev;
    constexpr int bytes = 2 * (TM + TN) * 128;
    if (once.pending(&dev)) {
        if (hipFuncSetAttribute((const void *)linear_e4m3_kernel<TM, TN, WM, WN, T>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
            hipSuccess)
            return fail(PHONLP_ERR_LAUNCH, "linear_e4m3: hipFuncSetAttribute failed");
        once.mark(dev);
    }
    a.num_m = ceil_div(a.M, TM);
    a.num_n = ceil_div(a.N, TN);
    hipLaunchKernelGGL((linear_e4m3_kernel<TM, TN, WM, WN, T>), dim3(tile_grid(a.num_m, a.num_n, 1)), dim3(WM * WN * 64), bytes, st, a);
    return check_launch("linear_e4m3_kernel");
}

}  // namespace phonlp

using namespace phonlp;

extern "C" int phonlp_linear_e4m3(const void *x_codes, const uint8_t *x_exponents, const void *w_codes, const uint8_t *w_exponents,
                                  const float *bias, void *y, int type, uint32_t *bits, int M, int N, int K, int relu, void *stream) {
    if (!x_codes || !x_exponents || !w_codes || !w_exponents || !y || !type_ok(type) || M <= 0 || N <= 0 || K <= 0 || K > (1 << 22))
        return fail(PHONLP_ERR_SHAPE, "linear_e4m3: bad argument");
    if (((uintptr_t)x_codes & 15) || ((uintptr_t)w_codes & 15) || ((uintptr_t)x_exponents & 3) || ((uintptr_t)w_exponents & 3) ||
        ((uintptr_t)bias & 3) || ((uintptr_t)bits & 3) || (uintptr_t)y % type_bytes(type))
        return fail(PHONLP_ERR_SHAPE, "linear_e4m3: codes must be 16-byte aligned, exponents, bias and bits 4-byte, y to its type");
    if ((long)ceil_div(M, 32) * ceil_div(N, 32) > 0x3FFFFFFF) return fail(PHONLP_ERR_UNSUPPORTED, "linear_e4m3: M * N too large");
    E4m3Args a = {(const uint8_t *)x_codes, x_exponents, (const uint8_t *)w_codes, w_exponents, bias, y, bits, M, N, kp8_of(K), kb4_of(K),
                  0, 0, relu, ceil_div(N, 32)};
    hipStream_t st = as_stream(stream);
    ProfScope ps("linear_e4m3", st);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return launch_tile<128, 128, 2, 2, T>(a, st);
    });
}
