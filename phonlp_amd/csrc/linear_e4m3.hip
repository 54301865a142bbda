// Dense layer on e4m3 images (e4m3.h):  Y[m][n] = act(sum_k X^[m][k] W^[n][k] + bias[n]),  X^ / W^ the values of the images.
//
// Two matrix pipes.  The 8-bit one, v_mfma_scale_f32_32x32x64_f8f6f4, multiplies 64 codes of 32 rows of each operand at twice the
// bf16 rate (4.65 against 2.05 PFLOP/s in a loop of nothing else) and applies one E8M0 exponent per row and 32 codes, so the blocks'
// powers of two go in as they are.  It adds eight products at a time, each cut off 13 bits below the largest of the eight
// (measured: 2^16 + 2^2 loses the small one, products of different eights are added in fp32): enough where the sum is then rounded to
// 8 or 11 bits, too coarse for an fp32 result.  fp32 results take the bf16 pipe, v_mfma_f32_16x16x32_bf16, whose sums are fp32
// throughout: the values of an image are exact in bf16, converted with their scale from the codes as those leave LDS
// (v_cvt_scalef32_pk_bf16_fp8, two codes each).
// Both operands are K-contiguous and an instruction's K order is free (A and B share it).
#include <type_traits>

#include "e4m3.h"
#include "tile128.h"

namespace phonlp {

struct E4m3Args {
    const uint8_t *x, *xe, *w, *we;
    const float *bias;
    void *y;
    uint8_t *bits;
    int M, N, Kp, KB4, num_m, num_n, relu, row_bytes;  // row_bytes: of bits
};

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Eight codes times their block's scale -> the bf16 operand of v_mfma_f32_16x16x32_bf16.
__device__ __forceinline__ bf16x8 widen(int lo, int hi, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float scale_of(int exponents) { return __int_as_float((exponents & 0xFF) << 23); }  // e + 127 >= 1

// Bias, ReLU and the rounding to T of four neighbouring values.
template <class T>
__device__ __forceinline__ typename Vec<T, 4>::type finish(f32x4 v, const float (&bias)[4], int relu) {
    typename Vec<T, 4>::type t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x = v[i] + bias[i];
        if (relu) x = x < 0.f ? 0.f : x;  // keeps NaN
        t[i] = (T)x;
    }
    return t;
}

// Up to 16 bytes of a row of Y, and their bits (column n in bit n % 8 of byte n / 8 of a row: the words of phonlp_linear_e4m3).
template <class T>
__device__ __forceinline__ void store_row(const E4m3Args &a, int m, int n, const typename Vec<T, 16 / sizeof(T)>::type &v) {
    constexpr int VEC = 16 / sizeof(T);
    if (m >= a.M) return;
    T *y = (T *)a.y + (long)m * a.N + n;
    const int left = a.N - n;
    if (left >= VEC) {
        *reinterpret_cast<typename Vec<T, VEC>::type *>(y) = v;
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < left) y[i] = v[i];
    }
    if (!a.bits) return;
    int b = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) b |= i < left && (float)v[i] > 0.f ? 1 << i : 0;
    if (VEC == 4) {  // a byte is two lanes' four columns
        b |= __shfl_down(b, 1) << 4;
        if (n & 4) return;
    }
    if (n >> 3 < a.row_bytes) a.bits[(long)m * a.row_bytes + (n >> 3)] = (uint8_t)b;
}

// Tile of TM x TN, eight waves (4 x 2) of TM / 4 x TN / 2.  A block of 128 codes of every row comes by LDS-DMA in whole 128-byte lines
// into one of two buffers, and goes through registers in two parts of 64.  The codes of a part are read from LDS while the part
// before is multiplied, so one barrier a block, before its second part, does: there block kb + 1 has landed, and as every wave
// has all of block kb in registers, its buffer takes block kb + 2, a whole block's time ahead.
// Four blocks' exponents of a row are one dword; those of the tile's rows lie in a ring of four LDS slots, and each block brings a
// quarter of the next slot's.
//
// LDS image of a block: row r at r * 128, its 16-byte chunk c at slot c ^ ((r >> 1) & 7): sixteen rows' chunks c lie in all 64 banks.
template <int TM, int TN, class T>
__global__ __launch_bounds__(512) void linear_e4m3_kernel(E4m3Args a) {
    constexpr bool PIPE8 = sizeof(T) == 2;  // which matrix pipe (above)
    constexpr int ROWS = TM + TN, SIDE = PIPE8 ? 32 : 16, FA = TM / 4 / SIDE, FB = TN / 2 / SIDE, LOADS = ROWS / 64, SIZE = ROWS * 128;
    extern __shared__ uint8_t lds[];  // [2][ROWS][128] codes, [4][ROWS] exponents; then the waves' output patches
    uint8_t *slots = lds + 2 * SIZE;
    int tm, tn, split;
    if (!tile_of(blockIdx.x, a.num_m, a.num_n, 1, 8, &tm, &tn, &split)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave >> 1, wn = wave & 1, ls = lane & (SIDE - 1), lg = lane / SIDE, m0 = tm * TM, n0 = tn * TN;
    const int blocks = a.Kp / 128, groups = a.KB4 / 4;

    // rows behind the matrix read its last row: their products are not stored
    const uint8_t *xb = a.x + (long)m0 * a.Kp, *wb = a.w + (long)n0 * a.Kp;
    uint32_t off[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
        const int r = (wave + k * 8) * 8 + (lane >> 3), c = (lane & 7) ^ ((r >> 1) & 7);
        off[k] = (uint32_t)(r < TM ? min(r, a.M - 1 - m0) : min(r - TM, a.N - 1 - n0)) * (uint32_t)a.Kp + c * 16;
    }
    auto load = [&](int kb, int k) {  // behind the end the last block again
        const int r8 = wave + k * 8;
        dma16((r8 * 8 < TM ? xb : wb) + min(kb, blocks - 1) * 128, off[k], lds + (kb & 1) * SIZE + r8 * 1024);
    };
    // Exponents of the group G of four blocks: of the eighth of the tile's rows that this wave brings, quarter z (of `of`).
    auto load_exponents = [&](int G, int z, int of) {
        const int to = (G & 3) * ROWS, g = min(G, groups - 1) * 4;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            const int rows = (w ? TN : TM) / 8 / of, r = (w ? TN : TM) / 8 * wave + z * rows, last = w ? a.N - 1 - n0 : a.M - 1 - m0;
            dma4((w ? a.we + (long)n0 * a.KB4 : a.xe + (long)m0 * a.KB4) + g, (uint32_t)min(r + lane, last) * (uint32_t)a.KB4,
                 slots + (to + (w ? TM : 0) + r) * 4, (1ull << rows) - 1);
        }
    };

    // lane (ls, lg) holds row ls of a fragment: of a part's 64 codes 32 from 32 lg (8-bit pipe), or 16 from 16 lg, eight for each of two
    // steps; fragments are multiples of 16 rows apart, which do not change the slot
    constexpr int H = PIPE8 ? 2 : 1;
    int at_a[2][H], at_b[2][H];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const int slot = ((p * 4 + (PIPE8 ? lg * 2 + h : lg)) ^ ((ls >> 1) & 7)) << 4;
            at_a[p][h] = (wm * (TM / 4) + ls) * 128 + slot;
            at_b[p][h] = (TM + wn * (TN / 2) + ls) * 128 + slot;
        }
    struct A {
        i32x4 f[FA][H];
    };
    i32x4 b[FB][H];
    struct Scales {
        int a[FA], b[FB];
    };
    auto read_a = [&](int kb, int p, int i, A &x) {
#pragma unroll
        for (int h = 0; h < H; ++h) x.f[i][h] = *reinterpret_cast<const i32x4 *>(lds + (kb & 1) * SIZE + at_a[p][h] + i * SIDE * 128);
    };
    auto read_b = [&](int kb, int p, int j) {
#pragma unroll
        for (int h = 0; h < H; ++h) b[j][h] = *reinterpret_cast<const i32x4 *>(lds + (kb & 1) * SIZE + at_b[p][h] + j * SIDE * 128);
    };
    auto read_scales = [&](int kb, Scales &s) {  // of block kb, in the lowest byte
        const int *e = reinterpret_cast<const int *>(slots) + ((kb >> 2) & 3) * ROWS + ls, shift = (kb & 3) * 8;
#pragma unroll
        for (int i = 0; i < FA; ++i) s.a[i] = (unsigned)e[wm * (TM / 4) + i * SIDE] >> shift;
#pragma unroll
        for (int j = 0; j < FB; ++j) s.b[j] = (unsigned)e[TM + wn * (TN / 2) + j * SIDE] >> shift;
    };

    typedef std::conditional_t<PIPE8, f32x16, f32x4> Acc;
    Acc acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j)
#pragma unroll
            for (int r = 0; r < SIDE * SIDE / 64; ++r) acc[i][j][r] = 0.f;

    // Part p of block kb: its codes are in `now` and b; loads, and LDS reads of the next part's codes into registers that are done
    // with, stand between its matrix instructions.
    auto part = [&](int kb, auto pc, A &now, A &next, const Scales &s) {
        constexpr int p = decltype(pc)::value;
        const int nk = kb + p;  // the next part: 1 - p of block nk
        if (p == 1) dma_wait_barrier<0>();
        auto loads = [&](int z, int of) {  // the share of step z of `of`
            if (p == 0) return;
#pragma unroll
            for (int k = LOADS * z / of; k < LOADS * (z + 1) / of; ++k) load(kb + 2, k);
            if (z == of - 1) load_exponents(((kb + 1) >> 2) + 1, (kb + 1) & 3, 4);
        };
        if constexpr (PIPE8) {
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                loads(j, FB);
                if (j == 0) {
#pragma unroll
                    for (int i = 0; i < FA; ++i) read_a(nk, 1 - p, i, next);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < FA; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        __builtin_shufflevector(b[j][0], b[j][1], 0, 1, 2, 3, 4, 5, 6, 7),
                        __builtin_shufflevector(now.f[i][0], now.f[i][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, 0, s.b[j], 0, s.a[i]);
                __builtin_amdgcn_sched_barrier(0);
                read_b(nk, 1 - p, j);
            }
        } else {
            constexpr int HB = FB / 2, STEPS = 4 * FA;  // half of B's fragments at a time: registers
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                bf16x8 fa[FA];
#pragma unroll
                for (int i = 0; i < FA; ++i) fa[i] = widen(now.f[i][0][2 * q], now.f[i][0][2 * q + 1], scale_of(s.a[i]));
#pragma unroll
                for (int jh = 0; jh < 2; ++jh) {
                    bf16x8 fb[HB];
#pragma unroll
                    for (int j = 0; j < HB; ++j) {
                        const i32x4 &c = b[jh * HB + j][0];
                        fb[j] = widen(c[2 * q], c[2 * q + 1], scale_of(s.b[jh * HB + j]));
                    }
                    if (q == 1) {  // these codes of this part are used up
#pragma unroll
                        for (int k = 0; k < HB; ++k) read_b(nk, 1 - p, jh * HB + k);
                        if (jh == 0) {
#pragma unroll
                            for (int k = 0; k < FA; ++k) read_a(nk, 1 - p, k, next);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < FA; ++i) {
                        loads((q * 2 + jh) * FA + i, STEPS);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int j = 0; j < HB; ++j)
                            acc[i][jh * HB + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][jh * HB + j], 0, 0, 0);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
            }
        }
    };

    load_exponents(0, 0, 1);
#pragma unroll
    for (int k = 0; k < LOADS; ++k) load(0, k);
    dma_wait_barrier<0>();
#pragma unroll
    for (int k = 0; k < LOADS; ++k) load(1, k);
    load_exponents(1, 0, 4);
    A a0, a1;
    Scales s;
#pragma unroll
    for (int i = 0; i < FA; ++i) read_a(0, 0, i, a0);
#pragma unroll
    for (int j = 0; j < FB; ++j) read_b(0, 0, j);
    read_scales(0, s);
    for (int kb = 0; kb < blocks; ++kb) {
        part(kb, std::integral_constant<int, 0>{}, a0, PIPE8 ? a1 : a0, s);
        part(kb, std::integral_constant<int, 1>{}, PIPE8 ? a1 : a0, a0, s);
        read_scales(kb + 1, s);  // a next group's came with blocks up to kb + 1, which have landed
    }
    dma_wait_barrier<0>();  // the repeated loads have landed and every wave is done with the buffers

    // Through LDS, a patch of SIDE rows per wave, so that Y is written in whole row segments of 16 bytes per lane.
    constexpr int VEC = 16 / sizeof(T), COLS = TN / 2, PITCH = COLS * sizeof(T) + 16, LANES = COLS / VEC;
    static_assert(8 * SIDE * PITCH <= 4 * ROWS * 64 + 4 * ROWS * 4, "the patches must fit");
    uint8_t *patch = lds + wave * (SIDE * PITCH);
#pragma unroll
    for (int i = 0; i < FA; ++i) {
#pragma unroll
        for (int j = 0; j < FB; ++j) {
#pragma unroll
            for (int q = 0; q < SIDE * SIDE / 256; ++q) {  // four neighbouring columns of row ls
                const int c = j * SIDE + (PIPE8 ? 8 * q + 4 * lg : 4 * lg), n = n0 + wn * COLS + c;
                float bias[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) bias[k] = a.bias && n + k < a.N ? a.bias[n + k] : 0.f;
                const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                *reinterpret_cast<typename Vec<T, 4>::type *>(patch + ls * PITCH + c * sizeof(T)) = finish<T>(v, bias, a.relu);
            }
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = lane / LANES; r < SIDE; r += 64 / LANES) {
            const int c = (lane % LANES) * VEC;
            const auto v = *reinterpret_cast<const typename Vec<T, VEC>::type *>(patch + r * PITCH + c * sizeof(T));
            store_row<T>(a, m0 + wm * (TM / 4) + i * SIDE + r, n0 + wn * COLS + c, v);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Few rows: a workgroup takes 32 x 32 of Y and its eight waves an eighth of the blocks each, straight from memory to registers (no
// LDS but for the sum over the waves, which is in a fixed order); bound by reading W, or by latency.  Always the bf16 pipe.
template <class T>
__global__ __launch_bounds__(512) void linear_e4m3_few_kernel(E4m3Args a) {
    __shared__ float sums[8][32][33];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 32, m0 = blockIdx.y * 32, blocks = a.Kp / 128;
    f32x4 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    long xr[2], wr[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        xr[i] = min(m0 + i * 16 + l16, a.M - 1);
        wr[i] = min(n0 + i * 16 + l16, a.N - 1);
    }
    for (int kb = wave; kb < blocks; kb += 8) {
        i32x4 x[2][2], w[2][2];  // 32 codes of a row per lane, from 32 g
        float sx[2], sw[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                x[i][h] = *reinterpret_cast<const i32x4 *>(a.x + xr[i] * a.Kp + kb * 128 + g * 32 + h * 16);
                w[i][h] = *reinterpret_cast<const i32x4 *>(a.w + wr[i] * a.Kp + kb * 128 + g * 32 + h * 16);
            }
            sx[i] = scale_of(a.xe[xr[i] * a.KB4 + kb]);
            sw[i] = scale_of(a.we[wr[i] * a.KB4 + kb]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                bf16x8 fx[2], fw[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    fx[i] = widen(x[i][h][2 * q], x[i][h][2 * q + 1], sx[i]);
                    fw[i] = widen(w[i][h][2 * q], w[i][h][2 * q + 1], sw[i]);
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[i], fw[j], acc[i][j], 0, 0, 0);
            }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][i * 16 + g * 4 + r][j * 16 + l16] = acc[i][j][r];
    __syncthreads();
    // 128 threads: eight columns of a row each; 512 threads: two, but a byte of bits stays with one thread
    if (threadIdx.x >= 128) return;
    const int r = threadIdx.x >> 2, c = (threadIdx.x & 3) * 8, m = m0 + r, waves = min(8, blocks);
    if (m >= a.M) return;
    int b = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int n = n0 + c + k;
        if (n >= a.N) continue;
        float v = 0.f;
        for (int w = 0; w < waves; ++w) v += sums[w][r][c + k];
        if (a.bias) v += a.bias[n];
        if (a.relu) v = v < 0.f ? 0.f : v;  // keeps NaN
        const T t = (T)v;
        ((T *)a.y)[(long)m * a.N + n] = t;
        b |= (float)t > 0.f ? 1 << k : 0;
    }
    if (a.bits && (n0 + c) >> 3 < a.row_bytes) a.bits[(long)m * a.row_bytes + ((n0 + c) >> 3)] = (uint8_t)b;
}

template <int TM, int TN, class T>
static int launch_tile(E4m3Args a, hipStream_t st) {
    static PerDeviceOnce once;
    int dev;
    constexpr int bytes = 4 * (TM + TN) * 64 + 4 * (TM + TN) * 4;
    if (once.pending(&dev)) {
        if (hipFuncSetAttribute((const void *)linear_e4m3_kernel<TM, TN, T>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
            return fail(PHONLP_ERR_LAUNCH, "linear_e4m3: hipFuncSetAttribute failed");
        once.mark(dev);
    }
    a.num_m = ceil_div(a.M, TM);
    a.num_n = ceil_div(a.N, TN);
    hipLaunchKernelGGL((linear_e4m3_kernel<TM, TN, T>), dim3(tile_grid(a.num_m, a.num_n, 1)), dim3(512), bytes, st, a);
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
    E4m3Args a = {(const uint8_t *)x_codes, x_exponents, (const uint8_t *)w_codes, w_exponents, bias, y, (uint8_t *)bits, M, N, kp8_of(K),
                  kb4_of(K), 0, 0, relu, ceil_div(N, 32) * 4};
    hipStream_t st = as_stream(stream);
    ProfScope ps("linear_e4m3", st);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        // tiles of 128 x 128 would leave most compute units without work
        if ((long)ceil_div(M, 32) * ceil_div(N, 32) <= 1024 && M <= 32 * 65535) {
            hipLaunchKernelGGL((linear_e4m3_few_kernel<T>), dim3(ceil_div(N, 32), ceil_div(M, 32)), dim3(512), 0, st, a);
            return check_launch("linear_e4m3_few_kernel");
        }
        if ((long)ceil_div(M, 256) * ceil_div(N, 256) >= 256) return launch_tile<256, 256, T>(a, st);
        return launch_tile<128, 128, T>(a, st);
    });
}
