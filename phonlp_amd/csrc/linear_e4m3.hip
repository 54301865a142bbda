// Dense layer on e4m3 images (e4m3.h):  Y[m][n] = act(sum_k X^[m][k] W^[n][k] + bias[n]),  X^ / W^ the values of the images.
//
// Products on v_mfma_f32_16x16x32_bf16, whatever the result's type: the values of an image are exact in bf16, converted with their scale
// from the codes as those leave LDS (v_cvt_scalef32_pk_bf16_fp8, two codes each), every product is exact and the sums are fp32
// throughout (what an operand has below 2^-133, bf16's smallest step, is lost).  The 8-bit pipe, v_mfma_scale_f32_32x32x64_f8f6f4, would
// be up to twice as fast, but adds eight products at a time, each cut off 13 bits below the largest of the eight (measured: 2^16 + 2^2
// loses the small one): where large products cancel, what is left of the result is lost, whatever its type.
// Both operands are K-contiguous and an instruction's K order is free (A and B share it).
#include <type_traits>

#include "e4m3.h"
#include "lds_dma.h"

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
__device__ __forceinline__ typename Vec<T, 4>::type finish(f32x4 v, const f32x4 &bias, int relu) {
    typename Vec<T, 4>::type t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x = v[i] + bias[i];
        if (relu) x = x < 0.f ? 0.f : x;  // keeps NaN
        t[i] = (T)x;
    }
    return t;
}

// Tile of TM x TN, eight waves (4 x 2) of TM / 4 x TN / 2.  A block of 128 codes of every row comes by LDS-DMA in whole 128-byte lines
// into one of two buffers, and goes through registers in two parts of 64.  The codes of a part are read from LDS while the part
// before is multiplied, so one barrier a block, before its second part, does: there block kb + 1 has landed, and as every wave
// has all of block kb in registers, its buffer takes block kb + 2, a whole block's time ahead.
// Four blocks' exponents of a row are one dword, brought with every fourth block into a ring of four LDS slots; the bias comes into
// LDS with the first block.
//
// LDS image of a block: row r at r * 128, its 16-byte chunk c at slot c ^ ((r >> 1) & 7): sixteen rows' chunks c lie in all 64 banks.
template <int TM, int TN>
struct E4m3Tile {
    static constexpr int ROWS = TM + TN, SIZE = ROWS * 128, SLOTS = 4 * ROWS * 4, PATCH = 2048;
    static constexpr int BIAS = TN * 4, BYTES = 2 * SIZE + SLOTS + BIAS;
    static_assert(8 * PATCH <= SIZE, "the patches take the codes' place");
};

template <int TM, int TN, class T>
__global__ __launch_bounds__(512) void linear_e4m3_kernel(E4m3Args a) {
    using Tile = E4m3Tile<TM, TN>;
    constexpr int ROWS = Tile::ROWS, SIZE = Tile::SIZE, FA = TM / 4 / 16, FB = TN / 2 / 16, LOADS = ROWS / 64;
    extern __shared__ uint8_t lds[];  // [2][ROWS][128] codes, [4][ROWS] exponents, [TN] bias; at the end the waves' output patches
    uint8_t *slots = lds + 2 * SIZE, *biases = slots + Tile::SLOTS;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave >> 1, wn = wave & 1, ls = lane & 15, lg = lane >> 4;
    const int blocks = a.Kp / 128;
    int tm, tn, split;
    if (!tile_of(blockIdx.x, a.num_m, a.num_n, 1, 8, &tm, &tn, &split)) return;
    const int m0 = tm * TM, n0 = tn * TN;

    // Where block kb is loaded from; rows behind the matrix read its last one: their products are not stored.
    const int last_m = min(TM, a.M - m0) - 1, last_n = min(TN, a.N - n0) - 1;
    const uint32_t last_x = (uint32_t)last_m * (uint32_t)a.Kp, last_w = (uint32_t)last_n * (uint32_t)a.Kp;  // byte offsets of the last rows
    const uint8_t *x = a.x + (long)m0 * a.Kp, *w = a.w + (long)n0 * a.Kp, *xe = a.xe + (long)m0 * a.KB4, *we = a.we + (long)n0 * a.KB4;
    // load k of a block: rows 8 (wave + 8 k) + lane / 8
    const uint32_t row0 = (uint32_t)(wave * 8 + (lane >> 3)) * (uint32_t)a.Kp, chunk = ((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7)) << 4;
    auto load = [&](int kb, int buf, int k) {
        const bool of_w = k >= TM / 64;
        const uint32_t row = row0 + (uint32_t)(of_w ? k - TM / 64 : k) * 64u * (uint32_t)a.Kp;
        dma16((of_w ? w : x) + kb * 128, min(row, of_w ? last_w : last_x) + chunk, lds + buf * SIZE + (wave + k * 8) * 1024);
    };
    // the exponents of block kb's group, of the eighth of the tile's rows that this wave brings
    auto load_exponents = [&](int kb, bool on) {
        static_assert(TM == TN, "both operands' rows alike");
        constexpr int each = TM / 8;
#pragma unroll
        for (int of_w = 0; of_w < 2; ++of_w)
            dma4((of_w ? we : xe) + (kb >> 2) * 4, (uint32_t)min(wave * each + lane, of_w ? last_n : last_m) * (uint32_t)a.KB4,
                 slots + ((kb >> 2 & 3) * ROWS + of_w * TM + wave * each) * 4, on ? (1ull << each) - 1 : 0ull);
    };
    auto load_bias = [&] {
        constexpr int each = TN / 8;
        dma4((const uint8_t *)(a.bias + n0), (uint32_t)min(wave * each + lane, last_n) * 4u, biases + wave * each * 4,
             a.bias ? (1ull << each) - 1 : 0ull);
    };

    // lane (ls, lg) holds row ls of a fragment: of a part's 64 codes 16 from 16 lg, eight for each of two steps; fragments are multiples of
    // 16 rows apart, which do not change the slot
    int at_a[2], at_b[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
        const int slot = ((p * 4 + lg) ^ ((ls >> 1) & 7)) << 4;
        at_a[p] = (wm * (TM / 4) + ls) * 128 + slot;
        at_b[p] = (TM + wn * (TN / 2) + ls) * 128 + slot;
    }
    i32x4 ca[FA], cb[FB];
    struct Scales {
        int a[FA], b[FB];
    };
    auto read_a = [&](int buf, int p, int i) { ca[i] = *reinterpret_cast<const i32x4 *>(lds + buf * SIZE + at_a[p] + i * 16 * 128); };
    auto read_b = [&](int buf, int p, int j) { cb[j] = *reinterpret_cast<const i32x4 *>(lds + buf * SIZE + at_b[p] + j * 16 * 128); };
    auto read_scales = [&](int kb, Scales &s) {  // of block kb, in the lowest byte
        const int *e = reinterpret_cast<const int *>(slots) + (kb >> 2 & 3) * ROWS + ls, shift = (kb & 3) * 8;
#pragma unroll
        for (int i = 0; i < FA; ++i) s.a[i] = (unsigned)e[wm * (TM / 4) + i * 16] >> shift;
#pragma unroll
        for (int j = 0; j < FB; ++j) s.b[j] = (unsigned)e[TM + wn * (TN / 2) + j * 16] >> shift;
    };

    f32x4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Part p of block kb: its codes are in ca and cb; loads, and LDS reads of the next part's codes into registers that are done with,
    // stand between its matrix instructions.  Behind the end the last block is loaded and read again.
    auto part = [&](int kb, auto pc, const Scales &s) {
        constexpr int p = decltype(pc)::value;
        const int buf = kb & 1, nbuf = buf ^ p;  // the next part: 1 - p of this block or the next
        const int ahead = min(kb + 2, blocks - 1);
        auto loads = [&](int z, int of) {  // the share of step z of `of`
            if (p == 0) return;
#pragma unroll
            for (int k = LOADS * z / of; k < LOADS * (z + 1) / of; ++k) load(ahead, buf, k);
            if (z == of - 1) load_exponents(ahead, kb + 2 < blocks && (ahead & 3) == 0);
        };
        constexpr int HB = FB / 2, STEPS = 4 * FA;  // half of B's fragments at a time: registers
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            bf16x8 fa[FA];
#pragma unroll
            for (int i = 0; i < FA; ++i) fa[i] = widen(ca[i][2 * q], ca[i][2 * q + 1], scale_of(s.a[i]));
#pragma unroll
            for (int jh = 0; jh < 2; ++jh) {
                bf16x8 fb[HB];
#pragma unroll
                for (int j = 0; j < HB; ++j) {
                    const i32x4 &c = cb[jh * HB + j];
                    fb[j] = widen(c[2 * q], c[2 * q + 1], scale_of(s.b[jh * HB + j]));
                }
                if (q == 1) {  // these codes of this part are used up
#pragma unroll
                    for (int k = 0; k < HB; ++k) read_b(nbuf, 1 - p, jh * HB + k);
                    if (jh == 0) {
#pragma unroll
                        for (int k = 0; k < FA; ++k) read_a(nbuf, 1 - p, k);
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
    };
    using first_part = std::integral_constant<int, 0>;
    using second_part = std::integral_constant<int, 1>;

#pragma unroll
    for (int k = 0; k < LOADS; ++k) load(0, 0, k);
    load_exponents(0, true);
    load_bias();
    dma_wait_barrier<0>();
#pragma unroll
    for (int k = 0; k < LOADS; ++k) load(min(1, blocks - 1), 1, k);
    Scales s;
#pragma unroll
    for (int i = 0; i < FA; ++i) read_a(0, 0, i);
#pragma unroll
    for (int j = 0; j < FB; ++j) read_b(0, 0, j);
    read_scales(0, s);
    for (int kb = 0; kb < blocks; ++kb) {
        part(kb, first_part{}, s);
        dma_wait_barrier<0>();
        part(kb, second_part{}, s);
        read_scales(min(kb + 1, blocks - 1), s);  // landed with the block
    }

    // Through LDS, a patch of a wave's own, so that Y is written in row segments of 64 (16-bit) or 128 bytes, a row's one after the
    // other: lines that two segments share are then whole before they leave L2 (32768 x 2447 x 868 fp32 178 us, all rows of a segment
    // first 209).
    dma_wait_barrier<0>();  // the repeated loads still write this workgroup's LDS
    uint8_t *patch = lds + wave * Tile::PATCH;
    constexpr int VEC = 16 / sizeof(T), LANES = 32 / VEC, ROWB = 32 * sizeof(T);
    auto swizzle = [](int r, int c) { return r * ROWB + ((sizeof(T) == 2 ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7)) << 4); };
#pragma unroll
    for (int i = 0; i < FA; ++i) {
        const int mw = m0 + wm * (TM / 4) + i * 16;
#pragma unroll
        for (int jq = 0; jq < FB / 2; ++jq) {
            const int nw = n0 + wn * (TN / 2) + jq * 32;
#pragma unroll
            for (int q = 0; q < 2; ++q) {  // four neighbouring columns of row ls
                const int c = 16 * q + 4 * lg;
                f32x4 bias = {0.f, 0.f, 0.f, 0.f};
                if (a.bias) bias = *reinterpret_cast<const f32x4 *>(biases + (wn * (TN / 2) + jq * 32 + c) * 4);
                *reinterpret_cast<typename Vec<T, 4>::type *>(patch + swizzle(ls, c / VEC) + (c % VEC) * sizeof(T)) =
                    finish<T>(acc[i][jq * 2 + q], bias, a.relu);
            }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int r0 = 0; r0 < 16; r0 += 64 / LANES) {
                const int r = r0 + lane / LANES, c = lane % LANES, m = mw + r, n = nw + c * VEC;
                if (m >= a.M) continue;
                const T *from = reinterpret_cast<const T *>(patch + swizzle(r, c));
                T *to = (T *)a.y + (long)m * a.N + n;
                const auto v = *reinterpret_cast<const typename Vec<T, VEC>::type *>(from);
                const int left = a.N - n;
                if (left >= VEC) *reinterpret_cast<typename Vec<T, VEC>::type *>(to) = v;
                else
#pragma unroll 1
                    for (int k = 0; k < left; ++k) to[k] = from[k];
                if (a.bits) {
                    int bits = 0;
#pragma unroll
                    for (int k = 0; k < VEC; ++k) bits |= (float)v[k] > 0.f ? 1 << k : 0;
                    if (left < VEC) bits &= (1 << max(left, 0)) - 1;
                    if (VEC == 4) bits |= __shfl_down(bits, 1) << 4;  // a byte is two lanes' four columns
                    if ((VEC == 8 || !(c & 1)) && (n >> 3) < a.row_bytes) a.bits[(long)m * a.row_bytes + (n >> 3)] = (uint8_t)bits;
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// Few rows: straight from memory to registers, the next block's codes on their way while one is multiplied.  A workgroup takes 16 MF rows
// of Y and 8 / KS groups of 32 columns; KS waves of a group take every KS-th block each, and their sums are added in a fixed order.  Bound
// by reading W, or by latency.
template <int MF, int KS, class T>
__global__ __launch_bounds__(512) void linear_e4m3_few_kernel(E4m3Args a) {
    constexpr int GROUPS = 8 / KS;
    __shared__ float sums[8][MF * 16][33];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (32 * GROUPS), m0 = blockIdx.y * (16 * MF), blocks = a.Kp / 128, nw = n0 + wave / KS * 32;
    f32x4 acc[MF][2];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    long xr[MF], wr[2];
#pragma unroll
    for (int i = 0; i < MF; ++i) xr[i] = min(m0 + i * 16 + l16, a.M - 1);
#pragma unroll
    for (int j = 0; j < 2; ++j) wr[j] = min(nw + j * 16 + l16, a.N - 1);
    struct Block {  // 32 codes of a row per lane, from 32 g
        i32x4 x[MF][2], w[2][2];
        int ex[MF], ew[2];
    };
    auto load = [&](int kb, Block &b) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int j = 0; j < 2; ++j) b.w[j][h] = *reinterpret_cast<const i32x4 *>(a.w + wr[j] * a.Kp + kb * 128 + g * 32 + h * 16);
#pragma unroll
            for (int i = 0; i < MF; ++i) b.x[i][h] = *reinterpret_cast<const i32x4 *>(a.x + xr[i] * a.Kp + kb * 128 + g * 32 + h * 16);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) b.ew[j] = a.we[wr[j] * a.KB4 + kb];
#pragma unroll
        for (int i = 0; i < MF; ++i) b.ex[i] = a.xe[xr[i] * a.KB4 + kb];
    };
    auto multiply = [&](const Block &b) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                bf16x8 fx[MF], fw[2];
#pragma unroll
                for (int i = 0; i < MF; ++i) fx[i] = widen(b.x[i][h][2 * q], b.x[i][h][2 * q + 1], scale_of(b.ex[i]));
#pragma unroll
                for (int j = 0; j < 2; ++j) fw[j] = widen(b.w[j][h][2 * q], b.w[j][h][2 * q + 1], scale_of(b.ew[j]));
#pragma unroll
                for (int i = 0; i < MF; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fx[i], fw[j], acc[i][j], 0, 0, 0);
            }
    };
    const int first = wave % KS;
    if (first < blocks && nw < a.N) {
        Block b0, b1;
        load(first, b0);
        for (int kb = first; kb < blocks; kb += 2 * KS) {  // two blocks a turn, so that each stands where it is
            load(min(kb + KS, blocks - 1), b1);
            multiply(b0);
            if (kb + KS >= blocks) break;
            load(min(kb + 2 * KS, blocks - 1), b0);
            multiply(b1);
        }
    }
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][i * 16 + g * 4 + r][j * 16 + l16] = acc[i][j][r];
    __syncthreads();
    // eight columns of a row a thread: a byte of bits is one thread's
    if (threadIdx.x >= MF * 16 * 4 * GROUPS) return;
    const int u = threadIdx.x % (4 * GROUPS), group = u >> 2, r = threadIdx.x / (4 * GROUPS), c = (u & 3) * 8, m = m0 + r, nc = n0 + group * 32 + c,
              waves = min(KS, blocks);
    if (m >= a.M) return;
    int b = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        const int n = nc + k;
        if (n >= a.N) continue;
        float v = 0.f;
        for (int w = 0; w < waves; ++w) v += sums[group * KS + w][r][c + k];
        if (a.bias) v += a.bias[n];
        if (a.relu) v = v < 0.f ? 0.f : v;  // keeps NaN
        const T t = (T)v;
        ((T *)a.y)[(long)m * a.N + n] = t;
        b |= (float)t > 0.f ? 1 << k : 0;
    }
    if (a.bits && nc >> 3 < a.row_bytes) a.bits[(long)m * a.row_bytes + (nc >> 3)] = (uint8_t)b;
}

template <int MF, int KS, class T>
static int launch_few(const E4m3Args &a, hipStream_t st) {
    hipLaunchKernelGGL((linear_e4m3_few_kernel<MF, KS, T>), dim3(ceil_div(a.N, 256 / KS), ceil_div(a.M, 16 * MF)), dim3(512), 0, st, a);
    return check_launch("linear_e4m3_few_kernel");
}

template <int TM, int TN, class T>
static int launch_tile(E4m3Args a, hipStream_t st) {
    using Tile = E4m3Tile<TM, TN>;
    static PerDeviceOnce once;
    int dev;
    if (once.pending(&dev)) {
        if (hipFuncSetAttribute((const void *)linear_e4m3_kernel<TM, TN, T>, hipFuncAttributeMaxDynamicSharedMemorySize, Tile::BYTES) !=
            hipSuccess)
            return fail(PHONLP_ERR_LAUNCH, "linear_e4m3: hipFuncSetAttribute failed");
        once.mark(dev);
    }
    a.num_m = ceil_div(a.M, TM);
    a.num_n = ceil_div(a.N, TN);
    hipLaunchKernelGGL((linear_e4m3_kernel<TM, TN, T>), dim3(tile_grid(a.num_m, a.num_n, 1)), dim3(512), Tile::BYTES, st, a);
    return check_launch("linear_e4m3_kernel");
}

// The tile with the least estimated time.  A tile takes so much per block and so much at its ends (us, measured on products of 128 to
// 4096 columns, 512 to 65536 rows): 256 x 256, a workgroup per compute unit, in whole rounds; 128 x 128, two workgroups per compute unit,
// whose ends fall into each other's blocks.  16-bit results: 16384 x 8192 x 4096 789 against 949 us, 8192 x 2448 x 868 54
// against 41, 2011 x 13464 x 408 40 against 37, 16384 x 4096 x 128 54 against 46; fp32: 826 against 986, 62 against 46, 47.5 against 43, 61
// against 62.
template <class T>
static bool large_tile(int M, int N, int Kp) {
    constexpr bool f32 = sizeof(T) == 4;
    const int blocks = Kp / 128;
    const double large = (double)ceil_div(M, 256) * ceil_div(N, 256) / 256., small = (double)ceil_div(M, 128) * ceil_div(N, 128) / 512. + 0.25;
    return (double)(long)(large + 0.999) * ((f32 ? 2.5 : 2.6) * blocks + (f32 ? 18. : 10.7)) <
           small * ((f32 ? 1.7 : 1.73) * blocks + (f32 ? 6.5 : 4.));
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
    // a grid holds less than 2^32 threads
    if ((M + 127L) / 128 * ((N + 127L) / 128) >= 1 << 23) return fail(PHONLP_ERR_UNSUPPORTED, "linear_e4m3: M * N too large");
    E4m3Args a = {(const uint8_t *)x_codes, x_exponents, (const uint8_t *)w_codes, w_exponents, bias, y, (uint8_t *)bits, M, N, kp8_of(K),
                  kb4_of(K), 0, 0, relu, ceil_div(N, 32) * 4};
    hipStream_t st = as_stream(stream);
    ProfScope ps("linear_e4m3", st);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        // Up to sixteen rows, one token's among them, W is read once, at most of memory's rate: 1 x 64000 x 768 10.7 us (tiles of 128 x 128
        // 16.5; 4.6 TB/s), 1 x 8192 x 8192 18 (61), 1 x 28672 x 4096 26.5 (36).  Two waves of a group where
        // there are many groups: 10.7 against 12.3 with eight; 1 x 13464 x 4096 26 against 16.
        if (M <= 16) return ceil_div(N, 32) > 640 ? launch_few<1, 2, T>(a, st) : launch_few<1, 8, T>(a, st);
        // Of more rows, up to so many 32 x 32 the few-row form is the faster one; tiles of 128 x 128 would leave most compute units without
        // work (fp32: 256 x 868 x 868 6.4 against 10.9 us, 256 x 2448 x 868, 616 of them, 10.8 against 11.3, 2048 x 400 x 768, 832, 11.9
        // against 10.6; 16-bit: 512 x 868 x 868, 448, 8.3 against 10.4, 256 x 2448 x 868 11.4 against 10.2)
        if ((long)ceil_div(M, 32) * ceil_div(N, 32) <= (sizeof(T) == 4 ? 640 : 512)) return launch_few<2, 8, T>(a, st);
        if (large_tile<T>(M, N, a.Kp)) return launch_tile<256, 256, T>(a, st);
        return launch_tile<128, 128, T>(a, st);
    });
}
