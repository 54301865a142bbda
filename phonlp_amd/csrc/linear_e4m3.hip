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
// A workgroup takes tile after tile (PERSIST): behind a tile's last block come the next tile's first two, so that they land while the
// results are written, and the first wait behind the results lets their stores go on.
// Four blocks' exponents of a row are one dword, brought with every fourth block into a ring of four LDS slots; the bias comes into
// LDS with a tile's first block.
//
// LDS image of a block: row r at r * 128, its 16-byte chunk c at slot c ^ ((r >> 1) & 7): sixteen rows' chunks c lie in all 64 banks.
template <int TM, int TN, class T>
struct E4m3Tile {
    static constexpr bool PIPE8 = sizeof(T) == 2;  // which matrix pipe (above)
    static constexpr int ROWS = TM + TN, SIZE = ROWS * 128, SLOTS = 4 * ROWS * 4, PATCH = 2048;
    // not the smaller tile, which shares a compute unit with a second workgroup, nor the bf16 pipe, whose registers are all in use
    static constexpr bool PERSIST = TM == 256 && PIPE8;
    static constexpr int BIAS = 2 * TN * 4, BYTES = 2 * SIZE + SLOTS + BIAS + (PERSIST ? 8 * PATCH : 0);
    static constexpr int STORES = (TM / 4) * (TN / 2) * (int)sizeof(T) / 1024;  // of a wave, for a whole tile without bits
};

template <int TM, int TN, class T>
__global__ __launch_bounds__(512) void linear_e4m3_kernel(E4m3Args a) {
    using Tile = E4m3Tile<TM, TN, T>;
    constexpr bool PIPE8 = Tile::PIPE8, PERSIST = Tile::PERSIST;
    constexpr int ROWS = Tile::ROWS, SIZE = Tile::SIZE, SIDE = PIPE8 ? 32 : 16, FA = TM / 4 / SIDE, FB = TN / 2 / SIDE, LOADS = ROWS / 64;
    extern __shared__ uint8_t lds[];  // [2][ROWS][128] codes, [4][ROWS] exponents, [2][TN] bias, the waves' output patches (or in the codes' place)
    uint8_t *slots = lds + 2 * SIZE, *biases = slots + Tile::SLOTS;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = wave >> 1, wn = wave & 1, ls = lane & (SIDE - 1), lg = lane / SIDE;
    const int blocks = a.Kp / 128, groups = a.KB4 / 4;

    struct Place {  // a tile's first row and column
        int m, n;
    };
    auto place = [&](int bid, Place &t) {
        int tm, tn, split;
        if (!tile_of(bid, a.num_m, a.num_n, 1, 8, &tm, &tn, &split)) return false;
        t.m = tm * TM;
        t.n = tn * TN;
        return true;
    };
    int bid = blockIdx.x;
    Place now, next;
    if (!place(bid, now)) return;

    // Where a tile's block kb is loaded from; rows behind the matrix read its last one: their products are not stored.
    struct From {
        const uint8_t *x, *w, *xe, *we;
        uint32_t last_x, last_w;  // byte offsets of the last rows
        int last_m, last_n;
    };
    auto from = [&](const Place &t, int kb) {
        From f;
        f.x = a.x + (long)t.m * a.Kp + kb * 128;
        f.w = a.w + (long)t.n * a.Kp + kb * 128;
        f.xe = a.xe + (long)t.m * a.KB4 + (kb >> 2) * 4;
        f.we = a.we + (long)t.n * a.KB4 + (kb >> 2) * 4;
        f.last_m = min(TM, a.M - t.m) - 1;
        f.last_n = min(TN, a.N - t.n) - 1;
        f.last_x = (uint32_t)f.last_m * (uint32_t)a.Kp;
        f.last_w = (uint32_t)f.last_n * (uint32_t)a.Kp;
        return f;
    };
    // load k of a block: rows 8 (wave + 8 k) + lane / 8
    const uint32_t row0 = (uint32_t)(wave * 8 + (lane >> 3)) * (uint32_t)a.Kp, chunk = ((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7)) << 4;
    auto load = [&](const From &f, int buf, int k) {
        const bool w = k >= TM / 64;
        const uint32_t row = row0 + (uint32_t)(w ? k - TM / 64 : k) * 64u * (uint32_t)a.Kp;
        dma16(w ? f.w : f.x, min(row, w ? f.last_w : f.last_x) + chunk, lds + buf * SIZE + (wave + k * 8) * 1024);
    };
    // the exponents of its group, of the eighth of the tile's rows that this wave brings
    auto load_exponents = [&](const From &f, int slot, bool on) {
        static_assert(TM == TN, "both operands' rows alike");
        constexpr int each = TM / 8;
#pragma unroll
        for (int w = 0; w < 2; ++w)
            dma4(w ? f.we : f.xe, (uint32_t)min(wave * each + lane, w ? f.last_n : f.last_m) * (uint32_t)a.KB4,
                 slots + ((slot & 3) * ROWS + w * TM + wave * each) * 4, on ? (1ull << each) - 1 : 0ull);
    };

    auto load_bias = [&](const Place &t, int which, bool on) {
        constexpr int each = TN / 8;
        dma4((const uint8_t *)(a.bias + t.n), (uint32_t)min(wave * each + lane, min(TN, a.N - t.n) - 1) * 4u,
             biases + (which * TN + wave * each) * 4, on && a.bias ? (1ull << each) - 1 : 0ull);
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
    auto read_a = [&](int buf, int p, int i, A &x) {
#pragma unroll
        for (int h = 0; h < H; ++h) x.f[i][h] = *reinterpret_cast<const i32x4 *>(lds + buf * SIZE + at_a[p][h] + i * SIDE * 128);
    };
    auto read_b = [&](int buf, int p, int j) {
#pragma unroll
        for (int h = 0; h < H; ++h) b[j][h] = *reinterpret_cast<const i32x4 *>(lds + buf * SIZE + at_b[p][h] + j * SIDE * 128);
    };
    auto read_scales = [&](int kb, int slot, Scales &s) {  // of block kb, in the lowest byte
        const int *e = reinterpret_cast<const int *>(slots) + (slot & 3) * ROWS + ls, shift = (kb & 3) * 8;
#pragma unroll
        for (int i = 0; i < FA; ++i) s.a[i] = (unsigned)e[wm * (TM / 4) + i * SIDE] >> shift;
#pragma unroll
        for (int j = 0; j < FB; ++j) s.b[j] = (unsigned)e[TM + wn * (TN / 2) + j * SIDE] >> shift;
    };

    typedef std::conditional_t<PIPE8, f32x16, f32x4> Acc;
    Acc acc[FA][FB];
    int buf = 0, slot = 0, which = 0;  // of the block at hand; of this tile's first group; of its bias

    // Part p of block kb: its codes are in `now_a` and b; loads, and LDS reads of the next part's codes into registers that are done
    // with, stand between its matrix instructions.
    auto part = [&](int kb, auto pc, A &now_a, A &next_a, const Scales &s) {
        constexpr int p = decltype(pc)::value;
        const int nbuf = buf ^ p;  // the next part: 1 - p of this block or the next
        const bool here = kb + 2 < blocks;  // block kb + 2, or the next tile's
        const int v = here ? kb + 2 : min(kb + 2 - blocks, blocks - 1);
        From f;
        if (p == 1) f = from(Place{here ? now.m : next.m, here ? now.n : next.n}, v);
        auto loads = [&](int z, int of) {  // the share of step z of `of`
            if (p == 0) return;
#pragma unroll
            for (int k = LOADS * z / of; k < LOADS * (z + 1) / of; ++k) load(f, buf, k);
            if (z == of - 1) {
                load_exponents(f, slot + (here ? 0 : groups) + (v >> 2), (v & 3) == 0);
                if (PERSIST) load_bias(next, which ^ 1, !here && v == 0);
            }
        };
        if constexpr (PIPE8) {
#pragma unroll
            for (int j = 0; j < FB; ++j) {
                loads(j, FB);
                if (j == 0) {
#pragma unroll
                    for (int i = 0; i < FA; ++i) read_a(nbuf, 1 - p, i, next_a);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i < FA; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
                        __builtin_shufflevector(b[j][0], b[j][1], 0, 1, 2, 3, 4, 5, 6, 7),
                        __builtin_shufflevector(now_a.f[i][0], now_a.f[i][1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, 0, s.b[j], 0, s.a[i]);
                __builtin_amdgcn_sched_barrier(0);
                read_b(nbuf, 1 - p, j);
            }
        } else {
            constexpr int HB = FB / 2, STEPS = 4 * FA;  // half of B's fragments at a time: registers
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                bf16x8 fa[FA];
#pragma unroll
                for (int i = 0; i < FA; ++i) fa[i] = widen(now_a.f[i][0][2 * q], now_a.f[i][0][2 * q + 1], scale_of(s.a[i]));
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
                        for (int k = 0; k < HB; ++k) read_b(nbuf, 1 - p, jh * HB + k);
                        if (jh == 0) {
#pragma unroll
                            for (int k = 0; k < FA; ++k) read_a(nbuf, 1 - p, k, next_a);
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
    using first_part = std::integral_constant<int, 0>;
    using second_part = std::integral_constant<int, 1>;

    {
        const From f = from(now, 0);
#pragma unroll
        for (int k = 0; k < LOADS; ++k) load(f, 0, k);
        load_exponents(f, 0, true);
        load_bias(now, 0, true);
    }
    dma_wait_barrier<0>();
    bool more = PERSIST && place(bid + gridDim.x, next), whole = false;
    if (!more) next = now;
    {
        const From f = from(blocks > 1 ? now : next, blocks > 1 ? 1 : 0);
#pragma unroll
        for (int k = 0; k < LOADS; ++k) load(f, 1, k);
        load_exponents(f, groups, blocks == 1);
    }
    A a0, a1;
    Scales s;
#pragma unroll
    for (int i = 0; i < FA; ++i) read_a(0, 0, i, a0);
#pragma unroll
    for (int j = 0; j < FB; ++j) read_b(0, 0, j);
    read_scales(0, 0, s);
    while (true) {
#pragma unroll
        for (int i = 0; i < FA; ++i)
#pragma unroll
            for (int j = 0; j < FB; ++j)
#pragma unroll
                for (int r = 0; r < SIDE * SIDE / 64; ++r) acc[i][j][r] = 0.f;
        auto block = [&](int kb, auto pc) {
            constexpr bool first = decltype(pc)::value;
            part(kb, first_part{}, a0, PIPE8 ? a1 : a0, s);
            // behind a whole tile's results the loads of block 1 are older than exactly its stores
            if (first && whole) dma_wait_barrier<Tile::STORES>();
            else dma_wait_barrier<0>();
            part(kb, second_part{}, PIPE8 ? a1 : a0, a0, s);
            buf ^= 1;
            const int v = kb + 1 < blocks ? kb + 1 : 0;
            read_scales(v, slot + (kb + 1 < blocks ? 0 : groups) + (v >> 2), s);  // landed with block kb + 1
        };
        if (PERSIST) block(0, std::true_type{});
        for (int kb = PERSIST; kb < blocks; ++kb) block(kb, std::false_type{});
        slot += groups;

        // Through LDS, a patch of a wave's own, so that Y is written in row segments of 64 (16-bit) or 128 bytes, a row's one after the
        // other: lines that two segments share are then whole before they leave L2 (32768 x 2447 x 868 fp32 178 us, all rows of a segment
        // first 209; 16384 x 8192 x 4096 bf16 456 against 476).
        if (!PERSIST) dma_wait_barrier<0>();  // the patches take the codes' place
        whole = now.m + TM <= a.M && now.n + TN <= a.N;
        uint8_t *patch = (PERSIST ? biases + Tile::BIAS : lds) + wave * Tile::PATCH;
        constexpr int VEC = 16 / sizeof(T), LANES = 32 / VEC, ROWB = 32 * sizeof(T), JJ = 32 / SIDE;
        auto swizzle = [](int r, int c) { return r * ROWB + ((sizeof(T) == 2 ? c ^ ((r >> 2) & 3) : c ^ ((r >> 1) & 7)) << 4); };
        constexpr int QUADS = SIDE * SIDE * JJ / 256;
#pragma unroll
        for (int i = 0; i < FA; ++i) {
            const int mw = now.m + wm * (TM / 4) + i * SIDE;
#pragma unroll
            for (int jq = 0; jq < FB / JJ; ++jq) {
                const int nw = now.n + wn * (TN / 2) + jq * 32;
                f32x4 bias[QUADS];  // of four neighbouring columns
#pragma unroll
                for (int q = 0; q < QUADS; ++q) {
                    bias[q] = f32x4{0.f, 0.f, 0.f, 0.f};
                    const int c = wn * (TN / 2) + jq * 32 + (PIPE8 ? 8 * q : 16 * q) + 4 * lg;
                    if (a.bias) bias[q] = *reinterpret_cast<const f32x4 *>(biases + (which * TN + c) * 4);
                }
#pragma unroll
                for (int q = 0; q < QUADS; ++q) {  // four neighbouring columns of row ls
                    const int c = (PIPE8 ? 8 * q : 16 * q) + 4 * lg, j = jq * JJ + (PIPE8 ? 0 : q), r = PIPE8 ? 4 * q : 0;
                    const f32x4 v = {acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]};
                    *reinterpret_cast<typename Vec<T, 4>::type *>(patch + swizzle(ls, c / VEC) + (c % VEC) * sizeof(T)) =
                        finish<T>(v, bias[q], a.relu);
                }
                __builtin_amdgcn_wave_barrier();
#pragma unroll
                for (int r0 = 0; r0 < SIDE; r0 += 64 / LANES) {
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
        if (!more) break;
        whole = whole && !a.bits;
        now = next;
        which ^= 1;
        bid += gridDim.x;
        more = place(bid + gridDim.x, next);
        if (!more) next = now;
    }
    dma_wait<0>();  // the repeated loads still write this workgroup's LDS
}

// Few rows: straight from memory to registers, the next block's codes on their way while one is multiplied.  A workgroup takes 16 MF rows
// of Y and 8 / KS groups of 32 columns; KS waves of a group take every KS-th block each, and their sums are added in a fixed order.  Bound
// by reading W, or by latency.  Always the bf16 pipe.
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
    using Tile = E4m3Tile<TM, TN, T>;
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
    int grid = tile_grid(a.num_m, a.num_n, 1);
    // one workgroup per compute unit; the loads look two blocks ahead, into the next tile alone, so a tile needs two
    if (Tile::PERSIST && a.Kp >= 256 && grid > 256) grid = 256;
    hipLaunchKernelGGL((linear_e4m3_kernel<TM, TN, T>), dim3(grid), dim3(512), Tile::BYTES, st, a);
    return check_launch("linear_e4m3_kernel");
}

// The tile with the least estimated time.  A tile takes so much per block and so much at its ends (us, measured on products of 128 to
// 4096 columns, 512 to 65536 rows): 256 x 256, a workgroup per compute unit, in whole rounds; 128 x 128, two workgroups per compute unit,
// whose ends fall into each other's blocks.  16-bit results: 16384 x 8192 x 4096 475 against 572 us, 8192 x 2448 x 868 35.6 against
// 28.2, 2011 x 13464 x 408 29.6 against 27.3; fp32: 810 against 970, 62.8 against 46.2, 50 against 42.
template <class T>
static bool large_tile(int M, int N, int Kp) {
    constexpr bool f32 = sizeof(T) == 4;
    const int blocks = Kp / 128;
    const double large = (double)ceil_div(M, 256) * ceil_div(N, 256) / 256., small = (double)ceil_div(M, 128) * ceil_div(N, 128) / 512. + 0.25;
    return (double)(long)(large + 0.999) * ((f32 ? 2.5 : 1.58) * blocks + (f32 ? 18. : 9.)) <
           small * ((f32 ? 1.7 : 0.98) * blocks + (f32 ? 6.5 : 4.3));
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
        // Up to sixteen rows, one token's among them, W is read once, at most of memory's rate: 1 x 64000 x 768 10.7 us (fp32 tiles of 128 x
        // 128 18.9, 16-bit 12.3; 4.6 TB/s), 1 x 8192 x 8192 18 (60; 40), 1 x 28672 x 4096 26.5 (38.5; 24.8).  Two waves of a group where
        // there are many groups: 10.7 against 12.3 with eight; 1 x 13464 x 4096 26 against 16.
        if (M <= 16) return ceil_div(N, 32) > 640 ? launch_few<1, 2, T>(a, st) : launch_few<1, 8, T>(a, st);
        // Of more rows, up to so many 32 x 32 the few-row form is the faster one; tiles of 128 x 128 would leave most compute units without
        // work (fp32: 256 x 868 x 868 6.4 against 10.9 us, 256 x 2448 x 868, 616 of them, 10.8 against 11.3, 2048 x 400 x 768, 832, 11.9
        // against 10.6; 16-bit: 256 x 868 x 868 6.3 against 7.3, 128 x 2448 x 868, 308, 8.0 against 7.2)
        if ((long)ceil_div(M, 32) * ceil_div(N, 32) <= (sizeof(T) == 4 ? 640 : 256)) return launch_few<2, 8, T>(a, st);
        if (large_tile<T>(M, N, a.Kp)) return launch_tile<256, 256, T>(a, st);
        return launch_tile<128, 128, T>(a, st);
    });
}
