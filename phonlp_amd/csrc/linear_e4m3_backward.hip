// Backward of the dense layer of linear_e4m3.hip from its 8-bit checkpoint (the input's image and one bit per output):
//   dZ = dY where the bit is set (ReLU) or dY;   dX = dZ W^;   dW = dZ^T X^;   db = column sums of dZ.
//
// Products on v_mfma_f32_16x16x32_bf16 (2.05 PFLOP/s in a loop of nothing else, 32x32x16 1.84).  The values of an image are exact in bf16
// (four significant bits, a power of two), and dZ is cut into bf16 pieces whose sum is dZ itself -- one for bf16, two for fp16 (11
// bits), three for fp32 (24 bits), by truncation, so no piece can round past bf16's largest --, so every product is exact and only the
// fp32 sums round.  (What an operand has below 2^-133, bf16's smallest step, is lost.)
#include <type_traits>

#include "e4m3.h"
#include "e4m3_backward.h"
#include "lds_dma.h"

namespace phonlp {

template <class T>
struct Pieces;
template <>
struct Pieces<float> { static constexpr int N = 3; };
template <>
struct Pieces<_Float16> { static constexpr int N = 2; };
template <>
struct Pieces<__bf16> { static constexpr int N = 1; };
static int pieces_of(int type) { return type == PHONLP_F32 ? 3 : type == PHONLP_F16 ? 2 : 1; }

// The first N bf16 pieces of v (bit patterns): each the rest truncated.  Infinities and NaN stand in the first piece alone.
template <int N>
__device__ __forceinline__ void cut(float v, uint16_t (&p)[N]) {
    const bool fine = (__float_as_int(v) & 0x7F800000) != 0x7F800000;
    const int nan = __float_as_int(v) | 0x400000;  // quiet: the bit that truncation keeps
    p[0] = (uint16_t)((v != v ? nan : __float_as_int(v)) >> 16);
#pragma unroll
    for (int i = 1; i < N; ++i) {
        v -= __int_as_float((int)((uint32_t)p[i - 1] << 16));
        p[i] = fine ? (uint16_t)(__float_as_int(v) >> 16) : (uint16_t)0;
    }
}

// The operands of the two products, in one launch of three kinds of blocks.
struct BwPrep {
    const void *dy;
    long lddy;
    const uint32_t *bits;
    uint16_t *planes;  // [P][Mp][Np]
    float *part;       // column sums of dz_rows rows, [blocks of rows][N]
    const uint8_t *codes[2], *exps[2];  // images of x and w
    __bf16 *wide[2];                    // their values, [rows up to a multiple of 32][Kp]
    int rows[2], wide_blocks[2];
    int words, M, N, Mp, Np, Kp, KB4, dz_rows, dz_m, dz_blocks;  // dz_rows: rows of a workgroup
};

// dY -> the pieces of dZ (zero behind M and N) and the column sums.  A workgroup takes dz_rows x 256 columns, a thread eight columns
// of every eighth row; the eight threads of a column group add in order.
template <class T>
__device__ __forceinline__ void prep_dz(const BwPrep &a, int bid, float (&sums)[8][256]) {
    constexpr int P = Pieces<T>::N;
    typedef typename Vec<T, 8>::type V;
    const int bm = bid % a.dz_m, bn = bid / a.dz_m;
    const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5, n = bn * 256 + cg * 8, m0 = bm * a.dz_rows + rl;
    float s[8] = {};
    if (n < a.Np) {
#pragma unroll 4
        for (int it = 0; it < a.dz_rows / 8; ++it) {
            const int m = m0 + it * 8;
            if (m >= a.Mp) break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            if (m < a.M) {
                const T *p = (const T *)a.dy + m * a.lddy + n;
                if (n + 8 <= a.N) {
                    const V t = *reinterpret_cast<const V *>(p);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n + i < a.N) v[i] = (float)p[i];
                }
                if (a.bits) {
                    const uint32_t b = n < a.N ? a.bits[(long)m * a.words + (n >> 5)] >> (n & 31) : 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = b >> i & 1 ? v[i] : 0.f;
                }
            }
            if (a.planes) {
                uint32_t w[P][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint16_t lo[P], hi[P];
                    cut<P>(v[2 * i], lo);
                    cut<P>(v[2 * i + 1], hi);
#pragma unroll
                    for (int q = 0; q < P; ++q) w[q][i] = lo[q] | (uint32_t)hi[q] << 16;
                }
#pragma unroll
                for (int q = 0; q < P; ++q)
                    *reinterpret_cast<uint4 *>(a.planes + ((long)q * a.Mp + m) * a.Np + n) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += v[i];
        }
    }
    if (!a.part || bm * a.dz_rows >= a.M) return;  // rows behind M, which only the planes have, make no sums
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[rl][cg * 8 + i] = s[i];
    __syncthreads();
    const int c = bn * 256 + threadIdx.x;
    if (c >= a.N) return;
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += sums[r][threadIdx.x];
    a.part[(long)bm * a.N + c] = t;
}

template <class T>
__global__ __launch_bounds__(256) void e4m3_bw_prep_kernel(BwPrep a) {
    __shared__ float sums[8][256];
    int bid = blockIdx.x;
    if (bid < a.dz_blocks) return prep_dz<T>(a, bid, sums);
    bid -= a.dz_blocks;
    // an image's values in bf16, sixteen codes per thread and turn
    const int k = bid < a.wide_blocks[0] ? 0 : 1;
    if (k) bid -= a.wide_blocks[0];
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const int per_row = a.Kp / 16, R = a.rows[k];
    const long total = (long)((R + 31) / 32 * 32) * per_row, step = a.wide_blocks[k] * 256L;
    for (long g = bid * 256L + threadIdx.x; g < total; g += step) {
        const long r = total < (1L << 31) ? (long)((unsigned)g / (unsigned)per_row) : g / per_row;
        const int c = (int)(g - r * per_row) * 16;
        i32x4 code = {0, 0, 0, 0};
        float scale = 1.f;
        if (r < R) {
            code = *reinterpret_cast<const i32x4 *>(a.codes[k] + r * a.Kp + c);
            scale = exp2_biased(a.exps[k][r * a.KB4 + (c >> 7)]);
        }
        int w[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            w[2 * i] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[i], scale, false));
            w[2 * i + 1] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[i], scale, true));
        }
        i32x4 *o = reinterpret_cast<i32x4 *>(a.wide[k] + r * a.Kp + c);
        o[0] = i32x4{w[0], w[1], w[2], w[3]};
        o[1] = i32x4{w[4], w[5], w[6], w[7]};
    }
}

// Up to four neighbouring values, rounded to T.
template <class T>
__device__ __forceinline__ void store_quad(T *p, const f32x4 &v, int left) {
    if (left >= 4) {
        typename Vec<T, 4>::type t;
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = (T)v[i];
        *reinterpret_cast<typename Vec<T, 4>::type *>(p) = t;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < left) p[i] = (T)v[i];
    }
}

// One of the two products,  C[i][j] = sum_p sum_r A_p(i, r) B[r][j]:  B the values of an image, bf16 rows r; A the pieces of dZ, for dX
// with i their rows and r their columns, for dW with r their rows and i their columns.
struct BwProduct {
    BwOperand a;
    const uint8_t *b;  // [R up to 32][pitch_b bytes]
    void *c;           // [I][J], or fp32 partial sums [S][I][J]
    long pitch_b;
    int I, J, R, num_i, num_j, per_split, splits, blocks;  // per_split: steps of 32 r
};
struct BwArgs {
    BwProduct x, w;
    const float *part;  // column sums of dZ
    float *db;
    int parts, N, db_blocks;
};

// LDS images.  Of a tile whose reduction runs along its rows, [i][32 r], 64 bytes a row: chunk c (16 bytes) of row i at slot
// c ^ ((i >> 2) & 3), so that the chunks c of sixteen rows lie in all 64 banks.  Of a tile whose reduction runs down its rows: turn().

// The operand of v_mfma_f32_16x16x32_bf16 out of such a tile: lane l gets column col + (l & 15), rows 8 (l >> 4) .. + 7.
// ds_read_b64_tr_b16: lane i of 16 points at four neighbouring columns of a row (four lanes a row, four rows) and receives four rows
// of its own column i.
template <int ROW>
__device__ __forceinline__ bf16x8 tr_operand(const uint8_t *tile, int col, int lane) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 *lds4;
    const int i = lane & 15, r = (lane >> 4) * 8 + (i >> 2), c = (col >> 3) + ((i & 3) >> 1);
    const uint8_t *p = tile + r * ROW + ((c ^ turn(r)) << 4) + (i & 1) * 8;  // the rows four further have the same turn
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * ROW));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Tile of 64 IF x 32 JF, eight waves (4 x 2) of 16 IF x 16 JF, steps of 32 r.  Both operands come by LDS-DMA into rings of four parts (a
// step and piece), and from there into one of two register sets while the other is multiplied; the waits count loads, so that two
// parts stay in flight across each barrier.
template <int P, bool TRANS, int IF, int JF, class T>
__device__ __forceinline__ void bw_product(const BwProduct &q, int bid, uint8_t *lds) {
    constexpr int TI = IF * 64, TJ = JF * 32, ROWA = TRANS ? TI * 2 : 64, ROWB = JF > 4 ? 512 : 256, SA = TI * 64, SB = 32 * ROWB;
    constexpr int NA = SA / 8192, NB = SB / 8192;  // loads per wave
    uint8_t *ta = lds, *tb = lds + 4 * SA;
    int ti, tj, split;
    if (!tile_of(bid, q.num_i, q.num_j, q.splits, 8, &ti, &tj, &split)) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wi = wave >> 1, wj = wave & 1, i0 = ti * TI, j0 = tj * TJ;
    const int first = split * q.per_split, last = min(first + q.per_split, ceil_div(q.R, 32)), steps = last - first, parts = steps * P;

    uint32_t oa[NA], ob[NB];
#pragma unroll
    for (int k = 0; k < NA; ++k) {
        const int u = wave + k * 8, row = u * 16 + (lane >> 2);
        oa[k] = TRANS ? tr_offset<ROWA>(u, lane, q.a.pitch, q.a.width - i0 * 2L)
                      : (uint32_t)min(row, q.I - 1 - i0) * (uint32_t)q.a.pitch + (((lane & 3) ^ ((row >> 2) & 3)) << 4);
    }
#pragma unroll
    for (int k = 0; k < NB; ++k) ob[k] = tr_offset<ROWB>(wave + k * 8, lane, q.pitch_b, q.pitch_b - j0 * 2L);
    const uint8_t *ab = q.a.at + (TRANS ? i0 * 2L : i0 * q.a.pitch), *bb = q.b + j0 * 2L;
    // Load `k` of part t: its A's NA, then, where a step begins, B's NB.  Behind the end the last part is loaded again: the number of
    // loads in flight stays what the waits count.
    auto load = [&](int t, int k) {
        const int slot = t & 3, slot_b = t / P & 3;
        t = min(t, parts - 1);
        const int s = t / P, p = t - s * P;
        if (k < NA)
            dma16(ab + p * q.a.plane + (first + s) * (TRANS ? 32 * q.a.pitch : 64L), oa[k < NA ? k : 0], ta + slot * SA + (wave + k * 8) * 1024);
        else
            dma16(bb + (first + s) * (32 * q.pitch_b), ob[k < NA ? 0 : k - NA], tb + slot_b * SB + (wave + (k - NA) * 8) * 1024);
    };
    f32x4 acc[IF][JF];
#pragma unroll
    for (int i = 0; i < IF; ++i)
#pragma unroll
        for (int j = 0; j < JF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    struct A {
        bf16x8 f[IF];
    };
    struct B {
        bf16x8 f[JF];
    };
    auto read_a = [&](int t, int i, A &x) {
        const uint8_t *tile = ta + (t & 3) * SA;
        const int row = (wi * IF + i) * 16;
        x.f[i] = TRANS ? tr_operand<ROWA>(tile, row, lane)
                       : *reinterpret_cast<const bf16x8 *>(tile + (row + l16) * 64 + ((g ^ ((l16 >> 2) & 3)) << 4));
    };
    auto read_b = [&](int s, int j, B &x) { x.f[j] = tr_operand<ROWB>(tb + (s & 3) * SB, (wj * JF + j) * 16, lane); };
    // Part t: its operands are in registers; those of part t + 1 are read while it is multiplied, and its own buffer is filled again.
    // Loads (60 to 180 cycles each to issue) and LDS reads stand between the matrix instructions, the reads well before the barrier.
    auto part = [&](int t, auto pc, const A &a, A &next_a, const B &b, B &next_b) {
        constexpr int p = decltype(pc)::value;
        constexpr int LOADS = NA + ((p + 4) % P == 0 ? NB : 0), READS = IF + (p + 1 == P ? JF : 0), EARLY = IF - (IF > 2 ? 1 : 0);
        // in flight behind part t + 1: parts t + 2 and t + 3, with B where a step begins
        dma_wait_barrier<2 * NA + (P == 1 ? 2 : P == 3 && p == 2 ? 0 : 1) * NB>();
#pragma unroll
        for (int i = 0; i < IF; ++i) {
#pragma unroll
            for (int k = LOADS * i / IF; k < LOADS * (i + 1) / IF; ++k) load(t + 4, k);
#pragma unroll
            for (int k = READS * i / EARLY; k < READS * (i + 1) / EARLY; ++k) {
                if (k >= READS) break;
                if (k < IF) read_a(t + 1, k, next_a);
                else read_b((t + 1) / P, k - IF, next_b);
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < JF; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.f[j], a.f[i], acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < NA + (t % P == 0 ? NB : 0); ++k) load(t, k);
    A a0, a1;
    B b0, b1;
    dma_wait_barrier<3 * NA + (P == 1 ? 3 : 1) * NB>();
#pragma unroll
    for (int j = 0; j < JF; ++j) read_b(0, j, b0);
#pragma unroll
    for (int i = 0; i < IF; ++i) read_a(0, i, a0);
    using p0 = std::integral_constant<int, 0>;
    using p1 = std::integral_constant<int, P == 1 ? 0 : 1>;
    using p2 = std::integral_constant<int, 2>;
    // two steps a turn, so that the two register sets stand where they are
    for (int t = 0; t < parts;) {
        if constexpr (P == 1) {
            part(t++, p0{}, a0, a1, b0, b1);
            if (t < parts) part(t++, p0{}, a1, a0, b1, b0);
        } else if constexpr (P == 2) {
            part(t++, p0{}, a0, a1, b0, b1);
            part(t++, p1{}, a1, a0, b0, b1);
            if (t < parts) {
                part(t++, p0{}, a0, a1, b1, b0);
                part(t++, p1{}, a1, a0, b1, b0);
            }
        } else {
            part(t++, p0{}, a0, a1, b0, b1);
            part(t++, p1{}, a1, a0, b0, b1);
            part(t++, p2{}, a0, a1, b0, b1);
            if (t < parts) {
                part(t++, p0{}, a1, a0, b1, b0);
                part(t++, p1{}, a0, a1, b1, b0);
                part(t++, p2{}, a1, a0, b1, b0);
            }
        }
    }
    dma_wait<0>();  // the repeated loads still write this workgroup's LDS
    // a lane holds four neighbouring columns j of row i
    const long out = q.splits > 1 ? split * ((long)q.I * q.J) : 0;
#pragma unroll
    for (int i = 0; i < IF; ++i) {
        const int ci = i0 + (wi * IF + i) * 16 + l16;
        if (ci >= q.I) continue;
#pragma unroll
        for (int j = 0; j < JF; ++j) {
            const int cj = j0 + (wj * JF + j) * 16 + g * 4;
            const long at = out + (long)ci * q.J + cj;
            if (q.splits > 1) store_quad((float *)q.c + at, acc[i][j], q.J - cj);
            else store_quad((T *)q.c + at, acc[i][j], q.J - cj);
        }
    }
}

// Both products and the last step of the column sums in one launch: blocks of dW (the longer ones), then of dX, then of db.
template <int P, int IF, int JF, class T>
__global__ __launch_bounds__(512) void e4m3_bw_kernel(BwArgs a) {
    extern __shared__ uint8_t lds[];
    int bid = blockIdx.x;
    if (bid < a.w.blocks) return bw_product<P, true, IF, JF, float>(a.w, bid, lds);
    bid -= a.w.blocks;
    if (bid < a.x.blocks) return bw_product<P, false, IF, JF, T>(a.x, bid, lds);
    bid -= a.x.blocks;
    // db: 32 columns, sixteen threads of a column add a sixteenth of the parts each
    float *sums = (float *)lds;
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, n = bid * 32 + c, per = ceil_div(a.parts, 16);
    float s = 0.f;
    const int end = min((r + 1) * per, a.parts);
    if (n < a.N)
        for (int t = r * per; t < end; t += 8) {  // eight loads in flight
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = a.part[(long)min(t + u, end - 1) * a.N + n];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += t + u < end ? v[u] : 0.f;
        }
    sums[r * 32 + c] = s;
    __syncthreads();
    if (r || n >= a.N) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) s += sums[k * 32 + c];
    a.db[n] = s;
}

// The partial sums of both products, added in ascending order.
struct BwJoin {
    const float *part;
    void *out;
    long total;
    int S, blocks;
};
template <class T>
__device__ __forceinline__ void bw_join(const BwJoin &q, int bid) {
    for (long at = (bid * 256L + threadIdx.x) * 4; at < q.total; at += q.blocks * 1024L) {
        const int left = (int)min(q.total - at, 4L);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (left == 4) {
            for (int s = 0; s < q.S; s += 8) {  // eight loads in flight
                f32x4 p[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) p[u] = *reinterpret_cast<const Vec<float, 4>::type *>(q.part + min(s + u, q.S - 1) * q.total + at);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (s + u < q.S) v += p[u];
            }
        } else {
            for (int s = 0; s < q.S; ++s)
                for (int i = 0; i < left; ++i) v[i] += q.part[s * q.total + at + i];
        }
        store_quad((T *)q.out + at, v, left);
    }
}
template <class T>
__global__ __launch_bounds__(256) void e4m3_bw_join_kernel(BwJoin x, BwJoin w) {
    if ((int)blockIdx.x < x.blocks) bw_join<T>(x, blockIdx.x);
    else bw_join<float>(w, blockIdx.x - x.blocks);
}

static inline int up_to(int v, int a) { return (v + a - 1) / a * a; }

// Tile and splits of both products: those with the least estimated time.  The workgroups of both go to 256 compute units, one each at
// a time; a reduction is cut into S ranges whose fp32 partial sums are joined in ascending order.  Tiles are 256 or 128 rows by 256, 224,
// 192 or 128 columns: over 4000 sizes, the logarithms even (M to 32768, N to 13464, K to 4096), 160 columns beside them take 0.3 % off the
// estimate (2 % or more in 4 % of the sizes) for a quarter more kernels; 256 and 128 columns alone add 0.7 % to it, and 2 % or more in
// every tenth.
struct Split {
    int S, per;
};
struct BwPlan {
    int IF, JF;
    Split sx, sw;
    size_t planes, part, wx, ww, px, pw, total;
};
// Rows of a workgroup that makes dZ: few rows a thread where there are few workgroups (a thread's rows come one after the other: 256 x 868
// fp32 7.2 us with 8, 9.8 with 32; 8191 x 400 12.5 with 16, 13.4 with 32), many where there are many, for fewer partial sums (32768 x
// 2448 bf16 85 us with 128, 98 with 16).
static int dz_rows_of(int M, int N) {
    const long blocks = (long)ceil_div(M, 32) * ceil_div(N, 256);
    return blocks >= 4096 ? 128 : blocks >= 2048 ? 64 : blocks >= 768 ? 32 : blocks >= 128 ? 16 : 8;
}
static double plan_split(int I, int J, int R, int P, int TI, int TJ, Split *out) {
    const double tiles = (double)ceil_div(I, TI) * ceil_div(J, TJ), part = (TI * TJ) / (256. * 256.) * 0.65 + 0.1;  // us of a part
    const int steps = ceil_div(R, 32), fill = tiles < 256 ? (int)(256 / tiles) : 1;
    double least = 1e300;
    const int tries[] = {1, fill / 2, fill, 2 * fill};
    for (int S : tries) {
        S = S < 1 ? 1 : S > 64 ? 64 : S > steps ? steps : S;
        const int per = ceil_div(steps, S);
        S = ceil_div(steps, per);
        const double one = per * P * part + 4.0, rounds = tiles * S / 256.;
        // the last round is rarely full: a share of a workgroup's time on top
        const double us = (rounds > 1. ? (rounds + 0.4) : 1.) * one + (S > 1 ? 4.0 + 8.0 * S * I * (double)J / 4.0e6 : 0.0);
        if (us < least) {
            least = us;
            *out = {S, per};
        }
    }
    return least;
}
static BwPlan plan_bw(int M, int N, int K, int type) {
    const int P = pieces_of(type);
    BwPlan p = {};
    double least = 1e300;
    for (int IF = 4; IF >= 2; IF -= 2)
        for (int JF = 8; JF >= 4; JF -= JF == 6 ? 2 : 1) {
            Split sx, sw;
            const double us = plan_split(M, K, N, P, IF * 64, JF * 32, &sx) + plan_split(N, K, M, P, IF * 64, JF * 32, &sw);
            if (us < least) {
                least = us;
                p.IF = IF;
                p.JF = JF;
                p.sx = sx;
                p.sw = sw;
            }
        }
    const size_t Kp = kp8_of(K);
    p.planes = align_up((size_t)P * up_to(M, 32) * up_to(N, 32) * 2, 256);
    p.part = align_up((size_t)ceil_div(M, dz_rows_of(M, N)) * N * 4, 256);
    p.wx = up_to(M, 32) * Kp * 2;
    p.ww = up_to(N, 32) * Kp * 2;
    p.px = p.sx.S > 1 ? align_up((size_t)p.sx.S * M * K * 4, 256) : 0;
    p.pw = p.sw.S > 1 ? align_up((size_t)p.sw.S * N * K * 4, 256) : 0;
    p.total = p.planes + p.part + p.wx + p.ww + p.px + p.pw;
    return p;
}

static void set_split(BwProduct &q, const Split &s, void *out, void *part) {
    q.splits = s.S;
    q.per_split = s.per;
    q.c = s.S > 1 ? part : out;
    q.blocks = tile_grid(q.num_i, q.num_j, s.S);
}

template <int P, int IF, int JF, class T>
static int launch_products(const BwArgs &g, hipStream_t st) {
    constexpr int bytes = 4 * (IF * 64 * 64 + 32 * (JF > 4 ? 512 : 256));
    static PerDeviceOnce once;
    int dev;
    if (once.pending(&dev)) {
        if (hipFuncSetAttribute((const void *)e4m3_bw_kernel<P, IF, JF, T>, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
            return fail(PHONLP_ERR_LAUNCH, "linear_e4m3_backward: hipFuncSetAttribute failed");
        once.mark(dev);
    }
    ProfScope ps("e4m3_bw", st);
    hipLaunchKernelGGL((e4m3_bw_kernel<P, IF, JF, T>), dim3(g.x.blocks + g.w.blocks + g.db_blocks), dim3(512), bytes, st, g);
    return check_launch("e4m3_bw_kernel");
}

}  // namespace phonlp

using namespace phonlp;

static bool bw_shape_ok(int M, int N, int K, int type) {
    return M > 0 && N > 0 && K > 0 && K <= (1 << 21) && N <= (1 << 21) && M <= (1 << 24) && type_ok(type) &&
           (long)ceil_div(M, 128) * ceil_div(K, 128) < (1L << 22) && (long)ceil_div(N, 128) * ceil_div(K, 128) < (1L << 22);
}

extern "C" size_t phonlp_linear_e4m3_backward_ws_bytes(int M, int N, int K, int type) {
    return bw_shape_ok(M, N, K, type) ? plan_bw(M, N, K, type).total : 0;
}

extern "C" int phonlp_linear_e4m3_backward(const void *dy, int type, long lddy, const uint32_t *bits, const void *x_codes,
                                           const uint8_t *x_exponents, const void *w_codes, const uint8_t *w_exponents, int M, int N, int K,
                                           void *dx, float *dw, float *db, void *ws, size_t ws_bytes, void *stream) {
    if (!dy || (dw && (!x_codes || !x_exponents)) || (dx && (!w_codes || !w_exponents)) || !bw_shape_ok(M, N, K, type) || lddy < N)
        return fail(PHONLP_ERR_SHAPE, "linear_e4m3_backward: bad argument");
    if (((uintptr_t)x_codes & 15) || ((uintptr_t)w_codes & 15) || ((uintptr_t)x_exponents & 3) || ((uintptr_t)w_exponents & 3) ||
        ((uintptr_t)bits & 3) || ((uintptr_t)dw & 3) || ((uintptr_t)db & 3) || (uintptr_t)dy % type_bytes(type) ||
        (uintptr_t)dx % type_bytes(type))
        return fail(PHONLP_ERR_SHAPE, "linear_e4m3_backward: codes must be 16-byte aligned, exponents, bits, dw and db 4-byte, dy and dx to their type");
    const BwPlan pl = plan_bw(M, N, K, type);
    if (!ws || ((uintptr_t)ws & 15) || ws_bytes < pl.total)
        return fail(PHONLP_ERR_WORKSPACE, "linear_e4m3_backward: workspace too small or not 16-byte aligned");
    if (!dx && !dw && !db) return PHONLP_OK;
    hipStream_t st = as_stream(stream);
    const int Mp = up_to(M, 32), Np = up_to(N, 32), Kp = kp8_of(K), dz_rows = dz_rows_of(M, N), parts = ceil_div(M, dz_rows);
    uint8_t *planes = (uint8_t *)ws, *p = planes + pl.planes;
    float *part = (float *)p;
    uint8_t *wx = p + pl.part, *ww = wx + pl.wx;
    float *px = (float *)(ww + pl.ww), *pw = (float *)((uint8_t *)px + pl.px);
    const bool direct = bw_direct(dy, type, lddy, bits, M, N);
    const bool make_planes = (dx || dw) && !direct;
    BwPrep prep = {dy, lddy, bits, make_planes ? (uint16_t *)planes : nullptr, !db ? nullptr : parts == 1 ? db : part,
                   {(const uint8_t *)x_codes, (const uint8_t *)w_codes}, {x_exponents, w_exponents}, {(__bf16 *)wx, (__bf16 *)ww}, {M, N},
                   {0, 0}, ceil_div(N, 32), M, N, Mp, Np, Kp, kb4_of(K), dz_rows, ceil_div(Mp, dz_rows), 0};
    if (make_planes || db) prep.dz_blocks = prep.dz_m * ceil_div(Np, 256);
    auto wide_blocks = [&](int rows) {
        const long blocks = ((long)up_to(rows, 32) * (Kp / 16) + 1023) / 1024;
        return (int)(blocks < 1024 ? blocks : 1024);
    };
    if (dw) prep.wide_blocks[0] = wide_blocks(M);
    if (dx) prep.wide_blocks[1] = wide_blocks(N);
    const BwOperand a = bw_dz(direct, dy, lddy, planes, N, Mp, Np);
    BwArgs g = {};
    const int TI = pl.IF * 64, TJ = pl.JF * 32;
    g.x = {a, ww, nullptr, Kp * 2L, M, K, N, ceil_div(M, TI), ceil_div(K, TJ), 0, 1, 0};
    g.w = {a, wx, nullptr, Kp * 2L, N, K, M, ceil_div(N, TI), ceil_div(K, TJ), 0, 1, 0};
    if (dx) set_split(g.x, pl.sx, dx, px);
    if (dw) set_split(g.w, pl.sw, dw, pw);
    g.part = part;
    g.db = db;
    g.parts = parts;
    g.N = N;
    g.db_blocks = db && parts > 1 ? ceil_div(N, 32) : 0;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int P = Pieces<T>::N;
        int rc;
        {
            ProfScope ps("e4m3_bw_prep", st);
            hipLaunchKernelGGL((e4m3_bw_prep_kernel<T>), dim3(prep.dz_blocks + prep.wide_blocks[0] + prep.wide_blocks[1]), dim3(256), 0, st,
                               prep);
            if ((rc = check_launch("e4m3_bw_prep_kernel"))) return rc;
        }
        if (g.x.blocks + g.w.blocks + g.db_blocks) {
            auto by_j = [&](auto f) {
                constexpr int IF = decltype(f)::value;
                switch (pl.JF) {
                    case 4: return launch_products<P, IF, 4, T>(g, st);
                    case 6: return launch_products<P, IF, 6, T>(g, st);
                    case 7: return launch_products<P, IF, 7, T>(g, st);
                    default: return launch_products<P, IF, 8, T>(g, st);
                }
            };
            rc = pl.IF == 2 ? by_j(std::integral_constant<int, 2>{}) : by_j(std::integral_constant<int, 4>{});
            if (rc) return rc;
        }
        const bool jx = dx && pl.sx.S > 1, jw = dw && pl.sw.S > 1;
        if (!jx && !jw) return PHONLP_OK;
        ProfScope ps("e4m3_bw_join", st);
        auto plan = [](bool on, const float *p, void *out, long total, int S) {
            const long blocks = on ? (total + 1023) / 1024 : 0;  // four values a thread and turn
            return BwJoin{p, out, total, S, (int)(blocks < 2048 ? blocks : 2048)};
        };
        const BwJoin x = plan(jx, px, dx, (long)M * K, pl.sx.S), w = plan(jw, pw, dw, (long)N * K, pl.sw.S);
        hipLaunchKernelGGL((e4m3_bw_join_kernel<T>), dim3(x.blocks + w.blocks), dim3(256), 0, st, x, w);
        return check_launch("e4m3_bw_join_kernel");
    });
}
