// Backward of the dense layer of linear_e4m3.hip from its 8-bit checkpoint (the input's image and one bit per output):
//   dZ = dY where the bit is set (ReLU) or dY;   dX = dZ W^;   dW = dZ^T X^;   db = column sums of dZ.
//
// Products on v_mfma_f32_16x16x32_bf16 (2.05 PFLOP/s in a loop of nothing else, 32x32x16 1.84).  The values of an image are exact in bf16 (four significant bits, a power of two), and dZ is
// cut into bf16 pieces whose sum is dZ itself -- one for bf16, two for fp16 (11 bits), three for fp32 (24 bits), by truncation, so no
// piece can round past bf16's largest --, so every product is exact and only the fp32 sums round.  (Values under 2^-126 may lose
// low bits.)
#include "e4m3.h"
#include "tile128.h"

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

// dY -> the pieces of dZ as rows [P][Mp][Np] (zero behind M and N), and the column sums of 128 rows part[block][n].  A workgroup takes
// 128 rows x 256 columns, a thread eight columns of every eighth row; the eight threads of a column group add in order.
template <class T>
__global__ __launch_bounds__(256) void e4m3_bw_dz_kernel(const T *dy, long lddy, const uint32_t *bits, int words, int M, int N, int Mp,
                                                         int Np, uint16_t *planes, float *part) {
    constexpr int P = Pieces<T>::N;
    typedef typename Vec<T, 8>::type V;
    __shared__ float sums[8][256];
    const int cg = threadIdx.x & 31, rl = threadIdx.x >> 5, n = blockIdx.y * 256 + cg * 8, m0 = blockIdx.x * 128 + rl;
    float s[8] = {};
    if (n < Np) {
#pragma unroll 4
        for (int it = 0; it < 16; ++it) {
            const int m = m0 + it * 8;
            if (m >= Mp) break;
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
            if (m < M) {
                const T *p = dy + m * lddy + n;
                if (n + 8 <= N) {
                    const V t = *reinterpret_cast<const V *>(p);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n + i < N) v[i] = (float)p[i];
                }
                if (bits) {
                    const uint32_t b = n < N ? bits[(long)m * words + (n >> 5)] >> (n & 31) : 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = b >> i & 1 ? v[i] : 0.f;
                }
            }
            if (planes) {
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
                    *reinterpret_cast<uint4 *>(planes + ((long)q * Mp + m) * Np + n) = make_uint4(w[q][0], w[q][1], w[q][2], w[q][3]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s[i] += v[i];
        }
    }
    if (!part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[rl][cg * 8 + i] = s[i];
    __syncthreads();
    const int c = blockIdx.y * 256 + threadIdx.x;
    if (c >= N) return;
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += sums[r][threadIdx.x];
    part[(long)blockIdx.x * N + c] = t;
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

// One of the two products,  C[i][j] = sum_p sum_r A_p(i, r) B[r][j]:  B the values of an image's rows r, columns j; A the pieces of dZ,
// for dX with i their rows and r their columns, for dW with r their rows and i their columns.
struct BwProduct {
    const uint8_t *a;            // [P][..][pitch bytes]
    const uint8_t *codes, *exps;  // image of B
    void *c;                     // [I][J], or fp32 partial sums [S][I][J]
    long pitch, plane;           // bytes
    int I, J, R, Kp, KB4, num_i, num_j, per_split, splits, blocks;  // per_split: steps of 64 r
};
struct BwArgs {
    BwProduct x, w;
    const float *part;  // column sums of dZ
    float *db;
    int parts, N, db_blocks;
};

// LDS image of a [64 r][128 columns] bf16 tile: row r at r * 256, its 16-byte chunk c at slot c ^ 4 (r & 3).  A transposing read takes 4
// rows x 32 bytes per 16 lanes: four different pairs of slots, no bank conflict.
__device__ __forceinline__ int tr_slot(int r, int c) { return r * 256 + ((c ^ ((r & 3) << 2)) << 4); }

// The operand of v_mfma_f32_16x16x32_bf16 whose reduction runs down the rows of such a tile: lane l gets column col + (l & 15), rows
// r0 + 8 (l >> 4) .. + 7.  ds_read_b64_tr_b16: lane i of 16 points at four neighbouring columns of a row (four lanes a row, four rows)
// and receives four rows of its own column i.
__device__ __forceinline__ bf16x8 tr_operand(const uint8_t *tile, int r0, int col, int lane) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 *lds4;
    const int i = lane & 15, r = r0 + (lane >> 4) * 8 + (i >> 2), c = (col >> 3) + ((i & 3) >> 1);
    const uint8_t *p = tile + tr_slot(r, c) + (i & 1) * 8;  // the rows four further have the same slot
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 4 * 256));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 128 x 128 tile, four waves of 64 x 64, steps of 64 r.  A comes by LDS-DMA; B's codes pass through registers, where they take their
// row's scale (128 columns are one block, so a row has one) and become bf16, eight instructions for sixteen codes.
template <int P, bool TRANS, class T>
__device__ __forceinline__ void bw_product(const BwProduct &q, int bid, uint8_t *lds) {
    uint8_t *ta = lds, *tb = lds + 2 * 16384;  // [2][16 KB] each
    int ti, tj;
    const int tiles8 = (q.num_i * q.num_j + 7) / 8 * 8, split = bid / tiles8;
    if (!tile_of(bid - split * tiles8, q.num_i, q.num_j, 8, &ti, &tj)) return;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, l16 = lane & 15, g = lane >> 4, wi = wave >> 1, wj = wave & 1;
    const int i0 = ti * 128, j0 = tj * 128;
    const int first = split * q.per_split, last = min(first + q.per_split, ceil_div(q.R, 64)), steps = last - first;

    uint32_t off[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int u = wave + k * 4;  // 1 KB of the tile: 8 rows of 128 bytes, or 4 of 256
        if (TRANS) off[k] = (uint32_t)(u * 4 + (lane >> 4)) * (uint32_t)q.pitch + (((lane & 15) ^ ((lane >> 4) << 2)) << 4);
        else off[k] = (uint32_t)min(u * 8 + (lane >> 3), q.I - 1 - i0) * (uint32_t)q.pitch + (((lane & 7) ^ (lane >> 3)) << 4);
    }
    const uint8_t *ab = q.a + (TRANS ? i0 * 2L : i0 * q.pitch);
    auto load_a = [&](int s, int p, int buf) {
        const uint8_t *base = ab + p * q.plane + (first + s) * (TRANS ? 64 * q.pitch : 128L);
#pragma unroll
        for (int k = 0; k < 4; ++k) dma16(base, off[k], ta + buf * 16384 + (wave + k * 4) * 1024);
    };
    // codes of rows tid / 8 and 32 + tid / 8, sixteen columns each
    const int br = tid >> 3, bc = tid & 7;
    i32x4 code[2];
    int exps[2];
    auto load_b = [&](int s) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int r = (first + s) * 64 + h * 32 + br, rr = min(r, q.R - 1);
            code[h] = *reinterpret_cast<const i32x4 *>(q.codes + (long)rr * q.Kp + j0 + bc * 16);
            exps[h] = q.exps[(long)rr * q.KB4 + tj];
            if (r >= q.R) code[h] = i32x4{0, 0, 0, 0};
        }
    };
    auto store_b = [&](int buf) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float scale = exp2_biased(exps[h]);
            int w[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w[2 * k] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[h][k], scale, false));
                w[2 * k + 1] = __builtin_bit_cast(int, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(code[h][k], scale, true));
            }
            uint8_t *t = tb + buf * 16384;
            const int r = h * 32 + br;
            *reinterpret_cast<i32x4 *>(t + tr_slot(r, bc * 2)) = i32x4{w[0], w[1], w[2], w[3]};
            *reinterpret_cast<i32x4 *>(t + tr_slot(r, bc * 2 + 1)) = i32x4{w[4], w[5], w[6], w[7]};
        }
    };

    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    load_a(0, 0, 0);
    load_b(0);
    store_b(0);
    int t = 0;
    for (int s = 0; s < steps; ++s) {
#pragma unroll
        for (int p = 0; p < P; ++p, ++t) {
            dma_wait_barrier();  // A of this part and B of this step are in LDS; everybody is done with the other buffers
            if (p + 1 < P) load_a(s, p + 1, (t + 1) & 1);
            else if (s + 1 < steps) load_a(s + 1, 0, (t + 1) & 1);
            if (p == 0 && s + 1 < steps) load_b(s + 1);
            const uint8_t *A = ta + (t & 1) * 16384, *B = tb + (s & 1) * 16384;
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                bf16x8 fa[4], fb[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    fa[i] = TRANS ? tr_operand(A, ks * 32, wi * 64 + i * 16, lane)
                                  : __builtin_bit_cast(bf16x8, tile_chunk(A, wi * 64 + i * 16 + l16, ks * 4 + g));
#pragma unroll
                for (int j = 0; j < 4; ++j) fb[j] = tr_operand(B, ks * 32, wj * 64 + j * 16, lane);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[j], fa[i], acc[i][j], 0, 0, 0);
            }
            if (p + 1 == P && s + 1 < steps) store_b((s + 1) & 1);
        }
    }
    // a lane holds four neighbouring columns j of row i
    const long out = q.splits > 1 ? split * ((long)q.I * q.J) : 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int ci = i0 + wi * 64 + i * 16 + l16;
        if (ci >= q.I) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int cj = j0 + wj * 64 + j * 16 + g * 4;
            const long at = out + (long)ci * q.J + cj;
            if (q.splits > 1) store_quad((float *)q.c + at, acc[i][j], q.J - cj);
            else store_quad((T *)q.c + at, acc[i][j], q.J - cj);
        }
    }
}

// Both products and the last step of the column sums in one launch: blocks of dX, then of dW, then of db.
template <int P, class T>
__global__ __launch_bounds__(256, 2) void e4m3_bw_kernel(BwArgs a) {
    extern __shared__ uint8_t lds[];  // 64 KB
    int bid = blockIdx.x;
    if (bid < a.x.blocks) return bw_product<P, false, T>(a.x, bid, lds);
    bid -= a.x.blocks;
    if (bid < a.w.blocks) return bw_product<P, true, float>(a.w, bid, lds);
    bid -= a.w.blocks;
    // db: 32 columns, eight threads of a column add an eighth of the parts each
    float *sums = (float *)lds;
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, n = bid * 32 + c, per = ceil_div(a.parts, 8);
    float s = 0.f;
    if (n < a.N)
        for (int t = r * per; t < min((r + 1) * per, a.parts); ++t) s += a.part[(long)t * a.N + n];
    sums[r * 32 + c] = s;
    __syncthreads();
    if (r || n >= a.N) return;
    s = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) s += sums[k * 32 + c];
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
        for (int s = 0; s < q.S; ++s) {
            const float *p = q.part + s * q.total + at;
            if (left == 4) v += *reinterpret_cast<const Vec<float, 4>::type *>(p);
            else
                for (int i = 0; i < left; ++i) v[i] += p[i];
        }
        store_quad((T *)q.out + at, v, left);
    }
}
template <class T>
__global__ __launch_bounds__(256) void e4m3_bw_join_kernel(BwJoin x, BwJoin w) {
    if ((int)blockIdx.x < x.blocks) bw_join<T>(x, blockIdx.x);
    else bw_join<float>(w, blockIdx.x - x.blocks);
}

// Few output tiles and a long reduction: the reduction is cut into S ranges.  S is the count with the least estimated time: rounds of
// 512 workgroups (two per compute unit) times a workgroup's steps, plus writing and reading the partial sums.
struct Split {
    int S, per;
};
static Split plan_split(int I, int J, int R, int P) {
    const long tiles = (long)ceil_div(I, 128) * ceil_div(J, 128);
    const int steps = ceil_div(R, 64);
    Split best = {1, steps};
    double least = 1e300;
    for (int S = 1; S <= 64 && S <= steps; ++S) {
        const int per = ceil_div(steps, S), n = ceil_div(steps, per);
        if (n != S) continue;
        // us: a step of one piece takes about 0.6 with two workgroups on a compute unit, start and end of a workgroup about 3
        const double rounds = (double)((tiles * S + 511) / 512), us = rounds * (per * P * 0.6 + 3.0) +
                                                                     (S > 1 ? 4.0 + 8.0 * S * I * (double)J / 4.0e6 : 0.0);
        if (us < least) {
            least = us;
            best = {S, per};
        }
    }
    return best;
}

static inline int up_to(int v, int a) { return (v + a - 1) / a * a; }

struct BwPlan {
    Split sx, sw;
    size_t planes, part, px, pw, total;
};
static BwPlan plan_bw(int M, int N, int K, int type) {
    const int P = pieces_of(type);
    BwPlan p;
    p.sx = plan_split(M, K, N, P);
    p.sw = plan_split(N, K, M, P);
    p.planes = align_up((size_t)P * up_to(M, 64) * up_to(N, 128) * 2, 256);
    p.part = align_up((size_t)ceil_div(M, 128) * N * 4, 256);
    p.px = p.sx.S > 1 ? align_up((size_t)p.sx.S * M * K * 4, 256) : 0;
    p.pw = p.sw.S > 1 ? align_up((size_t)p.sw.S * N * K * 4, 256) : 0;
    p.total = p.planes + p.part + p.px + p.pw;
    return p;
}

static void set_split(BwProduct &q, const Split &s, void *out, void *part) {
    q.splits = s.S;
    q.per_split = s.per;
    q.c = s.S > 1 ? part : out;
    q.blocks = tile_grid(q.num_i, q.num_j) * s.S;
}

}  // namespace phonlp

using namespace phonlp;

static bool bw_shape_ok(int M, int N, int K, int type) {
    return M > 0 && N > 0 && K > 0 && K <= (1 << 21) && N <= (1 << 21) && M <= (1 << 24) && type_ok(type) &&
           (long)ceil_div(M, 128) * ceil_div(K, 128) < (1L << 24) && (long)ceil_div(N, 128) * ceil_div(K, 128) < (1L << 24);
}

extern "C" size_t phonlp_linear_e4m3_backward_ws_bytes(int M, int N, int K, int type) {
    return bw_shape_ok(M, N, K, type) ? plan_bw(M, N, K, type).total : 0;
}

extern "C" int phonlp_linear_e4m3_backward(const void *dy, int type, long lddy, const uint32_t *bits, const void *x_codes,
                                           const uint8_t *x_exponents, const void *w_codes, const uint8_t *w_exponents, int M, int N, int K,
                                           void *dx, float *dw, float *db, void *ws, size_t ws_bytes, void *stream) {
    if (!dy || !x_codes || !x_exponents || !w_codes || !w_exponents || !bw_shape_ok(M, N, K, type) || lddy < N)
        return fail(PHONLP_ERR_SHAPE, "linear_e4m3_backward: bad argument");
    if (((uintptr_t)x_codes & 15) || ((uintptr_t)w_codes & 15) || ((uintptr_t)x_exponents & 3) || ((uintptr_t)w_exponents & 3) ||
        ((uintptr_t)bits & 3) || ((uintptr_t)dw & 3) || ((uintptr_t)db & 3) || (uintptr_t)dy % type_bytes(type) ||
        (uintptr_t)dx % type_bytes(type))
        return fail(PHONLP_ERR_SHAPE, "linear_e4m3_backward: codes must be 16-byte aligned, exponents, bits, dw and db 4-byte, dy and dx to their type");
    if (!ws || ((uintptr_t)ws & 15) || ws_bytes < phonlp_linear_e4m3_backward_ws_bytes(M, N, K, type))
        return fail(PHONLP_ERR_WORKSPACE, "linear_e4m3_backward: workspace too small or not 16-byte aligned");
    if (!dx && !dw && !db) return PHONLP_OK;
    hipStream_t st = as_stream(stream);
    const BwPlan pl = plan_bw(M, N, K, type);
    const int Mp = up_to(M, 64), Np = up_to(N, 128), Kp = kp8_of(K), KB4 = kb4_of(K), parts = ceil_div(M, 128);
    uint8_t *planes = (uint8_t *)ws;
    float *part = (float *)(planes + pl.planes), *px = (float *)((uint8_t *)part + pl.part), *pw = (float *)((uint8_t *)px + pl.px);
    // without a mask and with whole tiles, bf16 gradients are their own single piece
    const bool direct = type == PHONLP_BF16 && !bits && M % 64 == 0 && N % 128 == 0 && lddy % 8 == 0 && lddy < (1 << 24) && !((uintptr_t)dy & 15);
    const bool make_planes = (dx || dw) && !direct;
    const uint8_t *a = direct ? (const uint8_t *)dy : planes;
    const long pitch = direct ? lddy * 2 : Np * 2L, plane = (long)Mp * Np * 2;
    BwArgs g = {};
    g.x = {a, (const uint8_t *)w_codes, w_exponents, nullptr, pitch, plane, M, K, N, Kp, KB4, ceil_div(M, 128), ceil_div(K, 128), 0, 1, 0};
    g.w = {a, (const uint8_t *)x_codes, x_exponents, nullptr, pitch, plane, N, K, M, Kp, KB4, ceil_div(N, 128), ceil_div(K, 128), 0, 1, 0};
    if (dx) set_split(g.x, pl.sx, dx, px);
    if (dw) set_split(g.w, pl.sw, dw, pw);
    g.part = part;
    g.db = db;
    g.parts = parts;
    g.N = N;
    g.db_blocks = db && parts > 1 ? ceil_div(N, 32) : 0;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int P = Pieces<T>::N, bytes = 65536;
        int rc;
        if (make_planes || db) {
            ProfScope ps("e4m3_bw_dz", st);
            hipLaunchKernelGGL((e4m3_bw_dz_kernel<T>), dim3(ceil_div(Mp, 128), ceil_div(Np, 256)), dim3(256), 0, st, (const T *)dy, lddy,
                               bits, ceil_div(N, 32), M, N, Mp, Np, make_planes ? (uint16_t *)planes : nullptr,
                               !db ? nullptr : parts == 1 ? db : part);
            if ((rc = check_launch("e4m3_bw_dz_kernel"))) return rc;
        }
        const int blocks = g.x.blocks + g.w.blocks + g.db_blocks;
        if (blocks) {
            ProfScope ps("e4m3_bw", st);
            hipLaunchKernelGGL((e4m3_bw_kernel<P, T>), dim3(blocks), dim3(256), bytes, st, g);
            if ((rc = check_launch("e4m3_bw_kernel"))) return rc;
        }
        const bool jx = dx && pl.sx.S > 1, jw = dw && pl.sw.S > 1;
        if (!jx && !jw) return PHONLP_OK;
        ProfScope ps("e4m3_bw_join", st);
        auto plan = [](bool on, const float *p, void *out, long total, int S) {
            const long blocks = on ? (total + 1023) / 1024 : 0;
            return BwJoin{p, out, total, S, (int)(blocks < 2048 ? blocks : 2048)};
        };
        const BwJoin x = plan(jx, px, dx, (long)M * K, pl.sx.S), w = plan(jw, pw, dw, (long)N * K, pl.sw.S);
        hipLaunchKernelGGL((e4m3_bw_join_kernel<T>), dim3(x.blocks + w.blocks), dim3(256), 0, st, x, w);
        return check_launch("e4m3_bw_join_kernel");
    });
}
