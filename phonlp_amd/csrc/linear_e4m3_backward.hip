// Backward of the dense layer of linear_e4m3.hip from its 8-bit checkpoint (the input's image and one bit per output):
//   dZ = dY where the bit is set (ReLU) or dY;   dX = dZ W^;   dW = dZ^T X^;   db = column sums of dZ.
//
// Products on v_mfma_f32_32x32x16_bf16.  The values of an image are exact in bf16 (four significant bits, a power of two), and dZ is
// cut into bf16 pieces whose sum is dZ itself -- one for bf16, two for fp16 (11 bits), three for fp32 (24 bits), by truncation, so no
// piece can round past bf16's largest --, so every product is exact and only the fp32 sums round.  (Values under 2^-126 may lose
// low bits.)
#include "e4m3.h"
#include "tile128.h"

namespace phonlp {

constexpr int kStep = 64;  // reduction step: 64 bf16 = 128 bytes of a row

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

// dY -> the pieces of dZ, as rows [P][M][Np] and transposed [P][N][Mp] (both zero-padded to kStep), and each 64-row tile's column
// sums part[tile][n] (ascending rows).  One workgroup per 64 x 64 tile.
template <class T>
__global__ __launch_bounds__(256) void e4m3_bw_dz_kernel(const T *dy, long lddy, const uint32_t *bits, int words, int M, int N, int Mp,
                                                         int Np, uint16_t *rows, uint16_t *cols, float *part) {
    constexpr int P = Pieces<T>::N;
    __shared__ float tile[64][65];
    const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int r = ty; r < 64; r += 4) {
        const int m = m0 + r, n = n0 + tx;
        float v = 0.f;
        if (m < M && n < N) {
            v = (float)dy[m * lddy + n];
            if (bits && !(bits[(long)m * words + (n >> 5)] >> (n & 31) & 1)) v = 0.f;
        }
        tile[r][tx] = v;
        if (rows && m < M) {
            uint16_t p[P];
            cut<P>(v, p);
#pragma unroll
            for (int i = 0; i < P; ++i) rows[((long)i * M + m) * Np + n] = p[i];
        }
    }
    __syncthreads();
    if (cols)
        for (int c = ty; c < 64; c += 4) {
            const int n = n0 + c, m = m0 + tx;
            if (n >= N) break;
            uint16_t p[P];
            cut<P>(tile[tx][c], p);
#pragma unroll
            for (int i = 0; i < P; ++i) cols[((long)i * N + n) * Mp + m] = p[i];
        }
    if (part && threadIdx.x < 64 && n0 + tx < N) {
        float s = 0.f;
        for (int r = 0; r < 64; ++r) s += tile[r][tx];
        part[(long)blockIdx.x * N + n0 + tx] = s;
    }
}

// db[n] = sum over the tiles of part[tile][n], ascending
__global__ __launch_bounds__(256) void e4m3_bw_db_kernel(const float *part, int tiles, int N, float *db) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float s = 0.f;
    for (int t = 0; t < tiles; ++t) s += part[(long)t * N + n];
    db[n] = s;
}

// Values of an image [R][K], transposed: out[k][r] bf16, row pitch Rp, zero for r >= R.  One workgroup per 64 x 64 tile.
__global__ __launch_bounds__(256) void e4m3_bw_transpose_kernel(const uint8_t *codes, const uint8_t *exponents, int R, int K, int Kp,
                                                                int KB4, int Rp, __bf16 *out) {
    __shared__ float tile[64][65];
    const int r0 = blockIdx.x * 64, k0 = blockIdx.y * 64, tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    for (int i = ty; i < 64; i += 4) {
        const int r = r0 + i, k = k0 + tx;
        tile[i][tx] = r < R ? __builtin_amdgcn_cvt_f32_fp8(codes[(long)r * Kp + k], 0) *
                                  exp2_biased(max((int)exponents[(long)r * KB4 + (k >> 7)], 1))
                            : 0.f;
    }
    __syncthreads();
    for (int i = ty; i < 64; i += 4) {
        const int k = k0 + i, r = r0 + tx;
        if (k < K) out[(long)k * Rp + r] = (__bf16)tile[tx][i];
    }
}

struct Bf16Args {
    const uint8_t *a, *b;  // [P][I][R], [J][R] bf16
    void *c;               // [I][J] T, or fp32 partial sums [S][I][J]
    int I, J, R, num_m, num_n, per_split;  // per_split: reduction steps of one split
};

// C[i][j] = sum_p sum_r A[p][i][r] B[j][r] over this split's range of r.
template <int TM, int TN, int WM, int WN, int P, class T>
__global__ __launch_bounds__(WM *WN * 64) void e4m3_bw_nt_kernel(Bf16Args a) {
    constexpr int NW = WM * WN, RA = TM / WM / 32, RB = TN / WN / 32, LOADS = (TM + TN) / 8 / NW;
    extern __shared__ uint8_t lds[];
    int tm, tn;
    if (!tile_of(blockIdx.x, a.num_m, a.num_n, 8, &tm, &tn)) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    const int wm = wave / WN, wn = wave % WN, m0 = tm * TM, n0 = tn * TN;
    const long pitch = (long)a.R * 2;
    const uint8_t *ab = a.a + m0 * pitch, *bb = a.b + n0 * pitch;
    uint32_t off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (wave + i * NW) * 8 + (lane >> 3);
        const int row = r < TM ? min(r, a.I - 1 - m0) : min(r - TM, a.J - 1 - n0);
        off[i] = (uint32_t)row * (uint32_t)pitch + (((lane & 7) ^ (lane >> 3)) << 4);
    }
    const int first = blockIdx.y * a.per_split, last = min(first + a.per_split, a.R / kStep);
    const int steps = (last - first) * P;
    auto load = [&](int t, int buf) {
        const int s = first + t / P, p = t % P;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r8 = wave + i * NW;
            dma16((r8 * 8 < TM ? ab + p * (a.I * pitch) : bb) + s * 128L, off[i], lds + buf * (TM + TN) * 128 + r8 * 1024);
        }
    };
    f32x16 acc[RA][RB];
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
    load(0, 0);
    for (int t = 0; t < steps; ++t) {
        dma_wait_barrier();
        if (t + 1 < steps) load(t + 1, (t + 1) & 1);
        const uint8_t *A = lds + (t & 1) * (TM + TN) * 128, *B = A + TM * 128;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            bf16x8 fa[RA], fb[RB];
#pragma unroll
            for (int i = 0; i < RA; ++i) fa[i] = __builtin_bit_cast(bf16x8, tile_chunk(A, (wm * RA + i) * 32 + l32, s * 2 + half));
#pragma unroll
            for (int j = 0; j < RB; ++j) fb[j] = __builtin_bit_cast(bf16x8, tile_chunk(B, (wn * RB + j) * 32 + l32, s * 2 + half));
#pragma unroll
            for (int i = 0; i < RA; ++i)
#pragma unroll
                for (int j = 0; j < RB; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
        }
    }
    T *c = (T *)a.c + blockIdx.y * ((long)a.I * a.J);
#pragma unroll
    for (int i = 0; i < RA; ++i)
#pragma unroll
        for (int j = 0; j < RB; ++j) {
            const int n = n0 + (wn * RB + j) * 32 + l32;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int m = m0 + (wm * RA + i) * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
                if (m < a.I && n < a.J) c[(long)m * a.J + n] = (T)acc[i][j][r];
            }
        }
}

// out[idx] = sum over the splits of part[s][idx], ascending
template <class T>
__global__ __launch_bounds__(256) void e4m3_bw_join_kernel(const float *part, int S, long total, T *out) {
    for (long idx = blockIdx.x * 256L + threadIdx.x; idx < total; idx += (long)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < S; ++s) v += part[s * total + idx];
        out[idx] = (T)v;
    }
}

// Few output tiles and a long reduction: the reduction is cut into S ranges whose partial sums are joined in ascending order.
struct Split {
    int S, per;
};
static Split plan_split(int I, int J, int R) {
    const int tiles = ceil_div(I, 128) * ceil_div(J, 128), steps = R / kStep;
    int S = 512 / tiles;
    if (S > steps / 8) S = steps / 8;
    if (S < 1) S = 1;
    Split p;
    p.per = ceil_div(steps, S);
    p.S = ceil_div(steps, p.per);
    return p;
}

template <int P, class T>
static int nt_product(const char *tag, const void *A, const void *B, T *C, float *part, int I, int J, int R, hipStream_t st) {
    constexpr int TM = 128, TN = 128, bytes = 2 * (TM + TN) * 128;
    const Split sp = plan_split(I, J, R);
    Bf16Args a = {(const uint8_t *)A, (const uint8_t *)B, sp.S > 1 ? (void *)part : (void *)C, I, J, R, ceil_div(I, TM), ceil_div(J, TN),
                  sp.per};
    const dim3 grid(tile_grid(a.num_m, a.num_n), sp.S);
    {
        ProfScope ps(tag, st);
        if (sp.S > 1) hipLaunchKernelGGL((e4m3_bw_nt_kernel<TM, TN, 2, 2, P, float>), grid, dim3(256), bytes, st, a);
        else hipLaunchKernelGGL((e4m3_bw_nt_kernel<TM, TN, 2, 2, P, T>), grid, dim3(256), bytes, st, a);
        const int rc = check_launch("e4m3_bw_nt_kernel");
        if (rc || sp.S == 1) return rc;
    }
    ProfScope ps("e4m3_bw_join", st);
    const long total = (long)I * J, blocks = (total + 255) / 256;
    hipLaunchKernelGGL((e4m3_bw_join_kernel<T>), dim3((unsigned)(blocks < 2048 ? blocks : 2048)), dim3(256), 0, st, part, sp.S, total, C);
    return check_launch("e4m3_bw_join_kernel");
}

static inline int up_step(int v) { return (v + kStep - 1) / kStep * kStep; }

struct BwPlan {
    size_t rows, cols, wt, xt, part, splits, total;
};
static BwPlan plan_bw(int M, int N, int K, int type) {
    const size_t P = pieces_of(type), Mp = up_step(M), Np = up_step(N);
    BwPlan p;
    p.rows = align_up(P * M * Np * 2, 256);
    p.cols = align_up(P * N * Mp * 2, 256);
    p.wt = align_up(K * Np * 2, 256);
    p.xt = align_up(K * Mp * 2, 256);
    p.part = align_up((size_t)ceil_div(M, 64) * N * 4, 256);
    const Split sx = plan_split(M, K, (int)Np), sw = plan_split(N, K, (int)Mp);
    const size_t bx = sx.S > 1 ? (size_t)sx.S * M * K * 4 : 0, bw = sw.S > 1 ? (size_t)sw.S * N * K * 4 : 0;
    p.splits = align_up(bx > bw ? bx : bw, 256);
    p.total = p.rows + p.cols + p.wt + p.xt + p.part + p.splits;
    return p;
}

}  // namespace phonlp

using namespace phonlp;

static bool bw_shape_ok(int M, int N, int K, int type) {
    return M > 0 && N > 0 && K > 0 && K <= (1 << 21) && N <= (1 << 21) && M <= (1 << 24) && type_ok(type);
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
    hipStream_t st = as_stream(stream);
    const BwPlan pl = plan_bw(M, N, K, type);
    const int Mp = up_step(M), Np = up_step(N), Kp = kp8_of(K), KB4 = kb4_of(K), tiles = ceil_div(M, 64);
    char *p = (char *)ws;
    uint16_t *rows = (uint16_t *)p, *cols = (uint16_t *)(p + pl.rows);
    __bf16 *wt = (__bf16 *)(p + pl.rows + pl.cols), *xt = (__bf16 *)((char *)wt + pl.wt);
    float *part = (float *)((char *)xt + pl.xt), *splits = (float *)((char *)part + pl.part);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int P = Pieces<T>::N;
        int rc;
        {
            ProfScope ps("e4m3_bw_dz", st);
            hipLaunchKernelGGL((e4m3_bw_dz_kernel<T>), dim3(tiles, Np / 64), dim3(256), 0, st, (const T *)dy, lddy, bits, ceil_div(N, 32), M,
                               N, Mp, Np, dx ? rows : nullptr, dw ? cols : nullptr, db ? part : nullptr);
            if ((rc = check_launch("e4m3_bw_dz_kernel"))) return rc;
        }
        if (db) {
            ProfScope ps("e4m3_bw_db", st);
            hipLaunchKernelGGL(e4m3_bw_db_kernel, dim3(ceil_div(N, 256)), dim3(256), 0, st, part, tiles, N, db);
            if ((rc = check_launch("e4m3_bw_db_kernel"))) return rc;
        }
        if (dx) {
            {
                ProfScope ps("e4m3_bw_transpose", st);
                hipLaunchKernelGGL(e4m3_bw_transpose_kernel, dim3(Np / 64, ceil_div(K, 64)), dim3(256), 0, st, (const uint8_t *)w_codes,
                                   w_exponents, N, K, Kp, KB4, Np, wt);
                if ((rc = check_launch("e4m3_bw_transpose_kernel"))) return rc;
            }
            if ((rc = nt_product<P, T>("e4m3_bw:dX", rows, wt, (T *)dx, splits, M, K, Np, st))) return rc;
        }
        if (dw) {
            {
                ProfScope ps("e4m3_bw_transpose", st);
                hipLaunchKernelGGL(e4m3_bw_transpose_kernel, dim3(Mp / 64, ceil_div(K, 64)), dim3(256), 0, st, (const uint8_t *)x_codes,
                                   x_exponents, M, K, Kp, KB4, Mp, xt);
                if ((rc = check_launch("e4m3_bw_transpose_kernel"))) return rc;
            }
            if ((rc = nt_product<P, float>("e4m3_bw:dW", cols, xt, dw, splits, N, K, Mp, st))) return rc;
        }
        return PHONLP_OK;
    });
}
