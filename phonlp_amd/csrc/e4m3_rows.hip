// Matrix <-> e4m3 image (e4m3.h): the operand form of phonlp_linear_e4m3 and, at a quarter of fp32's bytes, the checkpoint of a
// layer's input that phonlp_linear_e4m3_backward reads.  One pass, memory-bound: a block of 128 columns is held by 32 (fp32) or 16
// (16-bit types) neighbouring lanes with one 16-byte load each, its largest magnitude is found with lane permutations, and the
// codes leave as one 4- or 8-byte store per lane.  32768 x 868 fp32: 29 us to the image, 26 back, 5 TB/s, the rate of a copy.
#include <type_traits>

#include "e4m3.h"

namespace phonlp {

// Largest value over the aligned group of 16 lanes that a lane belongs to (quads, then halves, then the row mirrored).
__device__ __forceinline__ int group16_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));   // quad_perm [1,0,3,2]
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));   // quad_perm [2,3,0,1]
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));  // row_half_mirror
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));  // row_mirror
    return v;
}

template <class T>
__global__ __launch_bounds__(256) void e4m3_rows_kernel(const T *x, long ldx, int M, int K, int KB, int KB4, uint8_t *codes,
                                                        uint8_t *exponents) {
    constexpr int VEC = 16 / sizeof(T), LANES = kBlock8 / VEC, UNROLL = 4;
    typedef typename Vec<T, VEC>::type V;
    const int sub = threadIdx.x & (LANES - 1);
    const long groups = (long)gridDim.x * (256 / LANES), total = (long)M * KB;
    for (long g = (long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES; g < total; g += groups * UNROLL) {
        float v[UNROLL][VEC];
        int row[UNROLL], blk[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long it = g + u * groups;
#pragma unroll
            for (int i = 0; i < VEC; ++i) v[u][i] = 0.f;
            if (it >= total) continue;
            row[u] = total < (1L << 31) ? (int)((unsigned)it / (unsigned)KB) : (int)(it / KB);
            blk[u] = (int)(it - (long)row[u] * KB);
            const int k = blk[u] * kBlock8 + sub * VEC;
            const T *p = x + row[u] * ldx + k;
            if (k + VEC <= K) {
                const V t = *reinterpret_cast<const V *>(p);
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[u][i] = (float)t[i];
            } else {
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (k + i < K) v[u][i] = (float)p[i];
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long it = g + u * groups;
            int a = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const int bits = __float_as_int(v[u][i]) & 0x7FFFFFFF;
                a = max(a, bits < 0x7F800000 ? bits : 0);
            }
            a = group16_max(a);
            if (LANES == 32) a = max(a, __shfl_xor(a, 16));
            // a = 1.m * 2^(E-127) <= 448 * 2^e = 1.75 * 2^(8+e)  <=>  e + 127 >= E - 8, one more if 1.m > 1.75
            const int e = max((a >> 23) - 8 + ((a & 0x7FFFFF) > 0x600000 ? 1 : 0), 1);
            if (it >= total) continue;
            const float scale = exp2_biased(254 - e);
            uint32_t out[VEC / 4];
#pragma unroll
            for (int q = 0; q < VEC / 4; ++q) {
                float s[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float t = v[u][4 * q + i];
                    float w = t * scale;
                    // e = 120: codes from 256 up would stand for values past fp32's largest
                    if (e == 247) w = fminf(fmaxf(w, -240.f), 240.f);
                    s[i] = (__float_as_int(t) & 0x7F800000) == 0x7F800000 ? __int_as_float(0x7FC00000) : w;
                }
                int w = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
                out[q] = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], w, true);
            }
            uint8_t *c = codes + (long)row[u] * (KB * kBlock8) + blk[u] * kBlock8 + sub * VEC;
            if (VEC == 4) *reinterpret_cast<uint32_t *>(c) = out[0];
            else *reinterpret_cast<uint2 *>(c) = make_uint2(out[0], out[VEC / 4 - 1]);
            // the block's exponent, and behind a row's last block the padding ones
            if (sub == 0) exponents[(long)row[u] * KB4 + blk[u]] = (uint8_t)e;
            else if (blk[u] == KB - 1 && sub < KB4 - KB + 1) exponents[(long)row[u] * KB4 + blk[u] + sub] = 127;
        }
    }
}

// Values of an image, in T.  16-bit types saturate: an e4m3 code may stand for a little more than the block's largest entry was
// (fp16: 65504 becomes 256 * 2^8).  fp32's largest is kept by the quantiser itself.  RAGGED: K is no multiple of VEC, and a row's last
// vector begins VEC columns before its end, some of them its neighbour's as well, perhaps in two blocks (32768 x 867 bf16: 17 us, one
// column a thread 57).
template <class T, int VEC, bool RAGGED>
__global__ __launch_bounds__(256) void e4m3_values_kernel(const uint8_t *codes, const uint8_t *exponents, int M, int K, int Kp, int KB4,
                                                          T *out) {
    typedef typename Vec<T, VEC>::type V;
    const int per_row = (K + VEC - 1) / VEC;
    const long total = (long)M * per_row, step = (long)gridDim.x * 256;
    constexpr int UNROLL = 4;
    for (long g = (long)blockIdx.x * 256 + threadIdx.x; g < total; g += step * UNROLL) {
        uint8_t c[UNROLL][VEC];
        uint8_t e[UNROLL], e2[UNROLL];
        int border[UNROLL];  // from this one on the vector's columns are the next block's
        long at[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const long it = g + u * step;
            if (it >= total) continue;
            const long row = total < (1L << 31) ? (long)((unsigned)it / (unsigned)per_row) : it / per_row;
            int k = (int)(it - row * per_row) * VEC;
            if (RAGGED) k = min(k, K - VEC);
            at[u] = row * K + k;
            __builtin_memcpy(c[u], codes + row * Kp + k, VEC);
            e[u] = exponents[row * KB4 + (k >> 7)];
            if (RAGGED) {
                e2[u] = exponents[row * KB4 + ((k + VEC - 1) >> 7)];
                border[u] = 128 - (k & 127);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (g + u * step >= total) continue;
            const float scale = exp2_biased(e[u] < 1 ? 1 : e[u]), scale2 = RAGGED ? exp2_biased(e2[u] < 1 ? 1 : e2[u]) : scale;
            V o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                float v = __builtin_amdgcn_cvt_f32_fp8(c[u][i], 0) * (RAGGED && i >= border[u] ? scale2 : scale);
                if (sizeof(T) == 2) {
                    const float top = __is_same(T, _Float16) ? 65504.f : 3.3895313892515355e38f;
                    v = v > top ? top : v < -top ? -top : v;  // keeps NaN
                }
                o[i] = (T)v;
            }
            *reinterpret_cast<V *>(out + at[u]) = o;
        }
    }
}

}  // namespace phonlp

using namespace phonlp;

extern "C" int phonlp_e4m3_kp(int K) { return K > 0 && K <= (1 << 22) ? kp8_of(K) : 0; }
extern "C" int phonlp_e4m3_kb(int K) { return K > 0 && K <= (1 << 22) ? kb4_of(K) : 0; }

static int rows_grid(long work_items, int per_block) {
    const long blocks = (work_items + per_block - 1) / per_block;
    return (int)(blocks < 2048 ? (blocks < 1 ? 1 : blocks) : 2048);
}

extern "C" int phonlp_e4m3_rows(const void *x, int type, long ldx, int rows, int K, void *codes, uint8_t *exponents, void *stream) {
    if (!x || !codes || !exponents || !type_ok(type) || rows <= 0 || K <= 0 || K > (1 << 22) || ldx < K)
        return fail(PHONLP_ERR_SHAPE, "e4m3_rows: bad argument");
    if ((uintptr_t)x % type_bytes(type) || ((uintptr_t)codes & 15) || ((uintptr_t)exponents & 3))
        return fail(PHONLP_ERR_SHAPE, "e4m3_rows: x must have its type's alignment, codes 16 bytes, exponents 4 bytes");
    hipStream_t st = as_stream(stream);
    ProfScope ps("e4m3_rows", st);
    const int KB = kp8_of(K) / kBlock8;
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        hipLaunchKernelGGL((e4m3_rows_kernel<T>), dim3(rows_grid((long)rows * KB, 256 / (kBlock8 * (int)sizeof(T) / 16))), dim3(256), 0,
                           st, (const T *)x, ldx, rows, K, KB, kb4_of(K), (uint8_t *)codes, exponents);
        return check_launch("e4m3_rows_kernel");
    });
}

extern "C" int phonlp_e4m3_values(const void *codes, const uint8_t *exponents, int rows, int K, int type, void *out, void *stream) {
    if (!codes || !exponents || !out || !type_ok(type) || rows <= 0 || K <= 0 || K > (1 << 22))
        return fail(PHONLP_ERR_SHAPE, "e4m3_values: bad argument");
    if ((uintptr_t)out % type_bytes(type) || ((uintptr_t)codes & 15) || ((uintptr_t)exponents & 3))
        return fail(PHONLP_ERR_SHAPE, "e4m3_values: out must have its type's alignment, codes 16 bytes, exponents 4 bytes");
    hipStream_t st = as_stream(stream);
    ProfScope ps("e4m3_values", st);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        constexpr int VEC = 16 / sizeof(T);
        const uint8_t *c = (const uint8_t *)codes;
        auto launch = [&](auto vec, auto ragged) {
            constexpr int V = decltype(vec)::value;
            hipLaunchKernelGGL((e4m3_values_kernel<T, V, decltype(ragged)::value>), dim3(rows_grid((long)rows * ((K + V - 1) / V), 256)),
                               dim3(256), 0, st, c, exponents, rows, K, kp8_of(K), kb4_of(K), (T *)out);
        };
        if (K % VEC == 0) launch(std::integral_constant<int, VEC>{}, std::false_type{});
        else if (K > VEC) launch(std::integral_constant<int, VEC>{}, std::true_type{});
        else launch(std::integral_constant<int, 1>{}, std::false_type{});
        return check_launch("e4m3_values_kernel");
    });
}
