// Images of matrices in 8-bit floating point (OCP e4m3) with one power-of-two scale per row and block of 128 columns.
//
// Block of x: a = its largest finite magnitude, e = the smallest integer >= -126 with a <= 448 * 2^e, code = e4m3(x * 2^-e)
// (nearest even).  A power of two, not a / 448: the scaling is then exact and the value code * 2^e is exact in fp32 and, from its
// smallest step 2^-133 on, in bf16 (the conversion v_cvt_scalef32 applies it), while e4m3 is a floating-point code whose relative
// precision does not depend on where in its range a block lies.
//   codes     [rows][Kp]   Kp = K rounded up to 128, zero behind K (one block = one 128-byte line)
//   exponents [rows][KB4]  e + 127 as a byte, KB4 = Kp / 128 rounded up to 4 (four blocks' exponents = one dword), 127 behind
#pragma once
#include "common.h"

namespace phonlp {

constexpr int kBlock8 = 128;

__host__ __device__ inline int kp8_of(int K) { return (K + 127) / 128 * 128; }
__host__ __device__ inline int kb4_of(int K) { return ((K + 127) / 128 + 3) / 4 * 4; }

inline int type_bytes(int type) { return type == PHONLP_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == PHONLP_F32 || type == PHONLP_BF16 || type == PHONLP_F16; }

// Calls f with a value of the element type `type` names.
template <class F>
inline int with_type(int type, F &&f) {
    switch (type) {
        case PHONLP_F32: return f(float{});
        case PHONLP_BF16: return f(__bf16{});
        default: return f(_Float16{});
    }
}

#ifdef __HIPCC__
// Vectors that need only their element's alignment (global memory takes dword-wide accesses at any address).
template <class T, int N>
struct Vec {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};

__device__ __forceinline__ float exp2_biased(int e) { return __int_as_float(e << 23); }  // 2^(e - 127), 1 <= e <= 254
#endif

}  // namespace phonlp
