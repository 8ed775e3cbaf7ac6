// The 8-bit products with a scale per token and per channel: what their kernels share.
//
// y[i][r] = s_i s_r sum_j q[i][j] w[r][j].  The sum is an exact 32-bit integer (k <= 131071: 2^14 k < 2^31), so it may be
// split over lanes, waves and matrix instructions in any order, K's order included: a lane's 16 bytes of a weight row meet
// the same 16 bytes of an activation row in v_mfma_i32_16x16x64_i8, whichever of the instruction's k they stand for.
// Only the scaling rounds: ((float)sum * s_i) * s_r, each step to 32 bits, then y's type.
#pragma once

#include "common.hpp"

namespace trk {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// C += A B: lane l holds 16 bytes of A's row l % 16 and of B's column l % 16 (the same k of both), and rows 4 (l / 16) ..
// + 3 of C's column l % 16.
__device__ __forceinline__ i32x4 mfma_i8(i32x4 a, i32x4 b, i32x4 c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}

// The first n (0..16) bytes of v, zeros behind them: 16-byte pieces past a row's end multiply to nothing.
__device__ __forceinline__ i32x4 first_bytes(i32x4 v, uint32_t n) {
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t b = n > 4 * j ? n - 4 * j : 0u;
        v[j] = b >= 4 ? v[j] : v[j] & (int)((1u << (8 * b)) - 1u);
    }
    return v;
}

__device__ __forceinline__ float i8_scaled(int32_t acc, float sx, float sw) { return ((float)acc * sx) * sw; }

// One value of an element type (TRK_DT_*), rounded to nearest even.
template <uint32_t DT>
struct Elem;
template <>
struct Elem<TRK_DT_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<TRK_DT_BF16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ uint16_t put(float v) { return __builtin_bit_cast(uint16_t, (__bf16)v); }
};
template <>
struct Elem<TRK_DT_F16> {
    typedef uint16_t T;
    static __device__ __forceinline__ float get(uint16_t v) { return h2f(v); }
    static __device__ __forceinline__ uint16_t put(float v) { return f2h(v); }
};

// silu(g) u in 32 bits
__device__ __forceinline__ float swiglu(float g, float u) { return silu512(g) * u; }

}  // namespace trk
