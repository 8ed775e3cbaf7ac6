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
typedef float f32x4 __attribute__((ext_vector_type(4)));

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

// U pieces of 64 bytes of an activation row and of NM matrices' rows, all requested before the first is needed.
template <uint32_t U, uint32_t NM>
__device__ __forceinline__ void strip_pieces(const int8_t* const (&wr)[NM], const int8_t* __restrict__ xr, uint32_t at,
                                             uint32_t step, i32x4 (&acc)[NM]) {
    i32x4 w[NM][U], x[U];
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
        x[u] = *reinterpret_cast<const i32x4*>(xr + at + u * step * 64);
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) w[i][u] = *reinterpret_cast<const i32x4*>(wr[i] + at + u * step * 64);
    }
    __builtin_amdgcn_sched_barrier(0);  // else some wait for others' registers
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) acc[i] = mfma_i8(w[i][u], x[u], acc[i]);
}

// The exact sums of 16 weight rows of NM matrices and 16 activation rows over this wave's share of K: every `step`-th 64
// bytes from the first-th on.  wr, xr: this lane's row of each (row lane % 16).
template <uint32_t NM>
__device__ __forceinline__ void strip_sums(const int8_t* const (&wr)[NM], const int8_t* __restrict__ xr, uint32_t k,
                                           uint32_t first, uint32_t step, uint32_t lane, i32x4 (&acc)[NM]) {
#pragma unroll
    for (uint32_t i = 0; i < NM; i++) acc[i] = i32x4{0, 0, 0, 0};
    const uint32_t kg = lane / 16 * 16, whole = k / 64;
    uint32_t n = first < whole ? (whole - first + step - 1) / step : 0, at = first * 64 + kg;  // whole pieces of this wave
    for (; n >= 8; n -= 8, at += 8 * step * 64) strip_pieces<8, NM>(wr, xr, at, step, acc);
    if (n & 4) strip_pieces<4, NM>(wr, xr, at, step, acc), at += 4 * step * 64;
    if (n & 2) strip_pieces<2, NM>(wr, xr, at, step, acc), at += 2 * step * 64;
    if (n & 1) strip_pieces<1, NM>(wr, xr, at, step, acc);
    if (k % 64 && whole % step == first) {  // the row's end
        const uint32_t o = whole * 64 + kg, oc = o < k ? o : 0;
        const i32x4 x = first_bytes(*reinterpret_cast<const i32x4*>(xr + oc), o < k ? (k - o < 16 ? k - o : 16) : 0);
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) acc[i] = mfma_i8(*reinterpret_cast<const i32x4*>(wr[i] + oc), x, acc[i]);
    }
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

// silu(g) u in 32 bits.  Below -80, where silu512's exponential is soon held (at 88.3) and silu would fall no further, it is
// g e^g (1 + e^g is 1 there): e^g = 2^n e^r, and the power of two goes in last, so that the product rounds once where it
// ends among the smallest numbers.  u may be 2^128, g e^r is below 2^10; below -400 nothing is left for any u.
__device__ __forceinline__ float swiglu_far(float g, float u) {
    g = __builtin_fmaxf(g, -400.0f);
    const float n = __builtin_rintf(g * 1.442695041f);
    const float r = __builtin_fmaf(-n, 1.42860677e-6f, __builtin_fmaf(-n, 0.693145752f, g));
    return __builtin_ldexpf(g * 0x1p-16f * exp512(r) * u, (int)n + 16);
}
__device__ __forceinline__ float swiglu(float g, float u) { return g < -80.0f ? swiglu_far(g, u) : silu512(g) * u; }
// Of four, with one test for the wave: a branch a value costs the tiles 3 % (4096 tokens of 10 in 512 225 -> 231 us), this
// under 1 %.
__device__ __forceinline__ void swiglu4(const float (&g)[4], const float (&u)[4], float (&v)[4]) {
    const float least = __builtin_fminf(__builtin_fminf(g[0], g[1]), __builtin_fminf(g[2], g[3]));
#pragma unroll
    for (int c = 0; c < 4; c++) v[c] = silu512(g[c]) * u[c];
    if (__builtin_expect(__ballot(least < -80.0f) != 0, 0))
#pragma unroll
        for (int c = 0; c < 4; c++) v[c] = g[c] < -80.0f ? swiglu_far(g[c], u[c]) : v[c];
}

}  // namespace trk
