// Rows of floating values as the quantising kernels read and write them.
#pragma once

#include "i8.hpp"

namespace trk {

// Rows go by in pieces of 8 values, which may lie at any address (a slice of a wider tensor).
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_f32 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// 8 values of a row as they lie in memory, n of them there
template <uint32_t DT>
struct QuantPiece {
    static constexpr int W = DT == TRK_DT_F32 ? 8 : 4;
    uint32_t w[W];
    __device__ __forceinline__ void load(const typename Elem<DT>::T* p, uint32_t n) {
        if (n >= 8) {
            if constexpr (DT == TRK_DT_F32) {
                const u32x4_f32 a = *reinterpret_cast<const u32x4_f32*>(p), b = *reinterpret_cast<const u32x4_f32*>(p + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = a[i], w[4 + i] = b[i];
            } else {
                const u32x4_any a = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = a[i];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < W; i++) w[i] = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) {
            if (i >= n) continue;
            if constexpr (DT == TRK_DT_F32)
                w[i] = __float_as_uint(p[i]);
            else
                w[i / 2] |= (uint32_t)p[i] << (16 * (i % 2));
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (DT == TRK_DT_F32) return __uint_as_float(w[i]);
        return Elem<DT>::get((typename Elem<DT>::T)(w[i / 2] >> (16 * (i % 2))));
    }
    // the largest magnitude so far, as bits of the type: two 16-bit ones side by side
    __device__ __forceinline__ uint32_t most(uint32_t top) const {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < W; i++) {
            if constexpr (DT == TRK_DT_F32) {
                const uint32_t b = w[i] & 0x7fffffffu;
                top = b > top ? b : top;
            } else {
                const u16x2 b = __builtin_bit_cast(u16x2, w[i] & 0x7fff7fffu);
                top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), b));
            }
        }
        return top;
    }
    static __device__ __forceinline__ uint32_t most32(uint32_t top) {  // as bits of a float
        if constexpr (DT == TRK_DT_F32) return top;
        const uint32_t lo = top & 0xffffu, hi = top >> 16;
        return __float_as_uint(Elem<DT>::get((typename Elem<DT>::T)(lo > hi ? lo : hi)));
    }
};

}  // namespace trk
