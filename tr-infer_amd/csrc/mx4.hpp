// Microscaled 4-bit rows and their products: what the kernels share.
//
// A row is blocks of 32 values: 16 bytes, two values a byte, the first in the low half, and a scale byte s that stands for
// 2^(s - 127) (255: NaN).  A value is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  The matrix instructions take both as they
// are: a lane's operand is one block of one row and its scale byte, and sum_32 a b 2^(sa + sb - 254) of the blocks goes into the 32-bit
// sum.  Which of the instruction's k a block stands for does not matter as long as both operands agree, so a lane may hold any.
//
// Products of two 4-bit values have at most six bits, a block's sum of them eleven: only adding blocks rounds.
#pragma once

#include "i8.hpp"

namespace trk {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr uint32_t MX_BLOCK = 32, MX_ONE = 127;  // values of a block; the scale byte of 1
constexpr int MX_FP4 = 4;                        // the operands' format

__host__ __device__ inline uint32_t mx_blocks(uint32_t k) { return k / MX_BLOCK + (k % MX_BLOCK ? 1u : 0u); }

__device__ __forceinline__ i32x8 mx_operand(i32x4 v) { return i32x8{v[0], v[1], v[2], v[3], 0, 0, 0, 0}; }

// C += A B: lane l holds a block of A's row l % 16 and of B's column l % 16, the four lane groups four blocks; rows 4 (l / 16)
// .. + 3 of C's column l % 16.
__device__ __forceinline__ f32x4 mfma_mx4(i32x4 a, uint32_t sa, i32x4 b, uint32_t sb, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(a), mx_operand(b), c, MX_FP4, MX_FP4, 0, (int)sa, 0, (int)sb);
}

// The sum is made here, by the whole wave: sunk into a branch that lanes part at, the instructions' operands would be made in the
// lanes that take it alone.
__device__ __forceinline__ void mx_here(f32x4& c) { asm volatile("" : "+v"(c)); }

// 2^(s - 127), NaN for 255
__device__ __forceinline__ float mx_scale(uint32_t s) {
    return s == 255u ? __builtin_nanf("") : s ? __uint_as_float(s << 23) : 0x1p-127f;
}

// A lane's row of a stack of 4-bit matrices
struct Mx4Row {
    const uint8_t *q, *s;
};

typedef uint32_t u32x4_s __attribute__((ext_vector_type(4), aligned(4)));  // sixteen scale bytes

// A unit of a row: sixteen blocks as four matrix instructions take them, lane group g the block 4 u + g of instruction u.  The
// scales come in one load (one byte a lane is a load as slow each); the lane's byte of word u is its group's.
constexpr uint32_t MX_UNIT = 16;
struct Mx4Unit {
    i32x4 q[4];
    u32x4_s s;
    __device__ __forceinline__ void load(const Mx4Row& w, uint32_t unit, uint32_t g) {
        const uint64_t b = (uint64_t)MX_UNIT * unit;
        s = *reinterpret_cast<const u32x4_s*>(w.s + b);
#pragma unroll
        for (int u = 0; u < 4; u++) q[u] = *reinterpret_cast<const i32x4*>(w.q + 16 * (b + 4 * u + g));
    }
    __device__ __forceinline__ uint32_t scale(int u, uint32_t g) const { return s[u] >> (8 * g); }
};
// A lane's block of the four from 4 q on (one at least is there), past the row's end the first and the scale 1: what it meets is zero.
// (The compiler has the scale's load in the lanes' choice and waits for it there: a row's end that is no whole unit costs a trip to
// memory for each four blocks and matrix.)
struct Mx4Block {
    i32x4 q;
    uint32_t s;
    __device__ __forceinline__ void load(const Mx4Row& w, uint32_t at, uint32_t g, uint32_t nb) {
        const uint64_t b = 4ull * at;
        const bool in = b + g < nb;
        q = *reinterpret_cast<const i32x4*>(w.q + 16 * (b + (in ? g : 0)));
        const uint32_t word = *reinterpret_cast<const uint32_t*>(w.s + b);
        s = in ? word >> (8 * g) : MX_ONE;
    }
};

// U units of NM matrices' rows and of an activation row, all requested before the first is needed.
template <uint32_t U, uint32_t NM>
__device__ __forceinline__ void mx4_units(const Mx4Row (&w)[NM], const Mx4Row& x, uint32_t at, uint32_t step, uint32_t g,
                                          f32x4 (&acc)[NM]) {
    Mx4Unit wu[NM][U], xu[U];
#pragma unroll
    for (uint32_t v = 0; v < U; v++) {
        xu[v].load(x, at + v * step, g);
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) wu[i][v].load(w[i], at + v * step, g);
    }
    __builtin_amdgcn_sched_barrier(0);  // else some wait for others' registers
#pragma unroll
    for (uint32_t v = 0; v < U; v++)
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (uint32_t i = 0; i < NM; i++) acc[i] = mfma_mx4(wu[i][v].q[u], wu[i][v].scale(u, g), xu[v].q[u], xu[v].scale(u, g), acc[i]);
}

// The sums of 16 weight rows of NM matrices and 16 activation rows over this wave's share of K (nb blocks a row): every `step`-th
// unit from the first-th on, and of what is left every `step`-th four blocks.  w, x: this lane's row of each (row lane % 16).
template <uint32_t NM>
__device__ __forceinline__ void mx4_strip(const Mx4Row (&w)[NM], const Mx4Row& x, uint32_t nb, uint32_t first, uint32_t step,
                                          uint32_t lane, f32x4 (&acc)[NM]) {
#pragma unroll
    for (uint32_t i = 0; i < NM; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t g = lane / 16, units = nb / MX_UNIT;
    uint32_t n = first < units ? (units - first + step - 1) / step : 0, at = first;  // this wave's units
    for (; n >= 2; n -= 2, at += 2 * step) mx4_units<2, NM>(w, x, at, step, g, acc);
    if (n) mx4_units<1, NM>(w, x, at, step, g, acc);
    for (uint32_t q = MX_UNIT / 4 * units + first; 4 * q < nb; q += step) {
        Mx4Block wl[NM], xl;
        xl.load(x, q, g, nb);
        if (4 * q + g >= nb) xl.q = i32x4{0, 0, 0, 0};
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) wl[i].load(w[i], q, g, nb);
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) acc[i] = mfma_mx4(wl[i].q, wl[i].s, xl.q, xl.s, acc[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < NM; i++) mx_here(acc[i]);
}

}  // namespace trk
