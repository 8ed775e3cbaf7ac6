// Rows quantised as a whole (trk_quantize_rows) and the dense int8 product (trk_gemm_i8).
#include "i8.hpp"

namespace trk {

namespace {

// ============================================================================================
// rows to int8
// ============================================================================================

// 127 x / top rounded to nearest, ties to even, as exact arithmetic would.  In 32 bits the quotient is off by
// at most 2 ulp of 128 (2^-15); within 2^-12 of a border (a half) it is taken again in 64 bits, where it is right: 127 x
// is exact, and a quotient of a 31-bit and a 24-bit integer that is no tie is further than 2^-32 from one.
__device__ __forceinline__ int32_t quant_one(float x, float top, float inv) {
    const float t = x * inv, r = __builtin_rintf(t);
    if (__builtin_fabsf(__builtin_fabsf(t - r) - 0.5f) > 0x1p-12f) return (int32_t)r;
    return (int32_t)::rint((double)x * 127.0 / (double)top);
}

constexpr float QUANT_LEAST = 127.0f * 0x1p-126f;  // the least magnitude whose scale is a normal number
constexpr uint32_t QUANT_T = 256;

template <uint32_t DT>
__global__ __launch_bounds__(QUANT_T) void quantize_whole_rows_kernel(const typename Elem<DT>::T* __restrict__ x,
                                                                      uint64_t ldx, uint32_t m, uint32_t k,
                                                                      int8_t* __restrict__ q, uint64_t ldq,
                                                                      float* __restrict__ scale) {
    __shared__ uint32_t part[QUANT_T / WAVE];
    const uint32_t row = run_id(), tid = threadIdx.x;
    if (row >= m) return;  // the whole workgroup
    const auto* xr = x + row * ldx;
    uint32_t top = 0;  // magnitudes as bit patterns: NaN above infinity above every number
    for (uint32_t i = tid; i < k; i += QUANT_T) {
        const uint32_t b = __float_as_uint(Elem<DT>::get(xr[i])) & 0x7fffffffu;
        top = b > top ? b : top;
    }
    top = wave_max_u32(top);
    if (tid % WAVE == 0) part[tid / WAVE] = top;
    __syncthreads();
#pragma unroll
    for (uint32_t i = 0; i < QUANT_T / WAVE; i++) top = part[i] > top ? part[i] : top;
    const float t = __uint_as_float(top);
    const bool poison = top >= 0x7f800000u, zero = poison || t < QUANT_LEAST;
    const float inv = zero ? 0.0f : 127.0f / t;
    if (tid == 0) scale[row] = poison ? __builtin_nanf("") : zero ? 0.0f : t / 127.0f;
    int8_t* qr = q + row * ldq;
    for (uint32_t i = tid; i < k; i += QUANT_T) qr[i] = zero ? 0 : (int8_t)quant_one(Elem<DT>::get(xr[i]), t, inv);
}

// ============================================================================================
// the dense product
// ============================================================================================

// A workgroup takes 16 weight rows and up to 16 tokens: its waves share K, 64 bytes at a time, and add their sums in
// LDS.
constexpr uint32_t ST_WAVES = 4;

template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES * WAVE) void gemm_i8_strip_kernel(I8Gemm g) {
    __shared__ int32_t part[ST_WAVES][16][16];  // [wave][token][weight row]
    const uint32_t strips = (g.rows + 15) / 16, id = run_id();
    const uint32_t r0 = id % strips * 16, t0 = id / strips * 16;
    if (t0 >= g.m) return;  // the whole workgroup
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, c = lane % 16, kg = lane / 16 * 16;
    const int8_t* wr = g.w + (r0 + c < g.rows ? r0 + c : g.rows - 1) * g.ldw;
    const int8_t* xr = g.q + (uint64_t)(t0 + c < g.m ? t0 + c : g.m - 1) * g.ldq;
    i32x4 acc = {0, 0, 0, 0};
    for (uint32_t at = wv * 64; at < g.k; at += ST_WAVES * 64) {
        const uint32_t o = at + kg, n = o < g.k ? (g.k - o < 16 ? g.k - o : 16) : 0, oc = n ? o : 0;
        acc = mfma_i8(*reinterpret_cast<const i32x4*>(wr + oc),
                      first_bytes(*reinterpret_cast<const i32x4*>(xr + oc), n), acc);
    }
    *reinterpret_cast<i32x4*>(&part[wv][c][lane / 16 * 4]) = acc;
    __syncthreads();
    const uint32_t t = t0 + threadIdx.x / 16, r = r0 + threadIdx.x % 16;
    if (t >= g.m || r >= g.rows) return;
    int32_t sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) sum += part[i][threadIdx.x / 16][threadIdx.x % 16];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(g.y) + t * g.ldy + r;
    float v = i8_scaled(sum, g.sx[t], g.sw[r]);
    if (g.bias) v += g.bias[r];
    if (g.accumulate) v += O::get(*y);
    *y = O::put(v);
}

}  // namespace

hipError_t launch_quantize_rows(const void* x, uint32_t dt, uint64_t ldx, uint32_t m, uint32_t k, int8_t* q,
                                uint64_t ldq, float* scale, hipStream_t st) {
    const geo::Grid2 g = geo::grid_run(m, QUANT_T);
    const dim3 grid(g.x, g.y);
    if (dt == TRK_DT_F32)
        quantize_whole_rows_kernel<TRK_DT_F32><<<grid, QUANT_T, 0, st>>>((const float*)x, ldx, m, k, q, ldq, scale);
    else if (dt == TRK_DT_BF16)
        quantize_whole_rows_kernel<TRK_DT_BF16><<<grid, QUANT_T, 0, st>>>((const uint16_t*)x, ldx, m, k, q, ldq, scale);
    else
        quantize_whole_rows_kernel<TRK_DT_F16><<<grid, QUANT_T, 0, st>>>((const uint16_t*)x, ldx, m, k, q, ldq, scale);
    return hipGetLastError();
}

hipError_t launch_gemm_i8(const I8Gemm& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.rows + 15) / 16) * (((uint64_t)a.m + 15) / 16);
    const geo::Grid2 g = geo::grid_run(wgs, ST_WAVES * WAVE);
    const dim3 grid(g.x, g.y);
    if (a.dt == TRK_DT_F32)
        gemm_i8_strip_kernel<TRK_DT_F32><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        gemm_i8_strip_kernel<TRK_DT_BF16><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    else
        gemm_i8_strip_kernel<TRK_DT_F16><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace trk
