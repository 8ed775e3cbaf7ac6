// Rows quantised as a whole (trk_quantize_rows) and the dense int8 product (trk_gemm_i8).
#include "i8tile.hpp"

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

constexpr uint32_t ST_WAVES = 4;  // 8 or 16 waves are as fast from one row of 2560 values to 16 of 10240

// A workgroup takes 16 weight rows and up to 16 tokens: its waves share K and add their sums in LDS.
template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES* WAVE) void gemm_i8_strip_kernel(I8Gemm g) {
    __shared__ int32_t part[ST_WAVES][16][16];  // [wave][token][weight row]
    const uint32_t strips = (g.rows + 15) / 16, id = run_id();
    const uint32_t r0 = id % strips * 16, t0 = id / strips * 16;
    if (t0 >= g.m) return;  // the whole workgroup
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, c = lane % 16;
    const int8_t* wr = g.w + (r0 + c < g.rows ? r0 + c : g.rows - 1) * g.ldw;
    const int8_t* xr = g.q + (uint64_t)(t0 + c < g.m ? t0 + c : g.m - 1) * g.ldq;
    const uint32_t t = t0 + threadIdx.x / 16, r = r0 + threadIdx.x % 16;
    const bool out = threadIdx.x < 256 && t < g.m && r < g.rows;
    float sx = 0.0f, sw = 0.0f, b = 0.0f;
    if (out) sx = g.sx[t], sw = g.sw[r], b = g.bias ? g.bias[r] : 0.0f;
    i32x4 acc[1];
    strip_sums<1>({wr}, xr, g.k, wv, ST_WAVES, lane, acc);
    *reinterpret_cast<i32x4*>(&part[wv][c][lane / 16 * 4]) = acc[0];
    __syncthreads();
    if (!out) return;
    int32_t sum = 0;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) sum += part[i][threadIdx.x / 16][threadIdx.x % 16];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(g.y) + t * g.ldy + r;
    float v = i8_scaled(sum, sx, sw);
    if (g.bias) v += b;
    if (g.accumulate) v += O::get(*y);
    *y = O::put(v);
}

void launch_strip(const I8Gemm& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.rows + 15) / 16) * (((uint64_t)a.m + 15) / 16);
    const geo::Grid2 g = geo::grid_run(wgs, ST_WAVES * WAVE);
    const dim3 grid(g.x, g.y);
    if (a.dt == TRK_DT_F32)
        gemm_i8_strip_kernel<TRK_DT_F32><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        gemm_i8_strip_kernel<TRK_DT_BF16><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    else
        gemm_i8_strip_kernel<TRK_DT_F16><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
}

// The tiles' place in the launch: panels of eight weight tiles, activation tiles after one another inside each, so that
// the tiles that run at once on an XCD (a contiguous run of them) share rows of both in its L2.
__device__ __forceinline__ void tile_place(uint32_t idx, uint32_t tn, uint32_t tm, uint32_t& n, uint32_t& m) {
    const uint32_t panel = idx / (8 * tm), left = tn - panel * 8, w = left < 8 ? left : 8, rem = idx - panel * 8 * tm;
    n = panel * 8 + rem % w, m = rem / w;
}

template <typename Tile, uint32_t DT>
__global__ __launch_bounds__(Tile::T) void gemm_i8_tile_kernel(I8Gemm g) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::LDS];
    const uint32_t tn = (g.rows + Tile::BN - 1) / Tile::BN, tm = (g.m + Tile::BM - 1) / Tile::BM;
    uint32_t idx, n, m;
    if (!xcd_order_1d(tn * tm, idx, run_id())) return;  // the whole workgroup
    tile_place(idx, tn, tm, n, m);
    const uint32_t r0 = n * Tile::BN, t0 = m * Tile::BM, rl = g.rows - r0 - 1, tl = g.m - t0 - 1;  // the last rows there are
    Tile t;
    i32x4 rw[Tile::NA];
    uint32_t wo[Tile::NA], xo[Tile::NB];
#pragma unroll
    for (int i = 0; i < Tile::NA; i++) {
        const uint32_t r = t.load_row(i);
        rw[i] = buffer_at(g.w + r0 * g.ldw), wo[i] = (r < rl ? r : rl) * (uint32_t)g.ldw;
    }
#pragma unroll
    for (int i = 0; i < Tile::NB; i++) {
        const uint32_t r = t.load_row(i);
        xo[i] = (r < tl ? r : tl) * (uint32_t)g.ldq;
    }
    t.run(lds, rw, wo, buffer_at(g.q + t0 * g.ldq), xo, g.k, [&](int i) { return t.wn + 16 * i; });
    // every scale first (rows past the end: the last one's), so that the stores wait for memory once
    typedef Elem<DT> O;
    float sw[Tile::FN][4], bias[Tile::FN][4], sx[Tile::FM];
    auto col = [&](int i, int c) {
        const uint32_t r = t.wn + 16 * i + t.lane / 16 * 4 + c;
        return r0 + (r < rl ? r : rl);
    };
#pragma unroll
    for (int i = 0; i < Tile::FN; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) sw[i][c] = g.sw[col(i, c)], bias[i][c] = g.bias ? g.bias[col(i, c)] : 0.0f;
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        const uint32_t row = t.wm + 16 * j + t.lane % 16;
        sx[j] = g.sx[t0 + (row < tl ? row : tl)];
    }
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        const uint32_t row = t0 + t.wm + 16 * j + t.lane % 16;
        if (row >= g.m) continue;
        typename O::T* y = reinterpret_cast<typename O::T*>(g.y) + row * g.ldy;
        float v[Tile::FN][4];
#pragma unroll
        for (int i = 0; i < Tile::FN; i++)
#pragma unroll
            for (int c = 0; c < 4; c++) {
                v[i][c] = i8_scaled(t.acc[i][j][c], sx[j], sw[i][c]);
                if (g.bias) v[i][c] += bias[i][c];
            }
        if (g.accumulate) {
            typename O::T old[Tile::FN][4];
#pragma unroll
            for (int i = 0; i < Tile::FN; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) old[i][c] = y[col(i, c)];
#pragma unroll
            for (int i = 0; i < Tile::FN; i++)
#pragma unroll
                for (int c = 0; c < 4; c++) v[i][c] += O::get(old[i][c]);
        }
#pragma unroll
        for (int i = 0; i < Tile::FN; i++) {
            const uint32_t r = r0 + t.wn + 16 * i + t.lane / 16 * 4;
            store4<DT>(y + r, v[i], r < g.rows ? g.rows - r : 0, g.vec);
        }
    }
}

template <typename Tile>
void launch_tile(const I8Gemm& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.rows + Tile::BN - 1) / Tile::BN) * (((uint64_t)a.m + Tile::BM - 1) / Tile::BM);
    const geo::Grid2 g = geo::grid_run(wgs, Tile::T);
    const dim3 grid(g.x, g.y);
    if (a.dt == TRK_DT_F32)
        gemm_i8_tile_kernel<Tile, TRK_DT_F32><<<grid, Tile::T, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        gemm_i8_tile_kernel<Tile, TRK_DT_BF16><<<grid, Tile::T, 0, st>>>(a);
    else
        gemm_i8_tile_kernel<Tile, TRK_DT_F16><<<grid, Tile::T, 0, st>>>(a);
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
    switch (geo::gemm_i8_form(a.m, a.rows, a.k, a.ldw, a.ldq)) {
    case geo::I8_TILE_256: launch_tile<I8Tile<256, 256, 64, 128, 2>>(a, st); break;
    case geo::I8_TILE_128: launch_tile<I8Tile<128, 128, 64, 64, 2>>(a, st); break;
    case geo::I8_TILE_64: launch_tile<I8Tile<64, 64, 32, 32, 4>>(a, st); break;
    case geo::I8_TILE_32: launch_tile<I8Tile<64, 32, 16, 32, 4>>(a, st); break;
    default: launch_strip(a, st);
    }
    return hipGetLastError();
}

}  // namespace trk
