// Rows quantised as a whole (trk_quantize_rows) and the dense int8 product (trk_gemm_i8).
#include "i8tile.hpp"
#include "rows.hpp"

namespace trk {

namespace {

// ============================================================================================
// rows to int8
// ============================================================================================

// 127 x / top rounded to nearest, ties to even, as exact arithmetic would.  In 32 bits the quotient carries three
// roundings, under 2^-15 in all; one that near to a border (a half) is taken again in 64 bits, where it is right: 127 x is
// exact, and a quotient of a 31-bit and a 24-bit integer that is no tie is further than 2^-32 from one.
__device__ __forceinline__ float quant_exact(float x, float top) { return (float)::rint((double)x * 127.0 / (double)top); }
constexpr float QUANT_BORDER = 0.5f - 0x1p-15f;  // |t - rint(t)| above it: near a border

constexpr float QUANT_LEAST = 127.0f * 0x1p-126f;  // the least magnitude whose scale is a normal number
constexpr uint32_t QUANT_T = 256, QUANT_LONG_T = 1024;
constexpr float QUANT_MAGIC = 12582912.0f;

struct QuantScale {
    float top, inv, scale;
};
__device__ __forceinline__ QuantScale quant_scale(uint32_t top) {  // a magnitude's bits: NaN above infinity above every number
    const float t = __uint_as_float(top);
    const bool poison = top >= 0x7f800000u, zero = poison || t < QUANT_LEAST;
    return QuantScale{t, zero ? 0.0f : 127.0f / t, poison ? __builtin_nanf("") : zero ? 0.0f : t / 127.0f};
}

// The largest of the workgroup's values (of a row's WAVES waves), or of the wave's where those are one.
template <uint32_t WAVES>
__device__ __forceinline__ uint32_t quant_top(uint32_t top, uint32_t* part) {
    top = wave_max_u32(top);
    if constexpr (WAVES > 1) {
        if (threadIdx.x % WAVE == 0) part[threadIdx.x / WAVE] = top;
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < WAVES; i++) top = part[i] > top ? part[i] : top;
    }
    return top;
}
// A piece of a row scaled, rounded and written, n of its values there: t + 1.5 2^23 has rint(t), as an 8-bit integer, in its
// low byte.
template <uint32_t DT>
__device__ __forceinline__ void quant_write(const QuantPiece<DT>& v, const QuantScale& s, int8_t* q, uint32_t n) {
    uint32_t r[8];
    float far = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float t = v.get(i) * s.inv, u = t + QUANT_MAGIC;
        r[i] = __float_as_uint(u);
        far = __builtin_fmaxf(far, __builtin_fabsf(t - (u - QUANT_MAGIC)));
    }
    if (far > QUANT_BORDER) {
        asm volatile("");  // else the compiler takes the 64-bit quotients of every value and selects: 40960 x 512 18 -> 23 us
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = (uint32_t)(int)quant_exact(v.get(i), s.top);
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {  // the low bytes of four words
        const uint32_t lo = __builtin_amdgcn_perm(r[4 * i + 1], r[4 * i], 0x0c0c0400u);
        const uint32_t hi = __builtin_amdgcn_perm(r[4 * i + 3], r[4 * i + 2], 0x04000c0cu);
        w[i] = s.inv == 0.0f ? 0 : lo | hi;
    }
    if (n >= 8) {
        *reinterpret_cast<u32x2_any*>(q) = u32x2_any{w[0], w[1]};
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++)
            if (i < n) q[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
    }
}

// Rows that TPR threads hold in registers, PC pieces a thread: read once, written once, for memory is what bounds it (8192 x
// 4096: bf16 24 us, 4.2 TB/s, f32 31 us, 5.4 TB/s; read twice, value by value, 57 in bf16).  Beside it stand 8 instructions a
// value.  Few rows take the time of one row's chain (4 x 2048: 2.4 us).  Rows over 16384 by 1024 threads: 1024 x 28672 in bf16 24
// us (held) against 69 by 256 threads that read them twice, value by value.
template <uint32_t DT, uint32_t TPR, uint32_t PC>
__global__ __launch_bounds__(TPR > QUANT_T ? TPR : QUANT_T) void quantize_held_rows_kernel(
    const typename Elem<DT>::T* __restrict__ x, uint64_t ldx, uint32_t m, uint32_t k, int8_t* __restrict__ q, uint64_t ldq,
    float* __restrict__ scale) {
    constexpr uint32_t T = TPR > QUANT_T ? TPR : QUANT_T;
    __shared__ uint32_t part[T / WAVE];
    const uint32_t row = run_id() * (T / TPR) + threadIdx.x / TPR, tid = threadIdx.x % TPR;
    if (row >= m) return;  // a whole wave, or the whole workgroup
    const auto* xr = x + row * ldx;
    QuantPiece<DT> v[PC];
#pragma unroll
    for (uint32_t p = 0; p < PC; p++) {
        const uint32_t at = (p * TPR + tid) * 8;
        v[p].load(xr + (at < k ? at : 0), at < k ? k - at : 0);
    }
    uint32_t top = 0;
#pragma unroll
    for (uint32_t p = 0; p < PC; p++) top = v[p].most(top);
    const QuantScale s = quant_scale(quant_top<TPR / WAVE>(QuantPiece<DT>::most32(top), part));
    if (tid == 0) scale[row] = s.scale;
    int8_t* qr = q + row * ldq;
#pragma unroll
    for (uint32_t p = 0; p < PC; p++) {
        const uint32_t at = (p * TPR + tid) * 8;
        if (at < k) quant_write(v[p], s, qr + at, k - at);
    }
}

// Rows too long to be held (over 32768): a workgroup each, every row read twice, the second time from a cache: 1024 x 65536 in
// bf16 60 us (3.4 TB/s), 300 x 131071 in f32 72.
template <uint32_t DT, uint32_t T, uint32_t PC>
__global__ __launch_bounds__(T) void quantize_long_rows_kernel(const typename Elem<DT>::T* __restrict__ x, uint64_t ldx,
                                                              uint32_t m, uint32_t k, int8_t* __restrict__ q, uint64_t ldq,
                                                              float* __restrict__ scale) {
    __shared__ uint32_t part[T / WAVE];
    const uint32_t row = run_id(), tid = threadIdx.x;
    if (row >= m) return;  // the whole workgroup
    const auto* xr = x + row * ldx;
    constexpr uint32_t STEP = PC * T * 8;
    QuantPiece<DT> v[PC];
    // the row from p on, `left` values of it: counted down, for sums of places near 2^32 do not fit 32 bits
    auto load = [&](const typename Elem<DT>::T* p, uint32_t left) {
#pragma unroll
        for (uint32_t i = 0; i < PC; i++) {
            const uint32_t at = (i * T + tid) * 8;
            v[i].load(p + (at < left ? at : 0), at < left ? left - at : 0);
        }
    };
    uint32_t top = 0;
    const auto* xp = xr;
    for (uint32_t left = k;; left -= STEP, xp += STEP) {
        load(xp, left);
#pragma unroll
        for (uint32_t i = 0; i < PC; i++) top = v[i].most(top);
        if (left <= STEP) break;
    }
    const QuantScale s = quant_scale(quant_top<T / WAVE>(QuantPiece<DT>::most32(top), part));
    if (tid == 0) scale[row] = s.scale;
    int8_t* qp = q + row * ldq;
    xp = xr;
    for (uint32_t left = k;; left -= STEP, xp += STEP, qp += STEP) {
        load(xp, left);
#pragma unroll
        for (uint32_t i = 0; i < PC; i++) {
            const uint32_t at = (i * T + tid) * 8;
            if (at < left) quant_write(v[i], s, qp + at, left - at);
        }
        if (left <= STEP) break;
    }
}

template <uint32_t DT>
void launch_quantize(const void* x, uint64_t ldx, uint32_t m, uint32_t k, int8_t* q, uint64_t ldq, float* scale,
                     hipStream_t st) {
    typedef typename Elem<DT>::T T;
    const uint32_t per = k <= 2048 ? QUANT_T / WAVE : 1;  // rows of a workgroup: a wave each while they fit its registers
    const uint32_t t = k <= 16384 ? QUANT_T : QUANT_LONG_T;
    const geo::Grid2 g = geo::grid_run(((uint64_t)m + per - 1) / per, t);
    const dim3 grid(g.x, g.y);
#define GO(TPR, PC) quantize_held_rows_kernel<DT, TPR, PC><<<grid, t, 0, st>>>((const T*)x, ldx, m, k, q, ldq, scale)
    if (k <= 512)
        GO(WAVE, 1);
    else if (k <= 1024)
        GO(WAVE, 2);
    else if (k <= 2048)
        GO(WAVE, 4);
    else if (k <= 4096)
        GO(QUANT_T, 2);
    else if (k <= 8192)
        GO(QUANT_T, 4);
    else if (k <= 16384)
        GO(QUANT_T, 8);
    else if (k <= 32768)
        GO(QUANT_LONG_T, 4);
    else
        quantize_long_rows_kernel<DT, QUANT_LONG_T, 4><<<grid, t, 0, st>>>((const T*)x, ldx, m, k, q, ldq, scale);
#undef GO
}

// ============================================================================================
// the dense product
// ============================================================================================

constexpr uint32_t ST_WAVES = 4;  // 8 or 16 waves are as fast from one row of 2560 values to 16 of 10240

// A workgroup takes 16 weight rows and up to 16 tokens: its waves share K and add their sums in LDS.  One trip to memory bounds
// it: [2560] x 1 token at k = 2560 4.2 us (3.6 where a cache holds the weights), at k = 12288 13.1 (10.4); [1024] x 16 at k = 512
// 2.7.
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

// Bound by the matrix cores where there are many rows (4096 x 12288 x 2560 126 us, 2050 TOP/s; 8192 cubed 433 us, 2540
// TOP/s: busy two thirds of the cycles, and the clock gives way, at 1.9 GHz), by their weights' way through the stages
// where there are few ([12288] x 1 at k = 2560 6.1 us from a cache, 10.3 from memory, 3.1 TB/s).  A workgroup per CU that
// goes on to its next tile, whose loads then fly while the last is written, was no faster (126.5 us, 436).
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
    t.template run<false, false>(lds, rw, wo, buffer_at(g.q + t0 * g.ldq), xo, g.k, 0, [&](int i) { return t.wn + 16 * i; });
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
    if (dt == TRK_DT_F32)
        launch_quantize<TRK_DT_F32>(x, ldx, m, k, q, ldq, scale, st);
    else if (dt == TRK_DT_BF16)
        launch_quantize<TRK_DT_BF16>(x, ldx, m, k, q, ldq, scale, st);
    else
        launch_quantize<TRK_DT_F16>(x, ldx, m, k, q, ldq, scale, st);
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
