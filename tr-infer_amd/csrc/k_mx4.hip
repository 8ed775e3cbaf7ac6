// Rows to microscaled 4-bit values and back (trk_quantize_mx4, trk_dequantize_mx4), and their dense product (trk_gemm_mx4).
#include "mx4tile.hpp"
#include "rows.hpp"

namespace trk {

namespace {

// ============================================================================================
// rows to 4-bit values, and back
// ============================================================================================

constexpr uint32_t MQ_T = 256, MQ_U = 4;  // threads; pieces of 8 values a thread

// The pieces of all rows in one run, `P` (a multiple of 4) a row: this thread's n-th is MQ_T behind the one before.
struct MxPlace {
    uint64_t row;
    uint32_t piece;
};
__device__ __forceinline__ MxPlace mx_first(uint32_t P) {
    const uint64_t f = (uint64_t)run_id() * (MQ_T * MQ_U);
    const uint64_t row = f / P;  // the workgroup's, as scalars
    const uint64_t piece = f - row * P + threadIdx.x;
    if (piece < P) return MxPlace{row, (uint32_t)piece};
    const uint32_t more = (uint32_t)piece / P;
    return MxPlace{row + more, (uint32_t)piece - more * P};
}
__device__ __forceinline__ void mx_next(MxPlace& p, uint32_t P, uint32_t rows, uint32_t pieces) {  // MQ_T = rows * P + pieces
    p.row += rows;
    if (p.piece >= P - pieces)
        p.row++, p.piece -= P - pieces;
    else
        p.piece += pieces;
}

// Four lanes hold a block, 8 values each; its largest magnitude by two DPP steps, its exponent from that one's bits, and the
// conversion instruction, which rounds to nearest even and holds magnitudes at 6, divides by the scale exactly (a power of two).
// One read, one write; a thread's four pieces are all requested before the first is needed.  8192 x 4096 bf16 15.9 us, 5.3 TB/s (the
// reads alone would be 11); 4 x 2048 f32 2.6: the trip to memory and back.
template <uint32_t DT>
__global__ __launch_bounds__(MQ_T) void quantize_mx4_kernel(const typename Elem<DT>::T* __restrict__ x, uint64_t ldx, uint32_t m,
                                                           uint32_t k, uint32_t P, uint32_t step_rows, uint32_t step_pieces,
                                                           uint8_t* __restrict__ q, uint64_t ldq, uint8_t* __restrict__ s,
                                                           uint64_t lds) {
    MxPlace at[MQ_U];
    QuantPiece<DT> v[MQ_U];
    at[0] = mx_first(P);
#pragma unroll
    for (uint32_t u = 1; u < MQ_U; u++) at[u] = at[u - 1], mx_next(at[u], P, step_rows, step_pieces);
#pragma unroll
    for (uint32_t u = 0; u < MQ_U; u++) {
        const uint64_t c = 8ull * at[u].piece;
        const bool in = at[u].row < m && c < k;
        v[u].load(x + (in ? at[u].row * ldx + c : 0), in ? (uint32_t)(k - c < 8 ? k - c : 8) : 0);
    }
#pragma unroll
    for (uint32_t u = 0; u < MQ_U; u++) {
        uint32_t top = QuantPiece<DT>::most32(v[u].most(0));
        auto more = [&](uint32_t o) { top = o > top ? o : top; };
        more((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xf, 0xf, false));  // lane ^ 1
        more((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xf, 0xf, false));  // lane ^ 2
        const bool poison = top >= 0x7f800000u;
        // floor(log2 top) - 2 + 127, from 0 on: a magnitude below 2^-125 is under 4 of the least scale, 2^-127
        const uint32_t e = top >> 23, scale = poison ? 255u : e < 2u ? 0u : e - 2u;
        const float f = mx_scale(poison ? MX_ONE : scale);
        uint32_t w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u].get(0), v[u].get(1), f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u].get(2), v[u].get(3), f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u].get(4), v[u].get(5), f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[u].get(6), v[u].get(7), f, 3);
        if (at[u].row >= m) continue;
        *reinterpret_cast<uint32_t*>(q + at[u].row * ldq + 4ull * at[u].piece) = poison ? 0u : w;
        if (at[u].piece % 4 == 0) s[at[u].row * lds + at[u].piece / 4] = (uint8_t)scale;
    }
}

// 8 values of a row, n of them there, at any address
template <uint32_t DT>
__device__ __forceinline__ void mx_store(typename Elem<DT>::T* y, const float (&v)[8], uint32_t n) {
    if (n >= 8) {
        if constexpr (DT == TRK_DT_F32) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                u32x4_f32 w;
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = __float_as_uint(v[4 * h + i]);
                *reinterpret_cast<u32x4_f32*>(y + 4 * h) = w;
            }
        } else {
            u32x4_any w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = (uint32_t)Elem<DT>::put(v[2 * i]) | (uint32_t)Elem<DT>::put(v[2 * i + 1]) << 16;
            *reinterpret_cast<u32x4_any*>(y) = w;
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; i++)
        if (i < n) y[i] = Elem<DT>::put(v[i]);
}

// The same pieces back; the conversion instruction multiplies by the scale, exactly.  8192 x 4096 to bf16 14.6 us, 5.8 TB/s, most
// of it the writes.
template <uint32_t DT>
__global__ __launch_bounds__(MQ_T) void dequantize_mx4_kernel(const uint8_t* __restrict__ q, uint64_t ldq,
                                                             const uint8_t* __restrict__ s, uint64_t lds, uint32_t m, uint32_t k,
                                                             uint32_t P, uint32_t step_rows, uint32_t step_pieces,
                                                             typename Elem<DT>::T* __restrict__ y, uint64_t ldy) {
    MxPlace at[MQ_U];
    uint32_t w[MQ_U], b[MQ_U];
    at[0] = mx_first(P);
#pragma unroll
    for (uint32_t u = 1; u < MQ_U; u++) at[u] = at[u - 1], mx_next(at[u], P, step_rows, step_pieces);
#pragma unroll
    for (uint32_t u = 0; u < MQ_U; u++) {
        const bool in = at[u].row < m;
        w[u] = *reinterpret_cast<const uint32_t*>(q + (in ? at[u].row * ldq + 4ull * at[u].piece : 0));
        b[u] = s[in ? at[u].row * lds + at[u].piece / 4 : 0];
    }
#pragma unroll
    for (uint32_t u = 0; u < MQ_U; u++) {
        const uint64_t c = 8ull * at[u].piece;
        if (at[u].row >= m || c >= k) continue;
        const float f = mx_scale(b[u] == 255u ? MX_ONE : b[u]);
        float v[8];
        auto two = [&](int i, auto t) { v[2 * i] = t[0], v[2 * i + 1] = t[1]; };
        two(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 0));
        two(1, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 1));
        two(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 2));
        two(3, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], f, 3));
        if (b[u] == 255u)
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __builtin_nanf("");
        mx_store<DT>(y + at[u].row * ldy + c, v, k - c < 8 ? (uint32_t)(k - c) : 8u);
    }
}

// What a launch over all pieces of m rows is given.
struct MxRun {
    dim3 grid;
    uint32_t P, rows, pieces;
};
MxRun mx_run(uint32_t m, uint32_t k) {
    const uint32_t P = 4 * mx_blocks(k);
    const uint64_t n = (uint64_t)m * P;
    const geo::Grid2 g = geo::grid_run((n + MQ_T * MQ_U - 1) / (MQ_T * MQ_U), MQ_T);
    return MxRun{dim3(g.x, g.y), P, MQ_T / P, MQ_T % P};
}

template <uint32_t DT>
void launch_rows(bool back, const void* x, uint64_t ldx, uint32_t m, uint32_t k, uint8_t* q, uint64_t ldq, uint8_t* s, uint64_t lds,
                 void* y, uint64_t ldy, hipStream_t st) {
    typedef typename Elem<DT>::T T;
    const MxRun r = mx_run(m, k);
    if (back)
        dequantize_mx4_kernel<DT><<<r.grid, MQ_T, 0, st>>>(q, ldq, s, lds, m, k, r.P, r.rows, r.pieces, (T*)y, ldy);
    else
        quantize_mx4_kernel<DT><<<r.grid, MQ_T, 0, st>>>((const T*)x, ldx, m, k, r.P, r.rows, r.pieces, q, ldq, s, lds);
}

// ============================================================================================
// the dense product
// ============================================================================================

constexpr uint32_t ST_WAVES = 4;

// A workgroup takes 16 weight rows and up to 16 tokens: its waves share K and add their sums in LDS.  For few rows and short K, where the
// trips to memory are all there is: two units of both rows a wave are requested at once.  [12288] x 1 row at k = 2560 4.3 us (3.9
// TB/s, the weights in the last cache), [512] x 1 at k = 512 2.3.
template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES* WAVE) void gemm_mx4_strip_kernel(Mx4Gemm g) {
    __shared__ float part[ST_WAVES][16][16];  // [wave][token][weight row]
    const uint32_t strips = (g.w.rows + 15) / 16, id = run_id();
    const uint32_t r0 = id % strips * 16, t0 = id / strips * 16;
    if (t0 >= g.m) return;  // the whole workgroup
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, c = lane % 16;
    const uint64_t wr = r0 + c < g.w.rows ? r0 + c : g.w.rows - 1, xr = t0 + c < g.m ? t0 + c : g.m - 1;
    const uint32_t t = t0 + threadIdx.x / 16, r = r0 + threadIdx.x % 16;
    const bool out = t < g.m && r < g.w.rows;
    const float b = out && g.bias ? g.bias[r] : 0.0f;
    f32x4 acc[1];
    mx4_strip<1>({Mx4Row{g.w.q + wr * g.w.ld, g.w.s + wr * g.w.lds}}, Mx4Row{g.x.q + xr * g.x.ld, g.x.s + xr * g.x.lds}, g.w.nb, wv,
                 ST_WAVES, lane, acc);
    *reinterpret_cast<f32x4*>(&part[wv][c][lane / 16 * 4]) = acc[0];
    __syncthreads();
    if (!out) return;
    float v = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) v += part[i][threadIdx.x / 16][threadIdx.x % 16];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(g.y) + t * g.ldy + r;
    if (g.bias) v += b;
    if (g.accumulate) v += O::get(*y);
    *y = O::put(v);
}

void launch_strip(const Mx4Gemm& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.w.rows + 15) / 16) * (((uint64_t)a.m + 15) / 16);
    const geo::Grid2 g = geo::grid_run(wgs, ST_WAVES * WAVE);
    const dim3 grid(g.x, g.y);
    if (a.dt == TRK_DT_F32)
        gemm_mx4_strip_kernel<TRK_DT_F32><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        gemm_mx4_strip_kernel<TRK_DT_BF16><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
    else
        gemm_mx4_strip_kernel<TRK_DT_F16><<<grid, ST_WAVES * WAVE, 0, st>>>(a);
}

// v += the four neighbouring values of a row at any address, `left` of them there
template <uint32_t DT>
__device__ __forceinline__ f32x4 load_add4(const typename Elem<DT>::T* y, f32x4 v, uint32_t left) {
    typedef uint16_t u16x4_h __attribute__((ext_vector_type(4), aligned(2)));
    typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
    if (left >= 4) {
        typename std::conditional<DT == TRK_DT_F32, f32x4_any, u16x4_h>::type o;
        o = *reinterpret_cast<const decltype(o)*>(y);
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) v[c] += Elem<DT>::get(o[c]);
        return v;
    }
#pragma unroll
    for (uint32_t c = 0; c < 4; c++)
        if (c < left) v[c] += Elem<DT>::get(y[c]);
    return v;
}

// The tiles' place in the launch: panels of eight weight tiles, activation tiles after one another inside each, so that
// the tiles that run at once on an XCD (a contiguous run of them) share rows of both in its L2.
__device__ __forceinline__ void tile_place(uint32_t idx, uint32_t tn, uint32_t tm, uint32_t& n, uint32_t& m) {
    const uint32_t panel = idx / (8 * tm), left = tn - panel * 8, w = left < 8 ? left : 8, rem = idx - panel * 8 * tm;
    n = panel * 8 + rem % w, m = rem / w;
}

// 4096 x 12288 x 2560 to bf16 81 us, 3.2 PFLOP/s; 8192 cubed 299, 3.7 (from registers alone the instruction reached 6.6 on random
// bits, 8.9 on constants).  What bounds it is the clock that random bits leave (1.6 GHz; 8192 cubed of zeros takes 208 us) with the matrix
// cores busy half of it, and beside them LDS: a stage of 256 x 256 reads 192 KB of fragments and writes 64, 2048 clocks, as many as
// its products take at the nominal rate.  And the scales: sixteen loads a wave for eight stages, whose row offsets do not fit beside
// the sums (256 registers, 68 bytes of scratch a lane): seven of them wait for an offset from scratch, and with it for all that
// is on its way, eight for a stride's scalar load.  Tiles of 256 x 256 halve the rows' traffic against 128 x 128, at one workgroup
// a CU.  Where whole tiles do not fill the CUs smaller ones do (geo::gemm_mx4_form).
template <typename Tile, uint32_t DT>
__global__ __launch_bounds__(Tile::T) void gemm_mx4_tile_kernel(Mx4Gemm g) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::LDS];
    const uint32_t tn = (g.w.rows + Tile::BN - 1) / Tile::BN, tm = (g.m + Tile::BM - 1) / Tile::BM;
    uint32_t idx, n, m;
    if (!xcd_order_1d(tn * tm, idx, run_id())) return;  // the whole workgroup
    tile_place(idx, tn, tm, n, m);
    const uint32_t r0 = n * Tile::BN, t0 = m * Tile::BM, rl = g.w.rows - r0 - 1, tl = g.m - t0 - 1;  // the last rows there are
    Tile t;
    i32x4 rw[Tile::NA];
    uint32_t wo[Tile::NA], xo[Tile::NB];
    const i32x4 bw = buffer_at((const int8_t*)g.w.q + r0 * g.w.ld), bx = buffer_at((const int8_t*)g.x.q + t0 * g.x.ld);
    const i32x4 bws = buffer_at((const int8_t*)g.w.s + r0 * g.w.lds), bxs = buffer_at((const int8_t*)g.x.s + t0 * g.x.lds);
#pragma unroll
    for (int i = 0; i < Tile::NA; i++) {
        const uint32_t r = t.load_row(i);
        rw[i] = bw, wo[i] = (r < rl ? r : rl) * (uint32_t)g.w.ld;
    }
#pragma unroll
    for (int i = 0; i < Tile::NB; i++) {
        const uint32_t r = t.load_row(i);
        xo[i] = (r < tl ? r : tl) * (uint32_t)g.x.ld;
    }
    auto scales = [&](int i, i32x4& rs, uint32_t& so) {
        const bool w = t.scale_load(i) < Tile::BN / Tile::SR;
        const uint32_t r = t.scale_row(i) - (w ? 0 : Tile::BN), l = w ? rl : tl;
        rs = w ? bws : bxs, so = (r < l ? r : l) * (uint32_t)(w ? g.w.lds : g.x.lds);
    };
    t.template run<false, false>(lds, rw, wo, bx, xo, scales, g.w.nb, 0, t.wn + t.lane % 32, 32);
    typedef Elem<DT> O;
    const uint32_t r = r0 + t.wn + t.lane % (Tile::WN / 4) * 4, left = r < g.w.rows ? g.w.rows - r : 0;
    const bool inside = !g.accumulate && r0 + Tile::BN <= g.w.rows && t0 + Tile::BM <= g.m;  // the workgroup as a whole
    f32x4 bias{0.0f, 0.0f, 0.0f, 0.0f};
    if (g.bias) {
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) bias[c] = g.bias[c < left ? r + c : g.w.rows - 1];
        asm volatile("" : "+v"(bias));  // here, or every store is waited for before the next
    }
    typename O::T* y0 = reinterpret_cast<typename O::T*>(g.y) + (uint64_t)(t0 + t.wm) * g.ldy + r;
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        float v[Tile::WN / 8][4];
#pragma unroll
        for (int i = 0; i < Tile::FN; i++)
#pragma unroll
            for (int q = 0; q < 16; q++) v[4 * i + q / 4][q % 4] = t.acc[i][j][q];
        if (inside)
            t.template turn<Tile::WN>(lds, v, [&](uint32_t tr, uint32_t, f32x4 x) {
                store4_any<DT>(y0 + (32 * j + tr) * g.ldy, g.bias ? x + bias : x, 4);
            });
        else
            t.template turn<Tile::WN>(lds, v, [&](uint32_t tr, uint32_t, f32x4 x) {
                if (t0 + t.wm + 32 * j + tr >= g.m || left == 0) return;
                typename O::T* y = y0 + (32 * j + tr) * g.ldy;
                if (g.bias) x += bias;
                if (g.accumulate) x = load_add4<DT>(y, x, left);
                store4_any<DT>(y, x, left);
            });
    }
}

template <typename Tile>
void launch_tile(const Mx4Gemm& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.w.rows + Tile::BN - 1) / Tile::BN) * (((uint64_t)a.m + Tile::BM - 1) / Tile::BM);
    const geo::Grid2 g = geo::grid_run(wgs, Tile::T);
    const dim3 grid(g.x, g.y);
    if (a.dt == TRK_DT_F32)
        gemm_mx4_tile_kernel<Tile, TRK_DT_F32><<<grid, Tile::T, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        gemm_mx4_tile_kernel<Tile, TRK_DT_BF16><<<grid, Tile::T, 0, st>>>(a);
    else
        gemm_mx4_tile_kernel<Tile, TRK_DT_F16><<<grid, Tile::T, 0, st>>>(a);
}

}  // namespace

hipError_t launch_rows_mx4(bool back, uint32_t dt, const void* x, uint64_t ldx, uint32_t m, uint32_t k, uint8_t* q, uint64_t ldq,
                           uint8_t* s, uint64_t lds, void* y, uint64_t ldy, hipStream_t st) {
    if (dt == TRK_DT_F32)
        launch_rows<TRK_DT_F32>(back, x, ldx, m, k, q, ldq, s, lds, y, ldy, st);
    else if (dt == TRK_DT_BF16)
        launch_rows<TRK_DT_BF16>(back, x, ldx, m, k, q, ldq, s, lds, y, ldy, st);
    else
        launch_rows<TRK_DT_F16>(back, x, ldx, m, k, q, ldq, s, lds, y, ldy, st);
    return hipGetLastError();
}

hipError_t launch_gemm_mx4(const Mx4Gemm& a, hipStream_t st) {
    switch (geo::gemm_mx4_form(a.m, a.w.rows, a.w.nb, a.w.ld, a.x.ld, a.w.lds, a.x.lds)) {
    case geo::I8_TILE_256: launch_tile<Mx4Tile<256, 256, 64, 128, 2, 8>>(a, st); break;
    case geo::I8_TILE_128: launch_tile<Mx4Tile<128, 128, 32, 64, 2>>(a, st); break;  // 64 x 64 a wave: [12288] x 512, k = 2560 16.8 us against 15.9
    case geo::I8_TILE_64: launch_tile<Mx4Tile<64, 64, 32, 32, 4>>(a, st); break;
    case geo::I8_TILE_32: launch_tile<Mx4Tile<64, 32, 32, 32, 4>>(a, st); break;
    default: launch_strip(a, st);
    }
    return hipGetLastError();
}

}  // namespace trk
