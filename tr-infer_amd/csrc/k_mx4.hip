// Rows to microscaled 4-bit values and back (trk_quantize_mx4, trk_dequantize_mx4), and their dense product (trk_gemm_mx4).
#include "mx4gemm.hpp"
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

// A workgroup takes 16 weight rows and up to 16 tokens: its waves share K and add their sums in LDS.
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
    static const int form = getenv("MX4_FORM") ? atoi(getenv("MX4_FORM")) : 0;  // PROBE
    switch (form) {
    case 1: launch_mx4_tile<Mx4Tile<64, 32, 32, 32, 4>>(a, st); break;
    case 2: launch_mx4_tile<Mx4Tile<64, 64, 32, 32, 4>>(a, st); break;
    case 3: launch_mx4_tile<Mx4Tile<128, 128, 64, 64, 2>>(a, st); break;
    case 4: launch_mx4_tile<Mx4Tile<256, 256, 64, 128, 2, 8>>(a, st); break;
    case 5: launch_mx4_tile<Mx4Tile<128, 64, 64, 32, 3>>(a, st); break;
    case 6: launch_mx4_tile<Mx4Tile<256, 128, 64, 64, 3>>(a, st); break;
    case 7: launch_gemm_mx4_wide(a, st); break;
    default: launch_strip(a, st);
    }
    return hipGetLastError();
}

}  // namespace trk
