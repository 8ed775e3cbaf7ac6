// The dense 4-bit product by tiles: the kernel, and its launch for one tile shape.
#pragma once

#include "mx4tile.hpp"

namespace trk {

// v[c] += y[c] for the n of four values that are there
template <uint32_t DT>
__device__ __forceinline__ void load_add4(const typename Elem<DT>::T* y, float (&v)[4], uint32_t n, bool vec) {
    if (n >= 4 && vec) {
        if constexpr (DT == TRK_DT_F32) {
            const float4 o = *reinterpret_cast<const float4*>(y);
            v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
        } else {
            const ushort4 o = *reinterpret_cast<const ushort4*>(y);
            v[0] += Elem<DT>::get(o.x), v[1] += Elem<DT>::get(o.y), v[2] += Elem<DT>::get(o.z), v[3] += Elem<DT>::get(o.w);
        }
        return;
    }
#pragma unroll
    for (uint32_t c = 0; c < 4; c++)
        if (c < n) v[c] += Elem<DT>::get(y[c]);
}

// The tiles' place in the launch: panels of eight weight tiles, activation tiles after one another inside each, so that
// the tiles that run at once on an XCD (a contiguous run of them) share rows of both in its L2.
__device__ __forceinline__ void tile_place(uint32_t idx, uint32_t tn, uint32_t tm, uint32_t& n, uint32_t& m) {
    const uint32_t panel = idx / (8 * tm), left = tn - panel * 8, w = left < 8 ? left : 8, rem = idx - panel * 8 * tm;
    n = panel * 8 + rem % w, m = rem / w;
}

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
    const bool inside = g.vec && !g.accumulate && r0 + Tile::BN <= g.w.rows && t0 + Tile::BM <= g.m;  // the workgroup as a whole
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
                store4_whole<DT>(y0 + (32 * j + tr) * g.ldy, g.bias ? x + bias : x);
            });
        else
            t.template turn<Tile::WN>(lds, v, [&](uint32_t tr, uint32_t, f32x4 x) {
                if (t0 + t.wm + 32 * j + tr >= g.m || left == 0) return;
                typename O::T* y = y0 + (32 * j + tr) * g.ldy;
                float o[4];
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) o[c] = g.bias ? x[c] + bias[c] : x[c];
                if (g.accumulate) load_add4<DT>(y, o, left, g.vec);
                store4<DT>(y, o, left, g.vec);
            });
    }
}

template <typename Tile>
void launch_mx4_tile(const Mx4Gemm& a, hipStream_t st) {
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

}  // namespace trk
