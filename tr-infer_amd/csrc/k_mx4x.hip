// The microscaled 4-bit products of each token with its experts (trk_experts_up_mx4, trk_experts_down_mx4).
#include "mx4tile.hpp"
#include "plan.hpp"

namespace trk {

namespace {

// ============================================================================================
// few entries: each by itself
// ============================================================================================

constexpr uint32_t ST_WAVES = 4;

// This lane's row of the 16 from r0 on
__device__ __forceinline__ Mx4Row strip_row(const Mx4Mat& w, uint32_t e, uint32_t r0, uint32_t lane) {
    const uint64_t r = r0 + lane % 16 < w.rows ? r0 + lane % 16 : w.rows - 1;
    return Mx4Row{w.q + e * w.stride + r * w.ld, w.s + e * w.sstride + r * w.lds};
}

// A workgroup takes 16 rows of gate and up and one entry; its waves share K.  Two trips to memory, ids and then every weight: 1 token of
// 10 in 512 (H = 2048, F = 512) 5.7 us, 4 tokens 9.8 (4.4 TB/s), 8 of 8 in 256 (F = 768) 22.
template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES* WAVE) void experts_up_mx4_strip_kernel(Mx4Up a) {
    __shared__ float part[2][ST_WAVES][16];  // [gate, up][wave][weight row]
    const uint32_t strips = (a.gate.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, en = id / strips;
    const uint32_t t = en / a.slots, j = en % a.slots;
    if (t >= a.m) return;  // the whole workgroup, here and below
    const uint32_t e = a.ids[(size_t)t * K_MAX + j], n = a.n_sel[t];
    if (j >= n || e >= a.gate.count) return;
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    f32x4 acc[2];
    // every column of the matrix instruction is this token's row
    mx4_strip<2>({strip_row(a.gate, e, r0, lane), strip_row(a.up, e, r0, lane)},
                 Mx4Row{a.x.q + t * a.x.ld, a.x.s + t * a.x.lds}, a.gate.nb, wv, ST_WAVES, lane, acc);
    if (lane % 16 == 0) {
        *reinterpret_cast<f32x4*>(&part[0][wv][lane / 16 * 4]) = acc[0];
        *reinterpret_cast<f32x4*>(&part[1][wv][lane / 16 * 4]) = acc[1];
    }
    __syncthreads();
    const uint32_t r = r0 + threadIdx.x;
    if (threadIdx.x >= 16 || r >= a.gate.rows) return;
    float g = 0.0f, u = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) g += part[0][i][threadIdx.x], u += part[1][i][threadIdx.x];
    typedef Elem<DT> O;
    reinterpret_cast<typename O::T*>(a.h)[en * a.ldh + r] = O::put(swiglu(g, u));
}

// A workgroup takes 16 down rows and one token: a wave per slot (several where there are fewer slots than waves, sharing
// K; in turn where there are more), then a thread per (slot, row) weights, and a thread per row adds in slot order: no second
// launch, and no order but the slots'.  1 token of 10 in 512 (2048, 512) 5.0 us, 4 tokens 7.4, 8 of 8 in 256 (F = 768) 15.8.
constexpr uint32_t DOWN_WAVES = 8;

template <uint32_t DT>
__global__ __launch_bounds__(DOWN_WAVES* WAVE) void experts_down_mx4_strip_kernel(Mx4Down a) {
    __shared__ float part[K_MAX * 4][16];  // [slot * share of K][weight row]
    __shared__ float term[K_MAX][16];
    const uint32_t strips = (a.down.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, t = id / strips;
    if (t >= a.m) return;
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t ks = DOWN_WAVES / a.slots >= 4 ? 4 : DOWN_WAVES / a.slots >= 2 ? 2 : 1;  // waves that share a slot
    const uint32_t* ids = a.ids + (size_t)t * K_MAX;
    const uint32_t ns = a.n_sel[t], n = ns < a.slots ? ns : a.slots;
    static_assert(DOWN_WAVES * WAVE >= K_MAX * 16, "a thread per (slot, row)");
    const uint32_t ri = threadIdx.x % 16, r = r0 + ri;
    const uint32_t j = threadIdx.x / 16, jc = j < a.slots ? j : 0;
    const bool there = j < n && ids[jc] < a.down.count;
    const float wt = a.w[(size_t)t * K_MAX + jc];
    for (uint32_t w = wv; w < a.slots * ks; w += DOWN_WAVES) {
        const uint32_t ew = ids[w / ks];
        if (w / ks >= n || ew >= a.down.count) continue;
        const uint64_t xr = (uint64_t)t * a.slots + w / ks;
        f32x4 acc[1];
        mx4_strip<1>({strip_row(a.down, ew, r0, lane)}, Mx4Row{a.x.q + xr * a.x.ld, a.x.s + xr * a.x.lds}, a.down.nb, w % ks, ks,
                     lane, acc);
        if (lane % 16 == 0) *reinterpret_cast<f32x4*>(&part[w][lane / 16 * 4]) = acc[0];
    }
    __syncthreads();
    if (j < n) {
        float v = 0.0f;
        if (there) {
            v = part[j * ks][ri];
            for (uint32_t c = 1; c < ks; c++) v += part[j * ks + c][ri];
            v *= wt;
        }
        term[j][ri] = v;
    }
    __syncthreads();
    if (threadIdx.x >= 16 || r >= a.down.rows) return;
    float v = 0.0f;
#pragma unroll 8
    for (uint32_t i = 0; i < n; i++) v += term[i][ri];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(a.y) + t * a.ldy + r;
    *y = O::put(a.accumulate ? O::get(*y) + v : v);
}

// ============================================================================================
// many entries: tiles of one expert's
// ============================================================================================

// What a tile loads: for its BN weight rows, the first `split` of one matrix and the rest of another (or the same), and for its
// activation rows, `row(i)` of all.  Before a tile's first load lie its plan's head and place, the entries of its activation rows'
// values, then those of their scales: a trip to memory each.
struct Mx4Side {
    i32x4 q, s;
    uint32_t ld, lds;
};
__device__ __forceinline__ Mx4Side mx4_side(const Mx4Mat& w, uint32_t e, uint64_t r0) {
    return Mx4Side{buffer_at((const int8_t*)w.q + e * w.stride + r0 * w.ld), buffer_at((const int8_t*)w.s + e * w.sstride + r0 * w.lds),
                   (uint32_t)w.ld, (uint32_t)w.lds};
}
template <typename Tile>
struct Mx4Loads {
    i32x4 rw[Tile::NA], rs[Tile::NS], rx;
    uint32_t wo[Tile::NA], xo[Tile::NB], so[Tile::NS];
    template <typename Row>
    __device__ __forceinline__ Mx4Loads(const Tile& t, const Mx4Side& w0, const Mx4Side& w1, uint32_t split, uint32_t last, const Mx4X& x,
                                        Row&& row) {
        rx = buffer_at((const int8_t*)x.q);
        const i32x4 rxs = buffer_at((const int8_t*)x.s);
#pragma unroll
        for (int i = 0; i < Tile::NB; i++) xo[i] = row(t.load_row(i)) * (uint32_t)x.ld;
#pragma unroll
        for (int i = 0; i < Tile::NA; i++) {
            const bool two = (i * Tile::NW + t.wv) * 8 >= split;
            const uint32_t r = t.load_row(i) - (two ? split : 0), rc = r < last ? r : last;
            rw[i] = two ? w1.q : w0.q, wo[i] = rc * (two ? w1.ld : w0.ld);
        }
#pragma unroll
        for (int i = 0; i < Tile::NS; i++) {
            const uint32_t p = t.scale_load(i) * Tile::SR, n = t.lane / Tile::SW;
            const bool mine = p >= Tile::BN, two = !mine && p >= split;
            if (mine) {
                rs[i] = rxs, so[i] = row(p - Tile::BN + n) * (uint32_t)x.lds;
            } else {
                const uint32_t r = p - (two ? split : 0) + n, rc = r < last ? r : last;
                rs[i] = two ? w1.s : w0.s, so[i] = rc * (two ? w1.lds : w0.lds);
            }
        }
    }
    template <bool ONCE>
    __device__ __forceinline__ void run(Tile& t, uint8_t* lds, uint32_t nb, uint32_t live, uint32_t a0, uint32_t astep) const {
        t.template run<true, ONCE>(lds, rw, wo, rx, xo, [&](int i, i32x4& r, uint32_t& o) { r = rs[i], o = so[i]; }, nb, live, a0, astep);
    }
};

// gate and up: a tile's weight rows are BN / 2 rows of gate, then the same rows of up.  A wave's 32 rows of a matrix instruction are
// 16 of each, so that a lane has both sums of its rows and SwiGLU is the epilogue.  ONCE: geo::experts_once.  2000 tokens of 8 in 128
// (H = 2048, F = 768) 78 us: 1.3 PFLOP/s, 2.7 TB/s of weights.  What bounds it is the latency of the weights' loads, two workgroups
// a CU with one to two stages each on their way (all loads from a few lines: 52), and beside it LDS: a stage of both workgroups reads and
// writes 1 us of it.  Without its matrix instructions it takes 75.
template <typename Tile, uint32_t DT, bool ONCE>
__global__ __launch_bounds__(Tile::T) void experts_up_mx4_tile_kernel(Mx4Up a, Plan P) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::LDS];
    constexpr uint32_t BR = Tile::BN / 2;
    static_assert(BR % 32 == 0, "a load takes rows of one matrix");
    PlanTile pt;
    uint32_t block;
    const PlanHead head = *P.head;
    if (!plan_fits(head, a.m, a.slots, a.gate.count))  // the whole workgroup, here and below
        return nan_rows<DT>(a, a.gate.count, a.h, a.gate.rows, a.ldh);
    if (!expert_tile(P, head, a.gate.count, (a.gate.rows + BR - 1) / BR, pt, block)) return;
    const uint32_t r0 = block * BR;
    Tile t;
    auto entry = [&](uint32_t i) { return P.ent[pt.row0 + (i < pt.rows ? i : pt.rows - 1)]; };
    const uint32_t wr = t.wn / 2, c = t.lane % 32;  // this wave's first row of both
    uint32_t en[Tile::FM];
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) en[j] = entry(t.wm + 32 * j + c);
    const uint32_t live = t.wm < pt.rows ? (pt.rows - t.wm + 31) / 32 : 0;
    const Mx4Loads<Tile> at(t, mx4_side(a.gate, pt.expert, r0), mx4_side(a.up, pt.expert, r0), BR, a.gate.rows - r0 - 1, a.x,
                            [&](uint32_t i) { return entry(i) / a.slots; });
    at.template run<ONCE>(t, lds, a.gate.nb, live, wr + (c < 16 ? c : BR + c - 16), 16);
    typedef Elem<DT> O;
    constexpr int CW = Tile::WN / 2;
    const uint32_t r = r0 + wr + t.lane % (CW / 4) * 4, left = r < a.gate.rows ? a.gate.rows - r : 0;
    const bool whole = r0 + BR <= a.gate.rows;  // the workgroup as a whole
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        if (j >= (int)live) break;  // the wave as a whole
        float v[CW / 8][4];
#pragma unroll
        for (int i = 0; i < Tile::FN; i++)
#pragma unroll
            for (int q = 0; q < 2; q++) {
                float g[4], u[4];
#pragma unroll
                for (int e = 0; e < 4; e++) g[e] = t.acc[i][j][4 * q + e], u[e] = t.acc[i][j][8 + 4 * q + e];
                swiglu4(g, u, v[2 * i + q]);
            }
        t.template turn<CW>(lds, v, [&](uint32_t tr, uint32_t, f32x4 x) {
            const uint32_t e = __shfl(en[j], tr);
            if (t.wm + 32 * j + tr >= pt.rows || left == 0) return;
            typename O::T* h = reinterpret_cast<typename O::T*>(a.h) + e * a.ldh + r;
            store4_any<DT>(h, x, whole ? 4 : left);
        });
    }
}

// down: the entries' weighted rows into work [m * slots][rows], in 32 bits, as they are then added: every sum stays in 32 bits and in
// slot order, whatever order the plan has.  ONCE: geo::experts_once.  4096 tokens of 10 in 512 (H = 2048, F = 512) 143 us for 285 MB
// of weights and 336 of outputs, 4.3 TB/s where a copy reaches 4.7; the combine reads them again in 57.
template <typename Tile, bool ONCE>
__global__ __launch_bounds__(Tile::T) void experts_down_mx4_tile_kernel(Mx4Down a, Plan P) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::LDS];
    PlanTile pt;
    uint32_t block;
    const PlanHead head = *P.head;
    if (!plan_fits(head, a.m, a.slots, a.down.count))  // the whole workgroup, here and below
        return nan_rows<TRK_DT_F32>(a, a.down.count, a.work, a.down.rows, a.down.rows);
    if (!expert_tile(P, head, a.down.count, (a.down.rows + Tile::BN - 1) / Tile::BN, pt, block)) return;
    const uint32_t r0 = block * Tile::BN;
    Tile t;
    auto entry = [&](uint32_t i) { return P.ent[pt.row0 + (i < pt.rows ? i : pt.rows - 1)]; };
    const uint32_t c = t.lane % 32;
    uint32_t en[Tile::FM];
    float w[Tile::FM];
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) en[j] = entry(t.wm + 32 * j + c);
    const uint32_t live = t.wm < pt.rows ? (pt.rows - t.wm + 31) / 32 : 0;
    const Mx4Side ws = mx4_side(a.down, pt.expert, r0);
    const Mx4Loads<Tile> at(t, ws, ws, Tile::BN, a.down.rows - r0 - 1, a.x, entry);
    // the entries' weights are asked for after the tile's own addresses: its first loads then wait for one trip to memory less
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) w[j] = a.w[(size_t)(en[j] / a.slots) * K_MAX + en[j] % a.slots];
    at.template run<ONCE>(t, lds, a.down.nb, live, t.wn + c, 32);
    const uint32_t r = r0 + t.wn + t.lane % (Tile::WN / 4) * 4, left = r < a.down.rows ? a.down.rows - r : 0;
    const bool whole = r0 + Tile::BN <= a.down.rows;  // the workgroup as a whole
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        if (j >= (int)live) break;  // the wave as a whole
        float v[Tile::WN / 8][4];
#pragma unroll
        for (int i = 0; i < Tile::FN; i++)
#pragma unroll
            for (int q = 0; q < 16; q++) v[4 * i + q / 4][q % 4] = t.acc[i][j][q] * w[j];
        t.template turn<Tile::WN>(lds, v, [&](uint32_t tr, uint32_t, f32x4 x) {
            const uint32_t e = __shfl(en[j], tr);
            if (t.wm + 32 * j + tr >= pt.rows || left == 0) return;
            float* y = a.work + (uint64_t)e * a.down.rows + r;
            store4_any<TRK_DT_F32>(y, x, whole ? 4 : left);
        });
    }
}

dim3 run_of(uint64_t wgs, uint32_t threads) {
    const geo::Grid2 g = geo::grid_run(wgs, threads);
    return dim3(g.x, g.y);
}

// The kernels number their workgroups by 32 bits: of entries beyond, so many tokens a launch.
uint32_t strip_tokens(uint32_t rows, uint32_t per_token) {
    const uint64_t t = 0x7fffffffull / ((rows + 15) / 16) / per_token;
    return t < 1 ? 1 : t > 0x7fffffffull ? 0x7fffffffu : (uint32_t)t;
}

void launch_up_strip(Mx4Up a, hipStream_t st) {
    const uint32_t m = a.m, step = strip_tokens(a.gate.rows, a.slots);
    const uint64_t size = a.dt == TRK_DT_F32 ? 4 : 2;
    for (uint64_t t = 0; t < m; t += step) {
        a.m = m - t < step ? m - (uint32_t)t : step;
        const dim3 g = run_of((uint64_t)((a.gate.rows + 15) / 16) * a.m * a.slots, ST_WAVES * WAVE);
        if (a.dt == TRK_DT_F32)
            experts_up_mx4_strip_kernel<TRK_DT_F32><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        else if (a.dt == TRK_DT_BF16)
            experts_up_mx4_strip_kernel<TRK_DT_BF16><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        else
            experts_up_mx4_strip_kernel<TRK_DT_F16><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        a.x.q += step * a.x.ld, a.x.s += step * a.x.lds, a.ids += (uint64_t)step * K_MAX, a.n_sel += step;
        a.h = (char*)a.h + (uint64_t)step * a.slots * a.ldh * size;
    }
}

void launch_down_strip(Mx4Down a, hipStream_t st) {
    const uint32_t m = a.m, step = strip_tokens(a.down.rows, 1);
    const uint64_t size = a.dt == TRK_DT_F32 ? 4 : 2;
    for (uint64_t t = 0; t < m; t += step) {
        a.m = m - t < step ? m - (uint32_t)t : step;
        const dim3 g = run_of((uint64_t)((a.down.rows + 15) / 16) * a.m, DOWN_WAVES * WAVE);
        if (a.dt == TRK_DT_F32)
            experts_down_mx4_strip_kernel<TRK_DT_F32><<<g, DOWN_WAVES * WAVE, 0, st>>>(a);
        else if (a.dt == TRK_DT_BF16)
            experts_down_mx4_strip_kernel<TRK_DT_BF16><<<g, DOWN_WAVES * WAVE, 0, st>>>(a);
        else
            experts_down_mx4_strip_kernel<TRK_DT_F16><<<g, DOWN_WAVES * WAVE, 0, st>>>(a);
        const uint64_t rows = (uint64_t)step * a.slots;
        a.x.q += rows * a.x.ld, a.x.s += rows * a.x.lds, a.ids += (uint64_t)step * K_MAX, a.w += (uint64_t)step * K_MAX;
        a.n_sel += step, a.y = (char*)a.y + step * a.ldy * size;
    }
}

template <typename Tile, bool ONCE = true>
void launch_up_tile(const Mx4Up& a, const Plan& P, uint64_t tiles, hipStream_t st) {
    const dim3 g = run_of((a.gate.rows + Tile::BN / 2 - 1) / (Tile::BN / 2) * tiles, Tile::T);
    if (a.dt == TRK_DT_F32)
        experts_up_mx4_tile_kernel<Tile, TRK_DT_F32, ONCE><<<g, Tile::T, 0, st>>>(a, P);
    else if (a.dt == TRK_DT_BF16)
        experts_up_mx4_tile_kernel<Tile, TRK_DT_BF16, ONCE><<<g, Tile::T, 0, st>>>(a, P);
    else
        experts_up_mx4_tile_kernel<Tile, TRK_DT_F16, ONCE><<<g, Tile::T, 0, st>>>(a, P);
}

template <typename Tile, bool ONCE = true>
void launch_down_tile(const Mx4Down& a, const Plan& P, uint64_t tiles, hipStream_t st) {
    const dim3 g = run_of((a.down.rows + Tile::BN - 1) / Tile::BN * tiles, Tile::T);
    experts_down_mx4_tile_kernel<Tile, ONCE><<<g, Tile::T, 0, st>>>(a, P);
}

// The tiles address values and scales by 32 bits, weight rows from their block's first, activation rows from the first of all.
bool tile_addresses(const Mx4Mat& w, const Mx4X& x, uint64_t rows) {
    return geo::i8_tile_addresses(w.ld, x.ld, rows) && geo::i8_tile_addresses(w.lds, x.lds, rows);
}

}  // namespace

hipError_t launch_experts_up_mx4(const Mx4Up& a, const uint32_t* plan, hipStream_t st) {
    const uint32_t E = a.gate.count;
    if (!plan || !tile_addresses(a.gate, a.x, a.m) || !tile_addresses(a.up, a.x, a.m)) {
        launch_up_strip(a, st);
        return hipGetLastError();
    }
    const uint32_t rows = geo::plan_rows(a.m, a.slots, E);
    const Plan P = plan_at(const_cast<uint32_t*>(plan), a.m, a.slots);
    const uint64_t tiles = geo::plan_tiles(a.m, a.slots, E, rows);
    const bool narrow = geo::experts_width(2 * a.gate.rows, tiles, false) == geo::X_NARROW;
    // us at 128 entries a tile, four waves of 64 x 64 / eight of 32 x 64, two workgroups on a CU either way / 256 x 128 by eight of 64 x
    // 64: 2000 tokens of 8 in 128 (H = 2048, F = 768) 89.7 / 87.4 / 92.4, 400 of 8 in 64 (1024, 512) - / 18.1 / 20.3, 3000 of 2 in 8 (2048, 1024)
    // 39.7 / 37.9 / 40.4, 4096 of 10 in 512 (2048, 512) 177 / 175 / 182
    if (rows == 32)
        narrow ? launch_up_tile<Mx4Tile<64, 32, 32, 32, 4>>(a, P, tiles, st)
               : launch_up_tile<Mx4Tile<128, 32, 32, 32, 3>>(a, P, tiles, st);
    else if (rows == 64)
        narrow ? launch_up_tile<Mx4Tile<64, 64, 32, 32, 4>>(a, P, tiles, st)
               : launch_up_tile<Mx4Tile<128, 64, 64, 32, 3>>(a, P, tiles, st);
    else if (geo::experts_once(a.m, a.slots, E, 64))
        narrow ? launch_up_tile<Mx4Tile<64, 128, 32, 64, 3>>(a, P, tiles, st)
               : launch_up_tile<Mx4Tile<128, 128, 32, 64, 2>>(a, P, tiles, st);
    else
        narrow ? launch_up_tile<Mx4Tile<64, 128, 32, 64, 3>, false>(a, P, tiles, st)
               : launch_up_tile<Mx4Tile<128, 128, 32, 64, 2>, false>(a, P, tiles, st);
    return hipGetLastError();
}

hipError_t launch_experts_down_mx4(const Mx4Down& a, const uint32_t* plan, hipStream_t st) {
    const uint32_t E = a.down.count;
    if (!plan || !tile_addresses(a.down, a.x, (uint64_t)a.m * a.slots)) {
        launch_down_strip(a, st);
        return hipGetLastError();
    }
    const uint32_t rows = geo::plan_rows(a.m, a.slots, E);
    const Plan P = plan_at(const_cast<uint32_t*>(plan), a.m, a.slots);
    const uint64_t tiles = geo::plan_tiles(a.m, a.slots, E, rows);
    const bool narrow = geo::experts_width(a.down.rows, tiles, false) == geo::X_NARROW;
    // An expert's rows are short: more workgroups on a CU are worth more than a third stage.  us, three stages / two: 512 tokens of 10 in
    // 512 (H = 2048, F = 512) 97 / 83, 150 of 6 in 60 (1100, 347) 18.8 / 17.2, 300 of 8 in 128 (2048, 768) 42.3 / 41.2; 2000 of 10 in 512 144 / 133.
    if (rows == 32)
        narrow ? launch_down_tile<Mx4Tile<64, 32, 32, 32, 4>>(a, P, tiles, st)
               : launch_down_tile<Mx4Tile<128, 32, 32, 32, 2>>(a, P, tiles, st);
    else if (rows == 64)
        narrow ? launch_down_tile<Mx4Tile<64, 64, 32, 32, 4>>(a, P, tiles, st)
               : launch_down_tile<Mx4Tile<128, 64, 32, 32, 2>>(a, P, tiles, st);
    else if (geo::experts_once(a.m, a.slots, E, 128))
        narrow ? launch_down_tile<Mx4Tile<64, 128, 32, 64, 3>>(a, P, tiles, st)
               : launch_down_tile<Mx4Tile<128, 128, 64, 64, 2>>(a, P, tiles, st);
    else
        narrow ? launch_down_tile<Mx4Tile<64, 128, 32, 64, 3>, false>(a, P, tiles, st)
               : launch_down_tile<Mx4Tile<128, 128, 64, 64, 2>, false>(a, P, tiles, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    I8Down c{};
    c.down.rows = a.down.rows, c.down.count = a.down.count;
    c.m = a.m, c.slots = a.slots, c.ids = a.ids, c.n_sel = a.n_sel, c.work = a.work;
    c.y = a.y, c.dt = a.dt, c.ldy = a.ldy, c.accumulate = a.accumulate, c.vec = a.vec;
    return launch_experts_combine(c, st);
}

}  // namespace trk
