// The int8 products of each token with its experts (trk_experts_plan, trk_experts_up_i8, trk_experts_down_i8).
#include "i8.hpp"

namespace trk {

namespace {

// ============================================================================================
// the plan: entries sorted by expert
// ============================================================================================

constexpr uint32_t PLAN_T = 1024;

// One workgroup: the entries of each expert counted in LDS, the counts summed to offsets, the entries put to their
// places and every expert's run cut into tiles.  The order of an expert's entries is that of the atomics and may change;
// nothing that the products write depends on it (an entry's row is computed by itself and kept at its own place).
__global__ __launch_bounds__(PLAN_T) void experts_plan_kernel(const uint32_t* __restrict__ ids,
                                                              const uint32_t* __restrict__ n_sel, uint32_t m,
                                                              uint32_t slots, uint32_t E, uint32_t rows,
                                                              uint32_t* __restrict__ plan) {
    __shared__ uint32_t cnt[PLAN_T], tcnt[PLAN_T], wsum[2][PLAN_T / WAVE];
    const uint32_t tid = threadIdx.x, lane = tid % WAVE, wv = tid / WAVE, n = m * slots;
    cnt[tid] = 0;
    __syncthreads();
    auto expert = [&](uint32_t i) {
        const uint32_t t = i / slots, j = i % slots;
        const uint32_t e = j < n_sel[t] ? ids[(size_t)t * K_MAX + j] : 0xffffffffu;
        return e < E ? e : 0xffffffffu;
    };
    for (uint32_t i = tid; i < n; i += PLAN_T) {
        const uint32_t e = expert(i);
        if (e != 0xffffffffu) atomicAdd(&cnt[e], 1u);
    }
    __syncthreads();
    const uint32_t c = cnt[tid], tc = (c + rows - 1) / rows;
    const uint32_t si = wave_incl_scan_u32(c), ti = wave_incl_scan_u32(tc);
    if (lane == WAVE - 1) wsum[0][wv] = si, wsum[1][wv] = ti;
    __syncthreads();
    uint32_t so = si - c, to = ti - tc;
    for (uint32_t i = 0; i < wv; i++) so += wsum[0][i], to += wsum[1][i];
    const Plan P = plan_at(plan, m, slots);
    for (uint32_t i = 0; i < tc; i++)
        P.tile[to + i] = PlanTile{tid, so + i * rows, c - i * rows < rows ? c - i * rows : rows, 0};
    if (tid == PLAN_T - 1) *P.n_tiles = to + tc;
    cnt[tid] = so;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += PLAN_T) {
        const uint32_t e = expert(i);
        if (e != 0xffffffffu) P.ent[atomicAdd(&cnt[e], 1u)] = i;
    }
}

// ============================================================================================
// few entries: each by itself
// ============================================================================================

constexpr uint32_t ST_WAVES = 4;

// This lane's row of the 16 from r0 on
__device__ __forceinline__ const int8_t* strip_row(const I8Mat& w, uint32_t e, uint32_t r0, uint32_t lane) {
    const uint32_t r = r0 + lane % 16;
    return w.ptr + e * w.stride + (r < w.rows ? r : w.rows - 1) * w.ld;
}

// A workgroup takes 16 rows of gate and up and a tile's (or, without a plan, one) entries; its waves share K.
template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES * WAVE) void experts_up_strip_kernel(I8Up a, Plan P) {
    __shared__ int32_t part[2][ST_WAVES][16][16];  // [gate, up][wave][entry][weight row]
    __shared__ uint32_t ent[16];
    const uint32_t strips = (a.gate.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, it = id / strips;
    uint32_t e, n;
    if (P.ent) {
        if (it >= *P.n_tiles) return;
        const PlanTile t = P.tile[it];
        e = t.expert, n = t.rows;
        if (threadIdx.x < 16) ent[threadIdx.x] = P.ent[t.row0 + (threadIdx.x < n ? threadIdx.x : 0)];
    } else {
        if (it >= a.m * a.slots || it % a.slots >= a.n_sel[it / a.slots]) return;
        e = a.ids[(size_t)(it / a.slots) * K_MAX + it % a.slots], n = 1;
        if (e >= a.gate.count) return;
        if (threadIdx.x < 16) ent[threadIdx.x] = it;
    }
    __syncthreads();
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, c = lane % 16;
    const int8_t* xr = a.q + (uint64_t)(ent[c] / a.slots) * a.ldq;
    *reinterpret_cast<i32x4*>(&part[0][wv][c][lane / 16 * 4]) = strip_sum(strip_row(a.gate, e, r0, lane), xr, a.gate.k, wv, ST_WAVES, lane);
    *reinterpret_cast<i32x4*>(&part[1][wv][c][lane / 16 * 4]) = strip_sum(strip_row(a.up, e, r0, lane), xr, a.gate.k, wv, ST_WAVES, lane);
    __syncthreads();
    const uint32_t ei = threadIdx.x / 16, ri = threadIdx.x % 16, r = r0 + ri;
    if (ei >= n || r >= a.gate.rows) return;
    int32_t sg = 0, su = 0;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) sg += part[0][i][ei][ri], su += part[1][i][ei][ri];
    const float sx = a.sx[ent[ei] / a.slots];
    const uint64_t ws = (uint64_t)e * a.gate.rows + r;
    typedef Elem<DT> O;
    reinterpret_cast<typename O::T*>(a.h)[ent[ei] * a.ldh + r] =
            O::put(swiglu(i8_scaled(sg, sx, a.gate.scale[ws]), i8_scaled(su, sx, a.up.scale[ws])));
}

// A workgroup takes 16 down rows and one token: a wave per slot in turn, the slots' rows added in order.
template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES * WAVE) void experts_down_strip_kernel(I8Down a) {
    __shared__ float part[K_MAX][16];
    const uint32_t strips = (a.down.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, t = id / strips;
    if (t >= a.m) return;
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t n = a.n_sel[t] < a.slots ? a.n_sel[t] : a.slots;
    for (uint32_t j = wv; j < n; j += ST_WAVES) {
        const uint32_t e = a.ids[(size_t)t * K_MAX + j];
        if (e >= a.down.count) continue;
        const uint64_t row = (uint64_t)t * a.slots + j;
        const i32x4 s = strip_sum(strip_row(a.down, e, r0, lane), a.q + row * a.ldq, a.down.k, 0, 1, lane);
        if (lane % 16 == 0)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t r = r0 + lane / 16 * 4 + i, rc = r < a.down.rows ? r : a.down.rows - 1;
                part[j][lane / 16 * 4 + i] =
                        i8_scaled(s[i], a.sx[row], a.down.scale[(uint64_t)e * a.down.rows + rc]) * a.w[(size_t)t * K_MAX + j];
            }
    }
    __syncthreads();
    const uint32_t r = r0 + threadIdx.x;
    if (threadIdx.x >= 16 || r >= a.down.rows) return;
    float v = 0.0f;
    for (uint32_t j = 0; j < n; j++)
        if (a.ids[(size_t)t * K_MAX + j] < a.down.count) v += part[j][threadIdx.x];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(a.y) + t * a.ldy + r;
    *y = O::put(a.accumulate ? O::get(*y) + v : v);
}

// ============================================================================================
// many entries: tiles of one expert's
// ============================================================================================

// 16 down rows of a tile's entries into work [m * slots][rows], weighted
__global__ __launch_bounds__(ST_WAVES * WAVE) void experts_down_tile_kernel(I8Down a, Plan P) {
    __shared__ int32_t part[ST_WAVES][16][16];
    __shared__ uint32_t ent[16];
    const uint32_t strips = (a.down.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, it = id / strips;
    if (it >= *P.n_tiles) return;
    const PlanTile t = P.tile[it];
    if (threadIdx.x < 16) ent[threadIdx.x] = P.ent[t.row0 + (threadIdx.x < t.rows ? threadIdx.x : 0)];
    __syncthreads();
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, c = lane % 16;
    *reinterpret_cast<i32x4*>(&part[wv][c][lane / 16 * 4]) =
            strip_sum(strip_row(a.down, t.expert, r0, lane), a.q + (uint64_t)ent[c] * a.ldq, a.down.k, wv, ST_WAVES, lane);
    __syncthreads();
    const uint32_t ei = threadIdx.x / 16, ri = threadIdx.x % 16, r = r0 + ri;
    if (ei >= t.rows || r >= a.down.rows) return;
    int32_t s = 0;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) s += part[i][ei][ri];
    const uint32_t en = ent[ei];
    a.work[(uint64_t)en * a.down.rows + r] =
            i8_scaled(s, a.sx[en], a.down.scale[(uint64_t)t.expert * a.down.rows + r]) *
            a.w[(size_t)(en / a.slots) * K_MAX + en % a.slots];
}

// y[t] (+)= the rows of its entries, in slot order
template <uint32_t DT>
__global__ __launch_bounds__(256) void experts_combine_kernel(I8Down a) {
    const uint32_t cols = (a.down.rows + 255) / 256, id = run_id(), t = id / cols, r = id % cols * 256 + threadIdx.x;
    if (t >= a.m || r >= a.down.rows) return;
    float v = 0.0f;
    const uint32_t n = a.n_sel[t] < a.slots ? a.n_sel[t] : a.slots;
    for (uint32_t j = 0; j < n; j++)
        if (a.ids[(size_t)t * K_MAX + j] < a.down.count) v += a.work[((uint64_t)t * a.slots + j) * a.down.rows + r];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(a.y) + t * a.ldy + r;
    *y = O::put(a.accumulate ? O::get(*y) + v : v);
}

dim3 run_of(uint64_t wgs, uint32_t threads) {
    const geo::Grid2 g = geo::grid_run(wgs, threads);
    return dim3(g.x, g.y);
}

}  // namespace

hipError_t launch_experts_plan(const uint32_t* ids, const uint32_t* n_sel, uint32_t m, uint32_t slots, uint32_t E,
                               uint32_t* plan, hipStream_t st) {
    experts_plan_kernel<<<1, PLAN_T, 0, st>>>(ids, n_sel, m, slots, E, geo::plan_rows(m, slots, E), plan);
    return hipGetLastError();
}

hipError_t launch_experts_up(const I8Up& a, const uint32_t* plan, hipStream_t st) {
    const uint32_t E = a.gate.count;
    Plan P{};
    uint64_t items = (uint64_t)a.m * a.slots;
    if (plan) {
        const uint32_t rows = geo::plan_rows(a.m, a.slots, E);
        P = plan_at(const_cast<uint32_t*>(plan), a.m, a.slots);
        items = geo::plan_tiles(a.m, a.slots, E, rows);
    }
    const dim3 g = run_of((a.gate.rows + 15) / 16 * items, ST_WAVES * WAVE);
    if (a.dt == TRK_DT_F32)
        experts_up_strip_kernel<TRK_DT_F32><<<g, ST_WAVES * WAVE, 0, st>>>(a, P);
    else if (a.dt == TRK_DT_BF16)
        experts_up_strip_kernel<TRK_DT_BF16><<<g, ST_WAVES * WAVE, 0, st>>>(a, P);
    else
        experts_up_strip_kernel<TRK_DT_F16><<<g, ST_WAVES * WAVE, 0, st>>>(a, P);
    return hipGetLastError();
}

hipError_t launch_experts_down(const I8Down& a, const uint32_t* plan, hipStream_t st) {
    const uint32_t E = a.down.count;
    if (!plan) {
        const dim3 g = run_of((uint64_t)((a.down.rows + 15) / 16) * a.m, ST_WAVES * WAVE);
        if (a.dt == TRK_DT_F32)
            experts_down_strip_kernel<TRK_DT_F32><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        else if (a.dt == TRK_DT_BF16)
            experts_down_strip_kernel<TRK_DT_BF16><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        else
            experts_down_strip_kernel<TRK_DT_F16><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        return hipGetLastError();
    }
    const uint32_t rows = geo::plan_rows(a.m, a.slots, E);
    const Plan P = plan_at(const_cast<uint32_t*>(plan), a.m, a.slots);
    experts_down_tile_kernel<<<run_of((a.down.rows + 15) / 16 * geo::plan_tiles(a.m, a.slots, E, rows),
                                      ST_WAVES * WAVE), ST_WAVES * WAVE, 0, st>>>(a, P);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const dim3 g = run_of((uint64_t)((a.down.rows + 255) / 256) * a.m, 256);
    if (a.dt == TRK_DT_F32)
        experts_combine_kernel<TRK_DT_F32><<<g, 256, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        experts_combine_kernel<TRK_DT_BF16><<<g, 256, 0, st>>>(a);
    else
        experts_combine_kernel<TRK_DT_F16><<<g, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace trk
