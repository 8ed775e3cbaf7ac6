// The int8 products of each token with its experts (trk_experts_plan, trk_experts_up_i8, trk_experts_down_i8).
#include "i8tile.hpp"
#include "plan.hpp"

namespace trk {

namespace {

// ============================================================================================
// the plan: entries sorted by expert
// ============================================================================================

// The expert of entry i, ~0 for a slot that is none.
__device__ __forceinline__ uint32_t entry_expert(const uint32_t* __restrict__ ids, const uint32_t* __restrict__ n_sel,
                                                 uint32_t slots, uint32_t E, uint32_t i, uint32_t n) {
    const uint32_t ic = i < n ? i : n - 1, t = ic / slots, j = ic % slots;
    const uint32_t e = ids[(size_t)t * K_MAX + j], c = n_sel[t];  // both requested before either is looked at
    return i < n && j < c && e < E ? e : 0xffffffffu;
}

// The counts of `per` * PLAN_T entries from i0 on, into cnt[] of LDS (zeroed here).
__device__ __forceinline__ void plan_count(const uint32_t* __restrict__ ids, const uint32_t* __restrict__ n_sel, uint32_t slots,
                                           uint32_t E, uint32_t n, uint32_t i0, uint32_t per, uint32_t* cnt) {
    cnt[threadIdx.x] = 0;
    __syncthreads();
    for (uint32_t p = 0; p < per; p += 4) {
        uint32_t e[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
            e[u] = p + u < per ? entry_expert(ids, n_sel, slots, E, i0 + (p + u) * PLAN_T + threadIdx.x, n) : 0xffffffffu;
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
            if (e[u] != 0xffffffffu) atomicAdd(&cnt[e[u]], 1u);
    }
    __syncthreads();
}

// The counts of each workgroup's share of the entries, for the next kernel's offsets.
__global__ __launch_bounds__(PLAN_T) void experts_count_kernel(const uint32_t* __restrict__ ids,
                                                               const uint32_t* __restrict__ n_sel, uint32_t m,
                                                               uint32_t slots, uint32_t E, uint32_t per,
                                                               uint32_t* __restrict__ counts) {
    __shared__ uint32_t cnt[PLAN_T];
    plan_count(ids, n_sel, slots, E, m * slots, blockIdx.x * per * PLAN_T, per, cnt);
    if (threadIdx.x < E) counts[blockIdx.x * E + threadIdx.x] = cnt[threadIdx.x];
}

// Counts summed to offsets (every workgroup for itself: `counts` [gridDim.x][E], or its own where it is the only one),
// this workgroup's entries put to their places, and (the first) every expert's run cut into tiles.  The order of an
// expert's entries is that of the LDS atomics and may change; nothing that the products write depends on it (an entry's
// row is computed by itself and kept at its own place).  What bounds it: trips to memory (40960 entries of 512 experts, both
// kernels, 9.1 us).
__global__ __launch_bounds__(PLAN_T) void experts_plan_kernel(const uint32_t* __restrict__ ids,
                                                              const uint32_t* __restrict__ n_sel, uint32_t m,
                                                              uint32_t slots, uint32_t E, uint32_t rows, uint32_t per,
                                                              const uint32_t* __restrict__ counts, Plan P) {
    __shared__ uint32_t cnt[PLAN_T], wsum[2][PLAN_T / WAVE];
    const uint32_t tid = threadIdx.x, lane = tid % WAVE, wv = tid / WAVE, n = m * slots, i0 = blockIdx.x * per * PLAN_T;
    uint32_t c = 0, before = 0;  // expert tid's entries, and those of the workgroups before this one
    if (gridDim.x == 1) {
        plan_count(ids, n_sel, slots, E, n, 0, per, cnt);
        c = cnt[tid];
    } else if (tid < E) {
#pragma unroll 8
        for (uint32_t b = 0; b < gridDim.x; b++) {
            const uint32_t v = counts[b * E + tid];
            c += v;
            before += b < blockIdx.x ? v : 0;
        }
    }
    const uint32_t tc = (c + rows - 1) / rows;
    const uint32_t si = wave_incl_scan_u32(c), ti = wave_incl_scan_u32(tc);
    if (lane == WAVE - 1) wsum[0][wv] = si, wsum[1][wv] = ti;
    __syncthreads();
    uint32_t so = si - c, to = ti - tc;
    for (uint32_t i = 0; i < wv; i++) so += wsum[0][i], to += wsum[1][i];
    cnt[tid] = so + before;
    __syncthreads();
    for (uint32_t p = 0; p < per; p += 4) {
        uint32_t e[4];
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
            e[u] = p + u < per ? entry_expert(ids, n_sel, slots, E, i0 + (p + u) * PLAN_T + tid, n) : 0xffffffffu;
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
            if (e[u] != 0xffffffffu) P.ent[atomicAdd(&cnt[e[u]], 1u)] = i0 + (p + u) * PLAN_T + tid;
    }
    if (blockIdx.x) return;
    for (uint32_t i = 0; i < tc; i++)
        P.tile[to + i] = PlanTile{tid, so + i * rows, c - i * rows < rows ? c - i * rows : rows, 0};
    if (tid == PLAN_T - 1) *P.head = PlanHead{to + tc, m, slots, E};
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

// A workgroup takes 16 rows of gate and up and one entry; its waves share K.  Two trips to memory, the ids' and the rows': one
// token of 10 in 512 experts (H = 2048, F = 512; 21 MB) 6.4 us where a cache holds the weights, 9.0 from memory.
template <uint32_t DT>
__global__ __launch_bounds__(ST_WAVES * WAVE) void experts_up_strip_kernel(I8Up a) {
    __shared__ int32_t part[2][ST_WAVES][16];  // [gate, up][wave][weight row]
    const uint32_t strips = (a.gate.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, en = id / strips;
    const uint32_t t = en / a.slots, j = en % a.slots;
    if (t >= a.m) return;  // the whole workgroup, here and below
    const uint32_t e = a.ids[(size_t)t * K_MAX + j], n = a.n_sel[t];
    if (j >= n || e >= a.gate.count) return;
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t r = r0 + threadIdx.x;
    const bool out = threadIdx.x < 16 && r < a.gate.rows;
    float sx = 0.0f, sg = 0.0f, su = 0.0f;
    if (out) sx = a.sx[t], sg = a.gate.scale[(uint64_t)e * a.gate.rows + r], su = a.up.scale[(uint64_t)e * a.gate.rows + r];
    i32x4 acc[2];
    // every column of the matrix instruction is this token's row
    strip_sums<2>({strip_row(a.gate, e, r0, lane), strip_row(a.up, e, r0, lane)}, a.q + (uint64_t)t * a.ldq, a.gate.k, wv,
                  ST_WAVES, lane, acc);
    if (lane % 16 == 0) {
        *reinterpret_cast<i32x4*>(&part[0][wv][lane / 16 * 4]) = acc[0];
        *reinterpret_cast<i32x4*>(&part[1][wv][lane / 16 * 4]) = acc[1];
    }
    __syncthreads();
    if (!out) return;
    int32_t g = 0, u = 0;
#pragma unroll
    for (uint32_t i = 0; i < ST_WAVES; i++) g += part[0][i][threadIdx.x], u += part[1][i][threadIdx.x];
    typedef Elem<DT> O;
    reinterpret_cast<typename O::T*>(a.h)[en * a.ldh + r] = O::put(swiglu(i8_scaled(g, sx, sg), i8_scaled(u, sx, su)));
}

// A workgroup takes 16 down rows and one token: a wave per slot (several where there are fewer slots than waves, sharing
// K; in turn where there are more), then a thread per (slot, row) scales and weights, and a thread per row adds in slot
// order.  Four tokens of 10 in 512 (41 MB) 9.4 us where a cache holds the weights, 11.7 from memory.
constexpr uint32_t DOWN_WAVES = 8;  // 12 and 16 are slower where timed: four tokens of ten slots 11.3, 13.1 and 13.2 us

template <uint32_t DT>
__global__ __launch_bounds__(DOWN_WAVES* WAVE) void experts_down_strip_kernel(I8Down a) {
    __shared__ int32_t part[K_MAX * 4][16];  // [slot * share of K][weight row]
    __shared__ float term[K_MAX][16];
    const uint32_t strips = (a.down.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, t = id / strips;
    if (t >= a.m) return;
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t ks = DOWN_WAVES / a.slots >= 4 ? 4 : DOWN_WAVES / a.slots >= 2 ? 2 : 1;  // waves that share a slot
    const uint32_t* ids = a.ids + (size_t)t * K_MAX;
    const uint32_t ns = a.n_sel[t], n = ns < a.slots ? ns : a.slots;
    static_assert(DOWN_WAVES * WAVE >= K_MAX * 16, "a thread per (slot, row)");
    const uint32_t ri = threadIdx.x % 16, r = r0 + ri, rc = r < a.down.rows ? r : a.down.rows - 1;
    const uint32_t j = threadIdx.x / 16, jc = j < a.slots ? j : 0, e = ids[jc];
    const bool there = j < n && e < a.down.count;
    const float sx = a.sx[(uint64_t)t * a.slots + jc], wt = a.w[(size_t)t * K_MAX + jc];
    const float sw = a.down.scale[(uint64_t)(there ? e : 0) * a.down.rows + rc];
    for (uint32_t w = wv; w < a.slots * ks; w += DOWN_WAVES) {
        const uint32_t ew = ids[w / ks];
        if (w / ks >= n || ew >= a.down.count) continue;
        i32x4 acc[1];
        strip_sums<1>({strip_row(a.down, ew, r0, lane)}, a.q + ((uint64_t)t * a.slots + w / ks) * a.ldq, a.down.k, w % ks, ks,
                      lane, acc);
        if (lane % 16 == 0) *reinterpret_cast<i32x4*>(&part[w][lane / 16 * 4]) = acc[0];
    }
    __syncthreads();
    if (j < n) {
        int32_t s = part[j * ks][ri];
        for (uint32_t c = 1; c < ks; c++) s += part[j * ks + c][ri];
        term[j][ri] = there ? i8_scaled(s, sx, sw) * wt : 0.0f;
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

// gate and up: a tile's weight rows are BN / 2 rows of gate, then the same rows of up, and a wave has both of each.  ONCE:
// geo::experts_once.  2000 tokens of 8 in 128 (H = 2048, F = 768; 432 MB, 101 G operations) 115 us; 4096 of 10 in 512 (F = 512;
// 1.1 GB) 232: memory, at 3.8 and 4.8 TB/s, beside the products.
template <typename Tile, uint32_t DT, bool ONCE>
__global__ __launch_bounds__(Tile::T) void experts_up_tile_kernel(I8Up a, Plan P) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::LDS];
    constexpr uint32_t BR = Tile::BN / 2, FR = Tile::FN / 2;
    static_assert(BR % (8 * Tile::NW) == 0 && Tile::WN % 32 == 0, "a load takes rows of one matrix");
    PlanTile pt;
    uint32_t block;
    const PlanHead head = *P.head;
    if (!plan_fits(head, a.m, a.slots, a.gate.count))  // the whole workgroup, here and below
        return nan_rows<DT>(a, a.gate.count, a.h, a.gate.rows, a.ldh);
    if (!expert_tile(P, head, a.gate.count, (a.gate.rows + BR - 1) / BR, pt, block)) return;
    const uint32_t r0 = block * BR, rl = a.gate.rows - r0 - 1;  // the last row there is
    Tile t;
    auto entry = [&](uint32_t i) { return P.ent[pt.row0 + (i < pt.rows ? i : pt.rows - 1)]; };
    const i32x4 bg = buffer_at(a.gate.ptr + pt.expert * a.gate.stride + r0 * a.gate.ld);
    const i32x4 bu = buffer_at(a.up.ptr + pt.expert * a.up.stride + r0 * a.up.ld);
    i32x4 rw[Tile::NA];
    uint32_t wo[Tile::NA], xo[Tile::NB];
#pragma unroll
    for (int i = 0; i < Tile::NB; i++) xo[i] = entry(t.load_row(i)) / a.slots * (uint32_t)a.ldq;
#pragma unroll
    for (int i = 0; i < Tile::NA; i++) {
        const bool up = i * Tile::NW * 8 >= BR;
        const uint32_t r = t.load_row(i) - (up ? BR : 0), rc = r < rl ? r : rl;
        rw[i] = up ? bu : bg, wo[i] = rc * (uint32_t)(up ? a.up.ld : a.gate.ld);
    }
    const uint32_t wr = t.wn / 2;  // this wave's first row of both
    // what the entries and rows are scaled with, before the loads that the products wait for
    float sg[FR][4], su[FR][4], sx[Tile::FM];
    uint32_t en[Tile::FM];
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) en[j] = entry(t.wm + 16 * j + t.lane % 16);
#pragma unroll
    for (uint32_t i = 0; i < FR; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t r = wr + 16 * i + t.lane / 16 * 4 + c;
            const uint64_t at = (uint64_t)pt.expert * a.gate.rows + r0 + (r < rl ? r : rl);
            sg[i][c] = a.gate.scale[at], su[i][c] = a.up.scale[at];
        }
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) sx[j] = a.sx[en[j] / a.slots];
    const uint32_t live = t.wm < pt.rows ? (pt.rows - t.wm + 15) / 16 : 0;
    t.template run<true, ONCE>(lds, rw, wo, buffer_at(a.q), xo, a.gate.k, live,
                               [&](int i) { return i < FR ? wr + 16 * i : BR + wr + 16 * (i - FR); });
    typedef Elem<DT> O;
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        if (t.wm + 16 * j + t.lane % 16 >= pt.rows) continue;
        typename O::T* h = reinterpret_cast<typename O::T*>(a.h) + en[j] * a.ldh;
#pragma unroll
        for (uint32_t i = 0; i < FR; i++) {
            const uint32_t r = r0 + wr + 16 * i + t.lane / 16 * 4;
            float g[4], u[4], v[4];
#pragma unroll
            for (int c = 0; c < 4; c++)
                g[c] = i8_scaled(t.acc[i][j][c], sx[j], sg[i][c]), u[c] = i8_scaled(t.acc[FR + i][j][c], sx[j], su[i][c]);
            swiglu4(g, u, v);
            store4<DT>(h + r, v, r < a.gate.rows ? a.gate.rows - r : 0, a.vec);
        }
    }
}

// down: the entries' weighted rows into work [m * slots][rows], in 32 bits, as they are then added.  ONCE: geo::experts_once.
// Memory bounds it: 4096 tokens of 10 in 512 (H = 2048, F = 512) read 560 MB and write 336 in some 225 us (239 under a trace).
template <typename Tile, bool ONCE>
__global__ __launch_bounds__(Tile::T) void experts_down_tile_kernel(I8Down a, Plan P) {
    __shared__ __attribute__((aligned(1024))) uint8_t lds[Tile::LDS];
    PlanTile pt;
    uint32_t block;
    const PlanHead head = *P.head;
    if (!plan_fits(head, a.m, a.slots, a.down.count))  // the whole workgroup, here and below
        return nan_rows<TRK_DT_F32>(a, a.down.count, a.work, a.down.rows, a.down.rows);
    if (!expert_tile(P, head, a.down.count, (a.down.rows + Tile::BN - 1) / Tile::BN, pt, block)) return;
    const uint32_t r0 = block * Tile::BN, rl = a.down.rows - r0 - 1;
    Tile t;
    auto entry = [&](uint32_t i) { return P.ent[pt.row0 + (i < pt.rows ? i : pt.rows - 1)]; };
    const i32x4 bw = buffer_at(a.down.ptr + pt.expert * a.down.stride + r0 * a.down.ld);
    i32x4 rw[Tile::NA];
    uint32_t wo[Tile::NA], xo[Tile::NB];
#pragma unroll
    for (int i = 0; i < Tile::NB; i++) xo[i] = entry(t.load_row(i)) * (uint32_t)a.ldq;
#pragma unroll
    for (int i = 0; i < Tile::NA; i++) {
        const uint32_t r = t.load_row(i);
        rw[i] = bw, wo[i] = (r < rl ? r : rl) * (uint32_t)a.down.ld;
    }
    float sw[Tile::FN][4], sx[Tile::FM], w[Tile::FM];
    uint32_t en[Tile::FM];
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) en[j] = entry(t.wm + 16 * j + t.lane % 16);
#pragma unroll
    for (int i = 0; i < Tile::FN; i++)
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const uint32_t r = t.wn + 16 * i + t.lane / 16 * 4 + c;
            sw[i][c] = a.down.scale[(uint64_t)pt.expert * a.down.rows + r0 + (r < rl ? r : rl)];
        }
#pragma unroll
    for (int j = 0; j < Tile::FM; j++)
        sx[j] = a.sx[en[j]], w[j] = a.w[(size_t)(en[j] / a.slots) * K_MAX + en[j] % a.slots];
    const uint32_t live = t.wm < pt.rows ? (pt.rows - t.wm + 15) / 16 : 0;
    t.template run<true, ONCE>(lds, rw, wo, buffer_at(a.q), xo, a.down.k, live, [&](int i) { return t.wn + 16 * i; });
#pragma unroll
    for (int j = 0; j < Tile::FM; j++) {
        if (t.wm + 16 * j + t.lane % 16 >= pt.rows) continue;
        float* y = a.work + (uint64_t)en[j] * a.down.rows;
#pragma unroll
        for (int i = 0; i < Tile::FN; i++) {
            const uint32_t r = r0 + t.wn + 16 * i + t.lane / 16 * 4;
            float v[4];
#pragma unroll
            for (int c = 0; c < 4; c++) v[c] = i8_scaled(t.acc[i][j][c], sx[j], sw[i][c]) * w[j];
            store4<TRK_DT_F32>(y + r, v, r < a.down.rows ? a.down.rows - r : 0, a.down.rows % 4 == 0);
        }
    }
}

// y[t] (+)= the rows of its entries, in slot order: a thread per four columns, several tokens a workgroup where a row is
// short.  Four slots' rows are requested before the first is added.  They are read once and for the last time: past the
// caches' replacement order, what a larger work leaves there is still there for its turn (4096 tokens of 10 in 512 309 -> 294
// us, 8192 of 10 567 -> 542, 4096 of 4 in 64 270 -> 262; 2000 of 8 in 128 134 -> 135, 8192 of 2 in 8 169 -> 172).
template <uint32_t DT>
__global__ __launch_bounds__(256) void experts_combine_kernel(I8Down a) {
    const uint32_t w = a.down.rows, q = (w + 3) / 4, per = q < 256 ? 256 / q : 1, cols = (q + 255) / 256, id = run_id();
    const uint32_t sub = q < 256 ? threadIdx.x / q : 0, t = id / cols * per + sub;
    const uint32_t r = 4 * (q < 256 ? threadIdx.x % q : id % cols * 256 + threadIdx.x);
    if (t >= a.m || r >= w || sub >= per) return;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint32_t n = a.n_sel[t] < a.slots ? a.n_sel[t] : a.slots;
    const float* s = a.work + (uint64_t)t * a.slots * w + r;
    // A row's last columns are read and added with those before them: lanes that read them one by one would have the wave wait twice
    // (150 tokens of 6 in 60, 1101 columns 6.5 -> 5.9 us; four loads of one column each 5.9, but 2000 of 8 in 128, 2047 columns 36 for 29).
    const uint32_t back = w >= 4 && r + 4 > w ? r + 4 - w : 0;
    for (uint32_t j0 = 0; j0 < n; j0 += 4) {
        float p[4][4];
        bool on[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) {
            const uint32_t jc = j0 + j < n ? j0 + j : n - 1;
            on[j] = j0 + j < n && a.ids[(size_t)t * K_MAX + jc] < a.down.count;
            if (j0 + j >= n) continue;  // a row of no entry is read (anything) and not added: no load waits for another
            const float* f = s + (uint64_t)jc * w;
            if (w >= 4) {
                typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
                const f32x4_any x = __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(f - back));
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) p[j][c] = x[c];
            } else {
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) p[j][c] = f[r + c < w ? c : 0];
            }
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
            if (on[j])
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) v[c] += p[j][c];
    }
    if (back & 2) v[0] = v[2], v[1] = v[3];
    if (back & 1) v[0] = v[1], v[1] = v[2], v[2] = v[3];
    typedef Elem<DT> O;
    typename O::T* y = reinterpret_cast<typename O::T*>(a.y) + t * a.ldy + r;
    if (a.accumulate)
#pragma unroll
        for (uint32_t c = 0; c < 4; c++)
            if (r + c < w) v[c] += O::get(y[c]);
    store4<DT>(y, v, w - r, a.vec);
}

dim3 run_of(uint64_t wgs, uint32_t threads) {
    const geo::Grid2 g = geo::grid_run(wgs, threads);
    return dim3(g.x, g.y);
}

}  // namespace

hipError_t launch_experts_plan(const uint32_t* ids, const uint32_t* n_sel, uint32_t m, uint32_t slots, uint32_t E,
                               uint32_t* plan, hipStream_t st) {
    const Plan P = plan_at(plan, m, slots);
    const uint32_t wgs = geo::plan_workgroups(m, slots), n = m * slots, per = (n + wgs * PLAN_T - 1) / (wgs * PLAN_T);
    uint32_t* counts = plan + geo::plan_counts_at(m, slots, E);
    if (wgs > 1) {
        experts_count_kernel<<<wgs, PLAN_T, 0, st>>>(ids, n_sel, m, slots, E, per, counts);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    experts_plan_kernel<<<wgs, PLAN_T, 0, st>>>(ids, n_sel, m, slots, E, geo::plan_rows(m, slots, E), per, counts, P);
    return hipGetLastError();
}

template <typename Tile, bool ONCE = true>
static void launch_up_tile(const I8Up& a, const Plan& P, uint64_t tiles, hipStream_t st) {
    const dim3 g = run_of((a.gate.rows + Tile::BN / 2 - 1) / (Tile::BN / 2) * tiles, Tile::T);
    if (a.dt == TRK_DT_F32)
        experts_up_tile_kernel<Tile, TRK_DT_F32, ONCE><<<g, Tile::T, 0, st>>>(a, P);
    else if (a.dt == TRK_DT_BF16)
        experts_up_tile_kernel<Tile, TRK_DT_BF16, ONCE><<<g, Tile::T, 0, st>>>(a, P);
    else
        experts_up_tile_kernel<Tile, TRK_DT_F16, ONCE><<<g, Tile::T, 0, st>>>(a, P);
}

// The kernels number their workgroups by 32 bits: of entries beyond, so many tokens a launch.
static uint32_t strip_tokens(uint32_t rows, uint32_t per_token) {
    const uint64_t t = 0x7fffffffull / ((rows + 15) / 16) / per_token;
    return t < 1 ? 1 : t > 0x7fffffffull ? 0x7fffffffu : (uint32_t)t;
}

static void launch_up_strip(I8Up a, hipStream_t st) {
    const uint32_t m = a.m, step = strip_tokens(a.gate.rows, a.slots);
    const uint64_t size = a.dt == TRK_DT_F32 ? 4 : 2;
    for (uint64_t t = 0; t < m; t += step) {
        a.m = m - t < step ? m - (uint32_t)t : step;
        const dim3 g = run_of((uint64_t)((a.gate.rows + 15) / 16) * a.m * a.slots, ST_WAVES * WAVE);
        if (a.dt == TRK_DT_F32)
            experts_up_strip_kernel<TRK_DT_F32><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        else if (a.dt == TRK_DT_BF16)
            experts_up_strip_kernel<TRK_DT_BF16><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        else
            experts_up_strip_kernel<TRK_DT_F16><<<g, ST_WAVES * WAVE, 0, st>>>(a);
        a.q += step * a.ldq, a.sx += step, a.ids += (uint64_t)step * K_MAX, a.n_sel += step;
        a.h = (char*)a.h + (uint64_t)step * a.slots * a.ldh * size;
    }
}

template <bool ONCE>
static void launch_up_128(const I8Up& a, const Plan& P, uint64_t tiles, geo::ExpertsWidth w, hipStream_t st) {
    if (w == geo::X_NARROW)
        launch_up_tile<I8Tile<64, 128, 32, 64, 3>, ONCE>(a, P, tiles, st);
    else
        w == geo::X_WIDE ? launch_up_tile<I8Tile<256, 128, 64, 64, 3>, ONCE>(a, P, tiles, st)
                         : launch_up_tile<I8Tile<128, 128, 64, 64, 2>, ONCE>(a, P, tiles, st);
}

hipError_t launch_experts_up(const I8Up& a, const uint32_t* plan, hipStream_t st) {
    const uint32_t E = a.gate.count;
    if (!plan || !geo::i8_tile_addresses(a.gate.ld, a.ldq, a.m) || !geo::i8_tile_addresses(a.up.ld, a.ldq, a.m)) {
        launch_up_strip(a, st);
        return hipGetLastError();
    }
    const uint32_t rows = geo::plan_rows(a.m, a.slots, E);
    const Plan P = plan_at(const_cast<uint32_t*>(plan), a.m, a.slots);
    const uint64_t tiles = geo::plan_tiles(a.m, a.slots, E, rows);
    const geo::ExpertsWidth w = geo::experts_width(2 * a.gate.rows, tiles, rows == 128);
    if (rows == 32)
        w == geo::X_NARROW ? launch_up_tile<I8Tile<64, 32, 32, 16, 4>>(a, P, tiles, st)
                           : launch_up_tile<I8Tile<128, 32, 32, 32, 3>>(a, P, tiles, st);
    else if (rows == 64)
        w == geo::X_NARROW ? launch_up_tile<I8Tile<64, 64, 32, 32, 4>>(a, P, tiles, st)
                           : launch_up_tile<I8Tile<128, 64, 64, 32, 2>>(a, P, tiles, st);
    else if (geo::experts_once(a.m, a.slots, E, 64))
        launch_up_128<true>(a, P, tiles, w, st);
    else
        launch_up_128<false>(a, P, tiles, w, st);
    return hipGetLastError();
}

static void launch_down_strip(I8Down a, hipStream_t st) {
    const uint32_t m = a.m, step = strip_tokens(a.down.rows, 1);
    const uint64_t size = a.dt == TRK_DT_F32 ? 4 : 2;
    for (uint64_t t = 0; t < m; t += step) {
        a.m = m - t < step ? m - (uint32_t)t : step;
        const dim3 g = run_of((uint64_t)((a.down.rows + 15) / 16) * a.m, DOWN_WAVES * WAVE);
        if (a.dt == TRK_DT_F32)
            experts_down_strip_kernel<TRK_DT_F32><<<g, DOWN_WAVES * WAVE, 0, st>>>(a);
        else if (a.dt == TRK_DT_BF16)
            experts_down_strip_kernel<TRK_DT_BF16><<<g, DOWN_WAVES * WAVE, 0, st>>>(a);
        else
            experts_down_strip_kernel<TRK_DT_F16><<<g, DOWN_WAVES * WAVE, 0, st>>>(a);
        const uint64_t rows = (uint64_t)step * a.slots;
        a.q += rows * a.ldq, a.sx += rows, a.ids += (uint64_t)step * K_MAX, a.w += (uint64_t)step * K_MAX, a.n_sel += step;
        a.y = (char*)a.y + step * a.ldy * size;
    }
}

template <typename Tile, bool ONCE = true>
static void launch_down_tile(const I8Down& a, const Plan& P, uint64_t tiles, hipStream_t st) {
    const dim3 g = run_of((a.down.rows + Tile::BN - 1) / Tile::BN * tiles, Tile::T);
    experts_down_tile_kernel<Tile, ONCE><<<g, Tile::T, 0, st>>>(a, P);
}

hipError_t launch_experts_down(const I8Down& a, const uint32_t* plan, hipStream_t st) {
    const uint32_t E = a.down.count;
    if (!plan || !geo::i8_tile_addresses(a.down.ld, a.ldq, (uint64_t)a.m * a.slots)) {
        launch_down_strip(a, st);
        return hipGetLastError();
    }
    const uint32_t rows = geo::plan_rows(a.m, a.slots, E);
    const Plan P = plan_at(const_cast<uint32_t*>(plan), a.m, a.slots);
    const uint64_t tiles = geo::plan_tiles(a.m, a.slots, E, rows);
    const bool narrow = geo::experts_width(a.down.rows, tiles, false) == geo::X_NARROW;
    if (rows == 32)
        narrow ? launch_down_tile<I8Tile<64, 32, 16, 32, 4>>(a, P, tiles, st)
               : launch_down_tile<I8Tile<128, 32, 32, 32, 3>>(a, P, tiles, st);
    else if (rows == 64)
        narrow ? launch_down_tile<I8Tile<64, 64, 32, 32, 4>>(a, P, tiles, st)
               : launch_down_tile<I8Tile<128, 64, 64, 32, 3>>(a, P, tiles, st);
    else if (geo::experts_once(a.m, a.slots, E, 128))
        narrow ? launch_down_tile<I8Tile<64, 128, 32, 64, 3>>(a, P, tiles, st)
               : launch_down_tile<I8Tile<128, 128, 64, 64, 2>>(a, P, tiles, st);
    else
        narrow ? launch_down_tile<I8Tile<64, 128, 32, 64, 3>, false>(a, P, tiles, st)
               : launch_down_tile<I8Tile<128, 128, 64, 64, 2>, false>(a, P, tiles, st);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess ? e : launch_experts_combine(a, st);
}

hipError_t launch_experts_combine(const I8Down& a, hipStream_t st) {
    const uint32_t q = (a.down.rows + 3) / 4, per = q < 256 ? 256 / q : 1;
    const dim3 g = run_of((uint64_t)((q + 255) / 256) * ((a.m + per - 1) / per), 256);
    if (a.dt == TRK_DT_F32)
        experts_combine_kernel<TRK_DT_F32><<<g, 256, 0, st>>>(a);
    else if (a.dt == TRK_DT_BF16)
        experts_combine_kernel<TRK_DT_BF16><<<g, 256, 0, st>>>(a);
    else
        experts_combine_kernel<TRK_DT_F16><<<g, 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace trk
