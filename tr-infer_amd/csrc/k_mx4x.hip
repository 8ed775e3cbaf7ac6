// The microscaled 4-bit products of each token with its experts (trk_experts_up_mx4, trk_experts_down_mx4).
#include "mx4.hpp"

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

// A workgroup takes 16 rows of gate and up and one entry; its waves share K.
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
// K; in turn where there are more), then a thread per (slot, row) weights, and a thread per row adds in slot order.
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

}  // namespace

hipError_t launch_experts_up_mx4(const Mx4Up& a, const uint32_t* plan, hipStream_t st) {
    launch_up_strip(a, st);
    return hipGetLastError();
}

hipError_t launch_experts_down_mx4(const Mx4Down& a, const uint32_t* plan, hipStream_t st) {
    launch_down_strip(a, st);
    return hipGetLastError();
}

}  // namespace trk
