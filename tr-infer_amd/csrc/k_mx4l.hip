// A whole MoE layer on microscaled 4-bit experts for a few tokens (trk_moe_mx4): the router's logits, the choice
// (trk_route_scores' kernel), gate and up with SwiGLU, down with the weighted sum.
//
// The experts' weights bound it: with few tokens each is met by few rows, and the matrix instructions' other columns are free.
// So the activations are not quantised to 4 bits: each value is split into nine 4-bit parts that take a column each,
// x = p0 + p1 + .., with a scale per block of 32 and part.  A block's largest magnitude lies in [2, 4) of its first scale; a part
// rounds to steps of at most 1 there and leaves at most 0.5, which is at most 4 of the next scale, 2^-3 of it.  Nine
// parts leave 2^-25 of the first scale, 2^-26 of the largest magnitude: what 32 bits hold.  (8-bit parts would be fewer, but
// the matrix instructions add 8-bit products with a few bits less: values split into five were off by 2e-5, into nine
// of 4 bits by 1e-7.)
#include "mx4.hpp"
#include "rows.hpp"

namespace trk {

namespace {

constexpr uint32_t MX_PARTS = 9, MX_STEP = 3;  // parts of a value; the next one's scale is 2^-MX_STEP of a part's

// Activation rows in LDS, cut into groups of 128 values: [group][part][64 bytes], and the scales [group][block of 4][16].
struct MxParts {
    static constexpr uint32_t GROUP = MX_PARTS * 64, SCALES = 4 * 16;
    uint8_t *v, *s;
    // a piece of 8 values: four neighbouring lanes have a block's.  piece: its place in the groups
    __device__ __forceinline__ void put(uint32_t piece, const float (&x)[8]) const {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
            top = b > top ? b : top;
        }
        auto more = [&](uint32_t o) { top = o > top ? o : top; };
        more((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xf, 0xf, false));  // lane ^ 1
        more((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xf, 0xf, false));  // lane ^ 2
        const bool poison = top >= 0x7f800000u;  // the block's products are NaN
        const int e = (int)(top >> 23) - 1;
        float r[8];
#pragma unroll
        for (int i = 0; i < 8; i++) r[i] = poison ? 0.0f : x[i];
#pragma unroll
        for (uint32_t p = 0; p < MX_PARTS; p++) {
            const int ep = e - (int)(MX_STEP * p), byte = ep > 0 ? ep : 0;
            const float f = mx_scale((uint32_t)byte);
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[0], r[1], f, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[2], r[3], f, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[4], r[5], f, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, r[6], r[7], f, 3);
            if (p + 1 < MX_PARTS) {  // what is left: exact
                auto less = [&](int i, auto t) { r[i] -= t[0], r[i + 1] -= t[1]; };
                less(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 0));
                less(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 1));
                less(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 2));
                less(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 3));
            }
            *reinterpret_cast<uint32_t*>(v + piece / 16 * GROUP + p * 64 + piece % 16 * 4) = w;
            if (piece % 4 == 0) s[piece / 4 * 16 + p] = poison ? 255 : (uint8_t)byte;
        }
    }
    // c += a lane's block of a weight row times the parts, a column each (columns beyond hold anything)
    __device__ __forceinline__ f32x4 mul(uint32_t group, uint32_t lane, i32x4 a, uint32_t sa, f32x4 c) const {
        const uint32_t g = lane / 16, p = lane % 16 < MX_PARTS ? lane % 16 : 0;
        return mfma_mx4(a, sa, *reinterpret_cast<const i32x4*>(v + group * GROUP + p * 64 + g * 16), s[(group * 4 + g) * 16 + p], c);
    }
};

// This lane's block of a row, and its scale; past the row's end, its first block and 1 (it meets zeros).
struct MxBlock {
    i32x4 q;
    uint32_t s;
};
__device__ __forceinline__ MxBlock mx_block(const Mx4Row& w, uint32_t b, uint32_t nb) {
    const bool in = b < nb;
    const uint64_t bc = in ? b : 0;
    const i32x4 q = *reinterpret_cast<const i32x4*>(w.q + 16 * bc);
    const uint32_t s = w.s[bc];
    return MxBlock{q, in ? s : MX_ONE};
}

__device__ __forceinline__ Mx4Row layer_row(const Mx4Mat& w, uint32_t e, uint32_t r0, uint32_t lane) {
    const uint64_t r = r0 + lane % 16 < w.rows ? r0 + lane % 16 : w.rows - 1;
    return Mx4Row{w.q + e * w.stride + r * w.ld, w.s + e * w.sstride + r * w.lds};
}

// ---- the router's logits, and the shared experts' gate ---------------------------------------------

constexpr uint32_t LG_WAVES = 4;

// A wave per row of the router and token.
template <uint32_t DT>
__global__ __launch_bounds__(LG_WAVES* WAVE) void layer_logits_kernel(Mx4Layer a, uint32_t rows) {
    const uint32_t id = run_id() * LG_WAVES + threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t r = id % rows, t = id / rows;
    if (t >= a.m) return;
    const bool shared = a.router ? r >= a.n_expert : true;
    const float* w = shared ? a.shared_gate : a.router + (uint64_t)r * a.hidden;
    const auto* x = reinterpret_cast<const typename Elem<DT>::T*>(a.x) + t * a.ldx;
    float acc = 0.0f;
    for (uint32_t p = lane; 8ull * p < a.hidden; p += WAVE) {
        const uint32_t c = 8 * p, n = a.hidden - c;
        QuantPiece<DT> xv;
        QuantPiece<TRK_DT_F32> wv;
        xv.load(x + c, n), wv.load(w + c, n);
#pragma unroll
        for (int i = 0; i < 8; i++) acc = __builtin_fmaf(xv.get(i), wv.get(i), acc);
    }
    acc = reduce16_lanes(rows4_sum(acc));
    if (lane) return;
    if (shared)
        a.shlog[t] = acc;
    else
        a.wlogits[(uint64_t)t * a.n_expert + r] = acc;
}

// ---- gate, up, SwiGLU ------------------------------------------------------------------------------

// Slot j of a token: its j-th expert, then the shared ones; none where the router chose fewer.
__device__ __forceinline__ bool layer_slot(const Mx4Layer& a, uint32_t t, uint32_t j, uint32_t& e) {
    const uint32_t k = a.slots - a.n_shared;
    e = j < k ? a.ids[(size_t)t * K_MAX + j] : a.n_expert + j - k;
    return j >= k || j < a.n_sel[t];
}

constexpr uint32_t LU_WAVES = 4, LU_SEG = 2048;  // values of a row in LDS at once: a piece a thread, four groups a wave

// A workgroup takes 16 rows of gate and up and one entry; its waves share K.
template <uint32_t DT>
__global__ __launch_bounds__(LU_WAVES* WAVE) void layer_up_kernel(Mx4Layer a) {
    constexpr uint32_t P = MX_PARTS, G = LU_SEG / 128 / LU_WAVES;
    __shared__ __attribute__((aligned(16))) uint8_t lv[LU_SEG / 128 * MxParts::GROUP], ls[LU_SEG / 128 * MxParts::SCALES];
    __shared__ float part[2][LU_WAVES][P][16];  // [gate, up][wave][part][weight row]
    const uint32_t strips = (a.gate.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, en = id / strips;
    const uint32_t t = en / a.slots, j = en % a.slots;
    uint32_t e;
    if (t >= a.m || !layer_slot(a, t, j, e)) return;  // the whole workgroup
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, nb = a.gate.nb;
    const auto* x = reinterpret_cast<const typename Elem<DT>::T*>(a.x) + t * a.ldx;
    const Mx4Row gr = layer_row(a.gate, e, r0, lane), ur = layer_row(a.up, e, r0, lane);
    const MxParts parts{lv, ls};
    f32x4 g{0.0f, 0.0f, 0.0f, 0.0f}, u = g;
    for (uint32_t b0 = 0; b0 < nb; b0 += LU_SEG / 32) {
        MxBlock gq[G], uq[G];
#pragma unroll
        for (uint32_t i = 0; i < G; i++) {
            const uint32_t b = b0 + (i * LU_WAVES + wv) * 4 + lane / 16;
            gq[i] = mx_block(gr, b, nb), uq[i] = mx_block(ur, b, nb);
        }
        const uint64_t c = 32ull * b0 + 8 * threadIdx.x;
        QuantPiece<DT> xv;
        xv.load(x + (c < a.hidden ? c : 0), c < a.hidden ? (uint32_t)(a.hidden - c) : 0);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = xv.get(i);
        if (b0) __syncthreads();  // the segment before has been read
        parts.put(threadIdx.x, f);
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < G; i++) {
            if (b0 + (i * LU_WAVES + wv) * 4 >= nb) break;  // the wave as a whole
            g = parts.mul(i * LU_WAVES + wv, lane, gq[i].q, gq[i].s, g);
            u = parts.mul(i * LU_WAVES + wv, lane, uq[i].q, uq[i].s, u);
        }
    }
    mx_here(g), mx_here(u);
    if (lane % 16 < P) {
        *reinterpret_cast<f32x4*>(&part[0][wv][lane % 16][lane / 16 * 4]) = g;
        *reinterpret_cast<f32x4*>(&part[1][wv][lane % 16][lane / 16 * 4]) = u;
    }
    __syncthreads();
    const uint32_t r = r0 + threadIdx.x;
    if (threadIdx.x >= 16 || r >= a.gate.rows) return;
    float gs = 0.0f, us = 0.0f;
#pragma unroll
    for (int p = P - 1; p >= 0; p--)  // the smallest first
#pragma unroll
        for (uint32_t i = 0; i < LU_WAVES; i++) gs += part[0][i][p][threadIdx.x], us += part[1][i][p][threadIdx.x];
    a.h[(uint64_t)en * a.gate.rows + r] = swiglu(gs, us);
}

// ---- down, and the sum -----------------------------------------------------------------------------

constexpr uint32_t LD_WAVES = 8, LD_SEG = 512;  // values of a slot's row in a wave's LDS at once: a piece a lane
constexpr uint32_t LD_SLOTS = 64;               // most slots

// A workgroup takes 16 down rows and one token: a wave per slot, in turn where there are more.  Then a thread per (slot, row)
// weights, and a thread per row adds in slot order.
template <uint32_t DT>
__global__ __launch_bounds__(LD_WAVES* WAVE) void layer_down_kernel(Mx4Layer a) {
    constexpr uint32_t P = MX_PARTS, G = LD_SEG / 128;
    __shared__ __attribute__((aligned(16))) uint8_t lv[LD_WAVES][G * MxParts::GROUP], ls[LD_WAVES][G * MxParts::SCALES];
    __shared__ float part[LD_SLOTS][P][16];
    const uint32_t strips = (a.down.rows + 15) / 16, id = run_id(), r0 = id % strips * 16, t = id / strips;
    if (t >= a.m) return;  // the whole workgroup
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, nb = a.down.nb, F = a.gate.rows;
    const MxParts parts{lv[wv], ls[wv]};
    for (uint32_t j = wv; j < a.slots; j += LD_WAVES) {
        uint32_t e;
        if (!layer_slot(a, t, j, e)) continue;
        const Mx4Row wr = layer_row(a.down, e, r0, lane);
        const float* h = a.h + ((uint64_t)t * a.slots + j) * F;
        f32x4 acc{0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t b0 = 0; b0 < nb; b0 += LD_SEG / 32) {
            MxBlock wq[G];
#pragma unroll
            for (uint32_t i = 0; i < G; i++) wq[i] = mx_block(wr, b0 + i * 4 + lane / 16, nb);
            const uint64_t c = 32ull * b0 + 8 * lane;
            QuantPiece<TRK_DT_F32> hv;
            hv.load(h + (c < F ? c : 0), c < F ? (uint32_t)(F - c) : 0);
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; i++) f[i] = hv.get(i);
            wave_sync();  // the segment before has been read
            parts.put(lane, f);
            wave_sync();
#pragma unroll
            for (uint32_t i = 0; i < G; i++) {
                if (b0 + i * 4 >= nb) break;
                acc = parts.mul(i, lane, wq[i].q, wq[i].s, acc);
            }
        }
        mx_here(acc);
        if (lane % 16 < P) *reinterpret_cast<f32x4*>(&part[j][lane % 16][lane / 16 * 4]) = acc;
    }
    __syncthreads();
    const uint32_t ri = threadIdx.x % 16, r = r0 + ri, k = a.slots - a.n_shared;
    for (uint32_t j = threadIdx.x / 16; j < a.slots; j += LD_WAVES * WAVE / 16) {
        uint32_t e;
        float v = 0.0f;
        if (layer_slot(a, t, j, e)) {
            const float w = j < k ? a.w[(size_t)t * K_MAX + j] : a.shared_gate ? sigmoid512(a.shlog[t]) : 1.0f;
#pragma unroll
            for (int p = P - 1; p >= 0; p--) v += part[j][p][ri];
            v *= w;
        }
        part[j][0][ri] = v;  // its own
    }
    __syncthreads();
    if (threadIdx.x >= 16 || r >= a.down.rows) return;
    float v = 0.0f;
#pragma unroll 8
    for (uint32_t j = 0; j < a.slots; j++) v += part[j][0][ri];
    typedef Elem<DT> O;
    reinterpret_cast<typename O::T*>(a.y)[t * a.ldy + r] = O::put(v);
}

dim3 run_of(uint64_t wgs, uint32_t threads) {
    const geo::Grid2 g = geo::grid_run(wgs, threads);
    return dim3(g.x, g.y);
}

template <uint32_t DT>
void launch_before(const Mx4Layer& a, hipStream_t st) {
    const uint32_t rows = (a.router ? a.n_expert : 0) + (a.shared_gate ? 1 : 0);
    if (rows) layer_logits_kernel<DT><<<run_of(((uint64_t)rows * a.m + LG_WAVES - 1) / LG_WAVES, LG_WAVES * WAVE), LG_WAVES * WAVE, 0, st>>>(a, rows);
}
template <uint32_t DT>
void launch_up(const Mx4Layer& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.gate.rows + 15) / 16) * a.m * a.slots;
    layer_up_kernel<DT><<<run_of(wgs, LU_WAVES * WAVE), LU_WAVES * WAVE, 0, st>>>(a);
}
template <uint32_t DT>
void launch_down(const Mx4Layer& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.down.rows + 15) / 16) * a.m;
    layer_down_kernel<DT><<<run_of(wgs, LD_WAVES * WAVE), LD_WAVES * WAVE, 0, st>>>(a);
}

}  // namespace

hipError_t launch_moe_mx4(const Mx4Layer& a, const float* bias, const ScorePolicy& p, hipStream_t st) {
    a.xdt == TRK_DT_F32    ? launch_before<TRK_DT_F32>(a, st)
    : a.xdt == TRK_DT_BF16 ? launch_before<TRK_DT_BF16>(a, st)
                           : launch_before<TRK_DT_F16>(a, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if ((e = launch_route_scores(a.logits, bias, a.m, a.n_expert, p, a.ids, a.w, a.n_sel, st)) != hipSuccess) return e;
    a.xdt == TRK_DT_F32    ? launch_up<TRK_DT_F32>(a, st)
    : a.xdt == TRK_DT_BF16 ? launch_up<TRK_DT_BF16>(a, st)
                           : launch_up<TRK_DT_F16>(a, st);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    a.ydt == TRK_DT_F32    ? launch_down<TRK_DT_F32>(a, st)
    : a.ydt == TRK_DT_BF16 ? launch_down<TRK_DT_BF16>(a, st)
                           : launch_down<TRK_DT_F16>(a, st);
    return hipGetLastError();
}

}  // namespace trk
