// A whole MoE layer on microscaled 4-bit experts for a few tokens (trk_moe_mx4), in three launches: the router's logits and
// the tokens' parts (below); the choice, gate and up with SwiGLU and the parts of h; down with the weighted sum.
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
#include "score.hpp"

namespace trk {

namespace {

// ---- rows in parts -----------------------------------------------------------------------------------

// A row in parts is units of sixteen blocks (512 values): four times nine times 64 bytes of 4-bit values, then the scales [lane
// group][16 parts][4], so that a lane has its four in a word.  Whole units, zeros past the row's end.
constexpr uint32_t MX_PARTS = 9, MX_STEP = 3;  // parts of a value; the next one's scale is 2^-MX_STEP of a part's
constexpr uint32_t PU_GROUP = MX_PARTS * 64, PU_VALUES = 4 * PU_GROUP, PU_BYTES = PU_VALUES + 256;

__host__ __device__ inline uint32_t mx_units(uint32_t nb) { return (nb + MX_UNIT - 1) / MX_UNIT; }
__host__ __device__ inline uint64_t parts_bytes(uint32_t nb) { return (uint64_t)mx_units(nb) * PU_BYTES; }
// Block b's 16 bytes of part p in its unit, and its scale
__device__ __forceinline__ uint32_t part_at(uint32_t b, uint32_t p) { return b / 4 % 4 * PU_GROUP + p * 64 + b % 4 * 16; }
__device__ __forceinline__ uint32_t part_scale_at(uint32_t b, uint32_t p) { return PU_VALUES + b % 4 * 64 + p * 4 + b / 4 % 4; }

// A block's scales from its largest magnitude's bits: the largest magnitude lies in [2, 4) of the first.  Where that is 2^126 a
// first part that rounds up to 4 of it is 2^128, which 32 bits do not hold: such a block's values are split by their halves,
// with halved scales (what a half among the smallest numbers loses is far below the last part).
struct MxScales {
    bool poison;  // the block's products are NaN
    uint32_t half;
    int e;
    __device__ __forceinline__ explicit MxScales(uint32_t top)
        : poison(top >= 0x7f800000u), half(top >= 0x7f000000u && !poison), e((int)(top >> 23) - 1) {}
    __device__ __forceinline__ uint32_t byte(uint32_t p) const {
        const int ep = e - (int)(MX_STEP * p);
        return ep > 0 ? (uint32_t)ep : 0u;
    }
    // what is split, and part p's scale for it
    __device__ __forceinline__ float start(float x) const { return poison ? 0.0f : x * (half ? 0.5f : 1.0f); }
    __device__ __forceinline__ float scale(uint32_t p) const { return mx_scale(byte(p) - half); }
};

// This lane's part of a unit (parts beyond the last: the first, whose sums nobody reads).
struct MxPart {
    i32x4 q[4];
    uint32_t s;
    __device__ __forceinline__ void load(const uint8_t* row, uint32_t unit, uint32_t lane) {
        const uint32_t g = lane / 16, p = lane % 16 < MX_PARTS ? lane % 16 : 0;
        const uint8_t* b = row + (uint64_t)unit * PU_BYTES;
        s = *reinterpret_cast<const uint32_t*>(b + PU_VALUES + g * 64 + p * 4);
#pragma unroll
        for (int u = 0; u < 4; u++) q[u] = *reinterpret_cast<const i32x4*>(b + u * PU_GROUP + p * 64 + g * 16);
    }
};
// c += a lane's block of a weight row times instruction U of a unit's parts
template <int U>
__device__ __forceinline__ f32x4 mfma_part(i32x4 a, uint32_t sa, const MxPart& x, f32x4 c) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(mx_operand(a), mx_operand(x.q[U]), c, MX_FP4, MX_FP4, 0, (int)sa, U, (int)x.s);
}
// A unit of NM weight rows times a row's parts; `whole`: the rows have all sixteen blocks.
template <uint32_t NM>
__device__ __forceinline__ void part_unit(const Mx4Row (&w)[NM], const uint8_t* x, uint32_t unit, uint32_t nb, uint32_t lane,
                                          f32x4 (&acc)[NM]) {
    const uint32_t g = lane / 16;
    MxPart xu;
    xu.load(x, unit, lane);
    if ((unit + 1) * MX_UNIT <= nb) {
        Mx4Unit wu[NM];
#pragma unroll
        for (uint32_t i = 0; i < NM; i++) wu[i].load(w[i], unit, g);
        __builtin_amdgcn_sched_barrier(0);  // else some wait for others' registers
        auto mul = [&](auto U) {
            constexpr int u = decltype(U)::value;
#pragma unroll
            for (uint32_t i = 0; i < NM; i++) acc[i] = mfma_part<u>(wu[i].q[u], wu[i].scale(u, g), xu, acc[i]);
        };
        mul(std::integral_constant<int, 0>{}), mul(std::integral_constant<int, 1>{});
        mul(std::integral_constant<int, 2>{}), mul(std::integral_constant<int, 3>{});
    } else {
        const uint32_t q0 = unit * (MX_UNIT / 4);
        Mx4Block wl[NM][4];
#pragma unroll
        for (uint32_t u = 0; u < 4; u++)
            if (4 * (q0 + u) < nb)  // the wave as a whole
#pragma unroll
                for (uint32_t i = 0; i < NM; i++) wl[i][u].load(w[i], q0 + u, g, nb);
        auto mul = [&](auto U) {
            constexpr int u = decltype(U)::value;
            if (4 * (q0 + u) >= nb) return;
#pragma unroll
            for (uint32_t i = 0; i < NM; i++) acc[i] = mfma_part<u>(wl[i][u].q, wl[i][u].s, xu, acc[i]);
        };
        mul(std::integral_constant<int, 0>{}), mul(std::integral_constant<int, 1>{});
        mul(std::integral_constant<int, 2>{}), mul(std::integral_constant<int, 3>{});
    }
}

__device__ __forceinline__ Mx4Row layer_row(const Mx4Mat& w, uint32_t e, uint32_t r0, uint32_t lane) {
    const uint64_t r = r0 + lane % 16 < w.rows ? r0 + lane % 16 : w.rows - 1;
    return Mx4Row{w.q + e * w.stride + r * w.ld, w.s + e * w.sstride + r * w.lds};
}

// ---- the router's logits, the shared experts' gate, the tokens' parts ---------------------------------

constexpr uint32_t LG_WAVES = 4;

// A piece of 8 values into its parts: four neighbouring lanes have a block's.
__device__ __forceinline__ void put_parts(uint8_t* row, uint32_t piece, const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const uint32_t b = __float_as_uint(x[i]) & 0x7fffffffu;
        top = b > top ? b : top;
    }
    auto more = [&](uint32_t o) { top = o > top ? o : top; };
    more((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0xB1, 0xf, 0xf, false));  // lane ^ 1
    more((uint32_t)__builtin_amdgcn_mov_dpp((int)top, 0x4E, 0xf, 0xf, false));  // lane ^ 2
    const MxScales sc(top);
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; i++) r[i] = sc.start(x[i]);
    uint8_t* b = row + (uint64_t)(piece / 64) * PU_BYTES;
#pragma unroll
    for (uint32_t p = 0; p < MX_PARTS; p++) {
        const float f = sc.scale(p);
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
        *reinterpret_cast<uint32_t*>(b + part_at(piece / 4, p) + piece % 4 * 4) = w;
        if (piece % 4 == 0) b[part_scale_at(piece / 4, p)] = sc.poison ? 255 : (uint8_t)sc.byte(p);
    }
}

// A wave per row of the router and token, then (workgroups from `logits` on) a thread per piece of a token's row: the two need
// only x, and share a launch.  512 + 1 rows of 2048, 1 token 4.6 us, 8 tokens of 256 + 0 4.8: the trip to memory and the wave's sum.
template <uint32_t DT>
__global__ __launch_bounds__(LG_WAVES* WAVE) void layer_logits_kernel(Mx4Layer a, uint32_t rows, uint32_t logits) {
    const uint32_t lane = threadIdx.x % WAVE;
    if (blockIdx.x >= logits) {
        const uint32_t P = mx_units(a.gate.nb) * 64, per = (P + LG_WAVES * WAVE - 1) / (LG_WAVES * WAVE);  // pieces, workgroups of a row
        const uint32_t id = blockIdx.x - logits, t = id / per, p = id % per * (LG_WAVES * WAVE) + threadIdx.x;
        if (p >= P) return;  // four lanes of a block together
        const uint64_t c = 8ull * p;
        QuantPiece<DT> xv;
        xv.load(reinterpret_cast<const typename Elem<DT>::T*>(a.x) + t * a.ldx + (c < a.hidden ? c : 0),
                c < a.hidden ? (uint32_t)(a.hidden - c) : 0);
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = xv.get(i);
        put_parts(a.xparts + t * parts_bytes(a.gate.nb), p, f);
        return;
    }
    const uint32_t id = blockIdx.x * LG_WAVES + threadIdx.x / WAVE, r = id % rows, t = id / rows;
    if (t >= a.m) return;
    const bool shared = a.router ? r >= a.n_expert : true;
    const float* w = shared ? a.shared_gate : a.router + (uint64_t)r * a.hidden;
    const auto* x = reinterpret_cast<const typename Elem<DT>::T*>(a.x) + t * a.ldx;
    float acc = 0.0f;
#pragma unroll 4
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

// ---- the choice, gate, up, SwiGLU --------------------------------------------------------------------

constexpr uint32_t LU_WAVES = 4;

// Slot j of a token: its j-th expert, then the shared ones; none where the router chose fewer.
__device__ __forceinline__ bool layer_slot(const Mx4Layer& a, uint32_t t, uint32_t j, uint32_t& e) {
    const uint32_t k = a.slots - a.n_shared;
    e = j < k ? a.ids[t * K_MAX + j] : a.n_expert + j - k;
    return j >= k || j < a.n_sel[t];
}

// A wave's choice of its workgroup's token, as route_scores_kernel makes it; the workgroup of a token's first rows and entry
// leaves it for the next launch.
template <int NJ, bool SOFT, bool BIAS, bool GROUPED>
struct LayerChoice {
    uint2 cand[SC_CAND];
    uint32_t ids[K_MAX], n_sel;
    float w[K_MAX];
    __device__ __forceinline__ bool slot(const Mx4Layer& a, const float* __restrict__ bias, const ScorePolicy& p, uint32_t t, uint32_t j,
                                         bool first, double* keys, uint32_t& e) {
        const uint32_t k = a.slots - a.n_shared, lane = threadIdx.x % WAVE;
        e = a.n_expert + j - k;
        if (j >= k) return true;
        if (threadIdx.x < WAVE) {
            const float* lg = a.logits + (uint64_t)t * a.n_expert;
            if (!score_row32<NJ, SOFT, BIAS, GROUPED>(lg, bias, a.n_expert, p, lane, cand, ids, w, &n_sel))
                score_row(lg, bias, a.n_expert, p, lane, keys, ids, w, &n_sel);
        }
        __syncthreads();
        if (first && j == 0) {
            if (threadIdx.x < k) a.ids[t * K_MAX + threadIdx.x] = ids[threadIdx.x], a.w[t * K_MAX + threadIdx.x] = w[threadIdx.x];
            if (threadIdx.x == 0) a.n_sel[t] = n_sel;
        }
        e = __builtin_amdgcn_readfirstlane(ids[j]);
        return j < n_sel;
    }
};
struct LayerChosen {  // by a launch before
    __device__ __forceinline__ bool slot(const Mx4Layer& a, const float*, const ScorePolicy&, uint32_t t, uint32_t j, bool, double*,
                                         uint32_t& e) {
        return layer_slot(a, t, j, e);
    }
};

// A workgroup takes 32 rows (a block of h) of gate and up and one entry; its waves share K, a unit of all rows at once each.  With the
// choice inside (some 3 us of it, which every workgroup makes for itself and no launch waits for) 1 token of 10 in 512 and a shared one
// (H = 2048, F = 512) 9.4 us; chosen before, 8 tokens of 8 in 256 and one (F = 768) 22.2, 5.4 TB/s counting each entry's weights.
// (Eight waves, four for each half of the rows, hold fewer registers and are slower: that layer 57 us against 53.)
template <typename Choice>
__global__ __launch_bounds__(LU_WAVES* WAVE) void layer_up_kernel(Mx4Layer a, const float* __restrict__ bias, ScorePolicy p) {
    extern __shared__ double keys[];  // [n_expert]
    __shared__ Choice choice;
    __shared__ float part[2][LU_WAVES][MX_PARTS][32];  // [gate, up][wave][part][weight row]
    const uint32_t strips = (a.gate.rows + 31) / 32, id = run_id(), r0 = id % strips * 32, en = id / strips;
    const uint32_t t = en / a.slots, j = en % a.slots;
    if (t >= a.m) return;  // the whole workgroup, here and below
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, nb = a.gate.nb;
    uint32_t e;
    if (!choice.slot(a, bias, p, t, j, r0 == 0, keys, e)) return;
    const uint8_t* x = a.xparts + t * parts_bytes(nb);
    const Mx4Row w[4] = {layer_row(a.gate, e, r0, lane), layer_row(a.gate, e, r0 + 16, lane), layer_row(a.up, e, r0, lane),
                         layer_row(a.up, e, r0 + 16, lane)};
    f32x4 acc[4];
#pragma unroll
    for (int i = 0; i < 4; i++) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t n = wv; n < mx_units(nb); n += LU_WAVES) part_unit<4>(w, x, n, nb, lane, acc);
#pragma unroll
    for (int i = 0; i < 4; i++) mx_here(acc[i]);
    if (lane % 16 < MX_PARTS)
#pragma unroll
        for (int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(&part[i / 2][wv][lane % 16][i % 2 * 16 + lane / 16 * 4]) = acc[i];
    __syncthreads();
    if (wv) return;
    float s = 0.0f;  // lanes 0 .. 31: gate's rows, 32 .. 63: up's
#pragma unroll
    for (int q = MX_PARTS - 1; q >= 0; q--)  // the smallest first
#pragma unroll
        for (uint32_t i = 0; i < LU_WAVES; i++) s += part[lane / 32][i][q][lane % 32];
    const float u = __shfl_xor(s, 32);
    // h's block and its parts, a value a lane (the upper half holds what the lower does)
    const float gv = lane < 32 ? s : u, uv = lane < 32 ? u : s;
    float h = swiglu(gv, uv);
    const uint32_t b = r0 / 32, nf = (a.gate.rows + 31) / 32;
    if (r0 + lane % 32 >= a.gate.rows) h = 0.0f;
    const MxScales sc(row32_allreduce(__float_as_uint(h) & 0x7fffffffu, [](uint32_t c, uint32_t d) { return c > d ? c : d; }));
    float r = sc.start(h);
    uint8_t* hp = a.hparts + en * parts_bytes(nf) + (uint64_t)(b / MX_UNIT) * PU_BYTES;
#pragma unroll
    for (uint32_t q = 0; q < MX_PARTS; q++) {
        const float f = sc.scale(q);
        const uint32_t v = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, r, r, f, 0);
        r -= __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(v, f, 0)[0];
        const uint32_t next = (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, false);  // lane ^ 1
        if (lane < 32 && lane % 2 == 0) hp[part_at(b, q) + lane / 2] = (uint8_t)((v & 15u) | (next & 15u) << 4);
        if (lane == 0) hp[part_scale_at(b, q)] = sc.poison ? 255 : (uint8_t)sc.byte(q);
    }
    // past the row's last block zeros, up to its unit's end
    if (b + 1 == nf)
        for (uint32_t z = nf; z % MX_UNIT; z++) {
            if (lane < MX_PARTS * 4) *reinterpret_cast<uint32_t*>(hp + part_at(z, lane / 4) + lane % 4 * 4) = 0u;
            if (lane < MX_PARTS) hp[part_scale_at(z, lane)] = 0;
        }
}

// ---- down, and the sum -------------------------------------------------------------------------------

// A workgroup takes 16 NR down rows and one token: a wave per slot, in turn where there are more (geo::layer_down_waves).  Then a
// thread per (slot, row) weights, and a thread per row adds in slot order.  Every workgroup reads its token's h, which is as long in
// parts as 12 rows of weights: more rows a workgroup read less of it.  1 token of 11 slots (H = 2048, F = 512) 5.3 us, 8 tokens of 9 (F =
// 768) 14.4, 4.2 TB/s counting each entry's weights.  (The next slot's loads before this one's sum: 8 tokens 46.4 -> 45.7 us a layer, but 4 tokens 31.4 -> 32.8, 1 token 18.8 -> 19.1.)
template <uint32_t DT, uint32_t WAVES, uint32_t NR>
__global__ __launch_bounds__(WAVES* WAVE) void layer_down_kernel(Mx4Layer a) {
    constexpr uint32_t ROWS = 16 * NR;
    extern __shared__ float lds[];
    float(*part)[MX_PARTS][ROWS] = reinterpret_cast<float(*)[MX_PARTS][ROWS]>(lds);  // [slots]
    const uint32_t strips = (a.down.rows + ROWS - 1) / ROWS, id = run_id(), r0 = id % strips * ROWS, t = id / strips;
    if (t >= a.m) return;  // the whole workgroup
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE, nb = a.down.nb;
    for (uint32_t j = wv; j < a.slots; j += WAVES) {
        uint32_t e;
        if (!layer_slot(a, t, j, e)) continue;
        Mx4Row w[NR];
        f32x4 acc[NR];
#pragma unroll
        for (uint32_t i = 0; i < NR; i++) w[i] = layer_row(a.down, e, r0 + 16 * i, lane), acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        const uint8_t* h = a.hparts + ((uint64_t)t * a.slots + j) * parts_bytes(nb);
        for (uint32_t n = 0; n < mx_units(nb); n++) part_unit<NR>(w, h, n, nb, lane, acc);
#pragma unroll
        for (uint32_t i = 0; i < NR; i++) mx_here(acc[i]);
        if (lane % 16 < MX_PARTS)
#pragma unroll
            for (uint32_t i = 0; i < NR; i++) *reinterpret_cast<f32x4*>(&part[j][lane % 16][16 * i + lane / 16 * 4]) = acc[i];
    }
    // A NaN or an infinity in x reaches y by any product.  Where there is none (its logits are then NaN as a rule, and nothing is
    // chosen) the token's scales say it.
    bool poison = false;
    if (!a.n_shared && a.n_sel[t] == 0) {  // the workgroup as a whole
        const uint8_t* x = a.xparts + t * parts_bytes(a.gate.nb);
        for (uint32_t b = threadIdx.x; b < a.gate.nb; b += WAVES * WAVE)
            poison |= x[(uint64_t)(b / MX_UNIT) * PU_BYTES + part_scale_at(b, 0)] == 255;
        poison = __syncthreads_or(poison);
    }
    __syncthreads();
    const uint32_t ri = threadIdx.x % ROWS, r = r0 + ri, k = a.slots - a.n_shared;
    for (uint32_t j = threadIdx.x / ROWS; j < a.slots; j += WAVES * WAVE / ROWS) {
        uint32_t e;
        float v = 0.0f;
        if (layer_slot(a, t, j, e)) {
            const float w = j < k ? a.w[t * K_MAX + j] : a.shared_gate ? sigmoid512(a.shlog[t]) : 1.0f;
#pragma unroll
            for (int p = MX_PARTS - 1; p >= 0; p--) v += part[j][p][ri];
            v *= w;
        }
        part[j][0][ri] = v;  // its own
    }
    __syncthreads();
    if (threadIdx.x >= ROWS || r >= a.down.rows) return;
    float v = 0.0f;
#pragma unroll 8
    for (uint32_t j = 0; j < a.slots; j++) v += part[j][0][ri];
    typedef Elem<DT> O;
    reinterpret_cast<typename O::T*>(a.y)[t * a.ldy + r] = O::put(poison ? __builtin_nanf("") : v);
}

dim3 run_of(uint64_t wgs, uint32_t threads) {
    const geo::Grid2 g = geo::grid_run(wgs, threads);
    return dim3(g.x, g.y);
}

template <uint32_t DT>
void launch_before(const Mx4Layer& a, hipStream_t st) {
    const uint32_t rows = (a.router ? a.n_expert : 0) + (a.shared_gate ? 1 : 0), lg = (rows * a.m + LG_WAVES - 1) / LG_WAVES;
    const uint32_t per = (mx_units(a.gate.nb) * 64 + LG_WAVES * WAVE - 1) / (LG_WAVES * WAVE);
    layer_logits_kernel<DT><<<lg + a.m * per, LG_WAVES * WAVE, 0, st>>>(a, rows ? rows : 1, lg);
}
template <int NJ>
void launch_up(const Mx4Layer& a, const float* bias, const ScorePolicy& p, hipStream_t st) {
    const dim3 grid = run_of((uint64_t)((a.gate.rows + 31) / 32) * a.m * a.slots, LU_WAVES * WAVE);
    const size_t lds = a.n_expert * sizeof(double);
#define GO(S, B, G) layer_up_kernel<LayerChoice<NJ, S, B, G>><<<grid, LU_WAVES * WAVE, lds, st>>>(a, bias, p)
    const bool b = bias, g = p.n_group > 1;
    if (p.score == TRK_SCORE_SOFTMAX)
        b ? (g ? GO(true, true, true) : GO(true, true, false)) : (g ? GO(true, false, true) : GO(true, false, false));
    else
        b ? (g ? GO(false, true, true) : GO(false, true, false)) : (g ? GO(false, false, true) : GO(false, false, false));
#undef GO
}
template <uint32_t DT>
void launch_down(const Mx4Layer& a, hipStream_t st) {
    const uint64_t wgs = (uint64_t)((a.down.rows + 15) / 16) * a.m;
    const size_t lds = a.slots * MX_PARTS * 16 * sizeof(float);  // 64 slots at most: 36 KB
    switch (geo::layer_down_waves(wgs, a.slots)) {
    case 4: layer_down_kernel<DT, 4, 1><<<run_of(wgs, 4 * WAVE), 4 * WAVE, lds, st>>>(a); break;
    case 8: {  // at most 32 slots
        const uint64_t wgs2 = (uint64_t)((a.down.rows + 31) / 32) * a.m;
        layer_down_kernel<DT, 8, 2><<<run_of(wgs2, 8 * WAVE), 8 * WAVE, 2 * lds, st>>>(a);
        break;
    }
    default: layer_down_kernel<DT, 12, 1><<<run_of(wgs, 12 * WAVE), 12 * WAVE, lds, st>>>(a);
    }
}

}  // namespace

uint64_t mx4_parts_bytes(uint32_t nb) { return parts_bytes(nb); }

hipError_t launch_moe_mx4(const Mx4Layer& a, const float* bias, const ScorePolicy& policy, hipStream_t st) {
    a.xdt == TRK_DT_F32    ? launch_before<TRK_DT_F32>(a, st)
    : a.xdt == TRK_DT_BF16 ? launch_before<TRK_DT_BF16>(a, st)
                           : launch_before<TRK_DT_F16>(a, st);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const uint64_t wgs = (uint64_t)((a.gate.rows + 31) / 32) * a.m * a.slots;
    if (geo::layer_routes_apart(wgs)) {
        if ((e = launch_route_scores(a.logits, bias, a.m, a.n_expert, policy, a.ids, a.w, a.n_sel, st)) != hipSuccess) return e;
        layer_up_kernel<LayerChosen><<<run_of(wgs, LU_WAVES * WAVE), LU_WAVES * WAVE, 0, st>>>(a, bias, policy);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        a.ydt == TRK_DT_F32    ? launch_down<TRK_DT_F32>(a, st)
        : a.ydt == TRK_DT_BF16 ? launch_down<TRK_DT_BF16>(a, st)
                               : launch_down<TRK_DT_F16>(a, st);
        return hipGetLastError();
    }
    ScorePolicy p = policy;
    const uint32_t nj = score_lanes(p, a.n_expert);
    if (nj <= 2)
        launch_up<2>(a, bias, p, st);
    else if (nj <= 4)
        launch_up<4>(a, bias, p, st);
    else if (nj <= 8)
        launch_up<8>(a, bias, p, st);
    else if (nj <= 16)
        launch_up<16>(a, bias, p, st);
    else
        launch_up<32>(a, bias, p, st);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    a.ydt == TRK_DT_F32    ? launch_down<TRK_DT_F32>(a, st)
    : a.ydt == TRK_DT_BF16 ? launch_down<TRK_DT_BF16>(a, st)
                           : launch_down<TRK_DT_F16>(a, st);
    return hipGetLastError();
}

}  // namespace trk
