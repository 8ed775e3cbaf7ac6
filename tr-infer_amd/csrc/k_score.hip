// Routing by scores (trk_route_scores): sigmoid or softmax scores, a bias that moves the choice but not the
// weights, groups, top-k, renormalised weights.  One wave per token.
#include "common.hpp"

namespace trk {

namespace {

constexpr uint32_t SC_WAVES = 4;  // tokens per workgroup

// the larger key, the lower index among equal ones; an index of ~0 is no candidate
__device__ __forceinline__ bool better(double ka, uint32_t ia, double kb, uint32_t ib) {
    return ka > kb || (ka == kb && ia < ib);
}

__device__ __forceinline__ void wave_best(double& k, uint32_t& i) {
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        const double ko = __shfl_xor(k, d);
        const uint32_t io = __shfl_xor(i, d);
        if (better(ko, io, k, i)) k = ko, i = io;
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Every key in 64 bits, the best ones by k rounds over the wave.  `key`: E doubles of LDS.
__device__ void score_row(const float* __restrict__ lg, const float* __restrict__ bias, uint32_t E, const ScorePolicy& p,
                          uint32_t lane, double* key, uint32_t* __restrict__ ids, float* __restrict__ w,
                          uint32_t* __restrict__ n_sel) {
    const double NONE = -__builtin_inf();
    const uint32_t gs = E / p.n_group;
    double mx = NONE, denom = 1.0;
    if (p.score == TRK_SCORE_SOFTMAX) {
        for (uint32_t i = lane; i < E; i += WAVE) mx = ::fmax(mx, (double)lg[i]);  // NaN loses
#pragma unroll
        for (int d = 32; d; d >>= 1) mx = ::fmax(mx, __shfl_xor(mx, d));
        double s = 0.0;
        for (uint32_t i = lane; i < E; i += WAVE)
            if (lg[i] > -__builtin_inff()) s += ::exp((double)lg[i] - mx);
        denom = wave_sum(s);
    }
    auto score = [&](float l) {
        return p.score == TRK_SCORE_SOFTMAX ? ::exp((double)l - mx) / denom : 1.0 / (1.0 + ::exp(-(double)l));
    };
    // what a group's best two are summed from: without a bias the keys are logits
    const bool by_score = !bias && p.n_group > 1 && p.group_top == 2;
    for (uint32_t i = lane; i < E; i += WAVE) {
        const float l = lg[i];
        double k = bias || by_score ? score(l) + (bias ? (double)bias[i] : 0.0) : (double)l;
        key[i] = l > -__builtin_inff() && k > NONE ? k : NONE;  // NaN compares false
    }
    wave_sync();
    uint32_t kept = p.n_group == 1 ? 1u : 0u;  // bit g: group g may be chosen from
    if (p.n_group > 1) {
        double worth = NONE;
        if (lane < p.n_group) {
            double a = NONE, b = NONE;
            for (uint32_t i = 0; i < gs; i++) {
                const double k = key[lane * gs + i];
                if (k > a)
                    b = a, a = k;
                else if (k > b)
                    b = k;
            }
            worth = p.group_top == 2 && b > NONE ? a + b : a;
        }
        for (uint32_t r = 0; r < p.topk_group; r++) {
            double bw = worth;
            uint32_t bi = lane < p.n_group && worth > NONE ? lane : 0xffffffffu;
            wave_best(bw, bi);
            if (bi == 0xffffffffu) break;
            kept |= 1u << bi;
            if (lane == bi) worth = NONE;
        }
        if (by_score) {  // the choice itself goes by the logits
            wave_sync();
            for (uint32_t i = lane; i < E; i += WAVE) key[i] = lg[i] > -__builtin_inff() ? (double)lg[i] : NONE;
            wave_sync();
        }
    }
    uint32_t n = 0, mine = 0xffffffffu;
    for (; n < p.k; n++) {
        double bk = NONE;
        uint32_t bi = 0xffffffffu;
        for (uint32_t i = lane; i < E; i += WAVE)
            if ((kept >> (i / gs) & 1u) && key[i] > NONE && better(key[i], i, bk, bi)) bk = key[i], bi = i;
        wave_best(bk, bi);
        if (bi == 0xffffffffu) break;
        if (bi % WAVE == lane) key[bi] = NONE;
        if (lane == n) mine = bi;
    }
    double s = lane < n ? score(lg[mine]) : 0.0;
    if (p.renorm) {
        const double sum = wave_sum(s);
        s = sum > 0.0 ? s / sum : sum;  // every score underflowed: zeros; NaN stays
    }
    if (lane < p.k) {
        ids[lane] = mine;
        w[lane] = lane < n ? (float)(s * (double)p.factor) : 0.0f;
    }
    if (lane == 0) *n_sel = n;
}

__global__ __launch_bounds__(SC_WAVES * WAVE) void route_scores_kernel(const float* __restrict__ logits,
                                                                       const float* __restrict__ bias, uint32_t m,
                                                                       uint32_t E, ScorePolicy p,
                                                                       uint32_t* __restrict__ ids, float* __restrict__ w,
                                                                       uint32_t* __restrict__ n_sel) {
    extern __shared__ double keys[];  // [SC_WAVES][E]
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t row = run_id() * SC_WAVES + wv;
    if (row >= m) return;
    score_row(logits + (size_t)row * E, bias, E, p, lane, keys + (size_t)wv * E, ids + (size_t)row * K_MAX,
              w + (size_t)row * K_MAX, n_sel + row);
}

}  // namespace

hipError_t launch_route_scores(const float* logits, const float* bias, uint32_t m, uint32_t E, const ScorePolicy& p,
                               uint32_t* ids, float* w, uint32_t* n_sel, hipStream_t st) {
    const geo::Grid2 g = geo::grid_run(((uint64_t)m + SC_WAVES - 1) / SC_WAVES, SC_WAVES * WAVE);
    route_scores_kernel<<<dim3(g.x, g.y), SC_WAVES * WAVE, (size_t)SC_WAVES * E * sizeof(double), st>>>(
            logits, bias, m, E, p, ids, w, n_sel);
    return hipGetLastError();
}

}  // namespace trk
