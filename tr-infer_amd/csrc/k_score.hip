// Routing by scores (trk_route_scores): one wave per token.
#include "score.hpp"

namespace trk {

namespace {

constexpr uint32_t SC_WAVES = 4;  // tokens per workgroup

// 1 token x 256 (8 groups) 4.0 us and 2048 x 512 (softmax) 4.7: the chain of a row; 16384 x 256 (8 groups) 17.4 us, 1 TB/s:
// some 540 vector instructions a row.  The weights' 64 bits are 1.5 us of those; every key in 64 bits took 62.
template <int NJ, bool SOFT, bool BIAS, bool GROUPED>
__global__ __launch_bounds__(SC_WAVES * WAVE) void route_scores_kernel(const float* __restrict__ logits,
                                                                       const float* __restrict__ bias, uint32_t m,
                                                                       uint32_t E, ScorePolicy p,
                                                                       uint32_t* __restrict__ ids, float* __restrict__ w,
                                                                       uint32_t* __restrict__ n_sel) {
    extern __shared__ double keys[];  // [SC_WAVES][E]
    __shared__ uint2 cand[SC_WAVES][SC_CAND];
    const uint32_t wv = threadIdx.x / WAVE, lane = threadIdx.x % WAVE;
    const uint32_t row = run_id() * SC_WAVES + wv;
    if (row >= m) return;
    const float* lg = logits + (size_t)row * E;
    if (!score_row32<NJ, SOFT, BIAS, GROUPED>(lg, bias, E, p, lane, cand[wv], ids + (size_t)row * K_MAX,
                                              w + (size_t)row * K_MAX, n_sel + row))
        score_row(lg, bias, E, p, lane, keys + (size_t)wv * E, ids + (size_t)row * K_MAX, w + (size_t)row * K_MAX,
                  n_sel + row);
}

template <int NJ>
void launch_scores(dim3 grid, size_t lds, hipStream_t st, const float* logits, const float* bias, uint32_t m, uint32_t E,
                   const ScorePolicy& p, uint32_t* ids, float* w, uint32_t* n_sel) {
#define GO(S, B, G) route_scores_kernel<NJ, S, B, G><<<grid, SC_WAVES * WAVE, lds, st>>>(logits, bias, m, E, p, ids, w, n_sel)
    const bool b = bias, g = p.n_group > 1;
    if (p.score == TRK_SCORE_SOFTMAX)
        b ? (g ? GO(true, true, true) : GO(true, true, false)) : (g ? GO(true, false, true) : GO(true, false, false));
    else
        b ? (g ? GO(false, true, true) : GO(false, true, false)) : (g ? GO(false, false, true) : GO(false, false, false));
#undef GO
}

}  // namespace

hipError_t launch_route_scores(const float* logits, const float* bias, uint32_t m, uint32_t E, const ScorePolicy& p,
                               uint32_t* ids, float* w, uint32_t* n_sel, hipStream_t st) {
    const geo::Grid2 g = geo::grid_run(((uint64_t)m + SC_WAVES - 1) / SC_WAVES, SC_WAVES * WAVE);
    const size_t lds = (size_t)SC_WAVES * E * sizeof(double);
    ScorePolicy q = p;
    const uint32_t nj = score_lanes(q, E);
    const dim3 grid(g.x, g.y);
#define GO(N) launch_scores<N>(grid, lds, st, logits, bias, m, E, q, ids, w, n_sel)
    if (nj <= 2)
        GO(2);
    else if (nj <= 4)
        GO(4);
    else if (nj <= 8)
        GO(8);
    else if (nj <= 16)
        GO(16);
    else
        GO(32);
#undef GO
    return hipGetLastError();
}

}  // namespace trk
