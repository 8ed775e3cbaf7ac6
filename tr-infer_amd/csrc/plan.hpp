// The experts' plan as the tile kernels follow it.
#pragma once

#include "i8.hpp"

namespace trk {

constexpr uint32_t PLAN_T = 1024;  // threads of the kernels that make it, and the most experts

// Whether a plan is one for these sizes: its entries are then below m * slots, and its tiles fit the launch.  One made for more
// experts is where each entry may have a tile of its own.  Nothing is read through another; what would be written is NaN.
__device__ __forceinline__ bool plan_fits(const PlanHead& h, uint32_t m, uint32_t slots, uint32_t E) {
    return h.m == m && h.slots == slots && (h.E == E || (h.E > E && h.E <= PLAN_T && m * slots <= E));
}

// A tile's place: entries of one expert (the plan's tile) x a block of weight rows, the blocks of a tile next to one
// another and each expert's tiles in turn on one XCD, whose L2 then holds the entries' rows and the expert's weights.
// E: the stack's experts.  No plan made for it names others; of a plan made for more they are passed over, like ids.
__device__ __forceinline__ bool expert_tile(const Plan& P, const PlanHead& h, uint32_t E, uint32_t blocks, PlanTile& t,
                                            uint32_t& block) {
    uint32_t idx;
    if (!xcd_order_1d(h.n_tiles * blocks, idx, run_id())) return false;
    t = P.tile[idx / blocks], block = idx % blocks;
    return t.expert < E;
}

// NaN into every entry's row of y [m * slots][rows], the workgroups taking them in turn
template <uint32_t DT, typename A>
__device__ __forceinline__ void nan_rows(const A& a, uint32_t count, void* y, uint32_t rows, uint64_t ldy) {
    typedef Elem<DT> O;
    const uint32_t n = a.m * a.slots;
    for (uint64_t i = run_id(); i < n; i += (uint64_t)gridDim.x * gridDim.y) {
        const uint32_t t = (uint32_t)i / a.slots, j = (uint32_t)i % a.slots;
        if (j >= a.n_sel[t] || a.ids[(size_t)t * K_MAX + j] >= count) continue;
        for (uint64_t r = threadIdx.x; r < rows; r += blockDim.x)
            reinterpret_cast<typename O::T*>(y)[i * ldy + r] = O::put(__builtin_nanf(""));
    }
}

}  // namespace trk
