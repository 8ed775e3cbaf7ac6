// The dense 4-bit product's largest tiles, built with the matrix instructions' sums in accumulator registers.
#include "mx4gemm.hpp"

namespace trk {

void launch_gemm_mx4_wide(const Mx4Gemm& a, hipStream_t st) { launch_mx4_tile<Mx4Tile<256, 256, 128, 128, 2, 8, true>>(a, st); }

}  // namespace trk
