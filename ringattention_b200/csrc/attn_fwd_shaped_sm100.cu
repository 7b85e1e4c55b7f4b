// The flash-attention forward (attn_fwd_kernel.cuh) with shaped scores: a soft cap, slopes on the distance, an open prefix.
#include "attn_fwd_kernel.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace {
template <int NQ, int DV, bool HALVES>
int launch_shape(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const ra::attn::FwdParams& p, int shape, long long grid,
                 cudaStream_t s) {
  switch (shape & 3) {
    case 0: return launch_fwd<NQ, 0, DV, false, HALVES, 4>(tq, tk, tv, tq, tk, p, grid, s);
    case 1: return launch_fwd<NQ, 0, DV, false, HALVES, 5>(tq, tk, tv, tq, tk, p, grid, s);
    case 2: return launch_fwd<NQ, 0, DV, false, HALVES, 6>(tq, tk, tv, tq, tk, p, grid, s);
    default: return launch_fwd<NQ, 0, DV, false, HALVES, 7>(tq, tk, tv, tq, tk, p, grid, s);
  }
}
}  // namespace

int ra::attn::launch_fwd_shaped(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const FwdParams& p, int D, bool halves, int shape,
                                long long grid, cudaStream_t s) {
  static_assert(kShapeCap == 1 && kShapeSlopes == 2 && kShapeOn == 4, "the bits that launch_shape tells apart");
  if (D == 128) return halves ? launch_shape<2, 128, true>(tq, tk, tv, p, shape, grid, s) : launch_shape<2, 128, false>(tq, tk, tv, p, shape, grid, s);
  return halves ? launch_shape<1, 64, true>(tq, tk, tv, p, shape, grid, s) : launch_shape<1, 64, false>(tq, tk, tv, p, shape, grid, s);
}
