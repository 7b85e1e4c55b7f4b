// The flash-attention backward (attn_bwd_kernel.cuh) with shaped scores: a soft cap, slopes on the distance, an open prefix.
#include "attn_bwd_kernel.cuh"

RA_BOUNDS_TRANSLATION_UNIT()

namespace ra {
namespace attn {

BwdKernel bwd_kernel_shaped(int D, int shape) {
  static_assert(kShapeCap == 1 && kShapeSlopes == 2 && kShapeOn == 4, "the bits that are told apart here");
  switch (shape & 3) {
    case 0: return D == 128 ? attn_bwd_kernel<128, 4> : attn_bwd_kernel<64, 4>;
    case 1: return D == 128 ? attn_bwd_kernel<128, 5> : attn_bwd_kernel<64, 5>;
    case 2: return D == 128 ? attn_bwd_kernel<128, 6> : attn_bwd_kernel<64, 6>;
    default: return D == 128 ? attn_bwd_kernel<128, 7> : attn_bwd_kernel<64, 7>;
  }
}

}  // namespace attn
}  // namespace ra
