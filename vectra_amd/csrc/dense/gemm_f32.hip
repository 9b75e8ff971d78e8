// Tiled products of float operands.
#include "gemm_launch.h"

namespace vectra_dense {
int launch_gemm_f32(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream) {
  return launch_gemm<float>(p, layout, tile, any, epi, splits, stream);
}
}  // namespace vectra_dense
