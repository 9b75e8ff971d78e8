// Tiled products of _Float16 operands.
#include "gemm_launch.h"

namespace vectra_dense {
int launch_gemm_f16(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream) {
  return launch_gemm<_Float16>(p, layout, tile, any, epi, splits, stream);
}
}  // namespace vectra_dense
