// Tiled products of __bf16 operands.
#include "gemm_launch.h"

namespace vectra_dense {
int launch_gemm_bf16(const GemmParams& p, int layout, int tile, bool any, int epi, int splits, hipStream_t stream) {
  return launch_gemm<__bf16>(p, layout, tile, any, epi, splits, stream);
}
}  // namespace vectra_dense
