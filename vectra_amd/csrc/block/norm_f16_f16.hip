// Norms of a _Float16 branch on a _Float16 stream.
#include "norm_impl.h"

namespace vectra_block {
int launch_norm_f16_f16(const NormParams& p, int cus, hipStream_t stream) { return launch_norm<_Float16, _Float16>(p, cus, stream); }
int launch_norm_grad_f16_f16(const NormGradParams& p, int workgroups, hipStream_t stream) {
  return launch_norm_grad<_Float16, _Float16>(p, workgroups, stream);
}
}  // namespace vectra_block
