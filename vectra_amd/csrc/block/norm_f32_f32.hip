// Norms of a float branch on a float stream.
#include "norm_impl.h"

namespace vectra_block {
int launch_norm_f32_f32(const NormParams& p, int cus, hipStream_t stream) { return launch_norm<float, float>(p, cus, stream); }
int launch_norm_grad_f32_f32(const NormGradParams& p, int workgroups, hipStream_t stream) {
  return launch_norm_grad<float, float>(p, workgroups, stream);
}
}  // namespace vectra_block
