// Norms of a __bf16 branch on a float stream.
#include "norm_impl.h"

namespace vectra_block {
int launch_norm_bf16_f32(const NormParams& p, int cus, hipStream_t stream) { return launch_norm<__bf16, float>(p, cus, stream); }
int launch_norm_grad_bf16_f32(const NormGradParams& p, int workgroups, hipStream_t stream) {
  return launch_norm_grad<__bf16, float>(p, workgroups, stream);
}
}  // namespace vectra_block
