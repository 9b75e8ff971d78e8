// Norms of a __bf16 branch on a __bf16 stream.
#include "norm_impl.h"

namespace vectra_block {
int launch_norm_bf16_bf16(const NormParams& p, int cus, hipStream_t stream) { return launch_norm<__bf16, __bf16>(p, cus, stream); }
int launch_norm_grad_bf16_bf16(const NormGradParams& p, int workgroups, hipStream_t stream) {
  return launch_norm_grad<__bf16, __bf16>(p, workgroups, stream);
}
}  // namespace vectra_block
