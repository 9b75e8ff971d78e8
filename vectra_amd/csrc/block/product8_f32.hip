// Products in 8 bits with float results.
#include "product8_impl.h"

namespace vectra_block {
int launch_product8_f32(const Product8Params& p, int tile, int epilogue, int parts, hipStream_t stream) {
  return launch_product8<float>(p, tile, epilogue, parts, stream);
}
int launch_few8_f32(const Product8Params& p, bool gated, hipStream_t stream) { return launch_few8<float>(p, gated, stream); }
}  // namespace vectra_block
