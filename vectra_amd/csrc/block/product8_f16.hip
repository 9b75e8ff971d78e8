// Products in 8 bits with _Float16 results.
#include "product8_impl.h"

namespace vectra_block {
int launch_product8_f16(const Product8Params& p, int tile, int epilogue, int parts, hipStream_t stream) {
  return launch_product8<_Float16>(p, tile, epilogue, parts, stream);
}
int launch_few8_f16(const Product8Params& p, bool gated, hipStream_t stream) { return launch_few8<_Float16>(p, gated, stream); }
}  // namespace vectra_block
