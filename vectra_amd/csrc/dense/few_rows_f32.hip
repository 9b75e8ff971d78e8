// Products of a few float rows.
#include "few_rows_impl.h"

namespace vectra_dense {
int launch_few_rows_f32(const FewRowsParams& p, bool gated, hipStream_t stream) {
  return launch_few_rows<float>(p, gated, stream);
}
}  // namespace vectra_dense
