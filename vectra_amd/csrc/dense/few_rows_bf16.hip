// Products of a few __bf16 rows.
#include "few_rows_impl.h"

namespace vectra_dense {
int launch_few_rows_bf16(const FewRowsParams& p, bool gated, hipStream_t stream) {
  return launch_few_rows<__bf16>(p, gated, stream);
}
}  // namespace vectra_dense
