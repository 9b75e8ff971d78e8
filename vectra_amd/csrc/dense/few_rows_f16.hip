// Products of a few _Float16 rows.
#include "few_rows_impl.h"

namespace vectra_dense {
int launch_few_rows_f16(const FewRowsParams& p, bool gated, hipStream_t stream) {
  return launch_few_rows<_Float16>(p, gated, stream);
}
}  // namespace vectra_dense
