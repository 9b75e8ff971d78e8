// Products of __bf16 rows with a weight in LDS, one case per kResidentSteps16.
#include "resident_impl.h"

namespace vectra_dense {
int launch_resident_bf16(const ResidentParams& p, int steps, int epi, bool with_dx, int workgroups, hipStream_t stream) {
  switch (steps) {
    case 2: return launch_resident_steps<__bf16, 2>(p, epi, with_dx, workgroups, stream);
    case 4: return launch_resident_steps<__bf16, 4>(p, epi, with_dx, workgroups, stream);
    case 8: return launch_resident_steps<__bf16, 8>(p, epi, with_dx, workgroups, stream);
    default: return VECTRA_DENSE_ERR_LAUNCH;
  }
}
}  // namespace vectra_dense
