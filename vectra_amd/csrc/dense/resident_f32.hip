// Products of float rows with a weight in LDS, one case per kResidentSteps32.
#include "resident_impl.h"

namespace vectra_dense {
int launch_resident_f32(const ResidentParams& p, int steps, int epi, bool with_dx, int workgroups, hipStream_t stream) {
  switch (steps) {
    case 2: return launch_resident_steps<float, 2>(p, epi, with_dx, workgroups, stream);
    case 4: return launch_resident_steps<float, 4>(p, epi, with_dx, workgroups, stream);
    case 6: return launch_resident_steps<float, 6>(p, epi, with_dx, workgroups, stream);
    case 9: return launch_resident_steps<float, 9>(p, epi, with_dx, workgroups, stream);
    case 12: return launch_resident_steps<float, 12>(p, epi, with_dx, workgroups, stream);
    case 16: return launch_resident_steps<float, 16>(p, epi, with_dx, workgroups, stream);
    default: return VECTRA_DENSE_ERR_LAUNCH;
  }
}
}  // namespace vectra_dense
