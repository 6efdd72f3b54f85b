// float16 instantiations of the shared-prefix decode kernels (prefix.h).
#include "prefix.h"

namespace helm {
hipError_t launch_prefix_f16(const PfParams& p, int D, hipStream_t st) {
  return launch_prefix_type<f16_t>(p, D, st);
}
}  // namespace helm
