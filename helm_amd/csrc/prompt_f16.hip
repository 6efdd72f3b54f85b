// float16 instantiations of the prompt kernel (prompt.h).
#include "prompt.h"

namespace helm {
hipError_t launch_prompt_f16(const PromptParams& p, int D, hipStream_t st) {
  return launch_prompt_type<f16_t>(p, D, st);
}
}  // namespace helm
