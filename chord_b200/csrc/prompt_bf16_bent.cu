// Instantiations of prompt.cuh.
#include "prompt_kernels.cuh"

namespace chord {

bool prompt_bf16_bent(int64_t dim, PromptVariant* out) { return prompt_variant_for<false, true>(dim, out); }

}  // namespace chord
