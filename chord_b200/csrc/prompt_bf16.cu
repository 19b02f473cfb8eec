// Instantiations of prompt.cuh.
#include "prompt_kernels.cuh"

namespace chord {

bool prompt_bf16(int64_t dim, PromptVariant* out) { return prompt_variant_for<false, false>(dim, out); }

}  // namespace chord
