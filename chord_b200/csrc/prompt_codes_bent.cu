// Instantiations of prompt.cuh.
#include "prompt_kernels.cuh"

namespace chord {

bool prompt_codes_bent(int64_t dim, PromptVariant* out) { return prompt_variant_for<true, true>(dim, out); }

}  // namespace chord
