// What the entry points need of each instantiation of prompt.cuh, which are compiled in several files.
#pragma once

#include "prompt_join.cuh"

namespace chord {

struct PromptVariant {
  void (*kernel)(PromptParams);
  void (*join)(PromptParams);
  int smem, threads, tiles, step_tokens, row_regs, other_regs;
  int64_t part_floats;
};

template <int kDim, bool kCodes, bool kBent>
PromptVariant prompt_variant() {
  using L = PromptLayout<kDim, kCodes>;
  return {prompt_attention_kernel<kDim, kCodes, kBent>, prompt_join_kernel<kDim, kCodes>, L::kSmem, L::kThreads, L::kTiles,
          L::kN, L::kRowRegs, L::kOtherRegs, prompt_part_floats<kDim, kCodes>()};
}

template <bool kCodes, bool kBent>
bool prompt_variant_for(int64_t dim, PromptVariant* out) {
  switch (dim) {
    case 64: *out = prompt_variant<64, kCodes, kBent>(); return true;
    case 96: *out = prompt_variant<96, kCodes, kBent>(); return true;
    case 128: *out = prompt_variant<128, kCodes, kBent>(); return true;
    case 192: *out = prompt_variant<192, kCodes, kBent>(); return true;
    case 256: *out = prompt_variant<256, kCodes, kBent>(); return true;
  }
  return false;
}

// prompt_<values><form>.cu
bool prompt_bf16(int64_t dim, PromptVariant* out);
bool prompt_bf16_bent(int64_t dim, PromptVariant* out);
bool prompt_codes(int64_t dim, PromptVariant* out);
bool prompt_codes_bent(int64_t dim, PromptVariant* out);

}  // namespace chord
