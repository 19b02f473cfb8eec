// The attention of one token per sequence, as other translation units call it.
#pragma once

#include <stdint.h>

#include "../../include/chord_b200.h"

namespace chord {

// Whether what the kernels make of a cap fits FP32.
inline bool cap_fits(const chord_b200_scores& s) {
  return s.cap == 0.0 || (s.cap >= 1e-30 && s.cap <= 1e30 && s.scale <= 1e36 * s.cap && -s.scale <= 1e36 * s.cap);
}

// chord_b200_paged_attention with results in BF16 (out) or FP32 (wide_out).  shaped: by the kernels that cap scores, lean
// on distance and can leave results in FP32; the others are called with neither.
int paged_attention(const void* q, int64_t q_batch, int64_t q_head, const chord_b200_kv_cache* cache, const int32_t* tables,
                    int64_t table_stride, int64_t max_pages, const int32_t* lengths, void* out, float* wide_out, float* lse,
                    int32_t* locks, int64_t num_locks, void* workspace, int64_t workspace_bytes, int32_t* status, int64_t batch,
                    int64_t heads, const chord_b200_scores& scores, bool shaped, void* stream);

}  // namespace chord
