// The paged cache as the kernels see it.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "../../include/chord_b200.h"
#include "common.h"

namespace chord {

// ORed into the status word when a kernel meets an index outside a cache or a table.
constexpr int32_t kStatusIndex = 32;

// n / d for n < 2^31, as a multiplication (T. Granlund and P. Montgomery, "Division by invariant integers using
// multiplication", 1994).
struct Divisor {
  uint32_t d = 1, mul = 0, shift = 0;  // mul == 0: division by one
  Divisor() = default;
  explicit Divisor(uint32_t divisor) : d(divisor) {
    if (divisor <= 1) return;
    uint32_t log = 1;
    while ((1ull << log) < divisor) ++log;
    mul = static_cast<uint32_t>((1ull << (31 + log)) / divisor) + 1;
    shift = log - 1;
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return mul == 0 ? n : __umulhi(n, mul) >> shift; }
};

struct Cache {
  uint8_t* k;
  uint8_t* v;
  float* k_scale;  // null: BF16 values; else codes
  float* v_scale;
  int64_t page, head, token;                    // strides in bytes, of k and v alike
  int64_t scale_page, scale_head, scale_token;  // strides in floats
  uint32_t page16, head16, token16;             // strides in units of 16 bytes
  int32_t num_pages, heads;
  Divisor page_size;
};

// Checks a descriptor of the C ABI and turns it into the kernels' form.
inline int make_cache(const chord_b200_kv_cache* c, Cache* out) {
  CHORD_REQUIRE(c != nullptr && c->k != nullptr && c->v != nullptr, "null cache pointer");
  CHORD_REQUIRE((c->k_scale == nullptr) == (c->v_scale == nullptr), "an 8-bit cache has scales of keys and of values");
  CHORD_REQUIRE(c->num_pages > 0 && c->num_pages < (1ll << 31) && c->page_size > 0 && c->page_size < (1ll << 31) &&
                    c->num_pages * c->page_size < (1ll << 31),
                "a cache holds from 1 to 2^31 - 1 tokens, got %lld pages of %lld", static_cast<long long>(c->num_pages),
                static_cast<long long>(c->page_size));
  CHORD_REQUIRE(c->heads > 0 && c->heads <= 65535, "the cache's heads must be in [1, 65535]");
  const int64_t size = c->k_scale == nullptr ? 2 : 1;
  const int64_t unit = 16 / size;
  CHORD_REQUIRE(c->head_dim > 0 && c->head_dim % 16 == 0 && c->head_dim <= 256,
                "head_dim must be a multiple of 16 up to 256, got %lld", static_cast<long long>(c->head_dim));
  CHORD_REQUIRE(c->stride_page >= 0 && c->stride_head >= 0 && c->stride_token >= 0 && c->stride_page % unit == 0 &&
                    c->stride_head % unit == 0 && c->stride_token % unit == 0,
                "the cache's strides must be multiples of 16 bytes");
  CHORD_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15u) == 0,
                "the cache must be 16-byte aligned");
  CHORD_REQUIRE(c->k_scale == nullptr || (c->scale_stride_page >= 0 && c->scale_stride_head >= 0 &&
                                          c->scale_stride_token >= 0),
                "the scales' strides must not be negative");
  constexpr int64_t kMost = 1ll << 32;
  CHORD_REQUIRE(c->stride_page * size / 16 < kMost && c->stride_head * size / 16 < kMost && c->stride_token * size / 16 < kMost &&
                    (c->k_scale == nullptr || (c->scale_stride_page < kMost && c->scale_stride_head < kMost && c->scale_stride_token < kMost)),
                "the cache's strides must be below 2^36 bytes, its scales' below 2^34");
  *out = Cache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale,
               c->stride_page * size, c->stride_head * size, c->stride_token * size,
               c->scale_stride_page, c->scale_stride_head, c->scale_stride_token,
               static_cast<uint32_t>(c->stride_page * size / 16), static_cast<uint32_t>(c->stride_head * size / 16),
               static_cast<uint32_t>(c->stride_token * size / 16),
               static_cast<int32_t>(c->num_pages), static_cast<int32_t>(c->heads),
               Divisor(static_cast<uint32_t>(c->page_size))};
  return kOk;
}

}  // namespace chord
