// Queries, keys and values between the projection and the attention: norms of each head with the
// position rotation, and the paged cache as it is written and read back.
#include <cuda_bf16.h>

#include "../../include/chord_b200.h"
#include "common.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {
namespace {

struct HeadsParams {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_token, q_head, k_token, k_head, v_token, v_head;  // strides in elements
  const __nv_bfloat16 *q_weight, *k_weight;
  const float* cos_sin;
  const int32_t* positions;
  __nv_bfloat16 *q_out, *k_out;  // contiguous
  const int32_t* slots;
  int32_t* status;
  Cache cache;
  int32_t items, q_heads, k_heads, v_heads, dim, rotary, max_positions;
  int32_t q_items, k_items;  // items of a token: its queries', keys' and
  Divisor items_per_token;   // all
  float eps, share;          // share: 1 / dim
  bool interleaved;
};

__device__ __forceinline__ void unpack8(const uint4 v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bf16_lo(w[i]);
    x[2 * i + 1] = bf16_hi(w[i]);
  }
}

__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7]));
}

// The larger magnitude; a NaN where there is one.
__device__ __forceinline__ float max_magnitude(float a, float b) {
  float c;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(fabsf(a)), "f"(fabsf(b)));
  return c;
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Eight codes round(x / scale) + 128 of a row whose largest |x| is `top`, scale = top / 127; halves go to the
// even code.  A half is common (x = top / 2 is 63.5 steps), and x * rate is off by up to 2^-17 there: the first
// sum rounds to steps of 2^-15, which brings it back, the second (1.5 * 2^23 + 128 in all) to whole numbers, the
// code in the low byte.
__device__ __forceinline__ uint2 quantise8(float (&x)[8], float top) {
  if (!(top > 0x1p-100f && top < 0x1p100f)) {  // (the reciprocal's range)
    const float factor = top < 1.0f ? 0x1p100f : 0x1p-64f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= factor;
    top = top > 0.0f ? top * factor : 1.0f;
  }
  const float inverse = __fdividef(1.0f, top);
  float rate = 127.0f * inverse;
  rate = fmaf(fmaf(-top, rate, 127.0f), inverse, rate);  // (as good as correctly rounded)
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    // Two at a time.
    asm("{\n .reg .b64 x, r, c;\n mov.b64 x, {%2, %3};\n mov.b64 r, {%4, %4};\n mov.b64 c, {%5, %5};\n fma.rn.f32x2 x, x, r, c;\n"
        " mov.b64 c, {%6, %6};\n add.rn.f32x2 x, x, c;\n mov.b64 {%0, %1}, x;\n}"
        : "=r"(w[i]), "=r"(w[i + 1])
        : "f"(x[i]), "f"(x[i + 1]), "f"(rate), "f"(384.0f), "f"(12583040.0f - 384.0f));
  }
  return make_uint2(low_bytes(w[0], w[1], w[2], w[3]), low_bytes(w[4], w[5], w[6], w[7]));
}

// kLanes lanes hold a row of up to 8 kLanes elements, 16 bytes each, so a warp works on 32 / kLanes
// rows at a time and on kRows of those sets, whose loads are all in flight at once.  An item is the
// rows of a warp: rows of one token, all queries, keys or values.  What an item's rows have in common is
// worked out once: with x' the element that x turns with, a result is rate * (A x + B x'), where A and B
// hold the norm's weights and the angles, and x' comes from its lane as the bits that were loaded.
// Everything between the load and the store is FP32; the result is rounded once, to BF16 or to the codes.
template <int kLanes, int kRows, bool kRotate, bool kWrite>
__global__ void __launch_bounds__(256, 4)
heads_kernel(const HeadsParams p) {
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, side = lane / kLanes;
  const int32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int32_t token = p.items_per_token.div(item);
  int32_t group = item - token * p.items_per_token.d;
  // Which of the three, and the first of the item's rows.
  const bool is_q = kRotate && group < p.q_items;
  if (!is_q) group -= p.q_items;
  const bool is_v = kWrite && !is_q && group >= p.k_items;
  if (is_v) group -= p.k_items;
  const int32_t rows = is_q ? p.q_heads : p.k_heads;
  const int32_t first = group * (kSide * kRows) + side;
  const bool inside = 8 * chunk < p.dim;
  const __nv_bfloat16* from = (is_q ? p.q + token * p.q_token : is_v ? p.v + token * p.v_token : p.k + token * p.k_token) + 8 * chunk;
  const int64_t stride = is_q ? p.q_head : is_v ? p.v_head : p.k_head;
  from += first * stride;
  ptx::grid_dependency_wait();

  // (the results may take the inputs' place)
  uint4 raw[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int32_t row = first + i * kSide;
    raw[i] = row < rows && inside ? load_once_coherent(from) : make_uint4(0, 0, 0, 0);
    from += kSide * stride;
  }

  float own[8], other[8];  // A, B
  int partner = lane;
  bool lost = false;
  if constexpr (kRotate) {
    if (!is_v) {
      const uint4* const weight = reinterpret_cast<const uint4*>(is_q ? p.q_weight : p.k_weight);
      const int32_t position = __ldg(p.positions + token), half = p.rotary / 2;
      lost = position < 0 || position >= p.max_positions;
      if (lost && p.status != nullptr && lane == 0) atomicOr(p.status, kStatusIndex);
      const bool turned = 8 * chunk < p.rotary, upper = 8 * chunk >= half;
      float w[8];
      unpack8(inside ? __ldg(weight + chunk) : make_uint4(0, 0, 0, 0), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) own[j] = w[j], other[j] = 0.0f;
      if (turned && !lost) {
        const float* const at = p.cos_sin + static_cast<int64_t>(position) * p.rotary + (p.interleaved ? 4 * chunk : 8 * chunk - (upper ? half : 0));
        const float4 c0 = __ldg(reinterpret_cast<const float4*>(at)), s0 = __ldg(reinterpret_cast<const float4*>(at + half));
        if (p.interleaved) {
          const float c[4] = {c0.x, c0.y, c0.z, c0.w}, s[4] = {s0.x, s0.y, s0.z, s0.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            own[2 * j] *= c[j], own[2 * j + 1] *= c[j];
            other[2 * j] = -s[j] * w[2 * j + 1], other[2 * j + 1] = s[j] * w[2 * j];
          }
        } else {
          const float4 c1 = __ldg(reinterpret_cast<const float4*>(at) + 1), s1 = __ldg(reinterpret_cast<const float4*>(at + half) + 1);
          const float c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
          const int away = upper ? -half / 8 : half / 8;
          partner = lane + away;
          unpack8(__ldg(weight + chunk + away), w);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            own[j] *= c[j];
            other[j] = (upper ? s[j] : -s[j]) * w[j];
          }
        }
      }
    }
  }
  int64_t page_offset = -1, scale_offset = 0;
  if constexpr (kWrite) {
    if (!is_q) {
      const int32_t slot = __ldg(p.slots + token);
      const uint32_t page = slot >= 0 ? p.cache.page_size.div(static_cast<uint32_t>(slot)) : 0;
      const uint32_t in_page = static_cast<uint32_t>(slot) - page * p.cache.page_size.d;
      if (slot >= 0 && page < static_cast<uint32_t>(p.cache.num_pages)) {
        page_offset = page * p.cache.page + in_page * p.cache.token;
        scale_offset = page * p.cache.scale_page + in_page * p.cache.scale_token;
      } else if (slot >= 0 && p.status != nullptr && lane == 0) {
        atomicOr(p.status, kStatusIndex);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int32_t row = first + i * kSide;
    if (row - side >= rows) break;  // (the whole warp)
    const bool mine = row < rows && inside;
    float x[8];
    unpack8(raw[i], x);
    if (kRotate && !is_v) {
      float square = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) square = fmaf(x[j], x[j], square);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
      const float rate = rsqrtf(fmaf(square, p.share, p.eps));
      uint4 turn = raw[i];
      if (p.interleaved) {
        turn.x = __byte_perm(turn.x, 0, 0x1032);
        turn.y = __byte_perm(turn.y, 0, 0x1032);
        turn.z = __byte_perm(turn.z, 0, 0x1032);
        turn.w = __byte_perm(turn.w, 0, 0x1032);
      } else {
        turn.x = __shfl_sync(0xffffffffu, turn.x, partner);
        turn.y = __shfl_sync(0xffffffffu, turn.y, partner);
        turn.z = __shfl_sync(0xffffffffu, turn.z, partner);
        turn.w = __shfl_sync(0xffffffffu, turn.w, partner);
      }
      float y[8];
      unpack8(turn, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = lost ? 0.0f : rate * fmaf(x[j], own[j], y[j] * other[j]);
    }
    if (is_q || !kWrite) {
      __nv_bfloat16* const to = is_q ? p.q_out : p.k_out;
      if (mine) *reinterpret_cast<uint4*>(to + (static_cast<int64_t>(token) * rows + row) * p.dim + 8 * chunk) = pack8(x);
    } else if constexpr (kWrite) {
      const bool keep = mine && page_offset >= 0;
      uint8_t* const at = (is_v ? p.cache.v : p.cache.k) + page_offset + row * p.cache.head;
      if (p.cache.k_scale == nullptr) {
        if (keep) *reinterpret_cast<uint4*>(at + 16 * chunk) = kRotate && !is_v ? pack8(x) : raw[i];
      } else {
        float top = max_magnitude(max_magnitude(max_magnitude(x[0], x[1]), max_magnitude(x[2], x[3])),
                                  max_magnitude(max_magnitude(x[4], x[5]), max_magnitude(x[6], x[7])));
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) top = max_magnitude(top, __shfl_xor_sync(0xffffffffu, top, d));
        // A row with an infinity or a NaN gets a scale of NaN, so that it reads back as NaN.
        const bool finite = top < INFINITY;
        if (keep) {
          const float scale = finite ? top * (1.0f / 127.0f) : __uint_as_float(0x7FC00000u);
          *reinterpret_cast<uint2*>(at + 8 * chunk) = finite ? quantise8(x, top) : make_uint2(0x80808080u, 0x80808080u);
          if (chunk == 0) (is_v ? p.cache.v_scale : p.cache.k_scale)[scale_offset + row * p.cache.scale_head] = scale;
        }
      }
    }
  }
}

struct ReadParams {
  Cache cache;
  const int32_t* tables;
  const int32_t* offsets;
  __nv_bfloat16 *k_out, *v_out;  // [total, heads, dim]
  int32_t* status;
  int64_t table_stride;
  int32_t items, batch, max_pages, total, dim;
  Divisor items_per_token;
};

// As heads_kernel: a warp reads rows of one token, its keys' heads and then its values'.
template <int kLanes, int kRows>
__global__ void __launch_bounds__(256, 4)
cache_read_kernel(const ReadParams p) {
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, side = lane / kLanes;
  const int32_t item = blockIdx.x * 8 + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int32_t token = p.items_per_token.div(item);
  const int32_t first = (item - token * static_cast<int32_t>(p.items_per_token.d)) * (kSide * kRows) + side;
  const int32_t rows = 2 * p.cache.heads;
  ptx::grid_dependency_wait();

  // The sequence: the last one that does not begin after the token; 32 at a time, coarse to fine.
  int32_t low = 0, count = p.batch;
  while (count > 1) {
    const int32_t step = (count + 31) / 32;
    const int32_t at = lane * step;
    const bool before = at < count && __ldg(p.offsets + low + at) <= token;
    const uint32_t votes = __ballot_sync(0xffffffffu, before);
    const int32_t last = votes == 0 ? 0 : 31 - __clz(votes);
    low += last * step;
    count = min(step, count - last * step);
  }
  const int32_t begin = __ldg(p.offsets + low);
  int64_t page_offset = -1, scale_offset = 0;
  if (token >= begin && token < __ldg(p.offsets + low + 1)) {
    const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(begin);
    const uint32_t index = p.cache.page_size.div(at), in_page = at - index * p.cache.page_size.d;
    const int32_t page = begin >= 0 && index < static_cast<uint32_t>(p.max_pages) ? __ldg(p.tables + low * p.table_stride + index) : -1;
    if (page >= 0 && page < p.cache.num_pages) {
      page_offset = page * p.cache.page + in_page * p.cache.token;
      scale_offset = page * p.cache.scale_page + in_page * p.cache.scale_token;
    } else if (p.status != nullptr && lane == 0) {
      atomicOr(p.status, kStatusIndex);
    }
  }
  const bool inside = 8 * chunk < p.dim;
  uint4 raw[kRows];
  float scale[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int32_t row = first + i * kSide;
    const bool is_v = row >= p.cache.heads;
    const int32_t head = is_v ? row - p.cache.heads : row;
    const bool there = row < rows && inside && page_offset >= 0;
    const uint8_t* at = (is_v ? p.cache.v : p.cache.k) + page_offset + head * p.cache.head;
    raw[i] = make_uint4(0, 0, 0, 0);
    scale[i] = 0.0f;
    if (there && p.cache.k_scale == nullptr) raw[i] = *reinterpret_cast<const uint4*>(at + 16 * chunk);
    if (there && p.cache.k_scale != nullptr) {
      const uint2 codes = *reinterpret_cast<const uint2*>(at + 8 * chunk);
      raw[i].x = codes.x;
      raw[i].y = codes.y;
      scale[i] = (is_v ? p.cache.v_scale : p.cache.k_scale)[scale_offset + head * p.cache.scale_head];
    }
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int32_t row = first + i * kSide;
    if (row >= rows || !inside) continue;
    const bool is_v = row >= p.cache.heads;
    const int32_t head = is_v ? row - p.cache.heads : row;
    uint4 value = raw[i];
    if (p.cache.k_scale != nullptr) {
      // (a byte as the low one of 2^23 + 128 + it)
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = (__uint_as_float(__byte_perm(j < 4 ? raw[i].x : raw[i].y, 0x4B000000u, 0x7440 | j % 4)) - 8388736.0f) * scale[i];
      }
      value = page_offset < 0 ? make_uint4(0, 0, 0, 0) : pack8(x);
    }
    *reinterpret_cast<uint4*>((is_v ? p.v_out : p.k_out) + (static_cast<int64_t>(token) * p.cache.heads + head) * p.dim + 8 * chunk) = value;
  }
}

int lanes_for(int64_t dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

// Warps with several sets of rows each once there are enough of them to fill the GPU.
bool many(int64_t tokens, int64_t rows, int lanes, int sm_count) {
  return tokens * ((rows * lanes + 31) / 32) >= 64ll * sm_count;
}

template <bool kRotate, bool kWrite>
int launch_heads(HeadsParams p, int64_t tokens, cudaStream_t stream) {
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  const int lanes = lanes_for(p.dim);
  const int64_t rows = p.q_heads + p.k_heads + p.v_heads;
  const bool wide = many(tokens, rows, lanes, device.sm_count);
  const int64_t per_item = 32 / lanes * (wide ? 4 : 1);
  const auto items = [&](int32_t heads) { return static_cast<int32_t>((heads + per_item - 1) / per_item); };
  p.q_items = items(p.q_heads);
  p.k_items = items(p.k_heads);
  const int64_t of_token = p.q_items + p.k_items + items(p.v_heads);
  CHORD_REQUIRE(tokens * of_token < (1ll << 31), "too many rows");
  p.items_per_token = Divisor(static_cast<uint32_t>(of_token));
  p.items = static_cast<int32_t>(tokens * of_token);
  p.share = 1.0f / static_cast<float>(p.dim);
  using Fn = void (*)(HeadsParams);
  static const Fn kernels[3][2] = {{heads_kernel<8, 1, kRotate, kWrite>, heads_kernel<8, 4, kRotate, kWrite>},
                                   {heads_kernel<16, 1, kRotate, kWrite>, heads_kernel<16, 4, kRotate, kWrite>},
                                   {heads_kernel<32, 1, kRotate, kWrite>, heads_kernel<32, 4, kRotate, kWrite>}};
  const int64_t blocks = (p.items + 7ll) / 8;
  OptionsReadLock guard(options_mutex());
  CHORD_CUDA(launch_kernel(kernels[lanes / 16][wide], dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,
                           options().pdl != 0, p));
  return kOk;
}

int check_rows(const char* name, const void* at, int64_t token, int64_t head) {
  CHORD_REQUIRE(at != nullptr, "null pointer %s", name);
  CHORD_REQUIRE((reinterpret_cast<uintptr_t>(at) & 15u) == 0 && token >= 0 && head >= 0 && token % 8 == 0 && head % 8 == 0,
                "%s must have rows on 16-byte boundaries", name);
  return kOk;
}

int fill_rotation(HeadsParams* p, const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                  int64_t k_head, const void* q_weight, const void* k_weight, const float* cos_sin, int64_t max_positions,
                  int64_t rotary, int interleaved, const int32_t* positions, void* q_out, int64_t tokens, int64_t heads,
                  int64_t kv_heads, int64_t dim, int32_t* status, double eps) {
  if (int rc = check_rows("q", q, q_token, q_head)) return rc;
  if (int rc = check_rows("k", k, k_token, k_head)) return rc;
  CHORD_REQUIRE(q_weight != nullptr && k_weight != nullptr && (cos_sin != nullptr || rotary == 0) && positions != nullptr &&
                    q_out != nullptr,
                "null pointer");
  CHORD_REQUIRE(((reinterpret_cast<uintptr_t>(q_weight) | reinterpret_cast<uintptr_t>(k_weight) |
                  reinterpret_cast<uintptr_t>(cos_sin) | reinterpret_cast<uintptr_t>(q_out)) & 15u) == 0,
                "the norms' weights, cos_sin and q_out must be 16-byte aligned");
  CHORD_REQUIRE(tokens >= 0 && tokens < (1ll << 31), "tokens out of range");
  CHORD_REQUIRE(heads > 0 && kv_heads > 0 && heads <= 65535 && kv_heads <= 65535, "heads must be in [1, 65535]");
  CHORD_REQUIRE(dim > 0 && dim % 16 == 0 && dim <= 256, "head_dim must be a multiple of 16 up to 256, got %lld",
                static_cast<long long>(dim));
  CHORD_REQUIRE(rotary >= 0 && rotary % 16 == 0 && rotary <= dim, "rotary_dim must be a multiple of 16 up to head_dim, got %lld",
                static_cast<long long>(rotary));
  CHORD_REQUIRE(max_positions > 0 && max_positions < (1ll << 31), "cos_sin must have a row for some position");
  CHORD_REQUIRE(eps >= 0.0, "eps must not be negative");
  p->q = static_cast<const __nv_bfloat16*>(q);
  p->q_token = q_token;
  p->q_head = q_head;
  p->k = static_cast<const __nv_bfloat16*>(k);
  p->k_token = k_token;
  p->k_head = k_head;
  p->q_weight = static_cast<const __nv_bfloat16*>(q_weight);
  p->k_weight = static_cast<const __nv_bfloat16*>(k_weight);
  p->cos_sin = cos_sin;
  p->positions = positions;
  p->q_out = static_cast<__nv_bfloat16*>(q_out);
  p->status = status;
  p->q_heads = static_cast<int32_t>(heads);
  p->k_heads = static_cast<int32_t>(kv_heads);
  p->dim = static_cast<int32_t>(dim);
  p->rotary = static_cast<int32_t>(rotary);
  p->max_positions = static_cast<int32_t>(max_positions);
  p->eps = static_cast<float>(eps);
  p->interleaved = interleaved != 0;
  return kOk;
}

int fill_values(HeadsParams* p, const void* v, int64_t v_token, int64_t v_head, const chord_b200_kv_cache* cache,
                const int32_t* slots) {
  if (int rc = check_rows("v", v, v_token, v_head)) return rc;
  if (int rc = make_cache(cache, &p->cache)) return rc;
  CHORD_REQUIRE(slots != nullptr, "null slots");
  p->v = static_cast<const __nv_bfloat16*>(v);
  p->v_token = v_token;
  p->v_head = v_head;
  p->slots = slots;
  p->k_heads = p->v_heads = p->cache.heads;
  p->dim = static_cast<int32_t>(cache->head_dim);
  return kOk;
}

}  // namespace
}  // namespace chord

extern "C" {

int chord_b200_qk_norm_rope(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token, int64_t k_head,
                            const void* q_weight, const void* k_weight, const float* cos_sin, int64_t max_positions,
                            int64_t rotary_dim, int interleaved, const int32_t* positions, void* q_out, void* k_out,
                            int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int32_t* status, double eps,
                            void* stream) {
  chord::HeadsParams p = {};
  if (tokens == 0) return chord::kOk;
  if (int rc = chord::fill_rotation(&p, q, q_token, q_head, k, k_token, k_head, q_weight, k_weight, cos_sin, max_positions,
                                    rotary_dim, interleaved, positions, q_out, tokens, heads, kv_heads, head_dim, status, eps))
    return rc;
  CHORD_REQUIRE(k_out != nullptr && (reinterpret_cast<uintptr_t>(k_out) & 15u) == 0, "k_out must be 16-byte aligned");
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  return chord::launch_heads<true, false>(p, tokens, static_cast<cudaStream_t>(stream));
}

int chord_b200_qk_norm_rope_write(const void* q, int64_t q_token, int64_t q_head, const void* k, int64_t k_token,
                                  int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const void* q_weight,
                                  const void* k_weight, const float* cos_sin, int64_t max_positions, int64_t rotary_dim,
                                  int interleaved, const int32_t* positions, void* q_out, const chord_b200_kv_cache* cache,
                                  const int32_t* slots, int64_t tokens, int64_t heads, int32_t* status, double eps,
                                  void* stream) {
  chord::HeadsParams p = {};
  if (tokens == 0) return chord::kOk;
  CHORD_REQUIRE(cache != nullptr, "null cache");
  if (int rc = chord::fill_rotation(&p, q, q_token, q_head, k, k_token, k_head, q_weight, k_weight, cos_sin, max_positions,
                                    rotary_dim, interleaved, positions, q_out, tokens, heads, cache->heads,
                                    cache->head_dim, status, eps))
    return rc;
  if (int rc = chord::fill_values(&p, v, v_token, v_head, cache, slots)) return rc;
  return chord::launch_heads<true, true>(p, tokens, static_cast<cudaStream_t>(stream));
}

int chord_b200_cache_write(const void* k, int64_t k_token, int64_t k_head, const void* v, int64_t v_token, int64_t v_head,
                           const chord_b200_kv_cache* cache, const int32_t* slots, int64_t tokens, int32_t* status,
                           void* stream) {
  chord::HeadsParams p = {};
  CHORD_REQUIRE(tokens >= 0 && tokens < (1ll << 31), "tokens out of range");
  if (tokens == 0) return chord::kOk;
  if (int rc = chord::check_rows("k", k, k_token, k_head)) return rc;
  if (int rc = chord::fill_values(&p, v, v_token, v_head, cache, slots)) return rc;
  p.k = static_cast<const __nv_bfloat16*>(k);
  p.k_token = k_token;
  p.k_head = k_head;
  p.status = status;
  return chord::launch_heads<false, true>(p, tokens, static_cast<cudaStream_t>(stream));
}

int chord_b200_cache_read(const chord_b200_kv_cache* cache, const int32_t* tables, int64_t table_stride, int64_t max_pages,
                          const int32_t* offsets, int64_t batch, void* k_out, void* v_out, int64_t total, int32_t* status,
                          void* stream) {
  using namespace chord;
  ReadParams p = {};
  if (int rc = make_cache(cache, &p.cache)) return rc;
  CHORD_REQUIRE(total >= 0 && total < (1ll << 31), "total out of range");
  if (total == 0) return kOk;
  CHORD_REQUIRE(tables != nullptr && offsets != nullptr && k_out != nullptr && v_out != nullptr, "null pointer");
  CHORD_REQUIRE(batch > 0 && batch < (1ll << 31), "batch must be positive");
  CHORD_REQUIRE(max_pages > 0 && max_pages < (1ll << 31) && table_stride >= 0, "a block table has a page or more");
  CHORD_REQUIRE(((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15u) == 0,
                "k_out and v_out must be 16-byte aligned");
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  p.tables = tables;
  p.table_stride = table_stride;
  p.max_pages = static_cast<int32_t>(max_pages);
  p.offsets = offsets;
  p.batch = static_cast<int32_t>(batch);
  p.k_out = static_cast<__nv_bfloat16*>(k_out);
  p.v_out = static_cast<__nv_bfloat16*>(v_out);
  p.total = static_cast<int32_t>(total);
  p.status = status;
  p.dim = static_cast<int32_t>(cache->head_dim);
  const int lanes = lanes_for(p.dim);
  const int64_t rows = 2 * cache->heads;
  const bool wide = many(total, rows, lanes, device.sm_count);
  const int64_t per_item = 32 / lanes * (wide ? 4 : 1);
  const int64_t of_token = (rows + per_item - 1) / per_item;
  CHORD_REQUIRE(total * of_token < (1ll << 31), "too many rows");
  p.items_per_token = Divisor(static_cast<uint32_t>(of_token));
  p.items = static_cast<int32_t>(total * of_token);
  using Fn = void (*)(ReadParams);
  static const Fn kernels[3][2] = {{cache_read_kernel<8, 1>, cache_read_kernel<8, 4>},
                                   {cache_read_kernel<16, 1>, cache_read_kernel<16, 4>},
                                   {cache_read_kernel<32, 1>, cache_read_kernel<32, 4>}};
  const int64_t blocks = (p.items + 7ll) / 8;
  OptionsReadLock guard(options_mutex());
  CHORD_CUDA(launch_kernel(kernels[lanes / 16][wide], dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                           static_cast<cudaStream_t>(stream), options().pdl != 0, p));
  return kOk;
}

}  // extern "C"
