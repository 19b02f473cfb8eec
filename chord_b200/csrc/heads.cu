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
  int64_t items;
  int32_t q_heads, k_heads, v_heads, dim, rotary, max_positions, items_per_token;
  float eps;
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

// Eight codes round(x / scale) + 128 of a row whose largest |x| is `top`, scale = top / 127.
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float top) {
  // (rows below 2^-100 are taken times 2^100, so that 127 / top stays finite)
  const float lift = top < 0x1p-100f ? 0x1p100f : 1.0f;
  const float rate = top > 0.0f ? 127.0f / (top * lift) : 0.0f;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t code = static_cast<uint32_t>(__float2int_rn(x[i] * lift * rate) + 128);
    w[i / 4] |= (code & 0xFFu) << (8 * (i % 4));
  }
  return make_uint2(w[0], w[1]);
}

// kLanes lanes hold a row of up to 8 kLanes elements, 16 bytes each, so a warp works on 32 / kLanes
// rows at a time and on kRows of those sets, whose loads are all in flight at once.  An item is the
// rows of a warp; all belong to one token, so the angles are read once.  Everything between the load
// and the store is FP32; the result is rounded once, to BF16 or to the codes.
template <int kLanes, int kRows, bool kRotate, bool kWrite>
__global__ void __launch_bounds__(256)
heads_kernel(const HeadsParams p) {
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, side = lane / kLanes;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int32_t token = static_cast<int32_t>(item / p.items_per_token);
  const int32_t first = static_cast<int32_t>(item % p.items_per_token) * (kSide * kRows) + side;
  const int32_t rows = p.q_heads + p.k_heads + p.v_heads;
  const bool inside = 8 * chunk < p.dim;
  ptx::grid_dependency_wait();

  // (the results may take the inputs' place)
  uint4 raw[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int32_t row = first + i * kSide;
    const __nv_bfloat16* at = p.q + token * p.q_token + row * p.q_head;
    if (row >= p.q_heads) at = p.k + token * p.k_token + (row - p.q_heads) * p.k_head;
    if (kWrite && row >= p.q_heads + p.k_heads) at = p.v + token * p.v_token + (row - p.q_heads - p.k_heads) * p.v_head;
    raw[i] = row < rows && inside ? load_once_coherent(at + 8 * chunk) : make_uint4(0, 0, 0, 0);
  }

  float cos[8], sin[8];
  bool turned = false, lost = false;
  int partner = lane;
  float sign = 0.0f;
  uint4 q_weight, k_weight;
  if constexpr (kRotate) {
    q_weight = k_weight = make_uint4(0, 0, 0, 0);
    if (inside) {
      q_weight = __ldg(reinterpret_cast<const uint4*>(p.q_weight) + chunk);
      k_weight = __ldg(reinterpret_cast<const uint4*>(p.k_weight) + chunk);
    }
    const int32_t position = __ldg(p.positions + token);
    lost = position < 0 || position >= p.max_positions;
    if (lost && p.status != nullptr && lane == 0) atomicOr(p.status, kStatusIndex);
    turned = 8 * chunk < p.rotary && !lost;
    const int32_t half = p.rotary / 2;
    const bool upper = 8 * chunk >= half;
#pragma unroll
    for (int i = 0; i < 8; ++i) cos[i] = 1.0f, sin[i] = 0.0f;
    if (turned) {
      const float* at = p.cos_sin + static_cast<int64_t>(position) * p.rotary +
                        (p.interleaved ? 4 * chunk : 8 * chunk - (upper ? half : 0));
      float4 c[2], s[2];
      c[0] = __ldg(reinterpret_cast<const float4*>(at));
      s[0] = __ldg(reinterpret_cast<const float4*>(at + half));
      c[1] = c[0];
      s[1] = s[0];
      if (!p.interleaved) {
        c[1] = __ldg(reinterpret_cast<const float4*>(at) + 1);
        s[1] = __ldg(reinterpret_cast<const float4*>(at + half) + 1);
        partner = upper ? lane - half / 8 : lane + half / 8;
        sign = upper ? 1.0f : -1.0f;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        cos[4 * i] = c[i].x, cos[4 * i + 1] = c[i].y, cos[4 * i + 2] = c[i].z, cos[4 * i + 3] = c[i].w;
        sin[4 * i] = s[i].x, sin[4 * i + 1] = s[i].y, sin[4 * i + 2] = s[i].z, sin[4 * i + 3] = s[i].w;
      }
    }
  }
  int64_t page_offset = -1, scale_offset = 0;
  if constexpr (kWrite) {
    const int32_t slot = __ldg(p.slots + token);
    if (slot >= 0) {
      const uint32_t page = p.cache.page_size.div(static_cast<uint32_t>(slot));
      const uint32_t in_page = static_cast<uint32_t>(slot) - page * p.cache.page_size.d;
      if (page < static_cast<uint32_t>(p.cache.num_pages)) {
        page_offset = page * p.cache.page + in_page * p.cache.token;
        scale_offset = page * p.cache.scale_page + in_page * p.cache.scale_token;
      } else if (p.status != nullptr && lane == 0) {
        atomicOr(p.status, kStatusIndex);
      }
    }
  }

#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int32_t row = first + i * kSide;
    if (row - side >= rows) break;  // (the whole warp)
    float x[8];
    unpack8(raw[i], x);
    const bool is_q = row < p.q_heads, is_v = kWrite && row >= p.q_heads + p.k_heads;
    if constexpr (kRotate) {
      float square = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) square = fmaf(x[j], x[j], square);
#pragma unroll
      for (int d = kLanes / 2; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
      const float rate = rsqrtf(square / static_cast<float>(p.dim) + p.eps);
      float w[8], y[8];
      unpack8(is_q ? q_weight : k_weight, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = x[j] * rate * w[j];
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = y[2 * j], b = y[2 * j + 1];
          y[2 * j] = a * cos[j] - b * sin[j];
          y[2 * j + 1] = b * cos[j] + a * sin[j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float other = __shfl_sync(0xffffffffu, y[j], partner);
          y[j] = turned ? y[j] * cos[j] + sign * other * sin[j] : y[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = is_v ? x[j] : lost ? 0.0f : y[j];
    }
    if (kRotate && is_q) {
      if (inside) {
        *reinterpret_cast<uint4*>(p.q_out + (static_cast<int64_t>(token) * p.q_heads + row) * p.dim + 8 * chunk) = pack8(x);
      }
    }
    if constexpr (!kWrite) {
      if (!is_q && row < rows && inside) {
        const int32_t head = row - p.q_heads;
        *reinterpret_cast<uint4*>(p.k_out + (static_cast<int64_t>(token) * p.k_heads + head) * p.dim + 8 * chunk) = pack8(x);
      }
    } else {
      const int32_t head = row - p.q_heads - (is_v ? p.k_heads : 0);
      const bool keep = !is_q && row < rows && inside && page_offset >= 0;
      uint8_t* at = (is_v ? p.cache.v : p.cache.k) + page_offset + head * p.cache.head;
      if (p.cache.k_scale == nullptr) {
        if (keep) *reinterpret_cast<uint4*>(at + 16 * chunk) = pack8(x);
      } else {
        // The largest |x| by its bits: infinities and NaNs come out on top, and such a row gets a scale
        // of NaN, so that it reads back as NaN.
        uint32_t bits = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) bits = max(bits, __float_as_uint(x[j]) & 0x7FFFFFFFu);
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) bits = max(bits, __shfl_xor_sync(0xffffffffu, bits, d));
        const bool finite = bits < 0x7F800000u;
        const float top = __uint_as_float(finite ? bits : 0x7FC00000u);
        if (keep) {
          *reinterpret_cast<uint2*>(at + 8 * chunk) = finite ? quantise8(x, top) : make_uint2(0x80808080u, 0x80808080u);
          if (chunk == 0) (is_v ? p.cache.v_scale : p.cache.k_scale)[scale_offset + head * p.cache.scale_head] = top / 127.0f;
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
  int64_t table_stride, items;
  int32_t batch, max_pages, total, dim, items_per_token;
};

// As heads_kernel: a warp reads rows of one token, its keys' heads and then its values'.
template <int kLanes, int kRows>
__global__ void __launch_bounds__(256)
cache_read_kernel(const ReadParams p) {
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, side = lane / kLanes;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int32_t token = static_cast<int32_t>(item / p.items_per_token);
  const int32_t first = static_cast<int32_t>(item % p.items_per_token) * (kSide * kRows) + side;
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
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t code = ((j < 4 ? raw[i].x : raw[i].y) >> (8 * (j % 4))) & 0xFFu;
        x[j] = page_offset < 0 ? 0.0f : static_cast<float>(static_cast<int32_t>(code) - 128) * scale[i];
      }
      value = pack8(x);
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
  p.items_per_token = static_cast<int32_t>((rows + per_item - 1) / per_item);
  p.items = tokens * p.items_per_token;
  using Fn = void (*)(HeadsParams);
  static const Fn kernels[3][2] = {{heads_kernel<8, 1, kRotate, kWrite>, heads_kernel<8, 4, kRotate, kWrite>},
                                   {heads_kernel<16, 1, kRotate, kWrite>, heads_kernel<16, 4, kRotate, kWrite>},
                                   {heads_kernel<32, 1, kRotate, kWrite>, heads_kernel<32, 4, kRotate, kWrite>}};
  const int64_t blocks = (p.items + 7) / 8;
  CHORD_REQUIRE(blocks < (1ll << 31), "too many rows");
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
  p.items_per_token = static_cast<int32_t>((rows + per_item - 1) / per_item);
  p.items = total * p.items_per_token;
  using Fn = void (*)(ReadParams);
  static const Fn kernels[3][2] = {{cache_read_kernel<8, 1>, cache_read_kernel<8, 4>},
                                   {cache_read_kernel<16, 1>, cache_read_kernel<16, 4>},
                                   {cache_read_kernel<32, 1>, cache_read_kernel<32, 4>}};
  const int64_t blocks = (p.items + 7) / 8;
  CHORD_REQUIRE(blocks < (1ll << 31), "too many rows");
  OptionsReadLock guard(options_mutex());
  CHORD_CUDA(launch_kernel(kernels[lanes / 16][wide], dim3(static_cast<unsigned>(blocks)), dim3(256), 0,
                           static_cast<cudaStream_t>(stream), options().pdl != 0, p));
  return kOk;
}

}  // extern "C"
