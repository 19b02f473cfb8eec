// Queries, keys and values between the projection and the attention: norms of each head with the
// position rotation, and the paged cache as it is written and read back.
#include <cuda_bf16.h>

#include "../../include/chord_b200.h"
#include "common.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {
namespace {

// Warps of a CTA, which work on their own: with few of them none of an SM's places waits for the longest (8192
// tokens rotated 53.4 us, 55.6 with eight; 16384 written and read 35.9 and 36.9).
constexpr int kWarps = 2;

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
  int32_t items, turns, q_heads, k_heads, v_heads, dim, rotary, max_positions;
  int32_t q_items, k_items;  // items of a token: its queries', keys' and
  Divisor items_per_token;   // all
  float eps, share;          // share: 1 / dim
  bool interleaved;
};

// Two FP32 numbers at a time.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mul.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n .reg .b64 a, b, c, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n mov.b64 c, {%6, %7};\n fma.rn.f32x2 d, a, b, c;\n"
      " mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %5};\n add.rn.f32x2 d, a, b;\n mov.b64 {%0, %1}, d;\n}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

__device__ __forceinline__ float2 unpack2(uint32_t pair) { return make_float2(bf16_lo(pair), bf16_hi(pair)); }

// Eight elements of a row, as two halves of four that the rotation takes with one another.
struct Eight {
  float2 a[2], b[2];
};

__device__ __forceinline__ Eight unpack8(const uint4 v) { return Eight{{unpack2(v.x), unpack2(v.y)}, {unpack2(v.z), unpack2(v.w)}}; }

__device__ __forceinline__ uint4 pack8(const Eight& e) {
  return make_uint4(pack_bf16(e.a[0].x, e.a[0].y), pack_bf16(e.a[1].x, e.a[1].y), pack_bf16(e.b[0].x, e.b[0].y), pack_bf16(e.b[1].x, e.b[1].y));
}

// Eight elements in order: the even ones first, then the odd ones; and back, as BF16 and as bytes.
__device__ __forceinline__ uint4 deal(const uint4 v) {
  return make_uint4(__byte_perm(v.x, v.y, 0x5410), __byte_perm(v.z, v.w, 0x5410), __byte_perm(v.x, v.y, 0x7632), __byte_perm(v.z, v.w, 0x7632));
}

__device__ __forceinline__ uint4 undeal(const uint4 v) {
  return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
}

__device__ __forceinline__ uint2 undeal(const uint2 v) { return make_uint2(__byte_perm(v.x, v.y, 0x5140), __byte_perm(v.x, v.y, 0x7362)); }

__device__ __forceinline__ uint2 load8_once_ordered(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p) : "memory");
  return v;
}

// The largest magnitude; a NaN where there is one.
__device__ __forceinline__ float max_magnitude(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// a / b where `inverse` is 1 / b to 2^-22: the product's residual, exact by one multiply-add, corrects it once (the
// last step of P. Markstein's division, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990).  What is left is the last rounding, 2^-24, and 2^-43.  Twice a division here took a write and read
// of 16384 tokens from 36.9 to 38.9 us.
__device__ __forceinline__ float corrected_quotient(float a, float b, float inverse) {
  const float q = a * inverse;
  return fmaf(fmaf(-b, q, a), inverse, q);
}

// Eight codes round(x / scale) + 128 of a row whose largest |x| is `top`, scale = top / 127; halves go to the
// even code.  A half is common (x = top / 2 is 63.5 steps), and x * rate is off by up to 2^-17 there: the first
// sum rounds to steps of 2^-15, which brings it back, the second (1.5 * 2^23 + 128 in all) to whole numbers, the
// code in the low byte.  (No quotient of two BF16 numbers that is not a half comes as near to one.)
__device__ __forceinline__ uint2 quantise8(Eight& e, float top) {
  const bool beyond = !(top > 0x1p-100f && top < 0x1p100f);  // (the reciprocal's range)
  if (__any_sync(0xffffffffu, beyond)) {
    const float factor = !beyond ? 1.0f : top < 1.0f ? 0x1p100f : 0x1p-64f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      e.a[i].x *= factor, e.a[i].y *= factor;
      e.b[i].x *= factor, e.b[i].y *= factor;
    }
    top = top > 0.0f ? top * factor : 1.0f;
  }
  float inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(top));
  const float rate = corrected_quotient(127.0f, top, inverse);
  const float2 rates = make_float2(rate, rate), fine = make_float2(384.0f, 384.0f);
  const float2 whole = make_float2(12583040.0f - 384.0f, 12583040.0f - 384.0f);
  const auto four = [&](const float2 x, const float2 y) {
    const float2 c = add2(fma2(x, rates, fine), whole), d = add2(fma2(y, rates, fine), whole);
    return low_bytes(__float_as_uint(c.x), __float_as_uint(c.y), __float_as_uint(d.x), __float_as_uint(d.y));
  };
  return make_uint2(four(e.a[0], e.a[1]), four(e.b[0], e.b[1]));
}

// What becomes of keys and values.
enum class Keep { kNothing, kNumbers, kCodes };

// kLanes lanes hold a row of up to 8 kLanes elements, eight each, so a warp works on 32 / kLanes rows at a
// time and on kRows of those sets, whose loads are all in flight at once, p.turns times.  An item is the rows of
// a warp: rows of one token, all queries, keys or values (without queries keys and then values).  A lane's eight
// elements are four and the four that they turn with, so that a rotation needs no other lane; what an item's rows
// have in common is worked out once: with the norm's weights w and the angles in their products, a result is
// rate * (x A + x' B).  Everything between the load and the store is FP32; the result is rounded once, to BF16 or to
// the codes.
//
// Memory bounds it once there are many tokens, and instructions just before: 8192 tokens of 64 + 8 heads of 128,
// 302 MB, 53 to 56 us from GPU to GPU = 5.4 to 5.7 TB/s, 82 to 87 % of a plain copy's rate (184 instructions for a set of rows took 60.2, 115
// take this); 16384 tokens of 8 heads of 128 written as codes and read back, 203 MB, 36 to 37 us, 85 % (44.8
// with 149 and 137 instructions for a set, now 105 and 69).  Three or two sets in flight are slower (8192 tokens
// 63 and 59 us), as are fewer warps with more registers (64 us); one token takes a launch and two round trips
// to memory, 1.9 us.
template <int kLanes, int kRows, bool kRotate, Keep kKeep>
__global__ void __launch_bounds__(kWarps * 32, 32 / kWarps)
heads_kernel(const HeadsParams p) {
  constexpr bool kWrite = kKeep != Keep::kNothing;
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, side = lane / kLanes;
  const int32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int32_t token = p.items_per_token.div(item);
  int32_t group = item - token * p.items_per_token.d;
  // Which of the three, and the item's rows.
  const bool is_q = kRotate && group < p.q_items;
  if (!is_q) group -= p.q_items;
  bool is_v = kWrite && !is_q && group >= p.k_items;
  if (is_v) group -= p.k_items;
  const int32_t begin = group * p.turns * (kSide * kRows) + side;
  int32_t row = begin;
  const int32_t end = min(is_q ? p.q_heads : p.k_heads, (group + 1) * p.turns * (kSide * kRows));
  const bool inside = 8 * chunk < p.dim;
  // The lane's two fours: side by side, or half the rotated part apart.
  const bool turns = kRotate && !is_v;
  const bool apart = turns && !p.interleaved, dealt = turns && p.interleaved;
  const bool turned = turns && 8 * chunk < p.rotary;
  const int32_t half = p.rotary / 2;
  const int32_t first = apart && turned ? 4 * chunk : 8 * chunk, second = apart && turned ? first + half : first + 4;
  int64_t stride = is_q ? p.q_head : is_v ? p.v_head : p.k_head;
  const __nv_bfloat16* from = (is_q ? p.q + token * p.q_token : is_v ? p.v + token * p.v_token : p.k + token * p.k_token) + row * stride + first;
  const int32_t away = second - first;
  ptx::grid_dependency_wait();

  uint4 raw[kRows];
  const auto load = [&] {  // (the results may take the inputs' place)
    if (apart) {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const bool there = row + i * kSide < end && inside;
        const uint2 a = there ? load8_once_ordered(from) : make_uint2(0, 0), b = there ? load8_once_ordered(from + away) : make_uint2(0, 0);
        raw[i] = make_uint4(a.x, a.y, b.x, b.y);
        from += kSide * stride;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        raw[i] = row + i * kSide < end && inside ? load_once_ordered(from) : make_uint4(0, 0, 0, 0);
        from += kSide * stride;
      }
    }
  };
  load();

  Eight own, other;  // A, B
  bool lost = false;
  if constexpr (kRotate) {
    if (!is_v) {
      const __nv_bfloat16* const weight = is_q ? p.q_weight : p.k_weight;
      const int32_t position = load_arg(p.positions + token);
      lost = position < 0 || position >= p.max_positions;
      if (lost && p.status != nullptr && lane == 0) atomicOr(p.status, kStatusIndex);
      uint2 w0 = make_uint2(0, 0), w1 = make_uint2(0, 0);
      if (inside) {
        w0 = load_arg(reinterpret_cast<const uint2*>(weight + first));
        w1 = load_arg(reinterpret_cast<const uint2*>(weight + second));
      }
      uint4 words = make_uint4(w0.x, w0.y, w1.x, w1.y);
      if (dealt) words = deal(words);
      own = unpack8(words);
      other = Eight{};
      if (lost) {
        own = Eight{};
      } else if (turned) {
        const float* const at = p.cos_sin + static_cast<int64_t>(position) * p.rotary + 4 * chunk;
        const float4 c = load_arg(reinterpret_cast<const float4*>(at)), s = load_arg(reinterpret_cast<const float4*>(at + half));
        const float2 cs[2] = {{c.x, c.y}, {c.z, c.w}}, sn[2] = {{s.x, s.y}, {s.z, s.w}}, minus[2] = {{-s.x, -s.y}, {-s.z, -s.w}};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          other.a[i] = mul2(own.b[i], minus[i]);
          other.b[i] = mul2(own.a[i], sn[i]);
          own.a[i] = mul2(own.a[i], cs[i]);
          own.b[i] = mul2(own.b[i], cs[i]);
        }
      }
    }
  }
  bool kept = false;
  int64_t offset = 0, scale_offset = 0;  // of the token's first row here
  if constexpr (kWrite) {
    if (!is_q) {
      const int32_t slot = load_arg(p.slots + token);
      const uint32_t page = slot >= 0 ? p.cache.page_size.div(static_cast<uint32_t>(slot)) : 0;
      const uint32_t in_page = static_cast<uint32_t>(slot) - page * p.cache.page_size.d;
      kept = slot >= 0 && page < static_cast<uint32_t>(p.cache.num_pages);
      if (kept) {
        offset = page * p.cache.page + in_page * p.cache.token + row * p.cache.head;
        scale_offset = page * p.cache.scale_page + in_page * p.cache.scale_token + row * p.cache.scale_head;
      } else if (slot >= 0 && p.status != nullptr && lane == 0) {
        atomicOr(p.status, kStatusIndex);
      }
    }
  }
  uint8_t* at = (is_v ? p.cache.v : p.cache.k) + offset;
  float* scale_at = (is_v ? p.cache.v_scale : p.cache.k_scale) + scale_offset;
  __nv_bfloat16* to = is_q ? p.q_out : p.k_out;
  if (is_q || !kWrite) to += (static_cast<int64_t>(token) * (is_q ? p.q_heads : p.k_heads) + row) * p.dim + first;

#pragma unroll 1
  while (true) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (row - side >= end) {  // (the whole warp)
        if constexpr (kRotate || kRows == 1) return;
        break;
      }
      const bool mine = row < end && inside;
      if (kRotate && lost) raw[i] = make_uint4(0, 0, 0, 0);
      Eight x = unpack8(kRotate && dealt ? deal(raw[i]) : raw[i]);
      if (kRotate && !is_v) {
        const float2 squares = fma2(x.b[1], x.b[1], fma2(x.b[0], x.b[0], fma2(x.a[1], x.a[1], mul2(x.a[0], x.a[0]))));
        float square = squares.x + squares.y;
#pragma unroll
        for (int d = kLanes / 2; d > 0; d >>= 1) square += __shfl_xor_sync(0xffffffffu, square, d);
        const float rate = lost ? 0.0f : rsqrtf(fmaf(square, p.share, p.eps));
        const float2 rates = make_float2(rate, rate);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float2 a = mul2(rates, fma2(x.a[j], own.a[j], mul2(x.b[j], other.a[j])));
          x.b[j] = mul2(rates, fma2(x.b[j], own.b[j], mul2(x.a[j], other.b[j])));
          x.a[j] = a;
        }
      }
      if (is_q || !kWrite) {
        uint4 v = pack8(x);
        if (dealt) v = undeal(v);
        if (mine) {
          if (apart) {
            *reinterpret_cast<uint2*>(to) = make_uint2(v.x, v.y);
            *reinterpret_cast<uint2*>(to + away) = make_uint2(v.z, v.w);
          } else {
            *reinterpret_cast<uint4*>(to) = v;
          }
        }
        to += kSide * p.dim;
      } else if constexpr (kWrite) {
        const bool keep = mine && kept;
        if constexpr (kKeep == Keep::kNumbers) {
          uint4 v = raw[i];
          if (kRotate && !is_v) {
            v = pack8(x);
            if (dealt) v = undeal(v);
          }
          if (keep) {
            if (apart) {
              *reinterpret_cast<uint2*>(at + 2 * first) = make_uint2(v.x, v.y);
              *reinterpret_cast<uint2*>(at + 2 * second) = make_uint2(v.z, v.w);
            } else {
              *reinterpret_cast<uint4*>(at + 16 * chunk) = v;
            }
          }
        } else {
          float top = max_magnitude(x.a[0].x, x.a[0].y, x.a[1].x);
          top = max_magnitude(top, x.a[1].y, x.b[0].x);
          top = max_magnitude(top, x.b[0].y, x.b[1].x);
          top = max_magnitude(top, x.b[1].y, 0.0f);
#pragma unroll
          for (int d = kLanes / 2; d > 0; d >>= 1) top = max_magnitude(top, __shfl_xor_sync(0xffffffffu, top, d), 0.0f);
          uint2 codes = quantise8(x, top);
          if (dealt) codes = undeal(codes);
          // A row with an infinity or a NaN gets a scale of NaN, so that it reads back as NaN.
          const bool finite = top < INFINITY;
          if (!finite) codes = make_uint2(0x80808080u, 0x80808080u);
          if (keep) {
            if (apart) {
              *reinterpret_cast<uint32_t*>(at + first) = codes.x;
              *reinterpret_cast<uint32_t*>(at + second) = codes.y;
            } else {
              *reinterpret_cast<uint2*>(at + 8 * chunk) = codes;
            }
          }
          if (keep && chunk == 0) *scale_at = finite ? corrected_quotient(top, 127.0f, 1.0f / 127.0f) : __uint_as_float(0x7FC00000u);
          scale_at += kSide * p.cache.scale_head;
        }
        at += kSide * p.cache.head;
      }
      row += kSide;
    }
    if (row - side >= end) {
      if (kRotate || kRows == 1 || is_v) return;  // (else the keys are followed by the values)
      is_v = true;
      row = begin;
      from = p.v + token * p.v_token + row * p.v_head + first;
      stride = p.v_head;
      at = p.cache.v + offset;
      scale_at = p.cache.v_scale + scale_offset;
    }
    load();
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

// As heads_kernel: a warp reads heads of one token, their keys and then their values; where a set is all that it
// reads (kRows is one), keys or values by blockIdx.y.
template <int kLanes, int kRows>
__global__ void __launch_bounds__(kWarps * 32, 32 / kWarps)
cache_read_kernel(const ReadParams p) {
  constexpr int kSide = 32 / kLanes;
  const int lane = threadIdx.x & 31, chunk = lane % kLanes, side = lane / kLanes;
  const int32_t item = blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (item >= p.items) return;
  const int32_t token = p.items_per_token.div(item);
  const int32_t heads = p.cache.heads;
  const int32_t first = (item - token * static_cast<int32_t>(p.items_per_token.d)) * (kSide * kRows) + side;
  const int32_t end = min(heads, first - side + kSide * kRows);
  ptx::grid_dependency_wait();

  // The sequence: the last one that does not begin after the token; 32 at a time, coarse to fine.
  int32_t low = 0, count = p.batch;
  while (count > 1) {
    const int32_t step = (count + 31) / 32;
    const int32_t at = lane * step;
    const bool before = at < count && load_arg(p.offsets + low + at) <= token;
    const uint32_t votes = __ballot_sync(0xffffffffu, before);
    const int32_t last = votes == 0 ? 0 : 31 - __clz(votes);
    low += last * step;
    count = min(step, count - last * step);
  }
  const int32_t begin = load_arg(p.offsets + low);
  int64_t page_offset = -1, scale_offset = 0;
  if (token >= begin && token < load_arg(p.offsets + low + 1)) {
    const uint32_t at = static_cast<uint32_t>(token) - static_cast<uint32_t>(begin);
    const uint32_t index = p.cache.page_size.div(at), in_page = at - index * p.cache.page_size.d;
    const int32_t page = begin >= 0 && index < static_cast<uint32_t>(p.max_pages) ? load_arg(p.tables + low * p.table_stride + index) : -1;
    if (page >= 0 && page < p.cache.num_pages) {
      page_offset = page * p.cache.page + in_page * p.cache.token;
      scale_offset = page * p.cache.scale_page + in_page * p.cache.scale_token;
    } else if (p.status != nullptr && lane == 0) {
      atomicOr(p.status, kStatusIndex);
    }
  }
  const bool inside = 8 * chunk < p.dim, known = page_offset >= 0;
  const int64_t out = (static_cast<int64_t>(token) * heads + first) * p.dim + 8 * chunk;
#pragma unroll 1
  for (int32_t kv = kRows == 1 ? blockIdx.y : 0; kv < (kRows == 1 ? static_cast<int32_t>(blockIdx.y) + 1 : 2); ++kv) {
    __nv_bfloat16* to = (kv ? p.v_out : p.k_out) + out;
    if (p.cache.k_scale == nullptr) {
      const uint8_t* at = (kv ? p.cache.v : p.cache.k) + page_offset + first * p.cache.head + 16 * chunk;
      uint4 raw[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        raw[i] = known && inside && first + i * kSide < end ? load_once(at) : make_uint4(0, 0, 0, 0);
        at += kSide * p.cache.head;
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (inside && first + i * kSide < end) *reinterpret_cast<uint4*>(to) = raw[i];
        to += kSide * p.dim;
      }
    } else {
      const uint8_t* at = (kv ? p.cache.v : p.cache.k) + page_offset + first * p.cache.head + 8 * chunk;
      const float* scale_at = (kv ? p.cache.v_scale : p.cache.k_scale) + scale_offset + first * p.cache.scale_head;
      uint2 raw[kRows];
      float scale[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const bool there = known && inside && first + i * kSide < end;
        raw[i] = there ? load_arg(reinterpret_cast<const uint2*>(at)) : make_uint2(0, 0);
        scale[i] = there ? load_arg(scale_at) : 0.0f;
        at += kSide * p.cache.head;
        scale_at += kSide * p.cache.scale_head;
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        // (a byte as the low one of 2^23 + 128 + it)
        const float2 offset = make_float2(-8388736.0f, -8388736.0f), scales = make_float2(scale[i], scale[i]);
        const auto two = [&](uint32_t codes, int select) {
          return mul2(add2(make_float2(__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7440 | select)),
                                       __uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7441 | select))), offset), scales);
        };
        const uint4 v = pack8(Eight{{two(raw[i].x, 0), two(raw[i].x, 2)}, {two(raw[i].y, 0), two(raw[i].y, 2)}});
        if (inside && first + i * kSide < end) *reinterpret_cast<uint4*>(to) = known ? v : make_uint4(0, 0, 0, 0);
        to += kSide * p.dim;
      }
    }
  }
}

int lanes_for(int64_t dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

// The sets of rows, a warp's at a time, for every SM.  From 48 on a warp takes four of them (one before): 512
// tokens of 64 + 8 heads of 128 6.1 us with four, 8.4 with one, 128 tokens 3.9 and 3.5.
int64_t sets_per_sm(int64_t tokens, int64_t rows, int lanes, int sm_count) { return tokens * ((rows * lanes + 31) / 32) / sm_count; }

template <bool kRotate, Keep kKeep>
int launch_heads(HeadsParams p, int64_t tokens, cudaStream_t stream) {
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  const int lanes = lanes_for(p.dim);
  const int64_t sets = sets_per_sm(tokens, p.q_heads + p.k_heads + p.v_heads, lanes, device.sm_count);
  const bool wide = sets >= 48;
  // Twice four from 512 on, where the queries are more than two times four sets: weights and angles are worked out
  // half as often, but the warps of a token's keys have less to do than its queries'.  8192 tokens of 64 + 8 heads of
  // 128 52.3 us like this, 56.2 with four; 1024 tokens 10.7 and 9.5; 8192 of 32 + 8 heads of 64 20.9 and 19.3.
  const int64_t four = 32 / lanes * 4;
  p.turns = kRotate && sets >= 512 && p.q_heads > 2 * four ? 2 : 1;
  const int64_t per_item = wide ? four * p.turns : 32 / lanes;
  const auto items = [&](int32_t heads) { return static_cast<int32_t>((heads + per_item - 1) / per_item); };
  p.q_items = items(p.q_heads);
  p.k_items = items(p.k_heads);
  const int64_t of_token = p.q_items + p.k_items + (kRotate || !wide ? items(p.v_heads) : 0);
  CHORD_REQUIRE(tokens * of_token < (1ll << 31), "too many rows");
  p.items_per_token = Divisor(static_cast<uint32_t>(of_token));
  p.items = static_cast<int32_t>(tokens * of_token);
  p.share = 1.0f / static_cast<float>(p.dim);
  using Fn = void (*)(HeadsParams);
  static const Fn kernels[3][2] = {{heads_kernel<8, 1, kRotate, kKeep>, heads_kernel<8, 4, kRotate, kKeep>},
                                   {heads_kernel<16, 1, kRotate, kKeep>, heads_kernel<16, 4, kRotate, kKeep>},
                                   {heads_kernel<32, 1, kRotate, kKeep>, heads_kernel<32, 4, kRotate, kKeep>}};
  const int64_t blocks = (p.items + kWarps - 1ll) / kWarps;
  CHORD_CUDA(launch_kernel(kernels[lanes / 16][wide], dim3(static_cast<unsigned>(blocks)), dim3(kWarps * 32), 0, stream,
                           kEarlyLaunch, p));
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
  return chord::launch_heads<true, chord::Keep::kNothing>(p, tokens, static_cast<cudaStream_t>(stream));
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
  return p.cache.k_scale != nullptr ? chord::launch_heads<true, chord::Keep::kCodes>(p, tokens, static_cast<cudaStream_t>(stream))
                                    : chord::launch_heads<true, chord::Keep::kNumbers>(p, tokens, static_cast<cudaStream_t>(stream));
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
  return p.cache.k_scale != nullptr ? chord::launch_heads<false, chord::Keep::kCodes>(p, tokens, static_cast<cudaStream_t>(stream))
                                    : chord::launch_heads<false, chord::Keep::kNumbers>(p, tokens, static_cast<cudaStream_t>(stream));
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
  const bool wide = sets_per_sm(total, 2 * cache->heads, lanes, device.sm_count) >= 48;
  const int64_t per_item = 32 / lanes * (wide ? 4 : 1);
  const int64_t of_token = (cache->heads + per_item - 1) / per_item;
  CHORD_REQUIRE(total * of_token < (1ll << 31), "too many rows");
  p.items_per_token = Divisor(static_cast<uint32_t>(of_token));
  p.items = static_cast<int32_t>(total * of_token);
  using Fn = void (*)(ReadParams);
  static const Fn kernels[3][2] = {{cache_read_kernel<8, 1>, cache_read_kernel<8, 4>},
                                   {cache_read_kernel<16, 1>, cache_read_kernel<16, 4>},
                                   {cache_read_kernel<32, 1>, cache_read_kernel<32, 4>}};
  const int64_t blocks = (p.items + kWarps - 1ll) / kWarps;
  CHORD_CUDA(launch_kernel(kernels[lanes / 16][wide], dim3(static_cast<unsigned>(blocks), wide ? 1 : 2), dim3(kWarps * 32), 0,
                           static_cast<cudaStream_t>(stream), kEarlyLaunch, p));
  return kOk;
}

}  // extern "C"
