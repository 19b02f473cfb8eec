// Attention of one new token for each sequence over its pages of keys and values.
#include <cuda_bf16.h>

#include <mutex>

#include "../../include/chord_b200.h"
#include "common.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCtasPerSm = 2;
constexpr int kMaxParts = 1024;  // CTAs of a launch at most

struct AttentionParams {
  Cache cache;
  const __nv_bfloat16* q;
  const int32_t* tables;
  const int32_t* lengths;
  __nv_bfloat16* out;  // [batch, heads, dim]
  float* lse;          // [batch, heads] or null
  float* partials;
  int32_t* locks;
  int32_t* status;
  int64_t q_batch, q_head, table_stride;
  int32_t batch, heads, group, head_blocks, capacity, window;
  float scale;  // of the scores, with log2(e)
};

// What follows from the head's width and the cache's type.  A warp takes kStep tokens at a time, whose
// keys and values are some 5 to 16 KB; kStages of them are on their way or in use.
template <int kDim, bool kCodes>
struct Layout {
  static constexpr int kRow = kDim * (kCodes ? 1 : 2);  // bytes of a row
  static constexpr int kPitch = kRow + 16;              // an odd number of 16-byte pieces: no bank conflicts
  static constexpr int kStep = kRow < 128 ? 32 : 16;
  static constexpr int kUnit = kStep * kWarps;          // tokens of a CTA's step
  static constexpr int kScaleBytes = kCodes ? 2 * kStep * 4 : 0;
  static constexpr int kStageBytes = 2 * kStep * kPitch + kScaleBytes;
  static constexpr int kCtas = kDim > 128 ? 1 : kMaxCtasPerSm;
  static constexpr int kFit = (kCtas == 1 ? 220 : 110) * 1024 / (kWarps * kStageBytes);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  static constexpr int kHeads = 16;                     // query heads of a CTA
  static_assert(kStages >= 2 && kSmem >= kWarps * kHeads * kDim * 4, "the partial sums of the warps take the ring's place");
};

__host__ __device__ constexpr int64_t partial_floats(int dim) { return 16 * dim + 32; }

template <bool kCodes>
__device__ __forceinline__ void codes_to_bf16(uint32_t four, uint32_t select_a, uint32_t select_b, uint32_t& a, uint32_t& b) {
  constexpr uint32_t kOffset = 0xC000C000u;  // -128 / 64, twice
  a = bf16x2_fma(__byte_perm(four, 0, select_a), kTwo127, kOffset);
  b = bf16x2_fma(__byte_perm(four, 0, select_b), kTwo127, kOffset);
}

__device__ __forceinline__ void ldmatrix_x4_at(uint32_t addr, uint32_t (&r)[4]) { ptx::ldmatrix_x4<0>(addr, r); }

__device__ __forceinline__ void cp_async_4(uint32_t dst, const void* src, bool valid) {
  const uint32_t bytes = valid ? 4u : 0u;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// One row of work is a sequence, one of its key-value heads and a block of up to 16 of the query heads
// that share it; the rows' tokens, in units of kUnit, are numbered through and dealt out to the CTAs in
// equal shares, so that lengths need not be alike.  A CTA's share is cut into segments at the rows'
// ends.  The four warps of a CTA take every fourth step of a segment, each with its own ring of
// cp.async stages, running maximum, sum and output, and meet only at its end.
//
// Products: scores S[heads 16, tokens] = Q K^T and O[heads, dim] += P V on mma.m16n8k16, whose score
// fragment is the operand fragment of P.  P is multiplied as the sum of two BF16 numbers (16 bits of
// it); with up to eight heads the second part travels in the operand's idle rows 8-15 and costs
// nothing (kWide == false).  Codes are exact in BF16, (code - 128) / 64; the keys' scales are applied
// to the scores, the values' to P.
template <int kDim, bool kCodes, bool kWide>
__global__ void __launch_bounds__(kThreads, (Layout<kDim, kCodes>::kCtas))
paged_attention_kernel(const AttentionParams p) {
  using L = Layout<kDim, kCodes>;
  constexpr int kTiles = L::kStep / 8;      // score tiles of eight tokens
  constexpr int kOut = kDim / 8;            // output tiles of eight dims
  constexpr int kChunks = kDim / 16;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float warp_max[kWarps][16], warp_sum[kWarps][16];
  __shared__ int64_t found[2];
  __shared__ int64_t scan[kWarps];
  __shared__ int32_t last_arrival;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q4 = lane & 3, r8 = lane >> 2;
  ptx::grid_dependency_wait();

  const int32_t rows_per_sequence = p.cache.heads * p.head_blocks;
  // Tokens of sequence b that are read, and the first of them.
  auto extent = [&](int32_t b, int32_t& begin) {
    int32_t length = __ldg(p.lengths + b);
    length = max(0, min(length, p.capacity));
    begin = p.window > 0 && length > p.window ? length - p.window : 0;
    return length - begin;
  };
  auto units_of = [&](int32_t b) {
    int32_t begin;
    return (extent(b, begin) + L::kUnit - 1) / L::kUnit;
  };

  // Where the shares begin: a scan over the sequences' units.
  const int32_t per_thread = (p.batch + kThreads - 1) / kThreads;
  const int32_t b0 = min(p.batch, static_cast<int32_t>(threadIdx.x) * per_thread), b1 = min(p.batch, b0 + per_thread);
  int64_t mine = 0;
  for (int32_t b = b0; b < b1; ++b) {
    const int32_t units = units_of(b);
    mine += static_cast<int64_t>(units) * rows_per_sequence;
    if (blockIdx.x == 0 && p.status != nullptr && __ldg(p.lengths + b) > p.capacity) atomicOr(p.status, kStatusIndex);
  }
  // Sequences with nothing to attend to.
  for (int32_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (units_of(b) != 0) continue;
    const int64_t row = static_cast<int64_t>(b) * p.heads;
    for (int32_t i = threadIdx.x; i < p.heads * (kDim / 8); i += kThreads) {
      *reinterpret_cast<uint4*>(p.out + row * kDim + 8 * static_cast<int64_t>(i)) = make_uint4(0, 0, 0, 0);
    }
    if (p.lse != nullptr) {
      for (int32_t h = threadIdx.x; h < p.heads; h += kThreads) p.lse[row + h] = -INFINITY;
    }
  }
  int64_t inclusive = mine;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t below = __shfl_up_sync(0xffffffffu, inclusive, d);
    if (lane >= d) inclusive += below;
  }
  if (lane == 31) scan[warp] = inclusive;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) inclusive += scan[w];
    total += scan[w];
  }
  const int64_t share = max((total + gridDim.x - 1) / static_cast<int64_t>(gridDim.x), static_cast<int64_t>(1));
  int64_t unit = blockIdx.x * share;
  const int64_t unit_end = min(unit + share, total);
  if (unit >= unit_end) return;
  if (unit >= inclusive - mine && unit < inclusive) {
    int64_t base = inclusive - mine;
    for (int32_t b = b0; b < b1; ++b) {
      const int64_t units = static_cast<int64_t>(units_of(b)) * rows_per_sequence;
      if (unit < base + units) {
        found[0] = b;
        found[1] = base;
        break;
      }
      base += units;
    }
  }
  __syncthreads();
  int32_t b = static_cast<int32_t>(found[0]);
  int64_t base = found[1];  // of sequence b

  uint8_t* const ring = smem + warp * (L::kStages * L::kStageBytes);
  const uint32_t ring_addr = ptx::smem_u32(ring);

  while (unit < unit_end) {
    int32_t begin;
    int32_t tokens = extent(b, begin);
    int32_t units = (tokens + L::kUnit - 1) / L::kUnit;
    while (unit >= base + static_cast<int64_t>(units) * rows_per_sequence) {  // on to the next sequence with tokens
      base += static_cast<int64_t>(units) * rows_per_sequence;
      ++b;
      tokens = extent(b, begin);
      units = (tokens + L::kUnit - 1) / L::kUnit;
    }
    const int32_t row = static_cast<int32_t>((unit - base) / units);
    const int64_t row_first = base + static_cast<int64_t>(row) * units;
    const int32_t first_unit = static_cast<int32_t>(unit - row_first);
    const int32_t steps = static_cast<int32_t>(min(unit_end, row_first + units) - unit);
    const int32_t kv_head = row / p.head_blocks;
    const int32_t head_block = row % p.head_blocks;
    const int32_t heads = min(p.group - head_block * 16, 16);
    const int32_t head0 = kv_head * p.group + head_block * 16;
    const int32_t end = begin + tokens;

    const int32_t* table = p.tables + static_cast<int64_t>(b) * p.table_stride;
    const uint8_t* k_head = p.cache.k + kv_head * p.cache.head;
    const uint8_t* v_head = p.cache.v + kv_head * p.cache.head;

    // The page of each of a step's tokens, a lane's own, looked up a step before it is needed; place -1:
    // no token.
    int32_t ref_page = 0, ref_place = -1;
    auto look_up = [&](int32_t step) {
      const int32_t token = begin + (first_unit + step) * L::kUnit + warp * L::kStep + lane % L::kStep;
      ref_place = -1;
      if (step < steps && token < end) {
        const uint32_t index = p.cache.page_size.div(token);
        ref_place = token - index * p.cache.page_size.d;
        ref_page = __ldg(table + index);
      }
    };
    auto load = [&](int32_t step) {
      if (step >= steps) return;
      const uint32_t stage = ring_addr + (step % L::kStages) * L::kStageBytes;
      if (static_cast<uint32_t>(ref_page) >= static_cast<uint32_t>(p.cache.num_pages) && ref_place >= 0) {
        if (p.status != nullptr) atomicOr(p.status, kStatusIndex);
        ref_place = -1;
      }
      constexpr int kPieces = L::kRow / 16;
      static_assert(L::kStep * kPieces % 32 == 0, "whole warps");
#pragma unroll
      for (int i = 0; i < L::kStep * kPieces / 32; ++i) {
        const int piece = i * 32 + lane, at = piece / kPieces, column = piece % kPieces;
        const int32_t page = __shfl_sync(0xffffffffu, ref_page, at);
        const int32_t place = __shfl_sync(0xffffffffu, ref_place, at);
        const bool there = place >= 0;
        const int64_t offset = there ? page * p.cache.page + place * p.cache.token + column * 16 : 0;
        const uint32_t dst = stage + at * L::kPitch + column * 16;
        ptx::cp_async_16(dst, k_head + offset, there);
        ptx::cp_async_16(dst + L::kStep * L::kPitch, v_head + offset, there);
      }
      if constexpr (kCodes) {
        const bool there = ref_place >= 0;
        const int64_t offset = there ? ref_page * p.cache.scale_page + kv_head * p.cache.scale_head + ref_place * p.cache.scale_token : 0;
        const uint32_t dst = stage + 2 * L::kStep * L::kPitch + (lane % L::kStep) * 4;
        if (lane < L::kStep) {
          cp_async_4(dst, p.cache.k_scale + offset, there);
          cp_async_4(dst + L::kStep * 4, p.cache.v_scale + offset, there);
        }
      }
    };

    look_up(0);
#pragma unroll
    for (int s = 0; s < L::kStages - 1; ++s) {
      load(s);
      look_up(s + 1);
      ptx::cp_async_commit();
    }

    // The queries' fragments: rows r8 (and r8 + 8) of the block's heads; codes want the dims of a
    // 16-byte piece in the order in which its bytes lie in the lanes.
    uint32_t qf[kChunks][kWide ? 4 : 2];
    {
      const __nv_bfloat16* q = p.q + b * p.q_batch + static_cast<int64_t>(head0) * p.q_head;
#pragma unroll
      for (int c = 0; c < kChunks; ++c) {
#pragma unroll
        for (int i = 0; i < (kWide ? 4 : 2); ++i) {
          const int head = kWide ? r8 + 8 * (i & 1) : r8;
          const int part = kWide ? i >> 1 : i;
          const int dim = 16 * c + (kCodes ? 4 * q4 + 2 * part : 2 * q4 + 8 * part);
          qf[c][i] = head < heads ? __ldg(reinterpret_cast<const uint32_t*>(q + head * p.q_head + dim)) : 0u;
        }
      }
    }

    float out[kOut][4] = {};
    float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

    for (int32_t step = 0; step < steps; ++step) {
      ptx::cp_async_wait_group<L::kStages - 2>();
      __syncwarp();
      load(step + L::kStages - 1);
      look_up(step + L::kStages);
      ptx::cp_async_commit();

      const int32_t token0 = begin + (first_unit + step) * L::kUnit + warp * L::kStep;
      if (token0 >= end) continue;  // (the whole warp)
      const uint32_t stage = ring_addr + (step % L::kStages) * L::kStageBytes;
      float s[kTiles][4] = {};
#pragma unroll
      for (int j = 0; j < L::kStep / 16; ++j) {
        if constexpr (!kCodes) {
          const uint32_t at = stage + (j * 16 + (lane & 7) + ((lane >> 4) << 3)) * L::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t kf[4];
            ldmatrix_x4_at(at + c * 32, kf);
            const uint32_t a[4] = {qf[c][0], kWide ? qf[c][1] : 0u, qf[c][kWide ? 2 : 1], kWide ? qf[c][kWide ? 3 : 0] : 0u};
            ptx::mma_m16n8k16(s[2 * j], a, kf[0], kf[1]);
            ptx::mma_m16n8k16(s[2 * j + 1], a, kf[2], kf[3]);
          }
        } else {
          const uint32_t at = stage + (j * 16 + (lane & 7) + ((lane >> 4) << 3)) * L::kPitch + ((lane >> 3) & 1) * 16;
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t kf[4];
            ldmatrix_x4_at(at + c * 16, kf);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int cc = c + (i & 1);
              uint32_t lo, hi;
              codes_to_bf16<kCodes>(kf[i], 0x4140, 0x4342, lo, hi);
              const uint32_t a[4] = {qf[cc][0], kWide ? qf[cc][1] : 0u, qf[cc][kWide ? 2 : 1], kWide ? qf[cc][kWide ? 3 : 0] : 0u};
              ptx::mma_m16n8k16(s[2 * j + (i >> 1)], a, lo, hi);
            }
          }
        }
      }
      // Scores times the scale and log2(e); minus infinity behind the last token.
      float high[2] = {-INFINITY, -INFINITY};
      float value_scale[kCodes ? kTiles : 1][2];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        float f[2] = {p.scale, p.scale};
        if constexpr (kCodes) {
          const float2 ks = *reinterpret_cast<const float2*>(ring + (step % L::kStages) * L::kStageBytes + 2 * L::kStep * L::kPitch + (8 * t + 2 * q4) * 4);
          const float2 vs = *reinterpret_cast<const float2*>(ring + (step % L::kStages) * L::kStageBytes + 2 * L::kStep * L::kPitch + L::kStep * 4 + (8 * t + 2 * q4) * 4);
          f[0] *= 64.0f * ks.x;
          f[1] *= 64.0f * ks.y;
          value_scale[t][0] = 64.0f * vs.x;
          value_scale[t][1] = 64.0f * vs.y;
        }
        const bool seen[2] = {token0 + 8 * t + 2 * q4 < end, token0 + 8 * t + 2 * q4 + 1 < end};
#pragma unroll
        for (int i = 0; i < (kWide ? 4 : 2); ++i) {
          s[t][i] = seen[i & 1] ? s[t][i] * f[i & 1] : -INFINITY;
          high[i >> 1] = fmaxf(high[i >> 1], s[t][i]);
        }
      }
      bool rises = false;
#pragma unroll
      for (int i = 0; i < (kWide ? 2 : 1); ++i) {
        high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], 1));
        high[i] = fmaxf(high[i], __shfl_xor_sync(0xffffffffu, high[i], 2));
        rises |= high[i] > top[i];
      }
      if (__any_sync(0xffffffffu, rises)) {
        float factor[2] = {1.0f, 1.0f};
#pragma unroll
        for (int i = 0; i < (kWide ? 2 : 1); ++i) {
          const float next = fmaxf(top[i], high[i]);
          factor[i] = next == -INFINITY ? 1.0f : exp2_approx(top[i] - next);
          top[i] = next;
          sum[i] *= factor[i];
        }
        if constexpr (!kWide) factor[1] = factor[0];
#pragma unroll
        for (int t = 0; t < kOut; ++t) {
          out[t][0] *= factor[0];
          out[t][1] *= factor[0];
          out[t][2] *= factor[1];
          out[t][3] *= factor[1];
        }
      }
      const float from[2] = {top[0] == -INFINITY ? 0.0f : top[0], top[1] == -INFINITY ? 0.0f : top[1]};
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
#pragma unroll
        for (int i = 0; i < (kWide ? 4 : 2); ++i) {
          s[t][i] = exp2_approx(s[t][i] - from[i >> 1]);
          sum[i >> 1] += s[t][i];
          if constexpr (kCodes) s[t][i] *= value_scale[t][i & 1];
        }
      }
#pragma unroll
      for (int j = 0; j < L::kStep / 16; ++j) {
        // P of these 16 tokens in two parts
        uint32_t part[2][kWide ? 4 : 2];
#pragma unroll
        for (int i = 0; i < (kWide ? 4 : 2); ++i) {
          const float* pair = &s[2 * j + (kWide ? i >> 1 : i)][kWide ? 2 * (i & 1) : 0];
          part[0][i] = pack_bf16(pair[0], pair[1]);
          part[1][i] = pack_bf16(pair[0] - bf16_lo(part[0][i]), pair[1] - bf16_hi(part[0][i]));
        }
        auto multiply = [&](float (&o)[4], uint32_t v0, uint32_t v1) {
          if constexpr (kWide) {
            ptx::mma_m16n8k16(o, {part[0][0], part[0][1], part[0][2], part[0][3]}, v0, v1);
            ptx::mma_m16n8k16(o, {part[1][0], part[1][1], part[1][2], part[1][3]}, v0, v1);
          } else {
            ptx::mma_m16n8k16(o, {part[0][0], part[1][0], part[0][1], part[1][1]}, v0, v1);
          }
        };
        const uint32_t at = stage + L::kStep * L::kPitch + (j * 16 + (lane & 15)) * L::kPitch + (lane >> 4) * 16;
        if constexpr (!kCodes) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t vf[4];
            ldmatrix_x4_trans(at + c * 32, vf);
            multiply(out[2 * c], vf[0], vf[1]);
            multiply(out[2 * c + 1], vf[2], vf[3]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t vf[4];
            ldmatrix_x4_trans(at + c * 16, vf);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              uint32_t even[2], odd[2];
              codes_to_bf16<kCodes>(vf[2 * i], 0x4240, 0x4341, even[0], odd[0]);
              codes_to_bf16<kCodes>(vf[2 * i + 1], 0x4240, 0x4341, even[1], odd[1]);
              multiply(out[2 * (c + i)], even[0], even[1]);
              multiply(out[2 * (c + i) + 1], odd[0], odd[1]);
            }
          }
        }
      }
    }
    ptx::cp_async_wait_group<0>();

    // The warps' results into one: the ring is free.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      if (q4 == 0 && (kWide || i == 0)) {
        warp_max[warp][r8 + 8 * i] = top[i];
        warp_sum[warp][r8 + 8 * i] = sum[i];
      }
    }
    __syncthreads();
    constexpr int kRows = kWide ? 16 : 8;
    float* const shared_out = reinterpret_cast<float*>(smem);  // [kWarps][kRows][kDim]
#pragma unroll
    for (int i = 0; i < (kWide ? 2 : 1); ++i) {
      const int head = r8 + 8 * i;
      float most = warp_max[0][head];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) most = fmaxf(most, warp_max[w][head]);
      const float factor = most == -INFINITY ? 0.0f : exp2_approx(top[i] - most);
      float* to = shared_out + (warp * kRows + head) * kDim;
#pragma unroll
      for (int t = 0; t < kOut; ++t) {
        float v0 = out[t][2 * i], v1 = out[t][2 * i + 1];
        if constexpr (!kWide) v0 += out[t][2], v1 += out[t][3];
        // even and odd dims of a 16-byte piece of codes are two tiles
        const int d0 = kCodes ? 16 * (t / 2) + 4 * q4 + t % 2 : 8 * t + 2 * q4;
        to[d0] = v0 * factor;
        to[d0 + (kCodes ? 2 : 1)] = v1 * factor;
      }
    }
    __syncthreads();
    const int64_t first_cta = row_first / share, last_cta = (row_first + units - 1) / share;
    const bool whole = first_cta == last_cta;
    float* slot = p.partials + (2 * static_cast<int64_t>(blockIdx.x) + (blockIdx.x == first_cta ? 1 : 0)) * partial_floats(kDim);
    auto head_state = [&](int head, float& most, float& all) {
      most = warp_max[0][head];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) most = fmaxf(most, warp_max[w][head]);
      all = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) all += most == -INFINITY ? 0.0f * warp_sum[w][head] : warp_sum[w][head] * exp2_approx(warp_max[w][head] - most);
    };
    auto finish = [&](int head, int dim, const float (&v)[4], float all) {
      const float rate = all == 0.0f ? 0.0f : 1.0f / all;
      __nv_bfloat16* to = p.out + (static_cast<int64_t>(b) * p.heads + head0 + head) * kDim + dim;
      *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(v[0] * rate, v[1] * rate), pack_bf16(v[2] * rate, v[3] * rate));
    };
    auto finish_lse = [&](int head, float most, float all) {
      if (p.lse != nullptr) p.lse[static_cast<int64_t>(b) * p.heads + head0 + head] = all == 0.0f ? -INFINITY : (most + log2f(all)) * 0.693147180559945309f;
    };
    for (int i = threadIdx.x; i < heads * (kDim / 4); i += kThreads) {
      const int head = i / (kDim / 4), dim = i % (kDim / 4) * 4;
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float4 x = *reinterpret_cast<const float4*>(shared_out + (w * kRows + head) * kDim + dim);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
      }
      float most, all;
      head_state(head, most, all);
      if (whole) {
        finish(head, dim, v, all);
        if (dim == 0) finish_lse(head, most, all);
      } else {
        __stcg(reinterpret_cast<float4*>(slot + head * kDim + dim), make_float4(v[0], v[1], v[2], v[3]));
        if (dim == 0) {
          __stcg(slot + 16 * kDim + head, most);
          __stcg(slot + 16 * kDim + 16 + head, all);
        }
      }
    }
    if (!whole) {
      // The last CTA of the row to arrive joins the parts, in their order.  The count goes back to zero.
      __threadfence();
      __syncthreads();
      const int32_t parts = static_cast<int32_t>(last_cta - first_cta) + 1;
      if (threadIdx.x == 0) {
        const int32_t before = atomicAdd(p.locks + first_cta, 1);
        last_arrival = before == parts - 1;
        if (last_arrival) p.locks[first_cta] = 0;
      }
      __syncthreads();
      if (last_arrival) {
        __threadfence();
        auto part_at = [&](int32_t part) {
          return p.partials + (2 * (first_cta + part) + (part == 0 ? 1 : 0)) * partial_floats(kDim);
        };
        float* weights = reinterpret_cast<float*>(smem);  // [parts][16]
        {
          const int head = threadIdx.x >> 3, sub = threadIdx.x & 7;
          float most = -INFINITY;
          if (head < heads) {
            for (int32_t i = sub; i < parts; i += 8) most = fmaxf(most, __ldcg(part_at(i) + 16 * kDim + head));
          }
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
          float all = 0.0f;
          if (head < heads) {
            for (int32_t i = sub; i < parts; i += 8) {
              const float high = __ldcg(part_at(i) + 16 * kDim + head);
              const float weight = most == -INFINITY ? 0.0f : exp2_approx(high - most);
              weights[i * 16 + head] = weight;
              all += weight * __ldcg(part_at(i) + 16 * kDim + 16 + head);
            }
          }
#pragma unroll
          for (int d = 1; d < 8; d <<= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
          if (sub == 0 && head < heads) {
            warp_sum[0][head] = all;
            finish_lse(head, most, all);
          }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < heads * (kDim / 4); i += kThreads) {
          const int head = i / (kDim / 4), dim = i % (kDim / 4) * 4;
          float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
          for (int32_t part = 0; part < parts; ++part) {
            const float weight = weights[part * 16 + head];
            const float4 x = __ldcg(reinterpret_cast<const float4*>(part_at(part) + head * kDim + dim));
            v[0] = fmaf(weight, x.x, v[0]);
            v[1] = fmaf(weight, x.y, v[1]);
            v[2] = fmaf(weight, x.z, v[2]);
            v[3] = fmaf(weight, x.w, v[3]);
          }
          finish(head, dim, v, warp_sum[0][head]);
        }
      }
    }
    __syncthreads();  // the shared memory is free again
    unit += steps;
  }
}

struct Variant {
  void (*kernel)(AttentionParams);
  int smem, unit, ctas;
};

template <int kDim, bool kCodes, bool kWide>
Variant variant() {
  using L = Layout<kDim, kCodes>;
  return {paged_attention_kernel<kDim, kCodes, kWide>, L::kSmem, L::kUnit, L::kCtas};
}

template <int kDim>
Variant variant_of(bool codes, bool wide) {
  if (codes) return wide ? variant<kDim, true, true>() : variant<kDim, true, false>();
  return wide ? variant<kDim, false, true>() : variant<kDim, false, false>();
}

bool variant_for(int64_t dim, bool codes, bool wide, Variant* out) {
  switch (dim) {
    case 64: *out = variant_of<64>(codes, wide); return true;
    case 96: *out = variant_of<96>(codes, wide); return true;
    case 128: *out = variant_of<128>(codes, wide); return true;
    case 192: *out = variant_of<192>(codes, wide); return true;
    case 256: *out = variant_of<256>(codes, wide); return true;
  }
  return false;
}

// Allows a kernel its shared memory, once per device.
int allow_smem(const Variant& v, int64_t dim, bool codes, bool wide, int device) {
  static std::mutex mutex;
  static bool done[64][5][2][2];
  std::lock_guard<std::mutex> guard(mutex);
  bool& known = done[device & 63][dim == 64 ? 0 : dim == 96 ? 1 : dim == 128 ? 2 : dim == 192 ? 3 : 4][codes][wide];
  if (known) return kOk;
  CHORD_CUDA(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem));
  known = true;
  return kOk;
}

}  // namespace
}  // namespace chord

extern "C" {

int chord_b200_paged_attention_lock_words(void) {
  chord::DeviceInfo device;
  if (chord::current_device_info(&device)) return -1;
  return device.sm_count * chord::kMaxCtasPerSm;
}

int64_t chord_b200_paged_attention_workspace_bytes(int64_t head_dim) {
  chord::DeviceInfo device;
  if (chord::current_device_info(&device)) return -1;
  if (head_dim <= 0 || head_dim > 256) return chord::fail(chord::kInvalidArgument, "head_dim out of range"), -1;
  return 2ll * device.sm_count * chord::kMaxCtasPerSm * chord::partial_floats(static_cast<int>(head_dim)) * 4;
}

int chord_b200_paged_attention(const void* q, int64_t q_batch, int64_t q_head, const chord_b200_kv_cache* cache,
                               const int32_t* tables, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
                               void* out, float* lse, int32_t* locks, int64_t num_locks, void* workspace,
                               int64_t workspace_bytes, int32_t* status, int64_t batch, int64_t heads, int64_t window,
                               double scale, void* stream) {
  using namespace chord;
  AttentionParams p = {};
  if (int rc = make_cache(cache, &p.cache)) return rc;
  CHORD_REQUIRE(batch >= 0 && batch < (1ll << 31), "batch out of range");
  if (batch == 0) return kOk;
  CHORD_REQUIRE(q != nullptr && tables != nullptr && lengths != nullptr && out != nullptr && locks != nullptr &&
                    workspace != nullptr,
                "null pointer");
  CHORD_REQUIRE(heads > 0 && heads <= 65535 && heads % cache->heads == 0,
                "the number of query heads (%lld) must be a multiple of the cache's (%lld)",
                static_cast<long long>(heads), static_cast<long long>(cache->heads));
  CHORD_REQUIRE(q_batch >= 0 && q_head >= 0 && q_batch % 8 == 0 && q_head % 8 == 0 &&
                    ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) |
                      reinterpret_cast<uintptr_t>(workspace)) & 15u) == 0,
                "q's rows, out and the workspace must lie on 16-byte boundaries");
  CHORD_REQUIRE(max_pages > 0 && table_stride >= 0 && max_pages < (1ll << 31), "a block table has a page or more");
  CHORD_REQUIRE(window >= 0 && window < (1ll << 31), "window out of range");
  CHORD_REQUIRE(scale == scale && scale - scale == 0.0, "scale must be finite");
  const bool codes = cache->k_scale != nullptr;
  const int64_t group = heads / cache->heads;
  const bool wide = group > 8;
  Variant v;
  CHORD_REQUIRE(variant_for(cache->head_dim, codes, wide, &v), "head_dim must be 64, 96, 128, 192 or 256, got %lld",
                static_cast<long long>(cache->head_dim));
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  if (int rc = allow_smem(v, cache->head_dim, codes, wide, device.device)) return rc;
  const int64_t head_blocks = (group + 15) / 16;
  // No more CTAs than there can be units of work.
  // (token numbers, those of the steps loaded ahead too, fit 32 bits)
  int64_t capacity = max_pages * cache->page_size;
  if (capacity > (1ll << 31) - 65536) capacity = (1ll << 31) - 65536;
  const int64_t longest = window > 0 && window < capacity ? window : capacity;
  const int64_t most = batch * cache->heads * head_blocks * ((longest + v.unit - 1) / v.unit);
  int64_t ctas = static_cast<int64_t>(device.sm_count) * v.ctas;
  if (ctas > most) ctas = most;
  const int64_t need = 2 * ctas * partial_floats(static_cast<int>(cache->head_dim)) * 4;
  CHORD_REQUIRE(num_locks >= ctas && ctas <= kMaxParts, "locks has %lld lock words, this launch needs %lld",
                static_cast<long long>(num_locks), static_cast<long long>(ctas));
  CHORD_REQUIRE(workspace_bytes >= need, "the workspace has %lld bytes, this launch needs %lld",
                static_cast<long long>(workspace_bytes), static_cast<long long>(need));
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_batch = q_batch;
  p.q_head = q_head;
  p.tables = tables;
  p.table_stride = table_stride;
  p.capacity = static_cast<int32_t>(capacity);
  p.lengths = lengths;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.lse = lse;
  p.partials = static_cast<float*>(workspace);
  p.locks = locks;
  p.status = status;
  p.batch = static_cast<int32_t>(batch);
  p.heads = static_cast<int32_t>(heads);
  p.group = static_cast<int32_t>(group);
  p.head_blocks = static_cast<int32_t>(head_blocks);
  p.window = static_cast<int32_t>(window);
  p.scale = static_cast<float>(scale * 1.4426950408889634074);
  OptionsReadLock guard(options_mutex());
  CHORD_CUDA(launch_kernel(v.kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), v.smem,
                           static_cast<cudaStream_t>(stream), options().pdl != 0, p));
  return kOk;
}

}  // extern "C"
