// What each token of the cache got of a new token's attention, and eviction by what has been gathered of it.
#include <mutex>
#include <set>
#include <utility>

#include "../../include/chord_b200.h"
#include "attention.h"
#include "common.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {
namespace {

constexpr float kLog2E = 1.44269504088896341f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------- weights --

struct WeighParams {
  Cache cache;
  const __nv_bfloat16* q;  // [batch, heads, dim]
  int64_t q_batch, q_head;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;
  const float* lse;      // [batch, heads]
  const float* slopes;   // [heads] or null
  float* weights;        // [batch, kv_heads, width]
  int64_t weight_batch, weight_head;
  int32_t* status;
  float scale, cap, over_cap;  // as of paged_attention
  int32_t heads, group, capacity, width, window, add;
  int32_t runs;    // of 64 tokens for a warp
  bool in_a_row;   // 16 tokens from a multiple of 16 lie one after another
};

constexpr int kWeighWarps = 4;
constexpr int kWeighRun = 64;  // tokens that a warp looks up at once

// What a lane has of a row: words (two elements) in the order of its loads.  A product's sum does not depend on the order of
// its terms, so a lane's words of a key and of a query, wherever they lie, stand for the columns that the instruction wants
// there, as long as they are the same dims.  Loads are of 16 bytes, the last one of 8 where codes of 96 dims leave no more.
// A warp has a ring of stages of 32 tokens, of wide rows 16, some 12 KB on their way or in use.
template <int kDim, bool kCodes>
struct WeighRow {
  static constexpr int kLoadDims = kCodes ? 64 : 32;  // of the four lanes of a row together
  static constexpr int kLoads = kDim / kLoadDims, kRest = kDim % kLoadDims / 32;
  static constexpr int kWords = kDim / 8;
  static constexpr int kBytes = kDim * (kCodes ? 1 : 2), kPieces = kBytes / 16;
  static constexpr int kGroups = kBytes <= 256 ? 2 : 1, kTokens = 16 * kGroups;
  static constexpr int kStage = kTokens * kBytes + (kCodes ? kTokens * 4 : 0);  // with the rows' scales
  static constexpr int kStages = 12 * 1024 / kStage < 2 ? 2 : 12 * 1024 / kStage > 6 ? 6 : 12 * 1024 / kStage;
  static constexpr int kSmem = kWeighWarps * kStages * kStage;
  // Rows of a multiple of 128 bytes: the lanes of an odd one read the other half of the banks.
  static __device__ __forceinline__ int place(int row, int piece) { return row * kBytes + (kBytes % 128 == 0 ? piece ^ (row & 1) << 2 : piece) * 16; }
};

// A warp takes p.runs times 64 tokens of one key-value head, 16 at a time as the rows of mma.m16n8k16, 8 of the heads that
// share it as columns.  The weights of a token's heads are summed in one order, so the same inputs give the same bits.
// Bounded by memory and by what is on its way (with fragments straight from memory into registers, three warps of a
// scheduler had 2 to 4 KB each on their way: 131072 tokens in 8 bits 50 us).  64 ragged sequences of up to 8192 tokens, 64 + 8 heads of
// 128 in BF16: 111 us, 96 % of the copy rate; 131072 tokens in 8 bits 31, 69 %, the issue slots 59 % busy.
template <int kDim, bool kCodes>
__global__ void __launch_bounds__(kWeighWarps * 32) attention_weights_kernel(const WeighParams p) {
  using R = WeighRow<kDim, kCodes>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q4 = lane & 3, r8 = lane >> 2;
  ptx::grid_dependency_wait();
  const int32_t b = blockIdx.z, kv_head = blockIdx.y;
  const int32_t given = load_arg(p.lengths + b), length = max(0, min(given, min(p.capacity, p.width)));
  if (given > min(p.capacity, p.width) && threadIdx.x == 0 && blockIdx.x == 0 && p.status != nullptr) atomicOr(p.status, kStatusIndex);
  const int32_t low = p.window > 0 ? max(0, length - p.window) : 0;
  const int32_t first = (blockIdx.x * kWeighWarps + warp) * (kWeighRun * p.runs);
  const int32_t last = min(first + kWeighRun * p.runs, p.width);
  float* const row = p.weights + b * p.weight_batch + kv_head * p.weight_head;
  if (first >= length || last <= low) {
    if (!p.add) {
      for (int32_t t = first + lane; t < last; t += 32) row[t] = 0.0f;
    }
    return;
  }
  uint8_t* const ring = smem + warp * (R::kStages * R::kStage);
  const uint32_t ring_at = ptx::smem_u32(ring);
  const int32_t* const table = p.tables + b * p.table_stride;

  // The loads, ahead of the products.  Pages are looked up for 64 tokens, two to a lane, one run before they are needed.
  int32_t page[2], place[2], ahead = first;
  int64_t offset[2] = {-1, -1}, scale_offset[2] = {0, 0};
  int load_stage = 0;
  auto look_up = [&](int32_t token0) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int32_t token = token0 + 32 * i + lane;
      place[i] = -1;
      if (token >= low && token < length && token < last) {
        const uint32_t index = p.cache.page_size.div(token);
        place[i] = token - index * p.cache.page_size.d;
        page[i] = load_arg(table + index);
      }
    }
  };
  auto load = [&]() {  // a stage's tokens from `ahead`
    if (ahead < last) {
      const int32_t inside = (ahead - first) % kWeighRun;
      if (inside == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          offset[i] = -1;
          if (place[i] >= 0) {
            if (static_cast<uint32_t>(page[i]) < static_cast<uint32_t>(p.cache.num_pages)) {
              offset[i] = page[i] * p.cache.page + place[i] * p.cache.token + kv_head * p.cache.head;
              if constexpr (kCodes) scale_offset[i] = page[i] * p.cache.scale_page + place[i] * p.cache.scale_token + kv_head * p.cache.scale_head;
            } else if (p.status != nullptr) {
              atomicOr(p.status, kStatusIndex);
            }
          }
        }
        look_up(ahead + kWeighRun);
      }
      // (a lane's token of the 32 that hold the stage's, and where these begin)
      const int64_t from = inside < 32 ? offset[0] : offset[1];
      const int32_t lane0 = R::kGroups == 2 ? 0 : inside % 32;
      const uint32_t to = ring_at + load_stage * R::kStage;
      const uint32_t there = __ballot_sync(0xffffffffu, from >= 0);
#pragma unroll
      for (int g = 0; g < R::kGroups; ++g) {
        const int32_t lane_of = lane0 + 16 * g;
        if (p.in_a_row && (there >> lane_of & 0xFFFFu) == 0xFFFFu) {
          // all there, one after another: a third of the instructions
          const uint8_t* const at0 = p.cache.k + __shfl_sync(0xffffffffu, from, lane_of) + lane * 16;
#pragma unroll
          for (int i = 0; i < R::kPieces / 2; ++i) {
            const int at = i * 32 + lane;
            ptx::cp_async_16(to + R::place(16 * g + at / R::kPieces, at % R::kPieces), at0 + i * 512, true);
          }
        } else {
#pragma unroll
          for (int i = 0; i < R::kPieces / 2; ++i) {
            const int at = i * 32 + lane, of = at / R::kPieces, piece = at % R::kPieces;
            const int64_t o = __shfl_sync(0xffffffffu, from, lane_of + of);
            ptx::cp_async_16(to + R::place(16 * g + of, piece), p.cache.k + (o < 0 ? 0 : o + piece * 16), o >= 0);
          }
        }
      }
      if constexpr (kCodes) {
        if (lane >= lane0 && lane < lane0 + R::kTokens) {
          const int64_t o = inside < 32 ? scale_offset[0] : scale_offset[1];
          cp_async_4(to + R::kTokens * R::kBytes + (lane - lane0) * 4, p.cache.k_scale + (from < 0 ? 0 : o), from >= 0);
        }
        __syncwarp();
      }
      load_stage = load_stage + 1 == R::kStages ? 0 : load_stage + 1;
      ahead += R::kTokens;
    }
    ptx::cp_async_commit();
  };
  look_up(first);
#pragma unroll
  for (int i = 0; i < R::kStages - 1; ++i) load();

  // Queries of the first eight heads (often all): head r8's.  Of the columns' heads, 2 q4 and the next: what the exponent
  // starts from, and the slope.
  const int64_t head0 = static_cast<int64_t>(kv_head) * p.group;
  uint32_t qw[R::kWords];
  float base[2], slope[2];
  auto load_heads = [&](int32_t h0) {
    const bool there = h0 + r8 < p.group;
    const __nv_bfloat16* const q = p.q + b * p.q_batch + (head0 + h0 + (there ? r8 : 0)) * p.q_head;
    constexpr int kStep = kCodes ? 8 : 4;  // words of a load
#pragma unroll
    for (int w = 0; w < R::kWords; w += 4) {
      const int of = w / kStep;
      const int dim = of < R::kLoads ? of * R::kLoadDims + q4 * (2 * kStep) + 2 * (w % kStep) : R::kLoads * R::kLoadDims + q4 * 8;
      const uint4 v = there ? load_once(q + dim) : make_uint4(0, 0, 0, 0);
      qw[w] = v.x, qw[w + 1] = v.y, qw[w + 2] = v.z, qw[w + 3] = v.w;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool here = h0 + 2 * q4 + i < p.group;
      const float lse = here ? load_arg(p.lse + static_cast<int64_t>(b) * p.heads + head0 + h0 + 2 * q4 + i) : -INFINITY;
      base[i] = lse == -INFINITY ? -INFINITY : -lse * kLog2E;  // (nothing was seen: no weight)
      slope[i] = here && p.slopes != nullptr ? load_arg(p.slopes + head0 + h0 + 2 * q4 + i) * kLog2E : 0.0f;
    }
  };
  load_heads(0);

  int stage = 0;
#pragma unroll 1
  for (int32_t token0 = first; token0 < last; token0 += R::kTokens) {
    ptx::cp_async_wait_group<R::kStages - 2>();
    __syncwarp();
    load();
    const uint8_t* const keys = ring + stage * R::kStage;
    stage = stage + 1 == R::kStages ? 0 : stage + 1;
    float factor[R::kGroups][2];  // a lane's tokens are r8 and r8 + 8 of each 16
#pragma unroll
    for (int g = 0; g < R::kGroups; ++g) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        factor[g][i] = p.scale;
        if constexpr (kCodes) factor[g][i] *= 64.0f * reinterpret_cast<const float*>(keys + R::kTokens * R::kBytes)[16 * g + 8 * i + r8];
      }
    }
    float sum[R::kGroups][2] = {};
#pragma unroll 1
    for (int32_t h0 = 0; h0 < p.group; h0 += 8) {
      if (p.group > 8) load_heads(h0);
#pragma unroll
      for (int g = 0; g < R::kGroups; ++g) {
        float s2[2][4] = {};  // (two sums, so that a product does not wait for the one before it)
        auto multiply = [&](uint32_t a, uint32_t b2, uint32_t c, uint32_t d, int word) {  // words of the two rows
          const uint32_t fragment[4] = {a, b2, c, d};
          ptx::mma_m16n8k16(s2[word / 2 % 2], fragment, qw[word], qw[word + 1]);
        };
        auto two = [](uint32_t four, uint32_t select) {  // codes as (code - 128) / 64
          constexpr uint32_t kOffset = 0xC000C000u;
          return bf16x2_fma(__byte_perm(four, 0, select), kTwo127, kOffset);
        };
#pragma unroll
        for (int c = 0; c < R::kLoads + R::kRest; ++c) {
          uint32_t a[4], b2[4];
          if (c < R::kLoads) {
            const uint4 x = *reinterpret_cast<const uint4*>(keys + R::place(16 * g + r8, 4 * c + q4));
            const uint4 y = *reinterpret_cast<const uint4*>(keys + R::place(16 * g + r8 + 8, 4 * c + q4));
            a[0] = x.x, a[1] = x.y, a[2] = x.z, a[3] = x.w;
            b2[0] = y.x, b2[1] = y.y, b2[2] = y.z, b2[3] = y.w;
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(keys + R::place(16 * g + r8, 4 * c) + 8 * q4);
            const uint2 y = *reinterpret_cast<const uint2*>(keys + R::place(16 * g + r8 + 8, 4 * c) + 8 * q4);
            a[0] = x.x, a[1] = x.y, b2[0] = y.x, b2[1] = y.y;
          }
          if constexpr (kCodes) {
#pragma unroll
            for (int i = 0; i < (c < R::kLoads ? 4 : 2); ++i) {
              multiply(two(a[i], 0x4140), two(b2[i], 0x4140), two(a[i], 0x4342), two(b2[i], 0x4342), 8 * c + 2 * i);
            }
          } else {
            multiply(a[0], b2[0], a[1], b2[1], 4 * c);
            multiply(a[2], b2[2], a[3], b2[3], 4 * c + 2);
          }
        }
        float x[2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int k = 0; k < 2; ++k) x[i][k] = (s2[0][2 * i + k] + s2[1][2 * i + k]) * factor[g][i];
        }
        if (p.cap > 0.0f) {
#pragma unroll
          for (int i = 0; i < 2; ++i) cap_pair(x[i][0], x[i][1], p.over_cap, p.cap);
        }
        if (p.slopes != nullptr) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float behind = static_cast<float>(length - 1 - (token0 + 16 * g + 8 * i + r8));
#pragma unroll
            for (int k = 0; k < 2; ++k) x[i][k] = fmaf(-slope[k], behind, x[i][k]);
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // (no weight where the head's sum is nothing, whatever the score)
          const float first_of = exp2_approx(x[i][0] + base[0]), second = exp2_approx(x[i][1] + base[1]);
          sum[g][i] += (base[0] == -INFINITY ? 0.0f : first_of) + (base[1] == -INFINITY ? 0.0f : second);
        }
      }
    }
    // Over the four lanes of a row's heads: each ends with the sum of one of the row's tokens (of one group, two do).
    float mine;
    int32_t place_of;
    if constexpr (R::kGroups == 2) {
      const bool odd = q4 & 1, upper = q4 & 2;
      const float a = odd ? sum[0][1] : sum[0][0], b2 = odd ? sum[1][1] : sum[1][0];
      const float a2 = a + __shfl_xor_sync(0xffffffffu, odd ? sum[0][0] : sum[0][1], 1);
      const float b3 = b2 + __shfl_xor_sync(0xffffffffu, odd ? sum[1][0] : sum[1][1], 1);
      mine = (upper ? b3 : a2) + __shfl_xor_sync(0xffffffffu, upper ? a2 : b3, 2);
      place_of = 16 * (q4 >> 1) + 8 * (q4 & 1) + r8;
    } else {
      const bool odd = q4 & 1;
      mine = (odd ? sum[0][1] : sum[0][0]) + __shfl_xor_sync(0xffffffffu, odd ? sum[0][0] : sum[0][1], 1);
      mine += __shfl_xor_sync(0xffffffffu, mine, 2);
      place_of = 8 * (q4 & 1) + r8;
    }
    const int32_t token = token0 + place_of;
    if (token < last && (R::kGroups == 2 || q4 < 2)) {
      const bool seen = token >= low && token < length;
      if (!p.add) {
        row[token] = seen ? mine : 0.0f;
      } else if (seen) {
        row[token] += mine;
      }
    }
  }
}

struct WeighKernel {
  void (*kernel)(WeighParams);
  int smem;
};

template <int kDim, bool kCodes>
WeighKernel weigh_variant() { return {attention_weights_kernel<kDim, kCodes>, WeighRow<kDim, kCodes>::kSmem}; }

template <bool kCodes>
WeighKernel weigh_kernel(int64_t dim) {
  switch (dim) {
    case 64: return weigh_variant<64, kCodes>();
    case 96: return weigh_variant<96, kCodes>();
    case 128: return weigh_variant<128, kCodes>();
    case 192: return weigh_variant<192, kCodes>();
    case 256: return weigh_variant<256, kCodes>();
  }
  return {nullptr, 0};
}

// Allows a kernel its shared memory, once per device.
int allow_smem(const void* kernel, int smem, int device) {
  static std::mutex mutex;
  static std::set<std::pair<int, const void*>> done;
  std::lock_guard<std::mutex> guard(mutex);
  if (done.count({device, kernel}) != 0) return kOk;
  CHORD_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  done.insert({device, kernel});
  return kOk;
}

// ------------------------------------------------------------------ eviction --

struct EvictParams {
  Cache cache;
  const int32_t* tables;
  const int32_t* new_tables;
  int64_t table_stride, new_stride;
  const int32_t* lengths;
  const float* weights;  // [batch, kv_heads, width]
  int64_t weight_batch, weight_head;
  int32_t* new_lengths;  // [batch]
  float* new_weights;    // [batch, kv_heads, new_width], contiguous
  int32_t* kept;         // [batch, kv_heads, places], as many as can be kept
  int32_t* status;
  int32_t capacity, new_capacity, width, new_width, keep, places, first, recent, row_bytes;
};

constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32;
constexpr int kBins = 2048;
// Order of weights as that of whole numbers: zeros alike, NaN above all.
__device__ __forceinline__ uint32_t rank_of(float w) {
  if (w != w) return 0xFFFFFFFFu;
  const uint32_t bits = __float_as_uint(w + 0.0f);
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

// The wanted-th largest of the counted ranks by their next digit: two bins to a thread, from the top.  Takes off `wanted`
// what lies in higher bins.
__device__ __forceinline__ uint32_t find_bin(const uint32_t* bins, uint32_t* of_warps, uint32_t* found, uint32_t& wanted) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int top = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
  const uint32_t high = bins[top], lower = bins[top - 1];
  uint32_t upto = high + lower;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const uint32_t below = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += below;
  }
  if (lane == 31) of_warps[warp] = upto;
  __syncthreads();
  const uint32_t before = upto - high - lower + __reduce_add_sync(0xffffffffu, lane < warp ? of_warps[lane] : 0);
  if (before < wanted && wanted <= before + high) {
    found[0] = top;
    found[1] = before;
  } else if (before + high < wanted && wanted <= before + high + lower) {
    found[0] = top - 1;
    found[1] = before + high;
  }
  __syncthreads();
  wanted -= found[1];
  return found[0];
}

// One CTA for a sequence's key-value head: the smallest weight that is kept, found by its digits (11, 11 and 10 bits),
// then the kept tokens in order.  Counts do not depend on the order in which they are counted.  A thread has up to kItems
// neighbours' weights in registers, which come coalesced, by way of shared memory; with kItems zero, for longer sequences,
// they are read from memory each time and a warp has a run of them.  Bounded by the latency of its steps: 128 CTAs of 16384
// weights 12 us (with the runs' ballots from shared memory 20).
template <int kItems>
__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictParams p) {
  extern __shared__ float held[];
  __shared__ uint32_t bins[3][kBins];
  __shared__ uint32_t of_warps[3][kSelectWarps];
  __shared__ uint32_t found[3][2];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < 3 * kBins; i += kSelectThreads) bins[0][i] = 0;
  ptx::grid_dependency_wait();
  const int32_t b = blockIdx.y, head = blockIdx.x;
  const int32_t given = load_arg(p.lengths + b), limit = min(p.capacity, p.width), length = max(0, min(given, limit));
  const int32_t count = min(length, p.keep);
  if (threadIdx.x == 0 && head == 0) {
    p.new_lengths[b] = count;
    if (given > limit && p.status != nullptr) atomicOr(p.status, kStatusIndex);
  }
  const float* const weights = p.weights + b * p.weight_batch + head * p.weight_head;
  const int64_t row = static_cast<int64_t>(b) * gridDim.x + head;
  float* const out = p.new_weights + row * p.new_width;
  int32_t* const kept = p.kept + row * p.places;
  if (length <= p.keep) {
    for (int32_t i = threadIdx.x; i < p.new_width; i += kSelectThreads) {
      if (i < count) kept[i] = i;
      out[i] = i < count ? load_arg(weights + i) : 0.0f;
    }
    return;
  }
  const int32_t begin = p.first, end = length - p.recent;
  const uint32_t between = end - begin;           // of these the largest
  uint32_t wanted = p.keep - p.first - p.recent;  // are kept, so many
  const bool any = wanted > 0;
  constexpr int kShift[3] = {21, 10, 0};
  auto digit_of = [&](uint32_t rank, int digit) { return rank >> kShift[digit] & (digit == 2 ? 0x3FFu : 0x7FFu); };
  uint32_t prefix = 0;

  if constexpr (kItems != 0) {
    static_assert(kItems * kSelectThreads <= 65536, "places in 16 bits");
    uint16_t* const places = reinterpret_cast<uint16_t*>(held + kItems * (kSelectThreads / 32 * 33));  // the kept ones'
    auto padded = [](int32_t i) { return i + (i >> 5); };  // (threads with 8, 16 or 32 neighbours each share no bank)
    constexpr int kAhead = kItems < 16 ? kItems : 16;      // loads of a thread on their way
#pragma unroll 1
    for (int32_t i0 = threadIdx.x; i0 < length; i0 += kAhead * kSelectThreads) {
      float w[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) w[k] = i0 + k * kSelectThreads < length ? load_arg(weights + i0 + k * kSelectThreads) : 0.0f;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (i0 + k * kSelectThreads < length) held[padded(i0 + k * kSelectThreads)] = w[k];
      }
    }
    for (int32_t i = count + threadIdx.x; i < p.new_width; i += kSelectThreads) out[i] = 0.0f;
    __syncthreads();
    const int32_t items = (length + kSelectThreads - 1) / kSelectThreads, mine = threadIdx.x * items;
    uint32_t rank[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      rank[k] = 0;
      if (k < items && mine + k < length) rank[k] = rank_of(held[padded(mine + k)]);
    }
    // The thread's items as bits: those there are, and those of which the largest are kept.
    auto bits_below = [&](int32_t i) {
      const int32_t n = max(0, min(i - mine, items));
      return n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1;
    };
    const uint32_t there = bits_below(length), inside = bits_below(end) & ~bits_below(begin);
    if (any) {
#pragma unroll
      for (int digit = 0; digit < 3; ++digit) {
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
          if ((inside >> k & 1) != 0 && (digit == 0 || rank[k] >> kShift[digit == 0 ? 0 : digit - 1] == prefix)) {
            atomicAdd(&bins[digit][digit_of(rank[k], digit)], 1u);
          }
        }
        __syncthreads();
        prefix = prefix << (digit == 2 ? 10 : 11) | find_bin(bins[digit], of_warps[digit], found[digit], wanted);
      }
    }
    // In order: `wanted` of those equal to the least, all above it, the first and the recent ones.
    uint32_t above = 0, level = 0;
    if (any) {
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        above |= static_cast<uint32_t>(rank[k] > prefix) << k;
        level |= static_cast<uint32_t>(rank[k] == prefix) << k;
      }
    }
    above = (above & inside) | (there & ~inside);
    level &= inside;
    const uint32_t my_above = __popc(above), my_level = __popc(level);
    uint32_t a = my_above, l = my_level;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const uint32_t x = __shfl_up_sync(0xffffffffu, a, d), y = __shfl_up_sync(0xffffffffu, l, d);
      if (lane >= d) a += x, l += y;
    }
    if (lane == 31) of_warps[0][warp] = a, of_warps[1][warp] = l;  // (last read before the barriers of the last digit)
    __syncthreads();
    a += __reduce_add_sync(0xffffffffu, lane < warp ? of_warps[0][lane] : 0) - my_above;
    l += __reduce_add_sync(0xffffffffu, lane < warp ? of_warps[1][lane] : 0) - my_level;
    // Of its equal ones the thread keeps the first, as many as those before it have left.
    uint32_t more = l < wanted ? min(wanted - l, my_level) : 0, chosen = above;
    for (; more != 0; --more) {
      chosen |= level & -level;
      level &= level - 1;
    }
    for (uint32_t at = a + min(l, wanted); chosen != 0; chosen &= chosen - 1) places[at++] = static_cast<uint16_t>(mine + __ffs(chosen) - 1);
    // (by way of shared memory: threads' own stores, each to lines of its own, took a third of the time)
    __syncthreads();
    for (int32_t i = threadIdx.x; i < count; i += kSelectThreads) {
      const int32_t place = places[i];
      kept[i] = place;
      out[i] = held[padded(place)];
    }
  } else {
    for (int32_t i = count + threadIdx.x; i < p.new_width; i += kSelectThreads) out[i] = 0.0f;
    __syncthreads();
    if (any) {
#pragma unroll
      for (int digit = 0; digit < 3; ++digit) {
#pragma unroll 8
        for (int32_t i = begin + threadIdx.x; i < end; i += kSelectThreads) {
          const uint32_t rank = rank_of(load_arg(weights + i));
          if (digit == 0 || rank >> kShift[digit == 0 ? 0 : digit - 1] == prefix) atomicAdd(&bins[digit][digit_of(rank, digit)], 1u);
        }
        __syncthreads();
        prefix = prefix << (digit == 2 ? 10 : 11) | find_bin(bins[digit], of_warps[digit], found[digit], wanted);
      }
    }
    const int32_t rows = (length + 32 * kSelectWarps - 1) / (32 * kSelectWarps);  // of 32 tokens, of a warp
    const int32_t from = warp * rows * 32, to = min(length, from + rows * 32);
    auto look = [&](int32_t i, float w, uint32_t& above, uint32_t& level) {
      const bool inside = static_cast<uint32_t>(i - begin) < between;
      const uint32_t rank = rank_of(w);
      above = __ballot_sync(0xffffffffu, i < to && (!inside || (any && rank > prefix)));
      level = __ballot_sync(0xffffffffu, i < to && inside && any && rank == prefix);
    };
    uint32_t all_above = 0, all_level = 0;
#pragma unroll 4
    for (int32_t r = 0; r < rows; ++r) {
      const int32_t i = from + 32 * r + lane;
      uint32_t above, level;
      look(i, i < to ? load_arg(weights + i) : 0.0f, above, level);
      all_above += __popc(above);
      all_level += __popc(level);
    }
    if (lane == 0) of_warps[0][warp] = all_above, of_warps[1][warp] = all_level;
    __syncthreads();
    uint32_t above_before = __reduce_add_sync(0xffffffffu, lane < warp ? of_warps[0][lane] : 0);
    uint32_t level_before = __reduce_add_sync(0xffffffffu, lane < warp ? of_warps[1][lane] : 0);
    const uint32_t below_lane = (1u << lane) - 1;
#pragma unroll 4
    for (int32_t r = 0; r < rows; ++r) {
      const int32_t i = from + 32 * r + lane;
      const float w = i < to ? load_arg(weights + i) : 0.0f;
      uint32_t above, level;
      look(i, w, above, level);
      const uint32_t l = level_before + __popc(level & below_lane);
      if ((above >> lane & 1) != 0 || ((level >> lane & 1) != 0 && l < wanted)) {
        const uint32_t at = above_before + __popc(above & below_lane) + min(l, wanted);
        kept[at] = i;
        out[at] = w;
      }
      above_before += __popc(above);
      level_before += __popc(level);
    }
  }
}

struct RowPlace {
  int64_t page, place;  // page < 0: none
};

__device__ __forceinline__ RowPlace row_place(const EvictParams& p, const int32_t* table, int32_t capacity, int32_t token) {
  if (token >= capacity) return {-1, 0};
  const uint32_t index = p.cache.page_size.div(token);
  const int32_t page = load_arg(table + index);
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(p.cache.num_pages)) return {-1, 0};
  return {page, token - index * p.cache.page_size.d};
}

constexpr int kCopyThreads = 256;

// Rows into other pages: every 16 bytes of keys and of values on their own.  16 sequences of 8 heads of 128
// in BF16, 4096 rows of 16384: 88 us, 93 % of the copy rate.
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictParams p) {
  ptx::grid_dependency_wait();
  const int32_t b = blockIdx.z, head = blockIdx.y, pieces = p.row_bytes / 16;
  const int32_t count = p.new_lengths[b];
  const int32_t* const kept = p.kept + (static_cast<int64_t>(b) * gridDim.y + head) * p.places;
  const int32_t* const from_table = p.tables + b * p.table_stride;
  const int32_t* const to_table = p.new_tables + b * p.new_stride;
  const int32_t rows = kCopyThreads / pieces;  // of a round
  const int32_t row = threadIdx.x / pieces, piece = threadIdx.x % pieces;
  if (row >= rows) return;
  for (int32_t i = blockIdx.x * rows + row; i < count; i += gridDim.x * rows) {
    const RowPlace from = row_place(p, from_table, p.capacity, kept[i]), to = row_place(p, to_table, p.new_capacity, i);
    if ((from.page < 0 || to.page < 0) && p.status != nullptr) atomicOr(p.status, kStatusIndex);
    if (to.page < 0) continue;
    const int64_t read = from.page * p.cache.page + from.place * p.cache.token + head * p.cache.head + piece * 16;
    const int64_t write = to.page * p.cache.page + to.place * p.cache.token + head * p.cache.head + piece * 16;
    uint4 k = make_uint4(0, 0, 0, 0), v = k;
    if (from.page >= 0) k = load_once(p.cache.k + read), v = load_once(p.cache.v + read);
    *reinterpret_cast<uint4*>(p.cache.k + write) = k;
    *reinterpret_cast<uint4*>(p.cache.v + write) = v;
    if (p.cache.k_scale != nullptr && piece == 0) {
      const int64_t read_scale = from.page * p.cache.scale_page + from.place * p.cache.scale_token + head * p.cache.scale_head;
      const int64_t write_scale = to.page * p.cache.scale_page + to.place * p.cache.scale_token + head * p.cache.scale_head;
      p.cache.k_scale[write_scale] = from.page >= 0 ? load_arg(p.cache.k_scale + read_scale) : 0.0f;
      p.cache.v_scale[write_scale] = from.page >= 0 ? load_arg(p.cache.v_scale + read_scale) : 0.0f;
    }
  }
}

constexpr int kShiftThreads = 1024;

// Keeps its place among the barriers and stores.
__device__ __forceinline__ float load_ordered(const float* p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p) : "memory");
  return v;
}

// Rows forward within their pages.  A kept token never moves back, so rows are moved in order, a round of them at a time,
// read whole before any of it is written; a CTA has some columns of a head's rows of its own (64 bytes or, of rows that
// do not divide so, 32 or 16), so that no two have to wait for each other.  One more takes the scales.  16 sequences of 8 heads of 128
// in BF16, 4096 rows of 16384, selection included: 226 us (into other pages 104); in 8 bits one of 32768 rows of 131072: 293 (138).  Bounded by
// the chain of a round, kept -> table -> row, between barriers.
__global__ void __launch_bounds__(kShiftThreads) evict_shift_kernel(const EvictParams p, int32_t slice_bytes) {
  __shared__ int32_t first_moved;
  ptx::grid_dependency_wait();
  const int32_t b = blockIdx.z, head = blockIdx.y, slices = p.row_bytes / slice_bytes;
  const int32_t count = p.new_lengths[b];
  const int32_t* const kept = p.kept + (static_cast<int64_t>(b) * gridDim.y + head) * p.places;
  const int32_t* const table = p.tables + b * p.table_stride;
  if (threadIdx.x == 0) {  // (kept[i] - i never falls)
    int32_t low = 0, high = count;
    while (low < high) {
      const int32_t middle = (low + high) / 2;
      if (kept[middle] == middle) low = middle + 1; else high = middle;
    }
    first_moved = low;
  }
  __syncthreads();
  const int32_t begin = first_moved;
  const bool of_scales = blockIdx.x == 2 * slices;
  const int32_t lanes = of_scales ? 2 : slice_bytes / 16, rows = kShiftThreads / lanes;
  const int32_t row = threadIdx.x / lanes, piece = threadIdx.x % lanes;
  uint8_t* const values = blockIdx.x < slices ? p.cache.k : p.cache.v;
  const int64_t column = static_cast<int64_t>(blockIdx.x % slices) * slice_bytes + piece * 16;
  float* const scales = piece == 0 ? p.cache.k_scale : p.cache.v_scale;
  auto place_of = [&](const RowPlace& at) { return at.page * p.cache.page + at.place * p.cache.token + head * p.cache.head + column; };
  auto scale_of = [&](const RowPlace& at) { return at.page * p.cache.scale_page + at.place * p.cache.scale_token + head * p.cache.scale_head; };
  uint4 ahead = make_uint4(0, 0, 0, 0);
  RowPlace ahead_to = {-1, 0};
  auto read = [&](int32_t i) {
    ahead_to.page = -1;
    if (i >= count) return;
    const RowPlace from = row_place(p, table, p.capacity, kept[i]);
    ahead_to = row_place(p, table, p.capacity, i);
    if ((from.page < 0 || ahead_to.page < 0) && p.status != nullptr) atomicOr(p.status, kStatusIndex);
    ahead = make_uint4(0, 0, 0, 0);
    if (from.page < 0) return;
    if (of_scales) ahead.x = __float_as_uint(load_ordered(scales + scale_of(from))); else ahead = load_once_ordered(values + place_of(from));
  };
  read(begin + row);
#pragma unroll 1
  for (int32_t i0 = begin; i0 < count; i0 += rows) {
    const uint4 now = ahead;
    const RowPlace to = ahead_to;
    read(i0 + rows + row);
    __syncthreads();  // the round has been read (and the next: its rows lie behind what is written now)
    if (to.page < 0) continue;
    if (of_scales) scales[scale_of(to)] = __uint_as_float(now.x); else *reinterpret_cast<uint4*>(values + place_of(to)) = now;
  }
}

}  // namespace
}  // namespace chord

extern "C" {

int chord_b200_attention_weights(const void* q, int64_t q_batch, int64_t q_head, const chord_b200_kv_cache* cache,
                                 const int32_t* tables, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
                                 const float* lse, float* weights, int64_t weight_batch, int64_t weight_head, int64_t width,
                                 int add, int32_t* status, int64_t batch, int64_t heads, const chord_b200_scores* scores,
                                 void* stream) {
  using namespace chord;
  WeighParams p = {};
  if (int rc = make_cache(cache, &p.cache)) return rc;
  CHORD_REQUIRE(batch >= 0 && batch <= 65535, "the batch must be in [0, 65535], got %lld", static_cast<long long>(batch));
  if (batch == 0 || width == 0) return kOk;
  CHORD_REQUIRE(q != nullptr && tables != nullptr && lengths != nullptr && lse != nullptr && weights != nullptr && scores != nullptr,
                "null pointer");
  CHORD_REQUIRE(heads > 0 && heads <= 65535 && heads % cache->heads == 0,
                "the number of query heads (%lld) must be a multiple of the cache's (%lld)", static_cast<long long>(heads),
                static_cast<long long>(cache->heads));
  CHORD_REQUIRE(q_batch >= 0 && q_head >= 0 && q_batch % 8 == 0 && q_head % 8 == 0 && (reinterpret_cast<uintptr_t>(q) & 15u) == 0,
                "q's rows must lie on 16-byte boundaries");
  CHORD_REQUIRE(max_pages > 0 && table_stride >= 0 && max_pages < (1ll << 31), "a block table has a page or more");
  CHORD_REQUIRE(width > 0 && width < (1ll << 31) - 65536 && weight_batch >= 0 && weight_head >= 0, "sizes of the weights out of range");
  CHORD_REQUIRE(scores->window >= 0 && scores->window < (1ll << 31), "window out of range");
  CHORD_REQUIRE(scores->scale - scores->scale == 0.0, "scale must be finite");
  CHORD_REQUIRE(cap_fits(*scores), "the cap must be zero or from 1e-30 to 1e30, and the scale no more than 1e36 of it");
  const WeighKernel kernel = cache->k_scale != nullptr ? weigh_kernel<true>(cache->head_dim) : weigh_kernel<false>(cache->head_dim);
  CHORD_REQUIRE(kernel.kernel != nullptr, "head_dim must be 64, 96, 128, 192 or 256, got %lld", static_cast<long long>(cache->head_dim));
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  if (int rc = allow_smem(reinterpret_cast<const void*>(kernel.kernel), kernel.smem, device.device)) return rc;
  const int64_t capacity = max_pages * cache->page_size;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_batch = q_batch;
  p.q_head = q_head;
  p.tables = tables;
  p.table_stride = table_stride;
  p.lengths = lengths;
  p.lse = lse;
  p.slopes = scores->slopes;
  p.weights = weights;
  p.weight_batch = weight_batch;
  p.weight_head = weight_head;
  p.status = status;
  p.scale = static_cast<float>(scores->scale * 1.4426950408889634074);
  p.cap = static_cast<float>(scores->cap * 1.4426950408889634074);
  p.over_cap = scores->cap > 0.0 ? static_cast<float>(1.0 / (scores->cap * 1.4426950408889634074)) : 0.0f;
  p.heads = static_cast<int32_t>(heads);
  p.group = static_cast<int32_t>(heads / cache->heads);
  p.capacity = static_cast<int32_t>(capacity < (1ll << 31) - 65536 ? capacity : (1ll << 31) - 65536);
  p.width = static_cast<int32_t>(width);
  p.window = static_cast<int32_t>(scores->window);
  p.add = add;
  // Several runs for a warp where that leaves a few warps for each of those that are resident: what a warp begins with is paid once.
  // (With one run always, 64 x 8192 in 8 bits 121 us for 103, 131072 38 for 31; with sixteen warps of an SM four, 64 x 1024 in BF16 38 for 26.)
  p.in_a_row = cache->page_size % 16 == 0 && p.cache.token == cache->head_dim * (cache->k_scale != nullptr ? 1 : 2);
  p.runs = 1;
  const int64_t warps = (width + kWeighRun - 1) / kWeighRun * cache->heads * batch;
  while (p.runs < 8 && warps / (2 * p.runs) >= device.sm_count * 16) p.runs *= 2;
  const int64_t tokens = kWeighWarps * kWeighRun * p.runs;
  const dim3 grid(static_cast<unsigned>((width + tokens - 1) / tokens), static_cast<unsigned>(cache->heads), static_cast<unsigned>(batch));
  CHORD_CUDA(launch_kernel(kernel.kernel, grid, dim3(kWeighWarps * 32), static_cast<size_t>(kernel.smem), static_cast<cudaStream_t>(stream), kEarlyLaunch, p));
  return kOk;
}

int64_t chord_b200_cache_evict_workspace_bytes(int64_t batch, int64_t kv_heads, int64_t keep) {
  using namespace chord;
  if (batch < 0 || kv_heads < 0 || keep < 0) return fail(kInvalidArgument, "no size may be negative"), -1;
  if (batch > 65535 || kv_heads > 65535 || keep >= (1ll << 28)) return fail(kInvalidArgument, "no sizes of an eviction"), -1;
  return batch * kv_heads * keep * 4;
}

int chord_b200_cache_evict(const chord_b200_kv_cache* cache, const int32_t* tables, int64_t table_stride, int64_t max_pages,
                           const int32_t* new_tables, int64_t new_stride, int64_t new_pages, const int32_t* lengths,
                           const float* weights, int64_t weight_batch, int64_t weight_head, int64_t width, int32_t* new_lengths,
                           float* new_weights, int64_t new_width, void* workspace, int64_t workspace_bytes, int32_t* status,
                           int64_t batch, int64_t keep, int64_t first, int64_t recent, void* stream) {
  using namespace chord;
  EvictParams p = {};
  if (int rc = make_cache(cache, &p.cache)) return rc;
  CHORD_REQUIRE(batch >= 0 && batch <= 65535, "the batch must be in [0, 65535], got %lld", static_cast<long long>(batch));
  if (batch == 0) return kOk;
  CHORD_REQUIRE(tables != nullptr && lengths != nullptr && weights != nullptr && new_lengths != nullptr && new_weights != nullptr &&
                    workspace != nullptr,
                "null pointer");
  CHORD_REQUIRE(max_pages > 0 && table_stride >= 0 && max_pages < (1ll << 31), "a block table has a page or more");
  CHORD_REQUIRE(new_tables == nullptr || (new_pages > 0 && new_stride >= 0 && new_pages < (1ll << 31)), "a block table has a page or more");
  CHORD_REQUIRE(keep > 0 && keep < (1ll << 28) && first >= 0 && recent >= 0 && first <= keep && recent <= keep - first,
                "keep is below 2^28, first and recent are at least zero and no more than keep, %lld, together, got %lld and %lld",
                static_cast<long long>(keep), static_cast<long long>(first), static_cast<long long>(recent));
  CHORD_REQUIRE(width > 0 && width < (1ll << 31) - 65536 && new_width > 0 && new_width < (1ll << 31) - 65536 && keep <= new_width &&
                    weight_batch >= 0 && weight_head >= 0,
                "sizes of the weights out of range");
  const int64_t places = keep < width ? keep : width, needed = chord_b200_cache_evict_workspace_bytes(batch, cache->heads, places);
  CHORD_REQUIRE(needed >= 0 && workspace_bytes >= needed && (reinterpret_cast<uintptr_t>(workspace) & 3u) == 0,
                "the workspace has %lld bytes, this launch needs %lld", static_cast<long long>(workspace_bytes),
                static_cast<long long>(needed));
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  const auto capacity = [&](int64_t pages) {
    const int64_t tokens = pages * cache->page_size;
    return static_cast<int32_t>(tokens < (1ll << 31) - 65536 ? tokens : (1ll << 31) - 65536);
  };
  p.tables = tables;
  p.table_stride = table_stride;
  p.new_tables = new_tables;
  p.new_stride = new_stride;
  p.lengths = lengths;
  p.weights = weights;
  p.weight_batch = weight_batch;
  p.weight_head = weight_head;
  p.new_lengths = new_lengths;
  p.new_weights = new_weights;
  p.kept = static_cast<int32_t*>(workspace);
  p.status = status;
  p.capacity = capacity(max_pages);
  p.new_capacity = new_tables != nullptr ? capacity(new_pages) : p.capacity;
  p.width = static_cast<int32_t>(width);
  p.new_width = static_cast<int32_t>(new_width);
  p.keep = static_cast<int32_t>(keep);
  p.places = static_cast<int32_t>(places);
  p.first = static_cast<int32_t>(first);
  p.recent = static_cast<int32_t>(recent);
  p.row_bytes = static_cast<int32_t>(cache->head_dim * (cache->k_scale != nullptr ? 1 : 2));
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const unsigned heads = static_cast<unsigned>(cache->heads), sequences = static_cast<unsigned>(batch);
  const int64_t most = width < p.capacity ? width : p.capacity;
  // As few weights to a thread as there are: 3 x 4 heads of 700 tokens (in place) 8.8 us with two, 10.2 with eight, 15.9 with 32,
  // 9.0 from memory; 16 x 8 of 8192 69 with eight, 71 with sixteen, 76 from memory; of 32768 246 with 32, 258 from memory.
  const auto select = [&](void (*kernel)(EvictParams), int items) {
    const int held = items * (kSelectThreads / 32 * 33 * 4 + kSelectThreads * 2);
    if (int rc = allow_smem(reinterpret_cast<const void*>(kernel), held, device.device)) return rc;
    CHORD_CUDA(launch_kernel(kernel, dim3(heads, sequences), dim3(kSelectThreads), static_cast<size_t>(held), s, kEarlyLaunch, p));
    return static_cast<int>(kOk);
  };
  const int rc = most <= 2 * kSelectThreads ? select(evict_select_kernel<2>, 2) : most <= 8 * kSelectThreads ? select(evict_select_kernel<8>, 8) :
                 most <= 16 * kSelectThreads ? select(evict_select_kernel<16>, 16) : most <= 32 * kSelectThreads ? select(evict_select_kernel<32>, 32) : select(evict_select_kernel<0>, 0);
  if (rc) return rc;
  if (new_tables != nullptr) {
    const int rows = kCopyThreads / (p.row_bytes / 16);
    const int64_t rounds = ((keep < most ? keep : most) + rows - 1) / rows;
    CHORD_CUDA(launch_kernel(evict_copy_kernel, dim3(static_cast<unsigned>((rounds + 3) / 4), heads, sequences), dim3(kCopyThreads), 0, s, kEarlyLaunch, p));
  } else {
    const int32_t slice = p.row_bytes % 64 == 0 ? 64 : p.row_bytes % 32 == 0 ? 32 : 16;
    const unsigned slices = static_cast<unsigned>(2 * (p.row_bytes / slice) + (cache->k_scale != nullptr ? 1 : 0));
    CHORD_CUDA(launch_kernel(evict_shift_kernel, dim3(slices, heads, sequences), dim3(kShiftThreads), 0, s, kEarlyLaunch, p, slice));
  }
  return kOk;
}

}  // extern "C"
