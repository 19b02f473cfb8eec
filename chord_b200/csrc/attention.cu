// Attention of one new token for each sequence over its pages of keys and values.
#include <cuda_bf16.h>

#include <mutex>

#include "../../include/chord_b200.h"
#include "common.h"
#include "join_plan.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kMaxCtasPerSm = 3;
constexpr int kMaxCtas = 480;      // of a launch: three on each of 160 SMs
// A lot's lock word: arrivals at the last join of the row that it is the first lot of (11 bits), and at the join of
// the group that it is the first of (6 bits).
constexpr int kRowShift = 0, kGroupShift = 11;
static_assert(kMaxCtas < (1 << 11) && kFan < (1 << 6), "the fields' widths");

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
  bool whole_groups;
};

// What follows from the head's width and the cache's type.  A warp takes kStep tokens at a time, whose
// keys and values are some 5 to 18 KB; kStages of them are on their way or in use.
template <int kDim, bool kCodes, int kTiles>
struct Layout {
  static constexpr int kRow = kDim * (kCodes ? 1 : 2);  // bytes of a row
  static constexpr int kPitch = kRow + 16;              // an odd number of 16-byte pieces: no bank conflicts
  static constexpr int kStep = kCodes && kDim <= 192 ? 32 : 16;
  static constexpr int kScaleBytes = kCodes ? 2 * kStep * 4 : 0;
  static constexpr int kStageBytes = 2 * kStep * kPitch + kScaleBytes;
  // CTAs of an SM: as many as have room for two stages and for their registers.  Heads of 192, 64 x 4096 and 256 x
  // 256 tokens: codes 111.0 and 44.8 us with two, 113.6 and 55.6 with one, BF16 184.5 and 62.7, 201.5 and 68.0.
  // Heads of 256, codes, with steps of 16 tokens two: 142.7 and 52.7, with 32 one: 136.2 and 58.9, 37 x 1000 31.4 and 34.0.
  // Heads of 64, codes: 47.4 and 25.6 with three, 52.9 and 28.2 with two, 46.5 and 24.4 with four, which lose where rows
  // are few (37 x 1000 of 12 heads 22.6, 18.7 with three).
  static constexpr int kCtas = kDim > 192 ? (kCodes ? 2 : 1) : kDim == 64 && kTiles == 1 ? 3 : 2;
  static constexpr int kFit = (kCtas == 1 ? 220 : kCtas == 2 ? 111 : 74) * 1024 / (kWarps * kStageBytes);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kSmem = kWarps * kStages * kStageBytes;
  static_assert(kStages >= 2 && kStages * kStageBytes >= 8 * kTiles * (kDim + 2) * 4, "a warp's part takes its ring's place");
};

// Part of a row: [dims, in the products' order][heads] values, the heads' maxima and their sums.
__host__ __device__ constexpr int64_t part_floats(int dim, int heads) { return heads * (dim + 2); }

// Floats of workspace: kSlots parts for each lot, one for each warp.
constexpr int64_t workspace_floats(int64_t ctas, int dim, int heads) {
  return ctas * (kSlots + kWarps) * part_floats(dim, heads);
}

// Two of four codes as BF16 pairs, (code - 128) / 64, exact.
__device__ __forceinline__ uint32_t two_codes(uint32_t four, uint32_t select) {
  constexpr uint32_t kOffset = 0xC000C000u;  // -128 / 64, twice
  return bf16x2_fma(__byte_perm(four, 0, select), kTwo127, kOffset);
}

__device__ __forceinline__ void ldmatrix_x4_at(uint32_t addr, uint32_t (&r)[4]) { ptx::ldmatrix_x4<0>(addr, r); }

__device__ __forceinline__ void cp_async_16_all(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// What a warp has of a row that does not lie in its share alone.
struct Part {
  float* at;
  int32_t b, row;
  int32_t first_lot, lots;  // that have parts of the row
  bool there, began;        // began: in an earlier share
};

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The logarithm of a sum, kept relative to 2^top.
__device__ __forceinline__ float lse_of(float top, float sum) {
  return sum == 0.0f ? -INFINITY : (top + log2f(sum)) * 0.693147180559945309f;
}

__device__ __forceinline__ void add_weighted(float4& v, const float4& weight, const float4& x) {
  v.x = fmaf(weight.x, x.x, v.x);
  v.y = fmaf(weight.y, x.y, v.y);
  v.z = fmaf(weight.z, x.z, v.z);
  v.w = fmaf(weight.w, x.w, v.w);
}

// Two numbers of at least zero as sums of two BF16 numbers each, to 2^-16.  Both parts of a number above zero are
// above zero (its last bit is set, the first part is cut off and not rounded), so that an infinity times the
// number is an infinity and not the difference of two, or zero times one.
__device__ __forceinline__ void positive_parts(float x, float y, uint32_t& coarse, uint32_t& fine) {
  const uint32_t a = __float_as_uint(x) | 1u, b = __float_as_uint(y) | 1u;
  coarse = __byte_perm(a, b, 0x7632);
  fine = pack_bf16(__uint_as_float(a) - __uint_as_float(a & 0xFFFF0000u), __uint_as_float(b) - __uint_as_float(b & 0xFFFF0000u));
}

// Reads of parts, in shared memory or written by another CTA.
__device__ __forceinline__ float4 read_part4(const float* p) {
  float4 v;
  asm volatile("ld.relaxed.gpu.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p) : "memory");
  return v;
}

__device__ __forceinline__ int32_t atomic_add_acq_rel(int32_t* p, int32_t v) {
  int32_t before;
  asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], %2;" : "=r"(before) : "l"(p), "r"(v) : "memory");
  return before;
}

// n / d, in 32 bits where they do.
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
  if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// What outputs are multiplied with: those of codes are 64ths.
template <bool kCodes>
__device__ __forceinline__ float rate_of(float sum) { return sum == 0.0f ? 0.0f : (kCodes ? 64.0f : 1.0f) / sum; }

__device__ __forceinline__ float power_of_two(int32_t exponent) { return __int_as_float((exponent + 127) << 23); }

// An 8x8 matrix of 16-bit elements, a row in four lanes, to its transpose.
__device__ __forceinline__ uint32_t transposed(uint32_t pair) {
  uint32_t t;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(t) : "r"(pair));
  return t;
}

// The query heads of a row of work, and its results.
struct Row {
  int64_t head0;  // of the batch's heads
  int32_t heads;
  __device__ __forceinline__ Row(const AttentionParams& p, int32_t b, int32_t row) {
    const int32_t kv_head = row / p.head_blocks, head_block = row % p.head_blocks;
    heads = min(p.group - head_block * 16, 16);
    head0 = static_cast<int64_t>(b) * p.heads + kv_head * p.group + head_block * 16;
  }
  // Four heads' values of one dim, the `place`-th of the products' order: with codes a 16-byte piece has
  // its even dims first.
  template <int kDim, bool kCodes>
  __device__ __forceinline__ void finish(const AttentionParams& p, int head, int place, const float4& v, const float4& all,
                                         const float4& most) const {
    const int dim = kCodes ? place / 16 * 16 + place % 8 * 2 + place % 16 / 8 : place;
    const float value[4] = {v.x, v.y, v.z, v.w}, sum[4] = {all.x, all.y, all.z, all.w}, top[4] = {most.x, most.y, most.z, most.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (head + i >= heads) break;
      p.out[(head0 + head + i) * kDim + dim] = __float2bfloat16(value[i] * rate_of<kCodes>(sum[i]));
      if (place == 0 && p.lse != nullptr) p.lse[head0 + head + i] = lse_of(top[i], sum[i]);
    }
  }
};

// A thread's values while a row's parts are joined: four heads' values of kItems dims, with the heads'
// maxima and sums.
template <int kDim, int kHeads>
struct Joined {
  static constexpr int kQuads = kHeads / 4;
  static constexpr int kItems = (kDim * kQuads + kThreads - 1) / kThreads;  // (dims, kThreads / kQuads apart)
  static constexpr bool kWhole = kDim * kQuads % kThreads == 0;  // every thread has all its items
  static __device__ __forceinline__ bool mine(int i) { return kWhole || threadIdx.x + i * kThreads < kDim * kQuads; }
  float4 value[kItems], top, sum;
  __device__ __forceinline__ Joined() {
#pragma unroll
    for (int i = 0; i < kItems; ++i) value[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    top = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
  }
  __device__ __forceinline__ void add(const float* from) {
    const int32_t quad = threadIdx.x % kQuads * 4;
    const float4 m = read_part4(from + kDim * kHeads + quad), l = read_part4(from + (kDim + 1) * kHeads + quad);
    float4 v[kItems];
#pragma unroll
    for (int i = 0; i < kItems; ++i) v[i] = mine(i) ? read_part4(from + 4 * (threadIdx.x + i * kThreads)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const float4 next = make_float4(fmaxf(top.x, m.x), fmaxf(top.y, m.y), fmaxf(top.z, m.z), fmaxf(top.w, m.w));
    const float4 old = factors(top, next), weight = factors(m, next);
    top = next;
    sum = make_float4(sum.x * old.x, sum.y * old.y, sum.z * old.z, sum.w * old.w);
    add_weighted(sum, weight, l);
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      value[i] = make_float4(value[i].x * old.x, value[i].y * old.y, value[i].z * old.z, value[i].w * old.w);
      add_weighted(value[i], weight, v[i]);
    }
  }
  static __device__ __forceinline__ float factor(float from, float to) { return to == -INFINITY ? 0.0f : exp2_approx(from - to); }
  static __device__ __forceinline__ float4 factors(const float4& from, const float4& to) {
    return make_float4(factor(from.x, to.x), factor(from.y, to.y), factor(from.z, to.z), factor(from.w, to.w));
  }
  // To a part, or to the results (to == null).
  template <bool kCodes>
  __device__ __forceinline__ void give(const AttentionParams& p, const Row& of, float* to) const {
    const int32_t head = threadIdx.x % kQuads * 4;
#pragma unroll
    for (int i = 0; i < kItems; ++i) {
      if (!mine(i)) break;
      const int32_t index = threadIdx.x + i * kThreads;
      if (to == nullptr) {
        of.template finish<kDim, kCodes>(p, head, index / kQuads, value[i], sum, top);
      } else {
        __stcg(reinterpret_cast<float4*>(to + 4 * index), value[i]);
      }
    }
    if (to != nullptr && threadIdx.x < kQuads) {
      __stcg(reinterpret_cast<float4*>(to + kDim * kHeads + head), top);
      __stcg(reinterpret_cast<float4*>(to + (kDim + 1) * kHeads + head), sum);
    }
  }
};

// Joins `count` (at most kFan) parts that other CTAs have written, source(j) the j-th of them, into a part or
// the results.  What they hold comes into shared memory by cp.async, all of it at once where there is room;
// the weights are worked out while the values are on their way, by every warp for itself.
template <int kDim, bool kCodes, int kHeads, int kSmem, typename Source>
__device__ __forceinline__ void join_parts(const AttentionParams& p, const Row& of, uint8_t* smem, int32_t count, float* to, Source source) {
  using Join = Joined<kDim, kHeads>;
  constexpr int kStats = 2 * kHeads * 4, kValues = kDim * kHeads * 4;  // bytes of a part
  constexpr int kRound = (kSmem - kFan * (kStats + kHeads * 4) - 2 * kHeads * 4) / kValues;
  static_assert(kRound >= 4 && kValues % 512 == 0, "room for some parts; whole pieces for a warp");
  float* const stats = reinterpret_cast<float*>(smem);           // [count][maxima, sums][heads]
  float* const weights = stats + kFan * 2 * kHeads;              // [count][heads]
  float* const result = weights + kFan * kHeads;                 // maxima, sums
  float* const values = result + 2 * kHeads;                     // [kRound][dims][heads]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

#pragma unroll 1
  for (int32_t e = threadIdx.x; e < count * (kStats / 16); e += kThreads) {
    const int32_t j = e / (kStats / 16), piece = e % (kStats / 16);
    cp_async_16_all(ptx::smem_u32(stats) + e * 16, source(j) + kDim * kHeads + piece * 4);
  }
  ptx::cp_async_commit();
  Join joined;
#pragma unroll 1
  for (int32_t j0 = 0; j0 < count; j0 += kRound) {
    const int32_t here = min(kRound, count - j0);
    if (j0 != 0) __syncthreads();
#pragma unroll 1
    for (int32_t j = warp; j < here; j += kWarps) {
      const float* const from = source(j0 + j) + lane * 4;
      const uint32_t dst = ptx::smem_u32(values) + j * kValues + lane * 16;
#pragma unroll
      for (int i = 0; i < kValues / 512; ++i) cp_async_16_all(dst + i * 512, from + i * 128);
    }
    ptx::cp_async_commit();
    if (j0 == 0) {
      ptx::cp_async_wait_group<1>();
      __syncthreads();
      constexpr int kSides = 32 / kHeads;
      const int head = lane % kHeads, side = lane / kHeads;
      float most = -INFINITY, all = 0.0f;
#pragma unroll 1
      for (int32_t j = side; j < count; j += kSides) most = fmaxf(most, stats[2 * j * kHeads + head]);
#pragma unroll
      for (int d = kHeads; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
#pragma unroll 1
      for (int32_t j = side; j < count; j += kSides) {
        const float weight = Join::factor(stats[2 * j * kHeads + head], most);
        weights[j * kHeads + head] = weight;  // (the same from every warp)
        all = fmaf(weight, stats[(2 * j + 1) * kHeads + head], all);
      }
#pragma unroll
      for (int d = kHeads; d < 32; d <<= 1) all += __shfl_xor_sync(0xffffffffu, all, d);
      if (side == 0) {
        result[head] = most;
        result[kHeads + head] = all;
      }
    }
    ptx::cp_async_wait_group<0>();
    __syncthreads();
    const int quad = threadIdx.x % Join::kQuads * 4;
#pragma unroll 4
    for (int32_t j = 0; j < here; ++j) {
      const float4 weight = *reinterpret_cast<const float4*>(weights + (j0 + j) * kHeads + quad);
#pragma unroll
      for (int i = 0; i < Join::kItems; ++i) {
        if (Join::mine(i)) {
          add_weighted(joined.value[i], weight, *reinterpret_cast<const float4*>(values + j * (kDim * kHeads) + 4 * (threadIdx.x + i * kThreads)));
        }
      }
    }
  }
  joined.top = *reinterpret_cast<const float4*>(result + threadIdx.x % Join::kQuads * 4);
  joined.sum = *reinterpret_cast<const float4*>(result + kHeads + threadIdx.x % Join::kQuads * 4);
  joined.template give<kCodes>(p, of, to);
}

// One row of work is a sequence, one of its key-value heads and a block of up to 16 of the query heads
// that share it; a step is kStep of its tokens.  A lot is a CTA's work.  Where there are few rows, each is
// cut into lots of its own; else the steps of all rows are numbered through and cut into equal lots, so
// that lengths need not be alike.  A warp goes through its quarter of a lot on its own: a ring of
// cp.async stages that runs ahead across the rows' ends, and a running maximum, sum and output.  Rows
// that lie in one quarter are finished by their warp; the others' parts are joined within the CTA once
// all its warps are done, and then, through memory, by the last CTA of a row to arrive (with more than
// kAtOnce parts by the last of each group of 8 or 24 neighbours, and the last of these).
//
// Products on mma.m16n8k16, keys and values as the 16-row operand, the heads (eight for each of kTiles)
// as columns: S[tokens, heads] = K Q^T and O[dims, heads] += V^T P, P by movmatrix from the score
// fragments.  (With the heads as rows, half of every product was idle with up to eight of them.)  P is multiplied
// as the sum of two BF16 numbers, 16 bits of it.
// Codes are exact in BF16; the keys' scales are applied to the scores, the values' to P.  The codes of
// values become (code - 128) / 64.  Those of keys are multiplied as they stand, as the BF16 numbers
// code * 2^-133, with queries times a power of two that takes the row's largest (finite) one to 2^111 or just
// above: the scores start from minus 128 times the query's sum, which saves a multiply-add for every two codes.
// Their additions are then off by FP32's roundings of up to 383 sum |q| steps (dim / 16 + 4 times 2^-22 of it), where the keys'
// own codes are off by up to half a step: under half a percent of that, however close to 128 the codes lie.
//
// The running maximum is raised, and the sums are scaled, only where a score passes it by more than
// 2^kSlack; until then P is up to 2^kSlack, which costs no precision, and no lane needs another's scores.
//
// Long rows are bounded by memory and by how unequally the SMs are served: 64 sequences of up to 8192 tokens in
// BF16, 64 + 8 heads of 128, 1.36 GB, 231 to 250 us from GPU to GPU = 5.4 to 5.9 TB/s, 83 to 90 % of a plain copy's rate (of 64 x 4096, equal lots, 12
// SMs were done after 127 us, 96 after 152, 40 after 174; lots by ticket or two and three times as many were no
// better).  Codes also by instructions, some 630 for 32 tokens: 131072 tokens of one sequence, 277 MB, 59 us =
// 4.7 TB/s, of which about 8 are the launch, the rings' filling and two joins.  Three CTAs of an SM with steps of 16
// tokens instead of two with 32 gain 9 % on 64 x 4096 of codes, and lose 10 % on that one and 40 % on 37 x 1000.  Short
// rows are bounded by latency: 333 tokens of 8 heads 8.4 us, some five dependent round trips to memory and one join.
template <int kDim, bool kCodes, int kTiles>
__global__ void __launch_bounds__(kThreads, (Layout<kDim, kCodes, kTiles>::kCtas))
paged_attention_kernel(const AttentionParams p) {
  using L = Layout<kDim, kCodes, kTiles>;
  constexpr int kChunks = kDim / 16;
  constexpr int kGroups = L::kStep / 16;  // of 16 tokens
  constexpr int kHeads = 8 * kTiles;
  constexpr float kSlack = 8.0f;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ int32_t answer[2];
  // Parts 2 w and 2 w + 1: what warp w holds of the row that its share begins inside of, and of the one
  // that its share ends inside of (the latter where both are one).
  __shared__ Part parts[2 * kWarps];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q4 = lane & 3, r8 = lane >> 2;
  constexpr int64_t kPartFloats = part_floats(kDim, kHeads);
  using Join = Joined<kDim, kHeads>;
  if (lane < 2) parts[2 * warp + lane].there = false;
  ptx::grid_dependency_wait();

  const int32_t rows_per_sequence = p.cache.heads * p.head_blocks;
  // The tokens of sequence b that are seen, from `begin` to the one returned; steps count from a
  // multiple of kStep.
  auto extent = [&](int32_t b, int32_t& begin) {
    const int32_t length = max(0, min(load_arg(p.lengths + b), p.capacity));
    begin = p.window > 0 && length > p.window ? length - p.window : 0;
    return length;
  };
  auto steps_between = [&](int32_t begin, int32_t end) { return (end - begin / L::kStep * L::kStep + L::kStep - 1) / L::kStep; };
  auto steps_of = [&](int32_t b) {
    int32_t begin;
    const int32_t end = extent(b, begin);
    return steps_between(begin, end);
  };

  // Where the warp's share begins: a scan over the sequences' steps, each warp for itself (with barriers
  // between four of them it took twice the time).
  const int32_t per_lane = (p.batch + 31) / 32;
  const int32_t b0 = min(p.batch, lane * per_lane), b1 = min(p.batch, b0 + per_lane);
  auto sum_up = [&](int64_t value) {  // inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t below = __shfl_up_sync(0xffffffffu, value, d);
      if (lane >= d) value += below;
    }
    return value;
  };
  int64_t mine = 0;
  int32_t most = 0;
#pragma unroll 1
  for (int32_t b = b0; b < b1; ++b) {
    const int32_t steps = steps_of(b);
    mine += static_cast<int64_t>(steps) * rows_per_sequence;
    most = max(most, steps);
  }
  int64_t upto = sum_up(mine);
  const int64_t before = upto - mine;
  const int64_t total = __shfl_sync(0xffffffffu, upto, 31);
  bool aligned = static_cast<int64_t>(p.batch) * rows_per_sequence <= gridDim.x;
  int64_t share = max(quotient(total + gridDim.x * kWarps - 1, gridDim.x * kWarps), static_cast<int64_t>(1));
  // Where there are few rows they stay in one lot each, if the longest then takes its warps no longer than equal
  // lots and a join with other lots, which is as long as four steps of 16 tokens.  Else each is cut into lots of its
  // own, as short as there are CTAs for all of them, or, where they would be kCut steps longer than equal lots, the
  // steps of all rows are numbered through.  (64 + 8 heads of 128 in BF16, 24 sequences with a window of 1000 tokens: lots
  // of their own 25.4 us, equal ones 29.3; 20 of them 25.0 and 26.4; 37 of up to 2000 tokens 44.4 and 46.7.  37 with a
  // window of 1000, 12 heads of 64, codes: whole 19.2, in equal lots 23.5.)
  const int32_t longest = __reduce_max_sync(0xffffffffu, most), whole = (longest + kWarps - 1) / kWarps;
  constexpr int32_t kAlone = L::kStep == 16 ? 4 : 3, kCut = L::kStep == 16 ? 16 : 6;
  if (aligned && whole < share + kAlone) share = max(share, static_cast<int64_t>(whole));
  const auto piece_for = [&](int64_t steps) { return static_cast<int32_t>(min(steps * kWarps, static_cast<int64_t>(1) << 30)); };
  int32_t piece = piece_for(share);  // a lot's steps
  int64_t lots = quotient(total + piece - 1, piece);
  auto pieces_of = [&](int32_t b) { return (steps_of(b) + piece - 1) / piece; };
  if (aligned) {
    int32_t longer = 0;
#pragma unroll 1
    do {
      piece = piece_for(share + longer);
      mine = 0;
#pragma unroll 1
      for (int32_t b = b0; b < b1; ++b) mine += static_cast<int64_t>(pieces_of(b)) * rows_per_sequence;
      lots = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(mine));
    } while (lots > gridDim.x && ++longer < kCut);
    aligned = lots <= gridDim.x;
    if (aligned) {
      share += longer;
      upto = sum_up(mine);
    } else {
      mine = upto - before;
      piece = piece_for(share);
      lots = quotient(total + piece - 1, piece);
    }
  }

  // Sequences with nothing to attend to, and lengths that the table cannot hold.
#pragma unroll 1
  for (int32_t b = blockIdx.x; b < p.batch; b += gridDim.x) {
    if (threadIdx.x == 0 && p.status != nullptr && load_arg(p.lengths + b) > p.capacity) atomicOr(p.status, kStatusIndex);
    if (steps_of(b) != 0) continue;
    const int64_t row = static_cast<int64_t>(b) * p.heads;
#pragma unroll 1
    for (int32_t i = threadIdx.x; i < p.heads * (kDim / 8); i += kThreads) {
      *reinterpret_cast<uint4*>(p.out + row * kDim + 8 * static_cast<int64_t>(i)) = make_uint4(0, 0, 0, 0);
    }
    if (p.lse != nullptr) {
#pragma unroll 1
      for (int32_t h = threadIdx.x; h < p.heads; h += kThreads) p.lse[row + h] = -INFINITY;
    }
  }
  const int32_t lot = blockIdx.x;
  if (lot >= lots) return;

  uint8_t* const ring = smem + warp * (L::kStages * L::kStageBytes);
  const uint32_t ring_addr = ptx::smem_u32(ring);
  float* const stash = p.partials + (kSlots * static_cast<int64_t>(gridDim.x) + blockIdx.x * kWarps + warp) * kPartFloats;

  // A place in the numbering: a row, its tokens and the next of its steps.
  struct Cursor {
    int32_t b, row, begin, end, token, left;
  };
  Cursor at;
  int32_t steps, row_first_lot = 0, row_lots = 0;
  const int64_t first_step = lot * static_cast<int64_t>(piece) + warp * share;
  {
    // (the warp's first step or, aligned, the lot)
    const int64_t wanted = aligned ? lot : min(first_step, total - 1);
    int32_t b = 0;
    int64_t base = upto - mine;
    const bool here = wanted >= base && wanted < upto;
    if (here) {
#pragma unroll 1
      for (b = b0; b < b1; ++b) {
        const int64_t count = static_cast<int64_t>(aligned ? pieces_of(b) : steps_of(b)) * rows_per_sequence;
        if (wanted < base + count) break;
        base += count;
      }
    }
    const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    at.b = __shfl_sync(0xffffffffu, b, from);
    base = __shfl_sync(0xffffffffu, base, from);
    at.end = extent(at.b, at.begin);
    const int32_t per_row = steps_between(at.begin, at.end);
    int32_t done;
    if (aligned) {
      row_lots = (per_row + piece - 1) / piece;
      const int32_t inside = static_cast<int32_t>(wanted - base);
      at.row = inside / row_lots;
      row_first_lot = lot - inside % row_lots;
      done = (inside % row_lots) * piece + warp * static_cast<int32_t>(share);
      steps = max(0, min(static_cast<int32_t>(share), per_row - done));
    } else {
      at.row = static_cast<int32_t>(quotient(wanted - base, per_row));
      done = static_cast<int32_t>(wanted - base - static_cast<int64_t>(at.row) * per_row);
      steps = static_cast<int32_t>(max(static_cast<int64_t>(0), min(share, total - first_step)));
    }
    at.token = (at.begin / L::kStep + done) * L::kStep;
    at.left = per_row - done;
  }
  if (steps > 0) {
    auto enter = [&](Cursor& c) {  // the first step of row c.row of sequence c.b, or of the next with tokens
      if (c.row == rows_per_sequence) {
        c.row = 0;
        do {
          c.end = extent(++c.b, c.begin);
        } while (c.end == 0);
      }
      c.token = c.begin / L::kStep * L::kStep;
      c.left = (c.end - c.token + L::kStep - 1) / L::kStep;
    };
    Cursor ahead = at;  // of the loads
    int32_t to_load = steps;
    int32_t load_stage = 0;

    // Pages are looked up a step before they are needed: that of a lane's own token or, where pages hold
    // whole groups of 16 tokens (p.whole_groups), of the first token of its group.
    constexpr int kPieces = L::kRow / 16;
    constexpr int kCopies = L::kStep * kPieces / 32;
    static_assert(16 * kPieces % 32 == 0, "whole warps");
    const int32_t own = lane % L::kStep;
    int32_t ref_page = 0, ref_place = -1;  // place -1: no token
    // What follows from the row: its part of the table and its head's offsets, in units of 16 bytes and in floats.
    const int32_t* row_table;
    uint64_t row_offset, row_scale = 0;
    auto enter_row = [&]() {
      const uint32_t kv_head = p.head_blocks == 1 ? ahead.row : ahead.row / p.head_blocks;
      row_table = p.tables + ahead.b * p.table_stride;
      row_offset = static_cast<uint64_t>(kv_head) * p.cache.head16;
      if constexpr (kCodes) row_scale = static_cast<uint64_t>(kv_head) * static_cast<uint32_t>(p.cache.scale_head);
    };
    auto look_up = [&]() {
      if (to_load == 0) return;
      const int32_t token = ahead.token + (p.whole_groups ? own / 16 * 16 : own);
      ref_place = -1;
      if (token < ahead.end && token + (p.whole_groups ? 15 : 0) >= ahead.begin) {
        const uint32_t index = p.cache.page_size.div(token);
        ref_place = token - index * p.cache.page_size.d;
        ref_page = load_arg(row_table + index);
      }
    };
    auto load = [&]() {
      if (to_load == 0) return;
      const uint32_t stage = ring_addr + load_stage * L::kStageBytes;
      load_stage = load_stage + 1 == L::kStages ? 0 : load_stage + 1;
      const bool there = ref_place >= 0 && static_cast<uint32_t>(ref_page) < static_cast<uint32_t>(p.cache.num_pages);
      if (ref_place >= 0 && !there && p.status != nullptr) atomicOr(p.status, kStatusIndex);
      const uint32_t page = ref_page, place = ref_place;
      const int64_t offset = there ? static_cast<int64_t>(row_offset + static_cast<uint64_t>(page) * p.cache.page16 + static_cast<uint64_t>(place) * p.cache.token16) << 4 : -1;
      const bool full = ahead.token >= ahead.begin && ahead.token + L::kStep <= ahead.end && __all_sync(0xffffffffu, there);
      if (p.whole_groups && full && p.cache.token == L::kRow) {
        // rows of a group follow one another
#pragma unroll
        for (int g = 0; g < L::kStep / 16; ++g) {
          const int64_t from = L::kStep == 16 ? offset : __shfl_sync(0xffffffffu, offset, 16 * g);
          const uint8_t* k = p.cache.k + from + lane * 16;
          const uint8_t* v = p.cache.v + from + lane * 16;
#pragma unroll
          for (int i = 0; i < kPieces / 2; ++i) {
            const int at_piece = i * 32 + lane, row = 16 * g + at_piece / kPieces, column = at_piece % kPieces;
            const uint32_t dst = stage + row * L::kPitch + column * 16;
            cp_async_16_all(dst, k + i * 512);
            cp_async_16_all(dst + L::kStep * L::kPitch, v + i * 512);
          }
        }
      } else {
        const int32_t stride = static_cast<int32_t>(p.cache.token);  // (in groups: fits)
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int at_piece = i * 32 + lane, row = at_piece / kPieces, column = at_piece % kPieces;
          int64_t from = __shfl_sync(0xffffffffu, offset, p.whole_groups ? row / 16 * 16 : row);
          const bool seen = from >= 0 && ahead.token + row >= ahead.begin && ahead.token + row < ahead.end;
          if (p.whole_groups) from += static_cast<int64_t>(row % 16) * stride;
          from = seen ? from + column * 16 : 0;
          const uint32_t dst = stage + row * L::kPitch + column * 16;
          ptx::cp_async_16(dst, p.cache.k + from, seen);
          ptx::cp_async_16(dst + L::kStep * L::kPitch, p.cache.v + from, seen);
        }
      }
      if constexpr (kCodes) {
        const bool seen = there && ahead.token + own >= ahead.begin && ahead.token + own < ahead.end;
        const uint64_t from = seen ? row_scale + static_cast<uint64_t>(page) * static_cast<uint32_t>(p.cache.scale_page) +
                                         static_cast<uint64_t>(place + (p.whole_groups ? own % 16 : 0)) * static_cast<uint32_t>(p.cache.scale_token)
                                   : 0;
        const uint32_t dst = stage + 2 * L::kStep * L::kPitch + own * 4;
        if (lane < L::kStep) {
          cp_async_4(dst, p.cache.k_scale + from, seen);
          cp_async_4(dst + L::kStep * 4, p.cache.v_scale + from, seen);
        }
      }
      --to_load;
      ahead.token += L::kStep;
      if (--ahead.left == 0 && to_load > 0) {
        ++ahead.row;
        enter(ahead);
        enter_row();
      }
    };

    enter_row();
    look_up();
#pragma unroll
    for (int s = 0; s < L::kStages - 1; ++s) {
      load();
      look_up();
      ptx::cp_async_commit();
    }

    uint32_t qf[kChunks][kTiles][2];
    float start[kTiles][2] = {};
    float of_scores = p.scale, of_codes = 1.0f;  // factors of the scores
    // A lane's heads are 8 n + 2 q4 and the next; of the dims it has rows r8 and r8 + 8 of each chunk.
    float out[kChunks][kTiles][4], top[kTiles][2], sum[kTiles][2];
    bool began = at.token > at.begin;  // in an earlier share
    bool fresh = true;
    int32_t stage_index = 0;

    for (int32_t step = 0; step < steps; ++step) {
      if (fresh) {
        // The queries' fragments: head 8 n + r8; codes want the dims of a 16-byte piece in the order in
        // which its bytes lie in the lanes.
        fresh = false;
        const Row of(p, at.b, at.row);
        const int32_t heads = of.heads;
        const __nv_bfloat16* q = p.q + at.b * p.q_batch + (of.head0 - static_cast<int64_t>(at.b) * p.heads) * p.q_head;
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          const int head = 8 * n + r8;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int dim = 16 * c + (kCodes ? 4 * q4 + 2 * i : 2 * q4 + 8 * i);
              qf[c][n][i] = head < heads ? load_arg(reinterpret_cast<const uint32_t*>(q + head * p.q_head + dim)) : 0u;
            }
          }
#pragma unroll
          for (int c = 0; c < kChunks; ++c) out[c][n][0] = out[c][n][1] = out[c][n][2] = out[c][n][3] = 0.0f;
          top[n][0] = top[n][1] = -INFINITY;
          sum[n][0] = sum[n][1] = 0.0f;
        }
        if constexpr (kCodes) {
          // The largest magnitude among the row's heads, infinities and NaN left out (their heads are NaN).
          uint32_t most_of_two = 0;
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
#pragma unroll
              for (int i = 0; i < 2; ++i) most_of_two = __vmaxu2(most_of_two, qf[c][n][i] & 0x7FFF7FFFu);
            }
          }
          uint32_t largest = __reduce_max_sync(0xffffffffu, max(most_of_two & 0xFFFFu, most_of_two >> 16));
          if (largest >= 0x7F80u) {
            largest = 0;
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
              for (int c = 0; c < kChunks; ++c) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                  const uint32_t low = qf[c][n][i] & 0x7FFFu, high = qf[c][n][i] >> 16 & 0x7FFFu;
                  largest = max(largest, max(low < 0x7F80u ? low : 0u, high < 0x7F80u ? high : 0u));
                }
              }
            }
            largest = __reduce_max_sync(0xffffffffu, largest);
          }
          // It lies below 2^(biased exponent - 126).  The queries' factor is 2^up, in two where one BF16 number does
          // not hold it; that of the scores 2^(133 - up), in two that FP32 holds whatever it is.
          const int32_t up = 238 - max(static_cast<int32_t>(largest >> 7), 1), rest = 133 - up;
          const uint32_t factor = static_cast<uint32_t>(min(up, 127) + 127) * 0x00800080u;
          const uint32_t factor2 = static_cast<uint32_t>(max(up - 127, 0) + 127) * 0x00800080u;
          of_codes = power_of_two(rest >> 1);
          of_scores = p.scale * power_of_two(rest - (rest >> 1));
          constexpr uint32_t kMinusZero = 0x80008000u;
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            float all = 0.0f;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                qf[c][n][i] = bf16x2_fma(qf[c][n][i], factor, kMinusZero);
                if (up > 127) qf[c][n][i] = bf16x2_fma(qf[c][n][i], factor2, kMinusZero);
                all += bf16_lo(qf[c][n][i]) + bf16_hi(qf[c][n][i]);
              }
            }
            all += __shfl_xor_sync(0xffffffffu, all, 1);
            all += __shfl_xor_sync(0xffffffffu, all, 2);
            all *= -0x1p-126f;  // -128 codes
            start[n][0] = __shfl_sync(0xffffffffu, all, 8 * q4);
            start[n][1] = __shfl_sync(0xffffffffu, all, 8 * q4 + 4);
          }
        }
      }

      ptx::cp_async_wait_group<L::kStages - 2>();
      __syncwarp();
      load();
      look_up();
      ptx::cp_async_commit();

      const uint32_t stage = ring_addr + stage_index * L::kStageBytes;
      const float* const scales = reinterpret_cast<const float*>(ring + stage_index * L::kStageBytes + 2 * L::kStep * L::kPitch);
      stage_index = stage_index + 1 == L::kStages ? 0 : stage_index + 1;
      float s[kGroups][kTiles][4];
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) s[j][n][0] = s[j][n][2] = start[n][0], s[j][n][1] = s[j][n][3] = start[n][1];
        const uint32_t k_at = stage + (j * 16 + (lane & 15)) * L::kPitch + (lane >> 4) * 16;
        if constexpr (!kCodes) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t a[4];
            ldmatrix_x4_at(k_at + c * 32, a);
#pragma unroll
            for (int n = 0; n < kTiles; ++n) ptx::mma_m16n8k16(s[j][n], a, qf[c][n][0], qf[c][n][1]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t kf[4];
            ldmatrix_x4_at(k_at + c * 16, kf);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const uint32_t a[4] = {__byte_perm(kf[2 * i], 0, 0x4140), __byte_perm(kf[2 * i + 1], 0, 0x4140),
                                     __byte_perm(kf[2 * i], 0, 0x4342), __byte_perm(kf[2 * i + 1], 0, 0x4342)};
#pragma unroll
              for (int n = 0; n < kTiles; ++n) ptx::mma_m16n8k16(s[j][n], a, qf[c + i][n][0], qf[c + i][n][1]);
            }
          }
        }
      }
      // Scores times the scale and log2(e); minus infinity before the first and behind the last token.
      // A lane's tokens are r8 and r8 + 8 of each 16.
      float value_scale[kCodes ? kGroups : 1][2];
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float f = of_scores;
          if constexpr (kCodes) {
            f = f * scales[16 * j + 8 * i + r8] * of_codes;
            value_scale[j][i] = scales[L::kStep + 16 * j + 8 * i + r8];
          }
#pragma unroll
          for (int n = 0; n < kTiles; ++n) s[j][n][2 * i] *= f, s[j][n][2 * i + 1] *= f;
        }
      }
      if (at.token < at.begin || at.token + L::kStep > at.end) {
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int32_t token = at.token + 16 * j + 8 * i + r8;
            if (token < at.begin || token >= at.end) {
#pragma unroll
              for (int n = 0; n < kTiles; ++n) s[j][n][2 * i] = s[j][n][2 * i + 1] = -INFINITY;
            }
          }
        }
      }
      float high[kTiles][2];
      bool rises = false;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          high[n][i] = fmaxf(s[0][n][i], s[0][n][2 + i]);
#pragma unroll
          for (int j = 1; j < kGroups; ++j) high[n][i] = fmaxf(high[n][i], fmaxf(s[j][n][i], s[j][n][2 + i]));
          rises |= high[n][i] > top[n][i] + kSlack;
        }
      }
      if (__any_sync(0xffffffffu, rises)) {
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          float factor[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) high[n][i] = fmaxf(high[n][i], __shfl_xor_sync(0xffffffffu, high[n][i], d));
            const float next = fmaxf(top[n][i], high[n][i]);
            factor[i] = next == -INFINITY ? 1.0f : exp2_approx(top[n][i] - next);
            top[n][i] = next;
            sum[n][i] *= factor[i];
          }
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
#pragma unroll
            for (int i = 0; i < 4; ++i) out[c][n][i] *= factor[i & 1];
          }
        }
      }
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
        const float from[2] = {top[n][0] == -INFINITY ? 0.0f : top[n][0], top[n][1] == -INFINITY ? 0.0f : top[n][1]};
#pragma unroll
        for (int j = 0; j < kGroups; ++j) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[j][n][i] = exp2_approx(s[j][n][i] - from[i & 1]);
            sum[n][i & 1] += s[j][n][i];
            if constexpr (kCodes) s[j][n][i] *= value_scale[j][i >> 1];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kGroups; ++j) {
        // P of these 16 tokens in two parts, tokens along the lane's registers
        uint32_t two[2][kTiles][2];
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float x = s[j][n][2 * i], y = s[j][n][2 * i + 1];
            uint32_t coarse, fine;
            if constexpr (kCodes) {
              coarse = pack_bf16(x, y);
              fine = pack_bf16(x - bf16_lo(coarse), y - bf16_hi(coarse));
            } else {
              positive_parts(x, y, coarse, fine);
            }
            two[0][n][i] = transposed(coarse);
            two[1][n][i] = transposed(fine);
          }
        }
        auto multiply = [&](int c, const uint32_t (&a)[4]) {
#pragma unroll
          for (int n = 0; n < kTiles; ++n) {
            ptx::mma_m16n8k16(out[c][n], a, two[0][n][0], two[0][n][1]);
            ptx::mma_m16n8k16(out[c][n], a, two[1][n][0], two[1][n][1]);
          }
        };
        const uint32_t v_at = stage + L::kStep * L::kPitch + (j * 16 + (lane & 7) + ((lane >> 4) << 3)) * L::kPitch + ((lane >> 3) & 1) * 16;
        if constexpr (!kCodes) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            uint32_t a[4];
            ldmatrix_x4_trans(v_at + c * 32, a);
            multiply(c, a);
          }
        } else {
#pragma unroll
          for (int c = 0; c < kChunks; c += 2) {
            uint32_t vf[4];
            ldmatrix_x4_trans(v_at + c * 16, vf);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              // even dims of the piece, then the odd ones
              multiply(c + i, {two_codes(vf[i], 0x4240), two_codes(vf[i], 0x4341), two_codes(vf[2 + i], 0x4240),
                               two_codes(vf[2 + i], 0x4341)});
            }
          }
        }
      }

      at.token += L::kStep;
      --at.left;
      if (at.left != 0 && step + 1 < steps) continue;

      // The end of the row, or of the share.
      const bool ended = at.left == 0;
#pragma unroll
      for (int n = 0; n < kTiles; ++n) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) sum[n][i] += __shfl_xor_sync(0xffffffffu, sum[n][i], d);
        }
      }
      if (ended && !began) {
        const Row of(p, at.b, at.row);
        const int32_t heads = of.heads;
        const int64_t head0 = of.head0;
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
          const float rate[2] = {rate_of<kCodes>(sum[n][0]), rate_of<kCodes>(sum[n][1])};
          __nv_bfloat16* to = p.out + (head0 + 8 * n + r8) * kDim;
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
            // dims 2 q4 and 2 q4 + 1 of head r8, of each half of the chunk
            const uint32_t a = transposed(pack_bf16(out[c][n][0] * rate[0], out[c][n][1] * rate[1]));
            const uint32_t b = transposed(pack_bf16(out[c][n][2] * rate[0], out[c][n][3] * rate[1]));
            if (8 * n + r8 < heads) {
              if constexpr (!kCodes) {
                *reinterpret_cast<uint32_t*>(to + 16 * c + 2 * q4) = a;
                *reinterpret_cast<uint32_t*>(to + 16 * c + 2 * q4 + 8) = b;
              } else {
                *reinterpret_cast<uint2*>(to + 16 * c + 4 * q4) = make_uint2(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int head = 8 * n + 2 * q4 + i;
            if (p.lse != nullptr && r8 == 0 && head < heads) p.lse[head0 + head] = lse_of(top[n][i], sum[n][i]);
          }
        }
      } else {
        // (the ring is free where the share ends)
        if (!ended) ptx::cp_async_wait_group<0>();
        __syncwarp();
        float* const part = ended ? stash : reinterpret_cast<float*>(ring);
#pragma unroll
        for (int n = 0; n < kTiles; ++n) {
#pragma unroll
          for (int c = 0; c < kChunks; ++c) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              *reinterpret_cast<float2*>(part + (16 * c + 8 * i + r8) * kHeads + 8 * n + 2 * q4) = make_float2(out[c][n][2 * i], out[c][n][2 * i + 1]);
            }
          }
          if (r8 == 0) {
            *reinterpret_cast<float2*>(part + kDim * kHeads + 8 * n + 2 * q4) = make_float2(top[n][0], top[n][1]);
            *reinterpret_cast<float2*>(part + (kDim + 1) * kHeads + 8 * n + 2 * q4) = make_float2(sum[n][0], sum[n][1]);
          }
        }
        if (lane == 0) {
          Part part_of = {part, at.b, at.row, row_first_lot, row_lots, true, began};
          if (!aligned) {
            const int32_t per_row = steps_between(at.begin, at.end);
            const int64_t row_first = first_step + step + 1 - (per_row - at.left);
            part_of.first_lot = static_cast<int32_t>(quotient(row_first, piece));
            part_of.lots = static_cast<int32_t>(quotient(row_first + per_row - 1, piece)) - part_of.first_lot + 1;
          }
          parts[2 * warp + (ended ? 0 : 1)] = part_of;
        }
      }
      began = false;
      fresh = true;
      if (step + 1 < steps) {
        ++at.row;
        enter(at);
      }
    }
  }
  __syncthreads();

  // Joins.  First the lot's own: parts of one row are neighbours, and a part at an even place ends its row.
  auto slot_of = [&](int32_t of_lot, int32_t which) { return p.partials + (kSlots * static_cast<int64_t>(of_lot) + which) * kPartFloats; };
  int32_t pending[2] = {0, 0}, waiting = 0;
  uint32_t there = 0;
#pragma unroll
  for (int32_t j = 0; j < 2 * kWarps; ++j) there |= static_cast<uint32_t>(parts[j].there) << j;
#pragma unroll 1
  while (there != 0) {
    const int32_t first = __ffs(there) - 1;
    bool ended = false;
    Join joined;
#pragma unroll 1
    while (there != 0 && !ended) {
      const int32_t j = __ffs(there) - 1;
      joined.add(parts[j].at);
      ended = j % 2 == 0;
      there &= there - 1;
    }
    const bool began = parts[first].began, whole = ended && !began;
    if (!whole) pending[waiting++] = first;
    const Row of(p, parts[first].b, parts[first].row);
    joined.template give<kCodes>(p, of, whole ? nullptr : slot_of(lot, began ? kSlotInside : kSlotFirst));
  }
  if (waiting == 0) return;

  // Then with other lots' parts, by the last CTA to arrive, in the parts' order; it leaves the counts at
  // zero.  (The barrier and the release order the parts before the count.)
#pragma unroll 1
  for (; waiting > 0; --waiting) {
    const Part part = parts[pending[waiting - 1]];
    const RowJoin join(part.first_lot, part.lots);
    const int32_t begin = join.group_of(lot), of_group = join.group_lots(begin);
    const Row of(p, part.b, part.row);
#pragma unroll 1
    for (int level = of_group > 1 ? 0 : 1; level < 2; ++level) {
      const int32_t count = level == 0 ? of_group : join.groups();
      __syncthreads();
      if (threadIdx.x == 0) {
        const int shift = level == 1 ? kRowShift : kGroupShift;
        int32_t* const word = p.locks + part.first_lot + (level == 0 ? begin : 0);
        const int32_t before = atomic_add_acq_rel(word, 1 << shift) >> shift & (level == 1 ? (1 << 11) - 1 : (1 << 6) - 1);
        answer[level] = before == count - 1;
        if (before == count - 1) atomicSub(word, count << shift);
      }
      __syncthreads();
      if (!answer[level]) break;
      float* const to = level == 0 ? slot_of(part.first_lot + begin, kSlotGroup) : nullptr;
      join_parts<kDim, kCodes, kHeads, L::kSmem>(p, of, smem, count, to, [&](int32_t j) {
        const PartPlace at_part = level == 0 ? join.part(begin, j) : join.joined(j);
        return slot_of(at_part.lot, at_part.slot);
      });
    }
  }
}

struct Variant {
  void (*kernel)(AttentionParams);
  int smem, step, ctas;
};

template <int kDim, bool kCodes, int kTiles>
Variant variant() {
  using L = Layout<kDim, kCodes, kTiles>;
  return {paged_attention_kernel<kDim, kCodes, kTiles>, L::kSmem, L::kStep, L::kCtas};
}

template <int kDim>
Variant variant_of(bool codes, bool wide) {
  if (codes) return wide ? variant<kDim, true, 2>() : variant<kDim, true, 1>();
  return wide ? variant<kDim, false, 2>() : variant<kDim, false, 1>();
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
  const int ctas = device.sm_count * chord::kMaxCtasPerSm;
  return ctas < chord::kMaxCtas ? ctas : chord::kMaxCtas;
}

int64_t chord_b200_paged_attention_workspace_bytes(int64_t head_dim, int64_t group) {
  using namespace chord;
  DeviceInfo device;
  if (current_device_info(&device)) return -1;
  Variant v, w;  // of either type of cache
  if (!variant_for(head_dim, false, group > 8, &v) || !variant_for(head_dim, true, group > 8, &w)) {
    return fail(kInvalidArgument, "head_dim must be 64, 96, 128, 192 or 256"), -1;
  }
  const int ctas = device.sm_count * (v.ctas > w.ctas ? v.ctas : w.ctas);
  return 4 * workspace_floats(ctas < kMaxCtas ? ctas : kMaxCtas, static_cast<int>(head_dim), group > 8 ? 16 : 8);
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
  // No more CTAs than there can be shares.
  // (token numbers, those of the steps loaded ahead too, fit 32 bits)
  int64_t capacity = max_pages * cache->page_size;
  if (capacity > (1ll << 31) - 65536) capacity = (1ll << 31) - 65536;
  const int64_t longest = window > 0 && window < capacity ? window : capacity;
  const int64_t most = batch * cache->heads * head_blocks * (((longest + v.step - 1) / v.step + kWarps) / kWarps);
  int64_t ctas = static_cast<int64_t>(device.sm_count) * v.ctas;
  if (ctas > kMaxCtas) ctas = kMaxCtas;
  if (ctas > most) ctas = most;
  const int64_t need = 4 * workspace_floats(ctas, static_cast<int>(cache->head_dim), wide ? 16 : 8);
  CHORD_REQUIRE(num_locks >= ctas, "locks has %lld lock words, this launch needs %lld",
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
  p.whole_groups = cache->page_size % 16 == 0 && p.cache.token < (1ll << 31);
  CHORD_CUDA(launch_kernel(v.kernel, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), v.smem,
                           static_cast<cudaStream_t>(stream), kEarlyLaunch, p));
  return kOk;
}

}  // extern "C"
