// How the work of prompt.cuh is dealt out.
#pragma once

#include "prompt_params.cuh"

namespace chord {

constexpr int32_t kPlanHeld = 1024;     // sequences and items that are kept in shared memory
// Steps that an item may take longer than its share before it is cut.  8 heads of 128 in BF16, one new token of one sequence after
// 128 tokens 9.7 us whole and 12.9 cut, after 512 15.3 and 15.5, after 1,024 22.3 and 17.6.  (Up to 16 instead of 4 steps: 16
// sequences after 640 tokens 18.5 us for 21.8, but one after 2,048 36.9 for 22.7.)
constexpr int32_t kPromptAlone = 4;

struct PromptPlanScratch {
  int64_t of_warps[32];
  int32_t longest_of[32];
  int32_t before[kPlanHeld];   // items of the sequences before each
  int4 sequences[kPlanHeld];   // begin, count, length, both_ways
  int32_t count, longest;
  int64_t steps;
};

// n / d for n, d >= 0, in 32 bits where they do.
__device__ __forceinline__ int64_t plan_quotient(int64_t n, int64_t d) {
  if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}

// A CTA of kThreads: the items of every sequence, the tokens that each of them sees, and where the main kernel's CTAs begin.
// Bounded by the latency of its loads, so sequences are kept in shared memory (with all of it in global memory the
// items of one sequence after another were some seven loads apart).
template <int kThreads>
struct PromptPlanner {
  static constexpr int kWarps = kThreads / 32;
  const PromptParams& p;
  PromptPlanScratch& s;
  const int32_t log_rows, log_tokens;  // of an item and of a step, both powers of two
  const int lane, warp;
  const bool by_token;  // an item's tokens do not follow from its first and last query token

  // The sum of `value` over the threads before this one, and of all.
  __device__ __forceinline__ int64_t sum_before(int64_t value, int64_t& all) {
    int64_t upto = value;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t below = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += below;
    }
    __syncthreads();  // (of_warps may still be read from the call before)
    if (lane == 31) s.of_warps[warp] = upto;
    __syncthreads();
    int64_t warps = lane < kWarps ? s.of_warps[lane] : 0;  // up to each one, inclusive
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t below = __shfl_up_sync(0xffffffffu, warps, d);
      if (lane >= d) warps += below;
    }
    all = __shfl_sync(0xffffffffu, warps, 31);
    const int64_t before = __shfl_sync(0xffffffffu, warps, max(warp - 1, 0));
    return (warp == 0 ? 0 : before) + upto - value;
  }

  __device__ __forceinline__ int4 load_sequence(int32_t b) const {
    const int32_t first = load_arg(p.offsets + b), last = load_arg(p.offsets + b + 1), tokens = load_arg(p.lengths + b);
    const int32_t prefix = p.prefixes == nullptr ? 0 : load_arg(p.prefixes + b);
    const bool wrong = tokens > p.capacity || first < 0 || last > p.tokens || last < first;
    int4 of;
    of.x = max(0, min(first, p.tokens));
    of.y = max(0, min(last, p.tokens) - of.x);
    of.z = max(0, min(tokens, p.capacity));
    of.w = min(prefix, of.z);
    if (wrong && p.status != nullptr) atomicOr(p.status, kStatusIndex);
    return of;
  }

  __device__ __forceinline__ PromptPlanner(const PromptParams& params, PromptPlanScratch& scratch, int32_t rows, int32_t tokens)
      : p(params), s(scratch), log_rows(rows), log_tokens(tokens), lane(threadIdx.x & 31), warp(threadIdx.x >> 5),
        by_token(params.starts != nullptr || (params.own != nullptr && params.window > 0)) {
    int64_t items = 0;
#pragma unroll 1
    for (int32_t b0 = 0; b0 < p.batch; b0 += kThreads) {
      const int32_t b = b0 + threadIdx.x;
      int64_t mine = 0;
      if (b < p.batch) {
        const int4 of = load_sequence(b);
        if (b < kPlanHeld) s.sequences[b] = of;
        mine = (static_cast<int64_t>(of.y) * p.group.d + (1 << log_rows) - 1) >> log_rows;
      }
      int64_t all;
      const int64_t before = items + sum_before(mine, all);
      if (b < p.batch) {
        const int32_t number = static_cast<int32_t>(min(before, static_cast<int64_t>(p.max_items)));
        if (b < kPlanHeld) s.before[b] = number; else p.tiles_before[b] = number;
      }
      items += all;
    }
    if (threadIdx.x == 0) {
      // (more only where offsets fall)
      s.count = static_cast<int32_t>(min(items, static_cast<int64_t>(p.max_items)));
      if (items > p.max_items && p.status != nullptr) atomicOr(p.status, kStatusIndex);
    }
    __syncthreads();
  }

  __device__ __forceinline__ int32_t before(int32_t b) const { return b < kPlanHeld ? s.before[b] : p.tiles_before[b]; }

  // An item but for its first step's number.  by_token: by eight lanes, number `part` of them.
  static constexpr int kSome = 8;
  __device__ __forceinline__ PromptItem make(int32_t item, int part) const {
    int32_t low = 0, high = p.batch - 1;  // the last sequence with before(b) <= item
    while (low < high) {
      const int32_t middle = (low + high + 1) / 2;
      if (before(middle) <= item) low = middle; else high = middle - 1;
    }
    const int4 of = low < kPlanHeld ? s.sequences[low] : load_sequence(low);
    PromptItem it;
    it.b = low;
    it.begin = of.x, it.count = of.y, it.length = of.z, it.both_ways = of.w;
    const int64_t row0 = static_cast<int64_t>(item - before(low)) << log_rows;
    const int64_t rows = min(static_cast<int64_t>(1 << log_rows), static_cast<int64_t>(it.count) * p.group.d - row0);
    it.row0 = static_cast<int32_t>(row0);
    it.rows = static_cast<int32_t>(max(rows, static_cast<int64_t>(0)));
    int32_t lo = INT32_MAX, hi = 0;
#pragma unroll
    for (int tile = 0; tile < 2; ++tile) {
      int32_t highest_lo = 0, lowest_hi = INT32_MAX;
      const int32_t r0 = it.row0 + tile * kPromptTile, r1 = min(it.row0 + it.rows, r0 + kPromptTile) - 1;
      if (r0 <= r1) {
        const int32_t t0 = p.group.div(r0), t1 = p.group.div(r1);
        if (by_token) {
#pragma unroll 2
          for (int32_t i = t0 + part; i <= t1; i += kSome) {
            const PromptView v(p, it, i);
            highest_lo = max(highest_lo, v.lo);
            lowest_hi = min(lowest_hi, v.hi);
            if (v.hi > v.lo) lo = min(lo, v.lo), hi = max(hi, v.hi);
          }
        } else {
          const PromptView a(p, it, t0), z(p, it, t1);  // (neither bound falls from token to token)
          highest_lo = z.lo;
          lowest_hi = a.hi;
          if (z.hi > a.lo) lo = min(lo, a.lo), hi = max(hi, z.hi);
        }
      }
      it.highest_lo[tile] = highest_lo;
      it.lowest_hi[tile] = lowest_hi;
    }
    if (by_token) {
#pragma unroll
      for (int d = 1; d < kSome; d <<= 1) {
        lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, d));
        hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, d));
#pragma unroll
        for (int tile = 0; tile < 2; ++tile) {
          it.highest_lo[tile] = max(it.highest_lo[tile], __shfl_xor_sync(0xffffffffu, it.highest_lo[tile], d));
          it.lowest_hi[tile] = min(it.lowest_hi[tile], __shfl_xor_sync(0xffffffffu, it.lowest_hi[tile], d));
        }
      }
    }
    it.lo = hi > lo ? lo : 0;
    it.hi = hi > lo ? hi : 0;
    it.steps = max(1, ((it.hi + (1 << log_tokens) - 1) >> log_tokens) - (it.lo >> log_tokens));
    it.first = 0;
    return it;
  }

  // Gives every item, with its first step's number, to keep(number, item), and counts steps.
  template <typename Keep>
  __device__ __forceinline__ void items(Keep keep) {
    // (eight lanes to an item, or one)
    const int32_t some = by_token ? kSome : 1, at_once = kThreads / some;
    int64_t steps = 0;
    int32_t longest = 0;
#pragma unroll 1
    for (int32_t i0 = 0; i0 < s.count; i0 += at_once) {
      const int32_t item = i0 + threadIdx.x / some;
      PromptItem it = make(min(item, s.count - 1), threadIdx.x % some);
      const bool mine = item < s.count && threadIdx.x % some == 0;
      int64_t all;
      it.first = steps + sum_before(mine ? it.steps : 0, all);
      if (mine) {
        keep(item, it);
        longest = max(longest, it.steps);
      }
      steps += all;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) s.longest_of[warp] = longest;
    __syncthreads();
    longest = __reduce_max_sync(0xffffffffu, lane < kWarps ? s.longest_of[lane] : 0);
    if (threadIdx.x == 0) {
      s.steps = steps;
      s.longest = longest;
    }
    __syncthreads();
  }

  // An item to a CTA where there are no more of them and the longest one takes hardly longer than equal runs and a join.
  __device__ __forceinline__ PromptPlan plan() const {
    const int64_t total = s.steps * p.kv_heads, runs = static_cast<int64_t>(s.count) * p.kv_heads;
    PromptPlan plan;
    plan.items = s.count;
    plan.head_steps = s.steps;
    plan.share = plan_quotient(total + p.ctas - 1, p.ctas);
    plan.cut = runs > p.ctas || s.longest > plan.share + kPromptAlone;
    return plan;
  }

  template <typename First, typename Steps>
  __device__ __forceinline__ PromptStart start(const PromptPlan& plan, int32_t cta, First first_of, Steps steps_of) const {
    const int64_t total = plan.head_steps * p.kv_heads;
    PromptStart at = {0, 0, 0, 0, 0, 0};
    if (!plan.cut) {
      if (cta < static_cast<int64_t>(plan.items) * p.kv_heads) {
        at.head = cta / plan.items;
        at.item = cta % plan.items;
        at.count = steps_of(at.item);
        at.begin = at.head * plan.head_steps + first_of(at.item);
      }
    } else if (cta * plan.share < total) {
      at.begin = cta * plan.share;
      at.count = min(plan.share, total - at.begin);
      at.head = static_cast<int32_t>(plan_quotient(at.begin, plan.head_steps));
      const int64_t wanted = at.begin - at.head * plan.head_steps;
      int32_t low = 0, high = plan.items - 1;  // the last item that begins there or before
      while (low < high) {
        const int32_t middle = (low + high + 1) / 2;
        if (first_of(middle) <= wanted) low = middle; else high = middle - 1;
      }
      at.item = low;
      at.step = static_cast<int32_t>(wanted - first_of(low));
    }
    return at;
  }
};

}  // namespace chord
