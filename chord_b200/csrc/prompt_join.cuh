// How parts of prompt.cuh's items are joined.
#pragma once

#include "prompt.cuh"

namespace chord {

// Joins the parts of the items that CTAs' runs have cut: block (x, y) does what CTA x + 1 finds cut at its begin, 128
// rows and 8 values of each, where x was the first of them.  Parts in their order, so the same inputs give the same bits.
// Bounded by latency: 12 us (and 17 MB) after the 250 us of 9 prompts, 16 where the 37 tokens of shared prefixes are joined.
template <int kDim, bool kCodes>
__global__ void __launch_bounds__(kPromptTile) prompt_join_kernel(const __grid_constant__ PromptParams p) {
  constexpr int64_t kPart = prompt_part_floats<kDim, kCodes>();
  ptx::grid_dependency_wait();
  const PromptPlan plan = *p.plan;
  if (!plan.cut) return;
  const PromptStart at = p.cta_starts[blockIdx.x + 1], before = p.cta_starts[blockIdx.x];
  if (at.count == 0 || at.step == 0) return;
  if (before.head == at.head && before.item == at.item && before.step > 0) return;  // its begin lies further back
  const PromptItem it = p.items[at.item];
  const int tile = blockIdx.y / (kDim / 8), dim = blockIdx.y % (kDim / 8) * 8;
  const int32_t row = threadIdx.x, r = tile * kPromptTile + row;
  if (r >= it.rows) return;
  const int64_t end = at.head * plan.head_steps + it.first + it.steps;

  // Parts: the last one of this CTA, then the first ones of those up to the item's end.  The highest maximum first, then all
  // values as they come: no load waits for another's.
  const int32_t parts = static_cast<int32_t>(plan_quotient(end - 1, plan.share)) - blockIdx.x + 1;
  auto part_of = [&](int32_t i) {
    return p.parts + (2 * static_cast<int64_t>(blockIdx.x + i) + (i == 0 ? 1 : 0)) * kPart + static_cast<int64_t>(tile) * kPromptTile * (kDim + 2) + row * 4;
  };
  const int stats = kDim * kPromptTile - row * 3;
  float o[8] = {}, top = -INFINITY, sum = 0.0f;
#pragma unroll 4
  for (int32_t i = 0; i < parts; ++i) top = fmaxf(top, __ldcg(part_of(i) + stats));
  const float to = top == -INFINITY ? 0.0f : top;
#pragma unroll 4
  for (int32_t i = 0; i < parts; ++i) {
    const float* const part = part_of(i);
    const float weight = exp2_fast(__ldcg(part + stats) - to);
    const float l = __ldcg(part + stats + kPromptTile);
    const float4 a = __ldcg(reinterpret_cast<const float4*>(part + dim * kPromptTile));
    const float4 b = __ldcg(reinterpret_cast<const float4*>(part + (dim + 4) * kPromptTile));
    sum = fmaf(l, weight, sum);
    const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = fmaf(v[k], weight, o[k]);
  }
  const int32_t token = p.group.div(it.row0 + r);
  const int64_t head = static_cast<int64_t>(at.head) * p.group.d + (it.row0 + r - token * static_cast<int32_t>(p.group.d));
  const int64_t result = (it.begin + static_cast<int64_t>(token)) * p.heads + head;
  PromptRates(p, result, top, sum, kCodes ? 64.0f : 1.0f, dim == 0).write(p, result * kDim + dim, o);
}

}  // namespace chord
