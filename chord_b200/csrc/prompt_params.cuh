// What the kernels of prompt.cuh are given.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "../../include/chord_b200.h"
#include "common.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {

// The rows of two tiles (or one) of one sequence, for each of its key-value heads, and the tokens that any of them sees.
struct __align__(16) PromptItem {
  int32_t b, row0, rows, steps;          // at least one step
  int32_t lo, hi, begin, count;          // tokens; the sequence's first query token and how many it has
  int32_t length, both_ways;             // tokens in the cache, and those seen by all
  int32_t highest_lo[2], lowest_hi[2];   // of each tile's rows: between them every row sees every token
  int64_t first;                         // number of its first step among those of a key-value head
};
static_assert(sizeof(PromptItem) == 64, "read as four vectors");

// Where a CTA begins, and how many steps it takes.
struct PromptStart {
  int32_t head, item, step, pad;
  int64_t count;
  int64_t begin;  // the step's number among all
};

struct PromptPlan {
  int32_t items, cut;  // cut: the CTAs take equal runs of steps; else an item each
  int64_t head_steps;  // of one key-value head
  int64_t share;       // where cut: steps of a CTA
};

struct PromptParams {
  CUtensorMap k_map, v_map;  // [pages][heads][page_size][dim], boxes of `box` tokens, 64 elements or a row of codes
  CUtensorMap q_map;         // [tokens][heads][dim], boxes of 64 elements of a group's heads of 128 / group tokens
  Cache cache;
  const __nv_bfloat16* q;  // [tokens, heads, dim]
  int64_t q_token, q_head;
  const int32_t* tables;
  int64_t table_stride;
  const int32_t* lengths;   // [batch] tokens in the cache
  const int32_t* offsets;   // [batch + 1] first query token of each
  const int32_t* starts;    // [tokens] or null
  const int32_t* prefixes;  // [batch] or null
  const int32_t* own;       // [tokens] or null: each query token stands behind so many more tokens of its own
  const float* slopes;      // [heads] or null
  const float* extra;       // [tokens, heads, dim] or null: what the tokens' own parts gave, with
  const float* extra_lse;   // [tokens, heads]
  __nv_bfloat16* out;       // [tokens, heads, dim]
  float* lse;               // [tokens, heads] or null
  int32_t* status;
  PromptPlan* plan;
  PromptStart* cta_starts;  // [ctas]
  PromptItem* items;        // [max_items]
  int32_t* tiles_before;    // [batch]
  float* parts;             // [ctas][2][tiles][dim / 4][128][4] sums, then [128] maxima and [128] sums of weights
  float scale, cap;         // the scale times log2(e); the cap times log2(e), or zero
  float cap_scale;          // the scale / the cap
  int32_t batch, tokens, heads, kv_heads, capacity, own_capacity, window, max_items, ctas;
  int32_t box;         // tokens of a TMA box of keys and values, which divides pages and steps; zero (codes): loaded as they are turned
  int32_t head_step;   // from head to head in k_map and v_map: zero where all heads are one
  int32_t page_step;   // the same of pages
  bool q_boxes;        // queries by TMA
  bool out_32;         // out lies on 32 bytes
  bool self;           // the main kernel's CTAs make the plan, each for itself
  Divisor group;
};

constexpr int kPromptTile = 128;  // rows
// The tokens of a sequence that its i-th query token sees, and where it stands.
struct PromptView {
  int32_t lo, hi, position;
  __device__ __forceinline__ PromptView() : lo(0), hi(INT32_MAX), position(0) {}
  __device__ __forceinline__ PromptView(const PromptParams& p, const PromptItem& of, int32_t i) {
    if (p.own != nullptr) {
      position = of.length + max(0, min(load_arg(p.own + of.begin + i), p.own_capacity)) - 1;
      hi = of.length;
    } else {
      position = of.length - of.count + i;
      hi = max(max(position + 1, 0), of.both_ways);
    }
    lo = p.window > 0 ? max(0, position + 1 - p.window) : 0;
    if (p.starts != nullptr) lo = max(lo, load_arg(p.starts + of.begin + i));
  }
};

}  // namespace chord
