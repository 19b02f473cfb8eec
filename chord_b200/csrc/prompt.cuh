// Attention of many query tokens over pages of keys and values on tcgen05: prompts, and the part of a batch's
// sequences that they share.
//
//   x = scale q . k,  x = cap tanh(x / cap),  x -= slope_h |p - j|,  out = sum_j softmax_j(x) v_j
//
// over the tokens j in [lo, hi) that a query token at position p sees.  A row is one query token and one of the heads
// that share a key-value head; 128 rows are the M dimension of the products.  An item is two such tiles (one where
// heads are wider than 128: 512 columns of tensor memory hold no more) of one sequence and key-value head, a step kN
// tokens of its keys and values.  A CTA takes a run of steps, which may begin and end inside items.
//
//   S = Q K^T      both from shared memory, K-major; FP32 in tensor memory
//   P = exp2(x - m) in BF16 over S, by one thread per row; m is raised, and O scaled, only where a score passes it by
//                  more than 2^kSlack
//   O += P V       P from tensor memory, V from shared memory as it lies there (MN-major)
//
// P is rounded to BF16 (2^-9 of each weight, at random, as the values it multiplies are), its sum is added up before
// that in FP32.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>

#include "../../include/chord_b200.h"
#include "common.h"
#include "kv_cache.cuh"
#include "warp_ops.cuh"

namespace chord {

// Two row tiles' worth of rows of one sequence, for each of its key-value heads, and the tokens that any of them sees.
struct PromptItem {
  int32_t b, row0, rows;
  int32_t lo, hi;
  int32_t steps;  // at least one
  int64_t first;  // number of its first step among those of a key-value head
};

// Where a CTA begins, and how many steps it takes.
struct PromptStart {
  int32_t head, item, step, pad;
  int64_t count;
  int64_t begin;  // the step's number among all
};

struct PromptPlan {
  int32_t items, cut;  // cut: the CTAs take equal runs of steps; else an item each
  int64_t head_steps;  // of one key-value head
};

struct PromptParams {
  CUtensorMap k_map, v_map;  // [pages][heads][page_size][dim], boxes of 64 elements of `box` tokens
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
  float* parts;             // [ctas][2][tiles][dim / 4][128][4] sums, then [ctas][2][tiles][2][128] maxima and sums
  float scale, cap;         // the scale times log2(e); the cap times log2(e), or zero
  float cap_scale;          // 2 log2(e) scale / cap
  int32_t batch, tokens, heads, kv_heads, capacity, own_capacity, window, max_items, ctas;
  int32_t box;    // tokens of a TMA box of keys and values, which divides pages and steps; zero: loaded by cp.async
  bool q_boxes;   // queries by TMA
  Divisor group;
};

constexpr int kPromptTile = 128;     // rows
constexpr int kPromptThreads = 512;  // two groups of four warps for the rows, one that loads, one of which a warp issues

template <int kDim, bool kCodes>
struct PromptLayout {
  static constexpr bool kTwo = kDim <= 128;  // row tiles of an item
  static constexpr int kTiles = kTwo ? 2 : 1;
  static constexpr int kN = kTwo ? 128 : 64;                // tokens of a step
  static constexpr int kBlocks = (kDim + 63) / 64;          // of 64 elements, 128 bytes
  static constexpr int kQBytes = kTiles * kBlocks * kPromptTile * 128;
  static constexpr int kSlotBytes = kBlocks * kN * 128;     // keys or values of a step
  static constexpr int kScaleBytes = kCodes ? 2 * kN * 4 : 0;
  static constexpr int kControl = 512;
  static constexpr int kFit = (232448 - kControl - kQBytes) / (kSlotBytes + kScaleBytes);
  static constexpr int kRing = kFit > 8 ? 8 : kFit;
  static constexpr int kSmem = kQBytes + kRing * (kSlotBytes + kScaleBytes) + kControl;
  static constexpr uint32_t kOutColumn = kTwo ? 256 : 128;  // of tensor memory; the scores' buffers come first
  // Of a CTA launched with 128 registers a thread: what the rows' warps have, and the others.
  static constexpr int kRowRegs = kCodes ? 168 : 184, kOtherRegs = kCodes ? 88 : 72;
  static_assert(kRing >= 4, "keys and values of two steps");
};

// Rows of a part of an item, as they lie in PromptParams::parts.
template <int kDim, bool kCodes>
__host__ __device__ constexpr int64_t prompt_part_floats() {
  return static_cast<int64_t>(PromptLayout<kDim, kCodes>::kTiles) * kPromptTile * (kDim + 2);
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The tokens of a sequence that its query token sees, and where it stands.
struct PromptView {
  int32_t lo, hi, position;
};

struct PromptSequence {
  int32_t begin, count, length, both_ways;  // query tokens, tokens in the cache, those seen by all
  __device__ __forceinline__ PromptSequence(const PromptParams& p, int32_t b) {
    begin = max(0, min(load_arg(p.offsets + b), p.tokens));
    count = max(0, min(load_arg(p.offsets + b + 1), p.tokens) - begin);
    length = max(0, min(load_arg(p.lengths + b), p.capacity));
    both_ways = p.prefixes == nullptr ? 0 : min(load_arg(p.prefixes + b), length);
  }
  __device__ __forceinline__ PromptView view(const PromptParams& p, int32_t i) const {
    PromptView v;
    if (p.own != nullptr) {
      v.position = length + max(0, min(load_arg(p.own + begin + i), p.own_capacity)) - 1;
      v.hi = length;
    } else {
      v.position = length - count + i;
      v.hi = max(max(v.position + 1, 0), both_ways);
    }
    v.lo = p.window > 0 ? max(0, v.position + 1 - p.window) : 0;
    if (p.starts != nullptr) v.lo = max(v.lo, load_arg(p.starts + begin + i));
    return v;
  }
};

// A warp's walk over its CTA's steps.
struct PromptWalk {
  int64_t left;
  int32_t head, item, step, items;
  __device__ __forceinline__ explicit PromptWalk(const PromptParams& p) {
    const PromptStart* const s = p.cta_starts + blockIdx.x;
    items = p.plan->items;
    left = s->count;
    head = s->head;
    item = s->item;
    step = s->step;
  }
  __device__ __forceinline__ int32_t here(const PromptItem& it) const {
    return static_cast<int32_t>(min(left, static_cast<int64_t>(it.steps - step)));
  }
  __device__ __forceinline__ void next(int32_t n) {
    left -= n;
    step = 0;
    if (++item == items) item = 0, ++head;
  }
};

__device__ __forceinline__ PromptItem load_item(const PromptParams& p, int32_t item) {
  const int4* const from = reinterpret_cast<const int4*>(p.items + item);
  const int4 a = __ldcg(from), b = __ldcg(from + 1);
  PromptItem it;
  it.b = a.x, it.row0 = a.y, it.rows = a.z, it.lo = a.w;
  it.hi = b.x, it.steps = b.y;
  it.first = 0;
  return it;
}

enum PromptStatus : int32_t { kPromptLoadTimeout = 1, kPromptIssueTimeout = 2, kPromptRowTimeout = 8 };

struct __align__(16) PromptControl {
  uint64_t q_full, q_empty, drained;
  uint64_t kv_full[8], kv_empty[8];
  uint64_t s_full[2], p_full[2], o_done[2], scanned[2];
  uint32_t tmem, abort;
  uint32_t skip[2];   // the product of P and V is made by the rows' warps
  uint32_t odd[2];    // number of the last look at values that found infinities or NaN
};
static_assert(sizeof(PromptControl) <= 512, "its place");

// Adds what a query token's own part gave, and writes a row's result.  o: its values from `dim0` on, not yet divided.
template <int kCount>
__device__ __forceinline__ void prompt_finish(const PromptParams& p, int64_t row, int dim0, int dims, float* o, float top, float sum,
                                              float unit, bool first) {
  float all = sum, weight = unit;
  if (p.extra != nullptr) {
    // (both parts' sums, relative to the larger one)
    const float other = load_arg(p.extra_lse + row) * 1.4426950408889634f;
    const float mine = sum == 0.0f ? -INFINITY : top;
    const float most = fmaxf(mine, other);
    const float to = most == -INFINITY ? 0.0f : most;
    const float w = exp2_fast(mine - to), e = exp2_fast(other - to);
    all = sum * w + e;
    weight = unit * w;
    const float* const from = p.extra + row * dims + dim0;
#pragma unroll
    for (int i = 0; i < kCount; i += 4) {
      const float4 x = load_arg(reinterpret_cast<const float4*>(from + i));
      o[i] = fmaf(o[i], weight, x.x * e);
      o[i + 1] = fmaf(o[i + 1], weight, x.y * e);
      o[i + 2] = fmaf(o[i + 2], weight, x.z * e);
      o[i + 3] = fmaf(o[i + 3], weight, x.w * e);
    }
    weight = 1.0f;
    top = to;
  }
  const float rate = all == 0.0f ? 0.0f : weight / all;
  uint4* const to = reinterpret_cast<uint4*>(p.out + row * dims + dim0);
#pragma unroll
  for (int i = 0; i < kCount; i += 8) {
    to[i / 8] = make_uint4(pack_bf16(o[i] * rate, o[i + 1] * rate), pack_bf16(o[i + 2] * rate, o[i + 3] * rate),
                           pack_bf16(o[i + 4] * rate, o[i + 5] * rate), pack_bf16(o[i + 6] * rate, o[i + 7] * rate));
  }
  if (first && p.lse != nullptr) p.lse[row] = all == 0.0f ? -INFINITY : (top + log2f(all)) * 0.693147180559945309f;
}

// The product of a tile's weights and values on the CUDA cores, for values among which are infinities or NaN that not all
// of its rows see: tokens of no weight are left out.  The scores lie in tensor memory at `s_at`; returns their sum.
template <int kDim, int kN>
__device__ __noinline__ float product_by_row(uint32_t s_at, uint32_t out_at, const uint8_t* v, float of_scores, float base, bool fresh) {
  float all = 0.0f;
#pragma unroll 1
  for (int dim = 0; dim < kDim; dim += 8) {
    float o[8];
    uint32_t bits[8];
    ptx::tmem_ld_32x32b_x8(out_at + dim, bits);
    ptx::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = fresh ? 0.0f : __uint_as_float(bits[i]);
    float sum = 0.0f;
#pragma unroll 1
    for (int t0 = 0; t0 < kN; t0 += 16) {
      uint32_t x[16];
      ptx::tmem_ld_32x32b_x16(s_at + t0, x);
      ptx::tmem_wait_ld();
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        const float e = exp2_fast(fmaf(__uint_as_float(x[t]), of_scores, base));
        sum += e;
        const int token = t0 + t;
        const uint4 w = *reinterpret_cast<const uint4*>(v + (dim / 64) * (kN * 128) + token * 128 + ((dim / 8 ^ token) & 7) * 16);
        if (e != 0.0f) {
          o[0] = fmaf(e, bf16_lo(w.x), o[0]), o[1] = fmaf(e, bf16_hi(w.x), o[1]);
          o[2] = fmaf(e, bf16_lo(w.y), o[2]), o[3] = fmaf(e, bf16_hi(w.y), o[3]);
          o[4] = fmaf(e, bf16_lo(w.z), o[4]), o[5] = fmaf(e, bf16_hi(w.z), o[5]);
          o[6] = fmaf(e, bf16_lo(w.w), o[6]), o[7] = fmaf(e, bf16_hi(w.w), o[7]);
        }
      }
      __syncwarp();
    }
    all = sum;
    ptx::tmem_st_32x32b_x8(out_at + dim, reinterpret_cast<const uint32_t*>(o));
    ptx::tmem_wait_st();
  }
  return all;
}

template <int kDim, bool kCodes, bool kBent>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_attention_kernel(const __grid_constant__ PromptParams p) {
  using L = PromptLayout<kDim, kCodes>;
  constexpr int kN = L::kN;
  constexpr int kRing = L::kRing;
  constexpr float kSlack = 8.0f;
  constexpr float kUnit = kCodes ? 64.0f : 1.0f;  // of values in shared memory (codes: (code - 128) / 64)
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const q_tile = smem;
  uint8_t* const slots = smem + L::kQBytes;
  float* const scales = reinterpret_cast<float*>(slots + kRing * L::kSlotBytes);  // [slot][of keys, of values][kN]
  PromptControl& c = *reinterpret_cast<PromptControl*>(smem + L::kSmem - L::kControl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t abort_at = ptx::smem_u32(&c.abort);
  uint32_t bad = 0;
  auto bar = [](const uint64_t& b) { return ptx::smem_u32(&b); };

  if ((ptx::smem_u32(smem) & 1023u) != 0) {  // (the tiles' swizzle counts from there)
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, kPromptIssueTimeout);
    return;
  }
  if (warp == 12) {
    ptx::tmem_alloc(bar(reinterpret_cast<const uint64_t&>(c.tmem)), 512);
    ptx::tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    ptx::mbar_init(bar(c.q_full), p.q_boxes ? 1 : p.box != 0 ? 3 : 4);
    ptx::mbar_init(bar(c.q_empty), 1);
    ptx::mbar_init(bar(c.drained), 1);
    for (int i = 0; i < 8; ++i) {
      ptx::mbar_init(bar(c.kv_full[i]), p.box != 0 ? 1 : 4);
      ptx::mbar_init(bar(c.kv_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(c.s_full[i]), 1);
      ptx::mbar_init(bar(c.p_full[i]), 4);
      ptx::mbar_init(bar(c.o_done[i]), 1);
      ptx::mbar_init(bar(c.scanned[i]), 4);
      c.skip[i] = 0;
      c.odd[i] = 0;
    }
    c.abort = 0;
    ptx::fence_barrier_init();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = c.tmem;
  ptx::grid_dependency_wait();

  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));

  if (warp >= 8 && warp < 12) {
    // ---- loads: queries once per item, keys and values step by step, each into a slot of the ring ----
    // By TMA where boxes of 8 tokens or more fit pages and steps: the first warp's lanes have a box each.  A step of
    // 128 tokens of 128 elements by cp.async takes its warps some 4700 cycles, the products 2000.  Boxes bring tokens
    // behind the last one with them; one outside the tokens that are seen, or whose page is not there, is asked for
    // behind the cache's last page, which gives zeros.
    const int w = warp - 8;
    const bool boxes = !kCodes && p.box != 0;
    constexpr int kOwn = kN / 4;  // tokens of a warp
    constexpr int kPieces = kDim * (kCodes ? 1 : 2) / 16;
    uint32_t slot = 0, slot_phase = 0, q_phase = 0;
    // Filled, but not yet said so: by cp.async, in order.
    uint32_t waiting[2] = {0, 0};
    auto publish = [&](uint32_t at) {
      ptx::fence_proxy_async();
      __syncwarp();
      ptx::mbar_arrive_lane0(at, lane);
    };
    auto flush = [&]() {
      ptx::cp_async_wait_group<0>();
      if (waiting[1] != 0) publish(waiting[1]);
      if (waiting[0] != 0) publish(waiting[0]);
      waiting[0] = waiting[1] = 0;
    };
    auto filled = [&](uint32_t at) {  // what has been issued since the last one
      ptx::cp_async_commit();
      if (waiting[1] != 0) {
        ptx::cp_async_wait_group<2>();
        publish(waiting[1]);
      }
      waiting[1] = waiting[0];
      waiting[0] = at;
    };
    auto wait_for = [&](uint32_t at, uint32_t parity) {
      if (__all_sync(0xffffffffu, ptx::mbar_try_wait<false>(at, parity))) return;
      flush();  // (who empties it may need what is on its way)
      ptx::mbar_wait_sticky<true>(at, parity, abort_at, bad);
    };
    auto advance = [&]() {
      if (++slot == kRing) slot = 0, slot_phase ^= 1;
    };

    PromptWalk walk(p);
    while (walk.left > 0 && bad == 0) {
      const PromptItem it = load_item(p, walk.item);
      const int32_t n = walk.here(it);
      const int32_t* const table = p.tables + it.b * p.table_stride;
      const int32_t token0 = (it.lo / kN + walk.step) * kN;
      const int64_t head_offset = static_cast<int64_t>(walk.head) * p.cache.head;
      const int32_t mine = boxes ? lane * p.box : w * kOwn + lane % kOwn;  // the token that the lane looks up
      const int32_t others = boxes ? p.box - 1 : 0;                        // and those with it
      int32_t page = 0, place = -1;
      auto look_up = [&](int32_t j) {
        const int32_t token = token0 + j * kN + mine;
        place = -1;
        if (j < n && token + others >= it.lo && token < it.hi && mine < kN) {
          const uint32_t index = p.cache.page_size.div(token);
          place = token - index * p.cache.page_size.d;
          page = load_arg(table + index);
        }
      };
      // The lane's token: its offset in bytes, negative for none.
      auto offset_of = [&]() {
        const bool there = place >= 0 && static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.num_pages);
        if (place >= 0 && !there && p.status != nullptr) atomicOr(p.status, kStatusIndex);
        return there ? static_cast<int64_t>(page) * p.cache.page + static_cast<int64_t>(place) * p.cache.token + head_offset : -1ll;
      };
      // Where the 16 bytes from element 8 * chunk of a token go.
      auto place_of = [](int token, int chunk) { return (chunk >> 3) * (kN * 128) + token * 128 + ((chunk ^ token) & 7) * 16; };
      auto load_rows = [&](const uint8_t* from, int64_t offset) {
        const uint32_t to = ptx::smem_u32(slots) + slot * L::kSlotBytes;
#pragma unroll
        for (int i = 0; i < kOwn * kPieces / 32; ++i) {
          const int at = i * 32 + lane, token = at / kPieces, piece = at % kPieces;
          const int64_t o = __shfl_sync(0xffffffffu, offset, token);
          ptx::cp_async_16(to + place_of(w * kOwn + token, piece), from + (o < 0 ? 0 : o + piece * 16), o >= 0);
        }
      };
      uint4 held[kCodes ? kOwn * kPieces / 32 : 1];
      auto fetch_codes = [&](const uint8_t* from, int64_t offset) {
        if constexpr (kCodes) {
#pragma unroll
          for (int i = 0; i < kOwn * kPieces / 32; ++i) {
            const int at = i * 32 + lane, token = at / kPieces, piece = at % kPieces;
            const int64_t o = __shfl_sync(0xffffffffu, offset, token);
            held[i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
            if (o >= 0) held[i] = load_once(from + o + piece * 16);
          }
        }
      };
      auto store_codes = [&]() {
        if constexpr (kCodes) {
          uint8_t* const to = slots + slot * L::kSlotBytes;
#pragma unroll
          for (int i = 0; i < kOwn * kPieces / 32; ++i) {
            const int at = i * 32 + lane, token = w * kOwn + at / kPieces, piece = at % kPieces;
            const uint32_t four[4] = {held[i].x, held[i].y, held[i].z, held[i].w};
            uint32_t v[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              constexpr uint32_t kOffset = 0xC000C000u;  // -128 / 64, twice
              v[2 * k] = bf16x2_fma(__byte_perm(four[k], 0, 0x4140), kTwo127, kOffset);
              v[2 * k + 1] = bf16x2_fma(__byte_perm(four[k], 0, 0x4342), kTwo127, kOffset);
            }
            *reinterpret_cast<uint4*>(to + place_of(token, 2 * piece)) = make_uint4(v[0], v[1], v[2], v[3]);
            *reinterpret_cast<uint4*>(to + place_of(token, 2 * piece + 1)) = make_uint4(v[4], v[5], v[6], v[7]);
          }
        }
      };
      auto load_boxes = [&](const CUtensorMap& map, uint32_t at, bool there) {
        if (lane == 0) ptx::mbar_arrive_expect_tx(at, L::kSlotBytes);
        __syncwarp();
        if (mine < kN) {
          const uint32_t to = ptx::smem_u32(slots) + slot * L::kSlotBytes + mine * 128;
#pragma unroll
          for (int b = 0; b < L::kBlocks; ++b) {
            ptx::tma_load_4d(to + b * (kN * 128), &map, at, 64 * b, there ? place : 0, walk.head, there ? page : p.cache.num_pages);
          }
        }
        __syncwarp();
      };
      auto load_query_boxes = [&]() {
        const PromptSequence of(p, it.b);
        const int tiles = L::kTwo && it.rows > kPromptTile ? 2 : 1;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(bar(c.q_full), tiles * (L::kBlocks * kPromptTile * 128));
          const int32_t token = of.begin + static_cast<int32_t>(p.group.div(it.row0)), per_tile = p.group.div(kPromptTile);
          for (int t = 0; t < tiles; ++t) {
#pragma unroll
            for (int b = 0; b < L::kBlocks; ++b) {
              ptx::tma_load_3d(ptx::smem_u32(q_tile) + (t * L::kBlocks + b) * (kPromptTile * 128), &p.q_map, bar(c.q_full), 64 * b,
                               walk.head * static_cast<int32_t>(p.group.d), token + t * per_tile);
            }
          }
        }
        __syncwarp();
      };
      auto load_queries = [&](int32_t of_warps, int32_t number) {  // as the number-th of so many warps
        const PromptSequence of(p, it.b);
        const uint32_t to = ptx::smem_u32(q_tile);
        constexpr int kQPieces = kDim / 8;
#pragma unroll 1
        for (int r0 = 32 * number; r0 < L::kTiles * kPromptTile; r0 += 32 * of_warps) {
          const int32_t r = it.row0 + r0 + lane;
          int64_t offset = -1;
          if (r < it.row0 + it.rows) {
            const int32_t i = p.group.div(r), h = r - i * p.group.d;
            offset = (of.begin + i) * p.q_token + (static_cast<int64_t>(walk.head) * p.group.d + h) * p.q_head;
          }
#pragma unroll 4
          for (int i = 0; i < kQPieces; ++i) {
            const int at = i * 32 + lane, row = at / kQPieces, piece = at % kQPieces, tile_row = r0 + row;
            const int64_t o = __shfl_sync(0xffffffffu, offset, row);
            const uint32_t dst = to + (tile_row / kPromptTile) * (L::kBlocks * kPromptTile * 128) + (piece >> 3) * (kPromptTile * 128) +
                                 (tile_row % kPromptTile) * 128 + ((piece ^ tile_row) & 7) * 16;
            ptx::cp_async_16(dst, p.q + (o < 0 ? 0 : o + piece * 8), o >= 0);
          }
        }
      };

      if (boxes) {
        if (w != 0) {
          if (!p.q_boxes) {
            wait_for(bar(c.q_empty), q_phase ^ 1);
            if (bad != 0) break;
            load_queries(3, w - 1);
            filled(bar(c.q_full));
            flush();
            q_phase ^= 1;
          }
          walk.next(n);
          continue;
        }
        look_up(0);
#pragma unroll 1
        for (int32_t j = 0; j < n; ++j) {
          const bool there = place >= 0 && static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.num_pages);
          if (place >= 0 && !there && p.status != nullptr) atomicOr(p.status, kStatusIndex);
          wait_for(bar(c.kv_empty[slot]), slot_phase ^ 1);
          if (bad != 0) break;
          load_boxes(p.k_map, bar(c.kv_full[slot]), there);
          advance();
          if (j == 0 && p.q_boxes) {
            wait_for(bar(c.q_empty), q_phase ^ 1);
            if (bad != 0) break;
            load_query_boxes();
            q_phase ^= 1;
          }
          wait_for(bar(c.kv_empty[slot]), slot_phase ^ 1);
          if (bad != 0) break;
          load_boxes(p.v_map, bar(c.kv_full[slot]), there);
          advance();
          look_up(j + 1);
        }
        walk.next(n);
        continue;
      }
      look_up(0);
#pragma unroll 1
      for (int32_t j = 0; j < n && bad == 0; ++j) {
        const int64_t offset = offset_of();
        float key_scale = 0.0f, value_scale = 0.0f;
        if constexpr (kCodes) {
          if (offset >= 0) {
            const int64_t at = page * p.cache.scale_page + place * p.cache.scale_token + walk.head * p.cache.scale_head;
            key_scale = load_arg(p.cache.k_scale + at);
            value_scale = load_arg(p.cache.v_scale + at);
          }
          fetch_codes(p.cache.k, offset);
        }
        look_up(j + 1);
        wait_for(bar(c.kv_empty[slot]), slot_phase ^ 1);
        if (bad != 0) break;
        if constexpr (kCodes) {
          store_codes();
          fetch_codes(p.cache.v, offset);
          publish(bar(c.kv_full[slot]));
        } else {
          load_rows(p.cache.k, offset);
          filled(bar(c.kv_full[slot]));
        }
        advance();
        if (j == 0) {
          wait_for(bar(c.q_empty), q_phase ^ 1);
          if (bad != 0) break;
          if (p.q_boxes) {
            if (w == 0) load_query_boxes();
          } else {
            load_queries(4, w);
            filled(bar(c.q_full));
            if constexpr (kCodes) flush();
          }
          q_phase ^= 1;
        }
        wait_for(bar(c.kv_empty[slot]), slot_phase ^ 1);
        if (bad != 0) break;
        if constexpr (kCodes) {
          store_codes();
          // scores times 64 (the keys' unit), the row's scale and what makes them logarithms to base 2 or the argument
          // of the cap's exponential
          if (lane < kOwn) {
            scales[slot * 2 * kN + mine] = key_scale * (64.0f * (kBent && p.cap > 0.0f ? p.cap_scale : p.scale));
            scales[slot * 2 * kN + kN + mine] = value_scale;
          }
          publish(bar(c.kv_full[slot]));
        } else {
          load_rows(p.cache.v, offset);
          filled(bar(c.kv_full[slot]));
        }
        advance();
      }
      walk.next(n);
    }
    flush();
    if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptLoadTimeout);
  } else if (warp == 12) {
    // ---- products ----
    constexpr uint32_t kBlock = L::kBlocks * kPromptTile * 128;
    const uint32_t q_at = ptx::smem_u32(q_tile), kv_at = ptx::smem_u32(slots);
    const uint32_t s_desc = ptx::idesc_bf16_f32(kPromptTile, kN);
    const uint32_t o_desc = ptx::idesc_bf16_f32(kPromptTile, kDim) | ptx::kIdescBMnMajor;
    const bool leader = ptx::elect_one();
    uint32_t taken = 0;  // slots before this item
    uint32_t p_phase = 0, q_phase = 0;
    auto wait = [&](uint32_t at, uint32_t parity) {
      ptx::mbar_wait_sticky<true>(at, parity, abort_at, bad);
      ptx::tc_fence_after();
    };
    auto wait_slot = [&](uint32_t number) { wait(bar(c.kv_full[number % kRing]), number / kRing & 1); };
    auto free_slot = [&](uint32_t number) {
      if (leader) ptx::mma_commit(bar(c.kv_empty[number % kRing]));
    };
    auto scores = [&](int tile, int buffer, uint32_t number) {
      if (leader) {
        const uint32_t q = q_at + tile * kBlock, k = kv_at + number % kRing * L::kSlotBytes, d = tmem + buffer * kN;
#pragma unroll
        for (int b = 0; b < L::kBlocks; ++b) {
          const uint64_t qd = ptx::smem_desc_k_sw128(q + b * kPromptTile * 128), kd = ptx::smem_desc_k_sw128(k + b * kN * 128);
          if (kDim - 64 * b >= 64) {
            ptx::mma_ss<4>(d, qd, kd, s_desc, b != 0);
          } else {
            ptx::mma_ss<kDim % 64 / 16>(d, qd, kd, s_desc, b != 0);
          }
        }
        ptx::mma_commit(bar(c.s_full[buffer]));
      }
    };
    auto values = [&](int tile, int buffer, uint32_t number, bool more) {
      const uint32_t skip = *const_cast<volatile uint32_t*>(&c.skip[tile]);
      if (leader) {
        if (skip == 0) {
          const uint64_t vd = ptx::smem_desc_mn_sw128(kv_at + number % kRing * L::kSlotBytes, kN * 128);
          ptx::mma_ts_mn<kN / 16>(tmem + L::kOutColumn + tile * kDim, tmem + buffer * kN, vd, o_desc, more);
        }
        ptx::mma_commit(bar(c.o_done[tile]));
      }
    };

    PromptWalk walk(p);
    while (walk.left > 0 && bad == 0) {
      const PromptItem it = load_item(p, walk.item);
      const int32_t n = walk.here(it);
      const int tiles = L::kTwo && it.rows > kPromptTile ? 2 : 1;
      wait(bar(c.q_full), q_phase);
      q_phase ^= 1;
      wait_slot(taken);
      if (bad != 0) break;
      for (int t = 0; t < tiles; ++t) scores(t, t, taken);
      free_slot(taken);
      if (n == 1 && leader) ptx::mma_commit(bar(c.q_empty));
#pragma unroll 1
      for (int32_t j = 0; j < n && bad == 0; ++j) {
        const uint32_t v = taken + 2 * j + 1, k = v + 1;
        const bool more = j + 1 < n;
        if (more) wait_slot(k);
        if constexpr (!L::kTwo) {
          // The next scores' buffer held weights that the product before has read (products run in order).
          if (bad != 0) break;
          if (more) scores(0, (j + 1) & 1, k);
        }
        wait_slot(v);
        if constexpr (L::kTwo) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= tiles) break;
            wait(bar(c.p_full[t]), p_phase >> t & 1);
            p_phase ^= 1u << t;
            if (bad != 0) break;
            values(t, t, v, j != 0);
            if (more) scores(t, t, k);
          }
        } else {
          const int buffer = j & 1;
          wait(bar(c.p_full[buffer]), p_phase >> buffer & 1);
          p_phase ^= 1u << buffer;
          if (bad != 0) break;
          values(0, buffer, v, j != 0);
        }
        if (bad != 0) break;
        free_slot(v);
        if (more) free_slot(k);
        if (j + 2 == n && leader) ptx::mma_commit(bar(c.q_empty));
      }
      taken += 2 * n;
      walk.next(n);
    }
    // All products, and what they arrive on, are done before the CTA ends.
    if (leader) ptx::mma_commit(bar(c.drained));
    __syncwarp();
    ptx::mbar_drain(bar(c.drained), 0);
    if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptIssueTimeout);
  } else if (warp < 4 * L::kTiles) {
    // ---- rows: a thread each ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRowRegs));  // (the host has checked that they are there)
    const int tile = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // its 32 lanes of tensor memory
    const uint32_t out_at = tmem + lanes + L::kOutColumn + tile * kDim;
    uint32_t s_phase = 0, outputs = 0, looks = 0, taken = 0;
    bool skipping = false;
    auto wait = [&](uint32_t at, uint32_t parity) { ptx::mbar_wait_sticky<true>(at, parity, abort_at, bad); };

    PromptWalk walk(p);
    while (walk.left > 0 && bad == 0) {
      const PromptItem it = load_item(p, walk.item);
      const int32_t n = walk.here(it);
      if (it.rows > tile * kPromptTile) {
        const PromptSequence of(p, it.b);
        // All rows of the tile, four to a lane, for what the tile's warps have to agree on.
        PromptView view = {0, INT32_MAX, 0};
        int32_t head = 0;
        int64_t result = -1;
        int32_t highest_lo = 0, lowest_hi = INT32_MAX;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int32_t r = tile * kPromptTile + 32 * i + lane;
          if (r < it.rows) {
            const int32_t token = p.group.div(it.row0 + r);
            const PromptView v = of.view(p, token);
            highest_lo = max(highest_lo, v.lo);
            lowest_hi = min(lowest_hi, v.hi);
            if (i == (warp & 3)) {
              view = v;
              head = walk.head * static_cast<int32_t>(p.group.d) + it.row0 + r - token * static_cast<int32_t>(p.group.d);
              result = static_cast<int64_t>(of.begin + token) * p.heads + head;
            }
          }
        }
        highest_lo = __reduce_max_sync(0xffffffffu, highest_lo);
        lowest_hi = __reduce_min_sync(0xffffffffu, lowest_hi);
        float slope = 0.0f;
        if constexpr (kBent) {
          if (p.slopes != nullptr && result >= 0) slope = load_arg(p.slopes + head) * 1.4426950408889634f;
        }

        float top = -INFINITY, sum = 0.0f;
        const int32_t token0 = (it.lo / kN + walk.step) * kN;
#pragma unroll 1
        for (int32_t j = 0; j < n; ++j) {
          const int32_t first = token0 + j * kN;
          const int buffer = L::kTwo ? tile : j & 1;
          const uint32_t s_at = tmem + lanes + buffer * kN;
          const uint32_t v_slot = (taken + 2 * j + 1) % kRing, v_phase = (taken + 2 * j + 1) / kRing & 1;
          if constexpr (kCodes) wait(bar(c.kv_full[v_slot]), v_phase);  // the scales lie there
          wait(bar(c.s_full[buffer]), s_phase >> buffer & 1);
          s_phase ^= 1u << buffer;
          if (bad != 0) break;
          ptx::tc_fence_after();
          uint32_t bits[kN];
#pragma unroll
          for (int i = 0; i < kN; i += 32) ptx::tmem_ld_32x32b_x32(s_at + i, bits + i);
          ptx::tmem_wait_ld();
          float (&x)[kN] = reinterpret_cast<float (&)[kN]>(bits);

          if constexpr (kCodes) {
            const float4* const factor = reinterpret_cast<const float4*>(scales + v_slot * 2 * kN);
#pragma unroll
            for (int i = 0; i < kN; i += 4) {
              const float4 f = factor[i / 4];
              x[i] *= f.x, x[i + 1] *= f.y, x[i + 2] *= f.z, x[i + 3] *= f.w;
            }
          }
          if constexpr (kBent) {
            if (p.cap > 0.0f) {
              const float factor = kCodes ? 1.0f : p.cap_scale, twice = -2.0f * p.cap;
#pragma unroll
              for (int i = 0; i < kN; ++i) x[i] = fmaf(twice, reciprocal_fast(exp2_fast(x[i] * factor) + 1.0f), p.cap);
            } else if constexpr (!kCodes) {
#pragma unroll
              for (int i = 0; i < kN; ++i) x[i] *= p.scale;
            }
            if (p.slopes != nullptr) {
              const float from = static_cast<float>(first - view.position);
#pragma unroll
              for (int i = 0; i < kN; ++i) x[i] = fmaf(-slope, fabsf(from + i), x[i]);
            }
          }
          const float of_scores = kBent || kCodes ? 1.0f : p.scale;
          if (highest_lo > first || lowest_hi < first + kN) {
            const uint32_t begin = view.lo - first, span = max(view.hi - view.lo, 0);
#pragma unroll
            for (int i = 0; i < kN; ++i) x[i] = i - begin < span ? x[i] : -INFINITY;
          }
          float high[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
          for (int i = 4; i < kN; ++i) high[i & 3] = fmaxf(high[i & 3], x[i]);
          const float highest = fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])) * of_scores;
          if (__any_sync(0xffffffffu, highest > top + kSlack)) {
            const float next = fmaxf(top, highest);
            const float factor = next == -INFINITY ? 1.0f : exp2_fast(top - next);
            top = next;
            sum *= factor;
            if (j != 0) {
              // (with two tiles the scores were made after the product before)
              if constexpr (!L::kTwo) wait(bar(c.o_done[tile]), (outputs - 1) & 1);
              if (bad != 0) break;
              ptx::tc_fence_after();
#pragma unroll 1
              for (int i = 0; i < kDim; i += 16) {
                uint32_t o[16];
                ptx::tmem_ld_32x32b_x16(out_at + i, o);
                ptx::tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * factor);
                ptx::tmem_st_32x32b_x16(out_at + i, o);
              }
            }
          }
          const float base = top == -INFINITY ? 0.0f : -top;
          if constexpr (!kCodes) {
            // Values that some rows do not see: zero times an infinity or a NaN would be a NaN for those rows too.  What
            // no row of the item sees (rows of a box outside its tokens) is set to zero.
            bool found = false;
            if (highest_lo > first || lowest_hi < first + kN) {
              wait(bar(c.kv_full[v_slot]), v_phase);
              uint32_t most = 0;
              uint8_t* const v = slots + v_slot * L::kSlotBytes + (warp & 3) * (kN / 4 * 128) + lane * 16;
              const int32_t token = first + (warp & 3) * (kN / 4) + lane / 8;
#pragma unroll
              for (int b = 0; b < L::kBlocks; ++b) {
#pragma unroll
                for (int i = 0; i < kN / 16; ++i) {
                  const int logical = (lane ^ (i * 4 + lane / 8)) & 7;  // the token's parity with its place
                  uint4* const at = reinterpret_cast<uint4*>(v + b * (kN * 128) + i * 512);
                  if (token + 4 * i < it.lo || token + 4 * i >= it.hi) {
                    *at = make_uint4(0, 0, 0, 0);
                  } else if (kDim - 64 * b >= 64 || 64 * b + 8 * logical < kDim) {
                    const uint4 w = *at;
                    most = __vmaxu2(__vmaxu2(most, __vmaxu2(w.x & 0x7FFF7FFFu, w.y & 0x7FFF7FFFu)),
                                    __vmaxu2(w.z & 0x7FFF7FFFu, w.w & 0x7FFF7FFFu));
                  }
                }
              }
              const bool any = __any_sync(0xffffffffu, (most & 0xFFFFu) >= 0x7F80u || (most >> 16) >= 0x7F80u);
              ptx::fence_proxy_async();
              ++looks;
              if (any && lane == 0) *const_cast<volatile uint32_t*>(&c.odd[tile]) = looks;
              __syncwarp();
              ptx::mbar_arrive_lane0(bar(c.scanned[tile]), lane);
              wait(bar(c.scanned[tile]), (looks - 1) & 1);
              if (bad != 0) break;
              found = *const_cast<volatile uint32_t*>(&c.odd[tile]) == looks;
            }
            if (found != skipping) {
              skipping = found;
              if ((warp & 3) == 0 && lane == 0) *const_cast<volatile uint32_t*>(&c.skip[tile]) = found;
            }
            if (found) {
              if constexpr (!L::kTwo) {
                if (j != 0) wait(bar(c.o_done[tile]), (outputs - 1) & 1);
                if (bad != 0) break;
                ptx::tc_fence_after();
              }
#pragma unroll
              for (int i = 0; i < kN; i += 32) ptx::tmem_st_32x32b_x32(s_at + i, bits + i);
              ptx::tmem_wait_st();
              sum += product_by_row<kDim, kN>(s_at, out_at, slots + v_slot * L::kSlotBytes, of_scores, base, j == 0);
              ptx::tc_fence_before();
              __syncwarp();
              ptx::mbar_arrive_lane0(bar(c.p_full[buffer]), lane);
              ++outputs;
              continue;
            }
          }
          float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          const float4* const value_factor = reinterpret_cast<const float4*>(scales + v_slot * 2 * kN + kN);
#pragma unroll
          for (int i = 0; i < kN; i += 32) {
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              float e[4];
#pragma unroll
              for (int l = 0; l < 4; ++l) {
                e[l] = exp2_fast(fmaf(x[i + k + l], of_scores, base));
                sums[l] += e[l];
              }
              if constexpr (kCodes) {
                const float4 f = value_factor[(i + k) / 4];
                // (a masked token's scale may be NaN)
                e[0] = e[0] == 0.0f ? 0.0f : e[0] * f.x, e[1] = e[1] == 0.0f ? 0.0f : e[1] * f.y;
                e[2] = e[2] == 0.0f ? 0.0f : e[2] * f.z, e[3] = e[3] == 0.0f ? 0.0f : e[3] * f.w;
              }
              w[k / 2] = pack_bf16(e[0], e[1]);
              w[k / 2 + 1] = pack_bf16(e[2], e[3]);
            }
            ptx::tmem_st_32x32b_x16(s_at + i / 2, w);
          }
          sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
          ptx::tmem_wait_st();
          ptx::tc_fence_before();
          __syncwarp();
          ptx::mbar_arrive_lane0(bar(c.p_full[buffer]), lane);
          ++outputs;
        }
        if (bad != 0) break;

        // The end of the item, or of the CTA's part of it.
        wait(bar(c.o_done[tile]), (outputs - 1) & 1);
        if (bad != 0) break;
        ptx::tc_fence_after();
        const bool whole = walk.step == 0 && n == it.steps;
        float* const part = p.parts + (2 * static_cast<int64_t>(blockIdx.x) + (walk.step == 0 ? 1 : 0)) * prompt_part_floats<kDim, kCodes>() +
                            static_cast<int64_t>(tile) * kPromptTile * (kDim + 2);
#pragma unroll 1
        for (int i = 0; i < kDim; i += 16) {
          uint32_t bits[16];
          __syncwarp();
          ptx::tmem_ld_32x32b_x16(out_at + i, bits);
          ptx::tmem_wait_ld();
          float (&o)[16] = reinterpret_cast<float (&)[16]>(bits);
          if (whole) {
            if (result >= 0) prompt_finish<16>(p, result, i, kDim, o, top, sum, kUnit, i == 0);
          } else {
#pragma unroll
            for (int k = 0; k < 16; k += 4) {
              __stcg(reinterpret_cast<float4*>(part) + (i + k) / 4 * kPromptTile + row, make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
            }
          }
        }
        if (!whole) {
          __stcg(part + kDim * kPromptTile + row, top);
          __stcg(part + (kDim + 1) * kPromptTile + row, sum);
        }
        ptx::tc_fence_before();
      }
      taken += 2 * n;
      walk.next(n);
    }
    if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptRowTimeout);
  }

  if (bad != 0) {
    // Whatever copies and products are on their way have long ended when the CTA does.
    ptx::cp_async_wait_all();
    for (int i = 0; i < 64; ++i) __nanosleep(20000);
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  if (warp == 12) ptx::tmem_dealloc(tmem, 512);
}

}  // namespace chord
