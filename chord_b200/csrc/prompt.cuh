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
//   P = exp2(x - m) in BF16 over S, by two threads per row, half of the step's tokens each; m is raised, and O scaled,
//                  only where a score passes it by more than kSlack (P is then 2^8 at most)
//   O += P V       P from tensor memory, V from shared memory as it lies there (MN-major)
//
// P is rounded to BF16 (by 2^-8 of each weight at most, as the values that it multiplies were; a second BF16 number for the
// rest would be a third product; see kFineSteps), its sum is added up before that in FP32.
//
// What bounds it: one prompt of 16,384 tokens, 64 + 8 heads of 128, 4.1 to 4.55 ms, 1.0 PFLOP/s of 1.4 that the library's products
// sustain.  At 4.45 ms and 1.72 GHz (the power limit; 1.965 without) a step of 256 rows and 128 tokens takes some 4300 cycles,
// of which its products take 2048 and its exponentials, on the four-lane units, 2048 others: what is left is the chain of a tile, maximum,
// weights, product, next scores, which the other tile covers in part.  With queries, keys and values by cp.async 5.6 ms.  Over codes with capped scores, 4 x 1,024 queries of
// 16 + 8 heads of 256 after 30,000 tokens, 1.9 to 2.2 ms: the rows' arithmetic on scores (scales, cap, maximum) and the turning of
// codes, 64 % of issue slots.  Short documents, 9 prompts of up to 2,048 tokens, 260 us for a floor of 72: 3,192 items of 1 to 4 steps, whose first step waits
// for its queries and keys and whose last one writes the rows (184 MB); products make up a quarter of the time.
#pragma once

#include "prompt_plan.cuh"

namespace chord {

// Warps: 16 for the rows, one that loads by TMA, one that issues products, two that look at values and load queries that
// TMA does not, and, over codes, those that turn these into BF16: four more, or the eight that one tile's rows leave (with
// four more there too, 4 x 1,024 queries of 16 heads of 256 after 30,000 tokens: 2.04 ms for 1.91).
constexpr int kLoadWarp = 16, kIssueWarp = 17, kLookWarp = 18, kLookWarps = 2;

template <int kDim, bool kCodes>
struct PromptLayout {
  static constexpr bool kTwo = kDim <= 128;  // row tiles of an item
  static constexpr int kTiles = kTwo ? 2 : 1;
  static constexpr int kTurnWarp = kTwo ? 20 : 8, kTurnWarps = kTwo ? 4 : 8;
  static constexpr int kThreads = 32 * (kCodes && kTwo ? 24 : 20);
  // Of a CTA launched with 96 registers a thread, 80 with 24 warps: what the first 16 warps have, and the others.
  static constexpr int kRowRegs = kCodes && kTwo ? 88 : 104, kOtherRegs = 64;
  static constexpr int kN = kTwo ? 128 : 64;             // tokens of a step
  static constexpr int kBlocks = (kDim + 63) / 64;       // of 64 elements, 128 bytes
  static constexpr int kQBytes = kTiles * kBlocks * kPromptTile * 128;
  static constexpr int kSlotBytes = kBlocks * kN * 128;  // keys or values of a step
  static constexpr int kRaw = kCodes ? 3 : 0;            // codes on their way
  static constexpr int kRawBytes = kN * kDim;
  static constexpr int kScales = kCodes ? 4 : 0;         // steps whose codes' scales are held
  static constexpr int kScaleBytes = 2 * kN * 4;
  static constexpr int kMaxBytes = 2 * 2 * kPromptTile * 4;
  static constexpr int kControl = 1024;
  static constexpr int kFit = (232448 - kControl - kMaxBytes - kQBytes - kRaw * kRawBytes - kScales * kScaleBytes) / kSlotBytes;
  static constexpr int kRing = kFit > 8 ? 8 : kFit;
  static constexpr int kSmem = kQBytes + kRing * kSlotBytes + kRaw * kRawBytes + kScales * kScaleBytes + kMaxBytes + kControl;
  static constexpr uint32_t kOutColumn = kTwo ? 256 : 128;  // of tensor memory; the scores' buffers come first
  static_assert(kTiles * kPromptTile == (kTwo ? 256 : 128) && kN == (kTwo ? 128 : 64), "the plan's logarithms");
  static_assert(kRing >= 3, "keys of one step and values of the one before, and one on its way");
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// Two at a time: x a + b, y a + b.
__device__ __forceinline__ void fma_pair(float& x, float& y, float a, float b) {
  asm("{\n .reg .b64 v, m, c;\n mov.b64 v, {%0, %1};\n mov.b64 m, {%2, %2};\n mov.b64 c, {%3, %3};\n fma.rn.f32x2 v, v, m, c;\n"
      " mov.b64 {%0, %1}, v;\n}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}

__device__ __forceinline__ void add_pair(float (&sum)[2], float x, float y) {
  asm("{\n .reg .b64 v, s;\n mov.b64 s, {%0, %1};\n mov.b64 v, {%2, %3};\n add.rn.f32x2 s, s, v;\n mov.b64 {%0, %1}, s;\n}"
      : "+f"(sum[0]), "+f"(sum[1])
      : "f"(x), "f"(y));
}

// A warp's walk over its CTA's steps.
struct PromptWalk {
  int64_t left;
  int32_t head, item, step, items, number;  // number: of the item among the CTA's
  __device__ __forceinline__ PromptWalk(const PromptStart& s, int32_t of)
      : left(s.count), head(s.head), item(s.item), step(s.step), items(of), number(0) {}
  __device__ __forceinline__ int32_t here(const PromptItem& it) const {
    return static_cast<int32_t>(min(left, static_cast<int64_t>(it.steps - step)));
  }
  __device__ __forceinline__ void next(int32_t n) {
    left -= n;
    step = 0;
    ++number;
    if (++item == items) item = 0, ++head;
  }
};

__device__ __forceinline__ PromptItem load_item(const PromptParams& p, int32_t item) {
  PromptItem it;
  const int4* const from = reinterpret_cast<const int4*>(p.items + item);
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<int4*>(&it)[i] = __ldcg(from + i);
  return it;
}

// Over codes a weight is rounded with its token's scale in it, the largest one of a row too, which is one otherwise.  Rows that see few
// tokens do not average that away, so in items of up to so many steps the rest goes into a product of its own, from the
// columns of tensor memory that the scores leave: off by 0.17 % of the results (their rounding to BF16) for 0.23 to 0.25 %.  With it in
// all items 4 x 1,024 queries after 30,000 tokens took 2.63 ms for 2.21.
constexpr int kFineSteps = 4;

enum PromptStatus : int32_t { kPromptLoadTimeout = 1, kPromptIssueTimeout = 2, kPromptRowTimeout = 8 };

struct __align__(16) PromptControl {
  PromptStart start;
  int32_t plan_items;
  PromptItem items[2];  // of the CTA, in turn
  uint64_t item_full[2], item_empty[2], q_full, q_empty, drained;
  uint64_t kv_full[8], kv_empty[8];  // by slot
  uint64_t looked[8];                // by the values' turn: there are no more than four of them in the ring
  uint64_t raw_full[4], raw_empty[4];
  uint64_t scales_empty[4];          // (they are there when the step has been looked at)
  uint64_t s_full[2], p_full[2][2];  // p_full: [half of the tokens][buffer]
  uint64_t o_done[2];                // by tile; of one tile's products, two in turn
  uint32_t odd[8];   // as looked, the values in turn: number of the values in which infinities or NaN were found, and one
  uint32_t skip[2];  // by buffer: the product of its P and V is made by the rows' warps
  uint32_t tmem, abort;
};
static_assert(sizeof(PromptControl) <= 1024, "its place");

// What a row's sums are multiplied with, and the results of its own part (PromptParams::extra); and the row's lse.
struct PromptRates {
  float mine, other;
  __device__ __forceinline__ PromptRates(const PromptParams& p, int64_t row, float top, float sum, float unit, bool first) {
    float all = sum, to = top;
    mine = unit, other = 0.0f;
    if (p.extra != nullptr) {
      // (relative to the larger one)
      const float beside = load_arg(p.extra_lse + row) * 1.4426950408889634f, here = sum == 0.0f ? -INFINITY : top;
      const float most = fmaxf(here, beside);
      to = most == -INFINITY ? 0.0f : most;
      const float w = exp2_fast(here - to);
      other = exp2_fast(beside - to);
      all = sum * w + other;
      mine = unit * w;
    }
    const float rate = all == 0.0f ? 0.0f : 1.0f / all;
    mine *= rate;
    other *= rate;
    if (first && p.lse != nullptr) p.lse[row] = all == 0.0f ? -INFINITY : (to + log2f(all)) * 0.693147180559945309f;
  }
  // Eight values of the row.
  __device__ __forceinline__ void write(const PromptParams& p, int64_t at, const float* o) const {
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = o[i] * mine;
    if (p.extra != nullptr) {
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const float4 x = load_arg(reinterpret_cast<const float4*>(p.extra + at + i));
        v[i] = fmaf(x.x, other, v[i]), v[i + 1] = fmaf(x.y, other, v[i + 1]);
        v[i + 2] = fmaf(x.z, other, v[i + 2]), v[i + 3] = fmaf(x.w, other, v[i + 3]);
      }
    }
    *reinterpret_cast<uint4*>(p.out + at) = make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
};

__device__ __forceinline__ void store_32_bytes(void* to, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Four lanes with a word for each of four places each: lane q receives the four lanes' words for place q.
__device__ __forceinline__ void exchange4(uint32_t (&w)[4], int q) {
#pragma unroll
  for (int d = 1; d < 4; d <<= 1) {
    // pairs of places that differ in bit d: the one that is not the lane's goes
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((i & d) != 0) continue;
      const bool upper = (q & d) != 0;
      const uint32_t gone = upper ? w[i] : w[i | d];
      const uint32_t come = __shfl_xor_sync(0xffffffffu, gone, d);
      if (upper) w[i] = come; else w[i | d] = come;
    }
  }
}

// Writes 64 or 32 values, from `dim` on, of a warp's 32 rows as BF16.  Rows are spread over four lanes each (with a row to a
// lane, every store touches 32 lines of memory: 6500 cycles for two tiles of 128 values, as long as two steps), which
// then write 128 or 64 bytes of it in one go, 32 bytes at a time where the results lie on 32 bytes, which a caller's need not
// (9 prompts of packed documents 257 us; 16 bytes at a time 271).
// `row`, `mine` and `other` are those of the lane's own row; row < 0: none.
template <int kCount>
__device__ __forceinline__ void write_rows(const PromptParams& p, uint32_t from, int dims, int dim, int64_t row, float mine, float other, int lane) {
  constexpr int kGroups = kCount / 8;
  const int q = lane & 3;
#pragma unroll
  for (int lower = 0; lower < 32; lower += 16) {
    uint32_t o[4 * kGroups];
    __syncwarp();
    if constexpr (kGroups == 8) ptx::tmem_ld_16x256b_x8(from + (static_cast<uint32_t>(lower) << 16), o);
    if constexpr (kGroups == 4) ptx::tmem_ld_16x256b_x4(from + (static_cast<uint32_t>(lower) << 16), o);
    ptx::tmem_wait_ld();
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int of = lower + 8 * r + lane / 4;
      const int64_t to = __shfl_sync(0xffffffffu, row, of);
      const float scale = __shfl_sync(0xffffffffu, mine, of);
      float v[2 * kGroups];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) {
        v[2 * g] = __uint_as_float(o[4 * g + 2 * r]) * scale;
        v[2 * g + 1] = __uint_as_float(o[4 * g + 2 * r + 1]) * scale;
      }
      if (p.extra != nullptr) {
        const float beside = __shfl_sync(0xffffffffu, other, of);
        if (to >= 0) {
          const float* const x = p.extra + to * dims + dim + 2 * q;
#pragma unroll
          for (int g = 0; g < kGroups; ++g) {
            v[2 * g] = fmaf(load_arg(x + 8 * g), beside, v[2 * g]);
            v[2 * g + 1] = fmaf(load_arg(x + 8 * g + 1), beside, v[2 * g + 1]);
          }
        }
        __syncwarp();
      }
      // Lane q gets groups 2 q and 2 q + 1 (of four groups, group q).
      uint32_t w[kGroups / 4][4];
#pragma unroll
      for (int g = 0; g < kGroups; ++g) w[g % (kGroups / 4)][g / (kGroups / 4)] = pack_bf16(v[2 * g], v[2 * g + 1]);
#pragma unroll
      for (int i = 0; i < kGroups / 4; ++i) exchange4(w[i], q);
      __nv_bfloat16* const at = p.out + to * dims + dim + q * (2 * kGroups);
      if (to >= 0) {
        if constexpr (kGroups == 8) {
          if (p.out_32) {
            store_32_bytes(at, &w[0][0]);
          } else {
            reinterpret_cast<uint4*>(at)[0] = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
            reinterpret_cast<uint4*>(at)[1] = make_uint4(w[1][0], w[1][1], w[1][2], w[1][3]);
          }
        }
        if constexpr (kGroups == 4) *reinterpret_cast<uint4*>(at) = make_uint4(w[0][0], w[0][1], w[0][2], w[0][3]);
      }
    }
  }
}

// The product of a tile's weights and values on the CUDA cores, for values among which are infinities or NaN that not all
// of its rows see: tokens of no weight are left out.  The scores lie in tensor memory at `s_at`; returns their weights' sum.
template <int kDim, int kN>
__device__ __noinline__ float product_by_row(uint32_t s_at, uint32_t out_at, const uint8_t* v, int dim0, float of_scores, float base, bool fresh) {
  float all = 0.0f;
#pragma unroll 1
  for (int dim = dim0; dim < dim0 + kDim / 2; dim += 8) {
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
      __syncwarp();
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
    }
    __syncwarp();
    all = sum;
    ptx::tmem_st_32x32b_x8(out_at + dim, reinterpret_cast<const uint32_t*>(o));
    ptx::tmem_wait_st();
  }
  return all;
}

// Sixteen codes as BF16 numbers (code - 128) / 64, exact.
__device__ __forceinline__ void decode16(const uint4& codes, uint4& low, uint4& high) {
  constexpr uint32_t kOffset = 0xC000C000u;  // -128 / 64, twice
  const uint32_t four[4] = {codes.x, codes.y, codes.z, codes.w};
  uint32_t v[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[2 * k] = bf16x2_fma(__byte_perm(four[k], 0, 0x4140), kTwo127, kOffset);
    v[2 * k + 1] = bf16x2_fma(__byte_perm(four[k], 0, 0x4342), kTwo127, kOffset);
  }
  low = make_uint4(v[0], v[1], v[2], v[3]);
  high = make_uint4(v[4], v[5], v[6], v[7]);
}

template <int kDim, bool kCodes, bool kBent>
__global__ void __launch_bounds__((PromptLayout<kDim, kCodes>::kThreads), 1) prompt_attention_kernel(const __grid_constant__ PromptParams p) {
  using L = PromptLayout<kDim, kCodes>;
  constexpr int kN = L::kN, kHalf = kN / 2, kChunks = kHalf / 32;
  constexpr int kRing = L::kRing;
  constexpr float kSlack = 8.0f;
  constexpr float kUnit = kCodes ? 64.0f : 1.0f;  // of values in shared memory (codes: (code - 128) / 64)
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t* const q_tile = smem;
  uint8_t* const slots = smem + L::kQBytes;
  uint8_t* const raw = slots + kRing * L::kSlotBytes;  // [kRaw][token][dim] codes
  float* const scales = reinterpret_cast<float*>(raw + L::kRaw * L::kRawBytes);  // [step][of keys, of values][kN]
  float* const maxima = reinterpret_cast<float*>(smem + L::kSmem - L::kControl - L::kMaxBytes);  // [tile or parity][half][row]
  PromptControl& c = *reinterpret_cast<PromptControl*>(smem + L::kSmem - L::kControl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t abort_at = ptx::smem_u32(&c.abort);
  uint32_t bad = 0;
  auto bar = [](const uint64_t& b) { return ptx::smem_u32(&b); };
  auto wait = [&](uint32_t at, uint32_t parity) { ptx::mbar_wait_sticky<true>(at, parity, abort_at, bad); };

  if ((ptx::smem_u32(smem) & 1023u) != 0) {  // (the tiles' swizzle counts from there)
    if (threadIdx.x == 0 && p.status != nullptr) atomicOr(p.status, kPromptIssueTimeout);
    return;
  }
  if (warp == kIssueWarp) {
    ptx::tmem_alloc(ptx::smem_u32(&c.tmem), 512);
    ptx::tmem_relinquish();
  }
  if (threadIdx.x == 32 * kLoadWarp) {
    ptx::prefetch_tensormap(&p.k_map);
    ptx::prefetch_tensormap(&p.v_map);
    if (p.q_boxes) ptx::prefetch_tensormap(&p.q_map);
  }
  if (threadIdx.x == 0) {
    ptx::mbar_init(bar(c.q_full), p.q_boxes ? 1 : kLookWarps);
    ptx::mbar_init(bar(c.q_empty), 1);
    ptx::mbar_init(bar(c.drained), 1);
    for (int i = 0; i < 8; ++i) {
      ptx::mbar_init(bar(c.kv_full[i]), kCodes ? L::kTurnWarps : 1);
      ptx::mbar_init(bar(c.kv_empty[i]), 1);
      ptx::mbar_init(bar(c.looked[i]), kLookWarps);
      c.odd[i] = 0;
    }
    for (int i = 0; i < 4; ++i) {
      ptx::mbar_init(bar(c.raw_full[i]), 1);
      ptx::mbar_init(bar(c.raw_empty[i]), L::kTurnWarps);
      ptx::mbar_init(bar(c.scales_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(bar(c.item_full[i]), 1);
      ptx::mbar_init(bar(c.item_empty[i]), 8 * L::kTiles + 1 + kLookWarps + (kCodes ? L::kTurnWarps : 0));
      ptx::mbar_init(bar(c.s_full[i]), 1);
      ptx::mbar_init(bar(c.p_full[0][i]), 4);
      ptx::mbar_init(bar(c.p_full[1][i]), 4);
      ptx::mbar_init(bar(c.o_done[i]), 1);
      c.skip[i] = 0;
    }
    c.abort = 0;
    ptx::fence_barrier_init();
  }
  ptx::tc_fence_before();
  __syncthreads();
  ptx::tc_fence_after();
  const uint32_t tmem = c.tmem;
  ptx::grid_dependency_wait();
  if (p.self) {
    // The plan, in the tiles' place: every CTA goes through all items and keeps those of its run.  (Several keep the same
    // ones, alike; a kernel of its own took 8 us and its launch.)
    static_assert(sizeof(PromptPlanScratch) % 16 == 0 && sizeof(PromptPlanScratch) + kPlanHeld * sizeof(PromptItem) <= L::kQBytes + kRing * L::kSlotBytes, "room");
    PromptPlanScratch& scratch = *reinterpret_cast<PromptPlanScratch*>(smem);
    PromptItem* const items = reinterpret_cast<PromptItem*>(smem + sizeof(PromptPlanScratch));
    PromptPlanner<L::kThreads> planner(p, scratch, L::kTwo ? 8 : 7, L::kTwo ? 7 : 6);
    planner.items([&](int32_t item, const PromptItem& it) { items[item] = it; });
    const PromptPlan plan = planner.plan();
    if (threadIdx.x == 0) {
      const PromptStart start =
          planner.start(plan, blockIdx.x, [&](int32_t item) { return items[item].first; }, [&](int32_t item) { return items[item].steps; });
      c.start = start;
      c.plan_items = plan.items;
      p.cta_starts[blockIdx.x] = start;  // (for the join)
      if (blockIdx.x == 0) *p.plan = plan;
    }
    __syncthreads();
    // Those of the run, of one key-value head or more.
    const int64_t begin = c.start.begin, end = begin + c.start.count;
#pragma unroll 1
    for (int32_t item = threadIdx.x; item < plan.items; item += L::kThreads) {
      const int64_t first = items[item].first, steps = items[item].steps;
      bool wanted = false;
      for (int64_t head = c.start.head; !wanted && head * plan.head_steps < end; ++head) {
        wanted = head * plan.head_steps + first < end && head * plan.head_steps + first + steps > begin;
      }
      if (wanted) p.items[item] = items[item];
    }
    __syncthreads();
    ptx::fence_proxy_async();  // (the tiles' copies come next)
    __syncthreads();
  } else {
    if (threadIdx.x == 0) {
      c.start = p.cta_starts[blockIdx.x];
      c.plan_items = p.plan->items;
    }
    __syncthreads();
  }

  // An item's description is read from global memory by the loading warp alone, which goes ahead of the others.
  auto item_of = [&](const PromptWalk& walk) {
    wait(bar(c.item_full[walk.number & 1]), walk.number >> 1 & 1);
    const PromptItem it = c.items[walk.number & 1];
    __syncwarp();
    ptx::mbar_arrive_lane0(bar(c.item_empty[walk.number & 1]), lane);
    return it;
  };
  // Whether some row of a tile does not see some token of a step.
  auto masked = [&](const PromptItem& it, int tile, int32_t first) { return it.highest_lo[tile] > first || it.lowest_hi[tile] < first + kN; };
  auto any_masked = [&](const PromptItem& it, int32_t first) {
    return masked(it, 0, first) || (L::kTwo && it.rows > kPromptTile && masked(it, 1, first));
  };
  // Where the 16 bytes from element 8 * chunk of a token go in a slot.
  auto place_of = [](int token, int chunk) { return (chunk >> 3) * (kN * 128) + token * 128 + ((chunk ^ token) & 7) * 16; };
  auto publish = [&](uint32_t at) {  // what the warp has written to shared memory is for products
    ptx::fence_proxy_async();
    __syncwarp();
    ptx::mbar_arrive_lane0(at, lane);
  };

  if (warp >= kLoadWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(L::kOtherRegs));

  if (warp == kLoadWarp) {
    // ---- loads: items, queries once per item, keys and values step by step, each into a slot of the ring ----
    // By TMA, a box of 1 to 128 tokens for each lane and round: as many as divide pages and steps.  (A step of 128 tokens of
    // 128 elements by cp.async took four warps some 4700 cycles, the products 2000.)  Boxes bring tokens behind the last one with
    // them; one outside the tokens that are seen, or whose page is not there, is asked for behind the cache's last
    // page, which gives zeros.  Codes come as they are into a ring of their own.
    constexpr int kSlots = kCodes ? L::kRaw : kRing;
    uint32_t slot = 0, slot_phase = 0, q_phase = 0;
    PromptWalk walk(c.start, c.plan_items);
    while (walk.left > 0 && bad == 0) {
      const PromptItem it = load_item(p, walk.item);
      const int32_t n = walk.here(it);
      const int32_t* const table = p.tables + it.b * p.table_stride;
      const int32_t token0 = (it.lo / kN + walk.step) * kN;
      const int32_t rounds = p.box == 0 ? 0 : (kN / p.box + 31) / 32;
      auto look_up = [&](int32_t j, int32_t box, int32_t& page, int32_t& place) {  // place -1: none
        const int32_t mine = box * p.box, token = token0 + j * kN + mine;
        place = -1;
        if (j < n && token + p.box > it.lo && token < it.hi && mine < kN) {
          const uint32_t index = p.cache.page_size.div(token);
          place = token - index * p.cache.page_size.d;
          page = load_arg(table + index);
        }
      };
      auto begin_item = [&]() {  // once the one before is done with
        wait(bar(c.item_empty[walk.number & 1]), (walk.number >> 1 & 1) ^ 1);
        if (bad != 0) return;
        if (lane < 4) reinterpret_cast<int4*>(&c.items[walk.number & 1])[lane] = __ldcg(reinterpret_cast<const int4*>(p.items + walk.item) + lane);
        __syncwarp();
        ptx::mbar_arrive_lane0(bar(c.item_full[walk.number & 1]), lane);
        if (!p.q_boxes) return;
        wait(bar(c.q_empty), q_phase ^ 1);
        q_phase ^= 1;
        if (bad != 0) return;
        const int tiles = L::kTwo && it.rows > kPromptTile ? 2 : 1;
        if (lane == 0) {
          ptx::mbar_arrive_expect_tx(bar(c.q_full), tiles * (L::kBlocks * kPromptTile * 128));
          const int32_t token = it.begin + static_cast<int32_t>(p.group.div(it.row0)), per_tile = p.group.div(kPromptTile);
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
      int32_t page = 0, place = -1;
      if (p.box != 0) look_up(0, lane, page, place);
      // (the queries of all but the first item wait for the one before; its first keys need not)
      const int first_which = walk.number == 0 ? 0 : 1;
#pragma unroll 1
      for (int32_t j = 0; j < n; ++j) {
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          if (j == 0 && which == first_which) begin_item();
          if (bad != 0) break;
          if (p.box == 0) continue;
          const uint32_t at = kCodes ? bar(c.raw_full[slot]) : bar(c.kv_full[slot]);
          wait(kCodes ? bar(c.raw_empty[slot]) : bar(c.kv_empty[slot]), slot_phase ^ 1);
          if (bad != 0) break;
          if (lane == 0) ptx::mbar_arrive_expect_tx(at, kCodes ? L::kRawBytes : L::kSlotBytes);
          __syncwarp();
          const CUtensorMap* const map = which == 0 ? &p.k_map : &p.v_map;
#pragma unroll 1
          for (int32_t round = 0; round < rounds; ++round) {
            const int32_t box = round * 32 + lane;
            int32_t of_page = page, of_place = place;
            if (round != 0) look_up(j, box, of_page, of_place);
            const bool there = of_place >= 0 && static_cast<uint32_t>(of_page) < static_cast<uint32_t>(p.cache.num_pages);
            if (of_place >= 0 && !there && p.status != nullptr) atomicOr(p.status, kStatusIndex);
            if (box * p.box < kN) {
              const int32_t head = walk.head * p.head_step, to_page = there ? of_page * p.page_step : p.cache.num_pages, to_place = there ? of_place : 0;
              if constexpr (kCodes) {
                ptx::tma_load_4d(ptx::smem_u32(raw) + slot * L::kRawBytes + box * p.box * kDim, map, at, 0, to_place, head, to_page);
              } else {
                const uint32_t to = ptx::smem_u32(slots) + slot * L::kSlotBytes + box * p.box * 128;
#pragma unroll
                for (int b = 0; b < L::kBlocks; ++b) ptx::tma_load_4d(to + b * (kN * 128), map, at, 64 * b, to_place, head, to_page);
              }
            }
            __syncwarp();
          }
          if (++slot == kSlots) slot = 0, slot_phase ^= 1;
        }
        if (bad != 0) break;
        if (p.box != 0) look_up(j + 1, lane, page, place);
      }
      walk.next(n);
    }
    if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptLoadTimeout);
  } else if (warp == kIssueWarp) {
    // ---- products ----
    constexpr uint32_t kBlock = L::kBlocks * kPromptTile * 128;
    const uint32_t q_at = ptx::smem_u32(q_tile), kv_at = ptx::smem_u32(slots);
    const uint32_t s_desc = ptx::idesc_bf16_f32(kPromptTile, kN);
    const uint32_t o_desc = ptx::idesc_bf16_f32(kPromptTile, kDim) | ptx::kIdescBMnMajor;
    const bool leader = ptx::elect_one();
    uint32_t taken = 0;  // slots before this item
    uint32_t p_phase = 0, q_phase = 0, products[2] = {0, 0};  // the latter: issued, by tile
    auto wait_to_issue = [&](uint32_t at, uint32_t parity) {
      wait(at, parity);
      ptx::tc_fence_after();
    };
    auto wait_slot = [&](uint32_t number) { wait_to_issue(bar(c.kv_full[number % kRing]), number / kRing & 1); };
    auto free_slot = [&](uint32_t number) {
      if (leader) ptx::mma_commit(bar(c.kv_empty[number % kRing]));
    };
    // Of two tiles over codes, a step's scores are made when its scales are there.  The rows of the second tile go past items
    // that have none, so they may come to a step while what has been looked at is items behind, of which the parity of
    // `looked` tells nothing; s_full does, and scales_empty, which waits for them, holds back what comes after.
    auto wait_scales = [&](uint32_t step) {
      if constexpr (kCodes && L::kTwo) wait_to_issue(bar(c.looked[step % 8]), step / 8 & 1);
    };
    // Scores go where weights were that the product before has read.  Products with other accumulators or of another
    // shape are not bound to run in order, so that one has to have ended.
    auto ended = [&](int tile) {  // the last one
      const uint32_t last = products[tile] - 1;
      wait_to_issue(bar(c.o_done[L::kTwo ? tile : last & 1]), (L::kTwo ? last : last >> 1) & 1);
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
    // The product with the weights of either half of a step's tokens as soon as they are there.
    auto values = [&](int tile, int buffer, uint32_t number, bool more, bool fine) {
      const uint64_t vd = ptx::smem_desc_mn_sw128(kv_at + number % kRing * L::kSlotBytes, kN * 128);
      const uint32_t phase = p_phase >> buffer & 1;
      p_phase ^= 1u << buffer;
      uint32_t skip = 0;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        wait_to_issue(bar(c.p_full[half][buffer]), phase);
        if (bad != 0) return;
        if (half == 0) skip = *const_cast<volatile uint32_t*>(&c.skip[buffer]);
        if (leader && skip == 0) {
#pragma unroll
          for (int chunk = 0; chunk < kChunks; ++chunk) {  // of 32 tokens: 16 columns of weights where 32 of scores were
            const int first = half * kHalf + 32 * chunk;
            ptx::mma_ts_mn<2>(tmem + L::kOutColumn + tile * kDim, tmem + buffer * kN + first, vd + (first * 128 >> 4), o_desc, more || first != 0);
            if (fine) ptx::mma_ts_mn<2>(tmem + L::kOutColumn + tile * kDim, tmem + buffer * kN + first + 16, vd + (first * 128 >> 4), o_desc, true);
          }
        }
      }
      if (leader) ptx::mma_commit(bar(c.o_done[L::kTwo ? tile : products[tile] & 1]));
      ++products[tile];
    };

    PromptWalk walk(c.start, c.plan_items);
    while (walk.left > 0 && bad == 0) {
      const PromptItem it = item_of(walk);
      if (bad != 0) break;
      const int32_t n = walk.here(it);
      const int tiles = L::kTwo && it.rows > kPromptTile ? 2 : 1;
      const bool fine = kCodes && it.steps <= kFineSteps;
      wait_to_issue(bar(c.q_full), q_phase);
      q_phase ^= 1;
      wait_slot(taken);
      wait_scales(taken / 2);
      if (bad != 0) break;
      for (int t = 0; t < tiles; ++t) scores(t, t, taken);
      free_slot(taken);
      if (n == 1 && leader) ptx::mma_commit(bar(c.q_empty));
#pragma unroll 1
      for (int32_t j = 0; j < n && bad == 0; ++j) {
        const uint32_t v = taken + 2 * j + 1, k = v + 1;
        const bool more = j + 1 < n;
        if (more) {
          wait_slot(k);
          wait_scales(k / 2);
        }
        if constexpr (!L::kTwo) {
          if (j != 0) ended(0);
          if (bad != 0) break;
          if (more) scores(0, (j + 1) & 1, k);
        }
        wait_slot(v);
        if constexpr (!kCodes) wait_to_issue(bar(c.looked[v / 2 % 8]), v / 16 & 1);
        if (bad != 0) break;
        if constexpr (L::kTwo) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t >= tiles) break;
            values(t, t, v, j != 0, fine);
            ended(t);
            if (bad != 0) break;
            if (more) scores(t, t, k);
          }
        } else {
          values(0, j & 1, v, j != 0, fine);
        }
        if (bad != 0) break;
        free_slot(v);
        if (kCodes && leader) ptx::mma_commit(bar(c.scales_empty[v / 2 % 4]));
        if (more) free_slot(k);
        if (j + 2 == n && leader) ptx::mma_commit(bar(c.q_empty));
      }
      if constexpr (!L::kTwo) {
        if (bad == 0) ended(0);
      }
      taken += 2 * n;
      walk.next(n);
    }
    // All products, and what they arrive on, are done before the CTA ends.
    if (leader) ptx::mma_commit(bar(c.drained));
    __syncwarp();
    ptx::mbar_drain(bar(c.drained), 0);
    if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptIssueTimeout);
  } else if (warp >= kLookWarp && warp < kLookWarp + kLookWarps) {
    // ---- queries that TMA does not load, and values that some rows do not see or, of codes, the scales ----
    // Zero times an infinity or a NaN would be a NaN for those rows too.  What no row of the item sees (rows of a box
    // outside its tokens) is set to zero; where something is left, the rows make the product themselves.  (Codes are
    // finite.  Their scales come here and not with the codes, so that a step's weights need not wait for its values.)
    const int w = warp - kLookWarp;
    uint32_t taken = 0, q_phase = 0;
    PromptWalk walk(c.start, c.plan_items);
    while (walk.left > 0 && bad == 0) {
      const PromptItem it = item_of(walk);
      if (bad != 0) break;
      const int32_t n = walk.here(it), token0 = (it.lo / kN + walk.step) * kN;
      if (!p.q_boxes) {
        wait(bar(c.q_empty), q_phase ^ 1);
        q_phase ^= 1;
        if (bad != 0) break;
        const uint32_t to = ptx::smem_u32(q_tile);
        constexpr int kQPieces = kDim / 8;
#pragma unroll 1
        for (int r0 = 32 * w; r0 < L::kTiles * kPromptTile && r0 < it.rows; r0 += 32 * kLookWarps) {
          const int32_t r = it.row0 + r0 + lane;
          int64_t offset = -1;
          if (r < it.row0 + it.rows) {
            const int32_t i = p.group.div(r), h = r - i * p.group.d;
            offset = (it.begin + i) * p.q_token + (static_cast<int64_t>(walk.head) * p.group.d + h) * p.q_head;
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
        ptx::cp_async_wait_all();
        publish(bar(c.q_full));
      }
      if constexpr (!kCodes) {
#pragma unroll 1
        for (int32_t j = 0; j < n; ++j) {
          const int32_t first = token0 + j * kN;
          const uint32_t number = taken + 2 * j + 1, slot = number % kRing, turn = number / 2 % 8;
          wait(bar(c.kv_full[slot]), number / kRing & 1);
          if (bad != 0) break;
          if (!any_masked(it, first)) {
            ptx::mbar_arrive_lane0(bar(c.looked[turn]), lane);
            continue;
          }
          uint8_t* const v = slots + slot * L::kSlotBytes;
          uint32_t most = 0;
          // (tokens from `low` to `high` are seen by all rows)
          const bool two = L::kTwo && it.rows > kPromptTile;
          const int32_t low = (two ? max(it.highest_lo[0], it.highest_lo[1]) : it.highest_lo[0]) - first;
          const int32_t high = (two ? min(it.lowest_hi[0], it.lowest_hi[1]) : it.lowest_hi[0]) - first;
#pragma unroll 2
          for (int i = w; i < L::kSlotBytes / 512; i += kLookWarps) {
            const int token0 = i * 4 % kN;
            if (token0 >= low && token0 + 4 <= high) continue;
            const int at = i * 512 + lane * 16, token = token0 + lane / 8, logical = (lane ^ token) & 7;
            uint4* const of = reinterpret_cast<uint4*>(v + at);
            if (first + token < it.lo || first + token >= it.hi) {
              *of = make_uint4(0, 0, 0, 0);
            } else if (kDim % 64 == 0 || at / (kN * 128) * 64 + 8 * logical < kDim) {
              const uint4 x = *of;
              most = __vmaxu2(__vmaxu2(most, __vmaxu2(x.x & 0x7FFF7FFFu, x.y & 0x7FFF7FFFu)), __vmaxu2(x.z & 0x7FFF7FFFu, x.w & 0x7FFF7FFFu));
            }
          }
          const bool any = __any_sync(0xffffffffu, (most & 0xFFFFu) >= 0x7F80u || (most >> 16) >= 0x7F80u);
          if (any && lane == 0) *const_cast<volatile uint32_t*>(&c.odd[turn]) = number + 1;
          publish(bar(c.looked[turn]));
        }
      } else {
        const int32_t* const table = p.tables + it.b * p.table_stride;
        constexpr int kEach = kN / kLookWarps / 32;
        int32_t page[kEach], place[kEach];
        auto look_up = [&](int32_t j) {
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            const int32_t token = token0 + j * kN + (w * kEach + e) * 32 + lane;
            place[e] = -1;
            if (j < n && token >= it.lo && token < it.hi) {
              const uint32_t index = p.cache.page_size.div(token);
              place[e] = token - index * p.cache.page_size.d;
              page[e] = load_arg(table + index);
            }
          }
        };
        look_up(0);
#pragma unroll 1
        for (int32_t j = 0; j < n; ++j) {
          float of_key[kEach], of_value[kEach];
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            of_key[e] = of_value[e] = 0.0f;
            if (place[e] < 0) continue;
            if (static_cast<uint32_t>(page[e]) < static_cast<uint32_t>(p.cache.num_pages)) {
              const int64_t at = page[e] * p.cache.scale_page + place[e] * p.cache.scale_token + walk.head * p.cache.scale_head;
              of_key[e] = load_arg(p.cache.k_scale + at);
              of_value[e] = load_arg(p.cache.v_scale + at);
            } else if (p.status != nullptr) {
              atomicOr(p.status, kStatusIndex);
            }
          }
          look_up(j + 1);
          const uint32_t step = taken / 2 + j;
          float* const to = scales + step % 4 * (2 * kN) + w * (32 * kEach) + lane;
          wait(bar(c.scales_empty[step % 4]), (step / 4 & 1) ^ 1);
          if (bad != 0) break;
          // scores times 64 (the keys' unit), the row's scale and what makes them logarithms to base 2 or fractions of the cap
          const float to_score = 64.0f * (kBent && p.cap > 0.0f ? p.cap_scale : p.scale);
#pragma unroll
          for (int e = 0; e < kEach; ++e) {
            to[32 * e] = of_key[e] * to_score;
            to[kN + 32 * e] = of_value[e];
          }
          __syncwarp();
          ptx::mbar_arrive_lane0(bar(c.looked[step % 8]), lane);
        }
      }
      taken += 2 * n;
      walk.next(n);
    }
    if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptLoadTimeout);
  } else if (kCodes && warp >= L::kTurnWarp) {
    if constexpr (kCodes) {
      // ---- codes into BF16, a quarter or an eighth of a step's tokens for each warp ----
      if constexpr (!L::kTwo) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRowRegs));
      const int w = warp - L::kTurnWarp;
      constexpr int kOwn = kN / L::kTurnWarps;
      constexpr int kPieces = kDim / 16;
      uint32_t slot = 0, slot_phase = 0, raw_slot = 0, raw_phase = 0;
      PromptWalk walk(c.start, c.plan_items);
      while (walk.left > 0 && bad == 0) {
        const PromptItem it = item_of(walk);
        if (bad != 0) break;
        const int32_t n = walk.here(it);
        const int32_t* const table = p.tables + it.b * p.table_stride;
        const int32_t token0 = (it.lo / kN + walk.step) * kN;
        // Turns the warp's tokens' codes into a slot: from the ring of codes or, where boxes do not fit, from memory.
        auto turn = [&](const uint8_t* from, int64_t offset) {
          uint8_t* const to = slots + slot * L::kSlotBytes;
          constexpr int kRounds = kOwn * kPieces / 32;
          auto put = [&](int at, const uint4& held) {
            const int token = w * kOwn + at / kPieces, piece = at % kPieces;
            uint4 low, high;
            decode16(held, low, high);
            // (lanes that write to the same 16 bytes of two blocks of 64 elements would share banks: odd blocks' second half first)
            const int swap = piece >> 2 & 1;
            *reinterpret_cast<uint4*>(to + place_of(token, 2 * piece + swap)) = swap ? high : low;
            *reinterpret_cast<uint4*>(to + place_of(token, 2 * piece + 1 - swap)) = swap ? low : high;
          };
          if (from == nullptr) {
            const uint8_t* const here = raw + raw_slot * L::kRawBytes + w * kOwn * kDim + lane * 16;
            constexpr int kAtOnce = kRounds % 4 == 0 ? 4 : kRounds % 3 == 0 ? 3 : 2;  // (all at once, they were spilled: 2.6 ms for 2.1)
            static_assert(kRounds % kAtOnce == 0, "whole batches");
#pragma unroll 1
            for (int i0 = 0; i0 < kRounds; i0 += kAtOnce) {
              uint4 held[kAtOnce];
#pragma unroll
              for (int i = 0; i < kAtOnce; ++i) held[i] = *reinterpret_cast<const uint4*>(here + (i0 + i) * 512);
#pragma unroll
              for (int i = 0; i < kAtOnce; ++i) put((i0 + i) * 32 + lane, held[i]);
            }
            return;
          }
#pragma unroll 2
          for (int i = 0; i < kRounds; ++i) {
            const int at = i * 32 + lane;
            const int64_t o = __shfl_sync(0xffffffffu, offset, at / kPieces);
            put(at, o >= 0 ? load_once(from + o + at % kPieces * 16) : make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u));
          }
        };
#pragma unroll 1
        for (int32_t j = 0; j < n && bad == 0; ++j) {
          int64_t offset = -1;  // of the token that the lane looks up (the scales' warps report pages that are not there)
          if (p.box == 0) {
            const int32_t token = token0 + j * kN + w * kOwn + lane % kOwn;
            if (token >= it.lo && token < it.hi) {
              const uint32_t index = p.cache.page_size.div(token);
              const int32_t page = load_arg(table + index);
              if (static_cast<uint32_t>(page) < static_cast<uint32_t>(p.cache.num_pages)) {
                offset = page * p.cache.page + (token - index * p.cache.page_size.d) * p.cache.token + walk.head * p.cache.head;
              }
            }
          }
#pragma unroll 1
          for (int which = 0; which < 2; ++which) {
            if (p.box != 0) wait(bar(c.raw_full[raw_slot]), raw_phase);
            wait(bar(c.kv_empty[slot]), slot_phase ^ 1);
            if (bad != 0) break;
            turn(p.box != 0 ? nullptr : which == 0 ? p.cache.k : p.cache.v, offset);
            publish(bar(c.kv_full[slot]));
            if (p.box != 0) {
              ptx::mbar_arrive_lane0(bar(c.raw_empty[raw_slot]), lane);
              if (++raw_slot == L::kRaw) raw_slot = 0, raw_phase ^= 1;
            }
            if (++slot == kRing) slot = 0, slot_phase ^= 1;
          }
        }
        walk.next(n);
      }
      if (bad != 0 && lane == 0 && p.status != nullptr) atomicOr(p.status, kPromptLoadTimeout);
    }
  } else if (warp < 8 * L::kTiles) {
    // ---- rows: two threads each, which have half of a step's tokens and, at an item's end, half of the values ----
    // Scores are taken 32 at a time; of all but the last 32, the highest one is found first and they are read from
    // tensor memory again for their weights: with all of them in registers some 150 bytes were spilled, to the
    // memory whose bandwidth the products use up.  (What the compiler still reports: none for heads of 192 and 256 and the plain
    // kernel of 64, 28 to 72 bytes for the other BF16 ones, 48 to 144 over codes.)
    // A wait that gives up does not take a warp out of its loops: both warps of 32 rows meet at their named barrier as often
    // as the item asks for, whatever has failed.
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(L::kRowRegs));  // (the host has checked that they are there)
    const int tile = warp >> 3, half = warp >> 2 & 1;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // its 32 lanes of tensor memory
    const uint32_t out_at = tmem + lanes + L::kOutColumn + tile * kDim;
    const uint32_t pair = 1 + tile * 4 + (warp & 3);
    uint32_t s_phase = 0, outputs = 0, taken = 0;
    uint32_t skipping = 0;  // by buffer, what c.skip holds
    // For the product of the last step.  A parity tells one product from the one before, no further: of one tile's, the last
    // but one may not have ended either, so these take turns at two barriers.
    auto product_ended = [&]() {
      const uint32_t last = outputs - 1;
      wait(bar(c.o_done[L::kTwo ? tile : last & 1]), (L::kTwo ? last : last >> 1) & 1);
      ptx::tc_fence_after();
    };

    PromptWalk walk(c.start, c.plan_items);
    while (walk.left > 0) {
      PromptItem it = item_of(walk);
      if (bad != 0) it = load_item(p, walk.item);
      const int32_t n = walk.here(it);
      if (it.rows > tile * kPromptTile) {
        PromptView view;
        int64_t result = -1;
        float slope = 0.0f;
        const int32_t r = tile * kPromptTile + row;
        if (r < it.rows) {
          const int32_t token = p.group.div(it.row0 + r);
          view = PromptView(p, it, token);
          const int32_t head = walk.head * static_cast<int32_t>(p.group.d) + it.row0 + r - token * static_cast<int32_t>(p.group.d);
          result = static_cast<int64_t>(it.begin + token) * p.heads + head;
          if constexpr (kBent) {
            if (p.slopes != nullptr) slope = load_arg(p.slopes + head) * 1.4426950408889634f;
          }
        }
        __syncwarp();

        float top = -INFINITY, sum = 0.0f;
        const int32_t token0 = (it.lo / kN + walk.step) * kN;
#pragma unroll 1
        for (int32_t j = 0; j < n; ++j) {
          const int32_t first = token0 + j * kN;
          const int buffer = L::kTwo ? tile : j & 1;
          const uint32_t s_at = tmem + lanes + buffer * kN + half * kHalf;
          const uint32_t v_number = taken + 2 * j + 1, v_slot = v_number % kRing;
          const bool partial = any_masked(it, first);
          bool odd = false;
          if (!kCodes && partial) {
            wait(bar(c.looked[v_number / 2 % 8]), v_number / 16 & 1);
            odd = *const_cast<volatile uint32_t*>(&c.odd[v_number / 2 % 8]) == v_number + 1;
          }
          wait(bar(c.s_full[buffer]), s_phase >> buffer & 1);
          s_phase ^= 1u << buffer;
          ptx::tc_fence_after();
          if constexpr (kCodes) wait(bar(c.looked[v_number / 2 % 8]), v_number / 16 & 1);  // (the scales)
          const float of_scores = kBent || kCodes ? 1.0f : p.scale;
          const bool changed = kBent || kCodes || partial;  // scores are kept as they become

          uint32_t bits[32];
          float (&x)[32] = reinterpret_cast<float (&)[32]>(bits);
          float highest = -INFINITY;
#pragma unroll
          for (int chunk = 0; chunk < kChunks; ++chunk) {
            ptx::tmem_ld_32x32b_x32(s_at + 32 * chunk, bits);
            ptx::tmem_wait_ld();
            if constexpr (kCodes) {
              const float4* const factor = reinterpret_cast<const float4*>(scales + v_number / 2 % 4 * (2 * kN) + half * kHalf + 32 * chunk);
#pragma unroll
              for (int i = 0; i < 32; i += 4) {
                const float4 f = factor[i / 4];
                x[i] *= f.x, x[i + 1] *= f.y, x[i + 2] *= f.z, x[i + 3] *= f.w;
              }
            }
            const uint32_t begin = view.lo - first - half * kHalf - 32 * chunk, span = max(view.hi - view.lo, 0);
            if constexpr (kBent) {
              if (p.cap > 0.0f) {
                // (by what the row itself sees, so that nothing else changes its bits)
                if (partial) {
#pragma unroll
                  for (int i = 0; i < 32; ++i) x[i] = i - begin < span ? x[i] : 0.0f;
                }
                float most = 0.0f;
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                  if constexpr (!kCodes) x[i] *= p.cap_scale, x[i + 1] *= p.cap_scale;
                  most = max3(most, fabsf(x[i]), fabsf(x[i + 1]));
                }
                if (most > kTanhBound) {
#pragma unroll
                  for (int i = 0; i < 32; ++i) x[i] = capped(x[i], p.cap);
                } else {
#pragma unroll
                  for (int i = 0; i < 32; i += 2) capped_pair(x[i], x[i + 1], p.cap);
                }
                __syncwarp();
              } else if constexpr (!kCodes) {
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] *= p.scale;
              }
              if (p.slopes != nullptr) {
                const float from = static_cast<float>(first + half * kHalf + 32 * chunk - view.position);
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = fmaf(-slope, fabsf(from + i), x[i]);
              }
            }
            if (partial) {
#pragma unroll
              for (int i = 0; i < 32; ++i) x[i] = i - begin < span ? x[i] : -INFINITY;
            }
            if ((changed && chunk + 1 < kChunks) || odd) ptx::tmem_st_32x32b_x32(s_at + 32 * chunk, bits);
            float high[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
            for (int i = 4; i + 8 <= 32; i += 8) {
#pragma unroll
              for (int k = 0; k < 4; ++k) high[k] = max3(high[k], x[i + 2 * k], x[i + 2 * k + 1]);
            }
            high[0] = max3(high[0], x[28], x[29]);
            high[1] = max3(high[1], x[30], x[31]);
            highest = fmaxf(highest, max3(fmaxf(high[0], high[1]), high[2], high[3]));
          }
          if (changed) {
            ptx::tmem_wait_st();
            ptx::tc_fence_before();
          }
          // The other half's: written before the barrier, not again before the other has arrived for its product.
          float* const shared = maxima + (L::kTwo ? tile : j & 1) * (2 * kPromptTile) + row;
          shared[half * kPromptTile] = highest;
          ptx::named_bar_sync(pair, 64);
          highest = fmaxf(highest, *const_cast<volatile float*>(shared + (1 - half) * kPromptTile)) * of_scores;
          if (__any_sync(0xffffffffu, highest > top + kSlack)) {
            const float next = highest > top + kSlack ? highest : top;  // (rows that need no other base keep theirs, and their bits)
            const float factor = next == -INFINITY ? 1.0f : exp2_fast(top - next);
            top = next;
            sum *= factor;
            if (j != 0 && half == 0) {  // (the products wait for this half)
              // (with two tiles the scores were made after the product before)
              if constexpr (!L::kTwo) product_ended();
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
            if (odd != (skipping >> buffer & 1)) {
              skipping ^= 1u << buffer;
              if (half == 0 && (warp & 3) == 0 && lane == 0) *const_cast<volatile uint32_t*>(&c.skip[buffer]) = odd;
            }
            if (odd) {
              // (all of it by the first half's warps, which have scaled what there is)
              ptx::tmem_wait_st();
              ptx::tc_fence_after();
              if (half == 0) {
                if constexpr (!L::kTwo) {
                  if (j != 0) product_ended();
                }
                const uint32_t scores_at = tmem + lanes + buffer * kN;
                sum += product_by_row<kDim, kN>(scores_at, out_at, slots + v_slot * L::kSlotBytes, 0, of_scores, base, j == 0);
                product_by_row<kDim, kN>(scores_at, out_at, slots + v_slot * L::kSlotBytes, kDim / 2, of_scores, base, j == 0);
              }
              ptx::tc_fence_before();
              __syncwarp();
              ptx::mbar_arrive_lane0(bar(c.p_full[half][buffer]), lane);
              ++outputs;
              continue;
            }
          }
          float sums[2][2] = {};
#pragma unroll
          for (int chunk = kChunks - 1; chunk >= 0; --chunk) {
            if (chunk + 1 < kChunks) {
              ptx::tmem_ld_32x32b_x32(s_at + 32 * chunk, bits);
              ptx::tmem_wait_ld();
            }
            const float4* const value_factor = reinterpret_cast<const float4*>(scales + v_number / 2 % 4 * (2 * kN) + kN + half * kHalf + 32 * chunk);
            uint32_t w[16];
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
              float e[4] = {x[k], x[k + 1], x[k + 2], x[k + 3]};
              fma_pair(e[0], e[1], of_scores, base);
              fma_pair(e[2], e[3], of_scores, base);
#pragma unroll
              for (int l = 0; l < 4; ++l) e[l] = exp2_fast(e[l]);
              add_pair(sums[0], e[0], e[1]);
              add_pair(sums[1], e[2], e[3]);
              if constexpr (kCodes) {
                const float4 f = value_factor[k / 4];
                // (a masked token's scale may be NaN)
                e[0] = e[0] == 0.0f ? 0.0f : e[0] * f.x, e[1] = e[1] == 0.0f ? 0.0f : e[1] * f.y;
                e[2] = e[2] == 0.0f ? 0.0f : e[2] * f.z, e[3] = e[3] == 0.0f ? 0.0f : e[3] * f.w;
              }
              w[k / 2] = pack_bf16(e[0], e[1]);
              w[k / 2 + 1] = pack_bf16(e[2], e[3]);
              if constexpr (kCodes) x[k] = e[0], x[k + 1] = e[1], x[k + 2] = e[2], x[k + 3] = e[3];
            }
            ptx::tmem_st_32x32b_x16(s_at + 32 * chunk, w);
            if constexpr (kCodes) {
              if (it.steps <= kFineSteps) {  // what the rounding has left
#pragma unroll
                for (int k = 0; k < 16; ++k) w[k] = pack_bf16(x[2 * k] - bf16_lo(w[k]), x[2 * k + 1] - bf16_hi(w[k]));
                ptx::tmem_st_32x32b_x16(s_at + 32 * chunk + 16, w);
              }
            }
          }
          sum += (sums[0][0] + sums[0][1]) + (sums[1][0] + sums[1][1]);
          ptx::tmem_wait_st();
          ptx::tc_fence_before();
          __syncwarp();
          ptx::mbar_arrive_lane0(bar(c.p_full[half][buffer]), lane);
          ++outputs;
        }

        // The end of the item, or of the CTA's part of it.
        float* const shared = maxima + (L::kTwo ? tile : n & 1) * (2 * kPromptTile) + row;
        ptx::named_bar_sync(pair, 64);  // (the other has read the last maximum)
        shared[half * kPromptTile] = sum;
        ptx::named_bar_sync(pair, 64);
        sum += *const_cast<volatile float*>(shared + (1 - half) * kPromptTile);
        product_ended();
        const bool whole = walk.step == 0 && n == it.steps;
        float* const part = p.parts + (2 * static_cast<int64_t>(blockIdx.x) + (walk.step == 0 ? 1 : 0)) * prompt_part_floats<kDim, kCodes>() +
                            static_cast<int64_t>(tile) * kPromptTile * (kDim + 2);
        if (whole) {
          const bool there = result >= 0;
          const PromptRates rates(p, there ? result : 0, top, sum, kUnit, there && half == 0);
          // in 64s while there are, the first half one more of them
          constexpr int kFirst = (kDim / 2 + 63) / 64 * 64 <= kDim ? (kDim / 2 + 31) / 32 * 32 : kDim / 2;
          const int begin = half == 0 ? 0 : kFirst, end = half == 0 ? kFirst : kDim;
#pragma unroll 1
          for (int i = begin; i < end; i += 64) {
            if (end - i >= 64) {
              write_rows<64>(p, out_at + i, kDim, i, result, rates.mine, rates.other, lane);
            } else {
              write_rows<32>(p, out_at + i, kDim, i, result, rates.mine, rates.other, lane);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < kDim / 2; i += 16) {
            uint32_t o[16];
            ptx::tmem_ld_32x32b_x16(out_at + half * (kDim / 2) + i, o);
            ptx::tmem_wait_ld();
            uint4* const to = reinterpret_cast<uint4*>(part) + (half * (kDim / 2) + i) / 4 * kPromptTile + row;
#pragma unroll
            for (int k = 0; k < 4; ++k) __stcg(to + k * kPromptTile, make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
          }
          if (half == 0) {
            __stcg(part + kDim * kPromptTile + row, top);
            __stcg(part + (kDim + 1) * kPromptTile + row, sum);
          }
        }
        ptx::tc_fence_before();
        ptx::named_bar_sync(pair, 64);  // the other has read the sum, and its values before the next item's are made
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
  if (warp == kIssueWarp) ptx::tmem_dealloc(tmem, 512);
}

}  // namespace chord
