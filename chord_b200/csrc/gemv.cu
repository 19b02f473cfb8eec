// Products of a few rows with packed 4-bit weights, without routing blocks: one weight for up to 16
// rows, or an expert of its own for every row.
#include <cuda_bf16.h>

#include <atomic>

#include "../../include/chord_b200.h"
#include "common.h"
#include "warp_ops.cuh"

namespace chord {
namespace {

constexpr int kGemvWarps = 8;  // of a CTA; kernels for up to four rows also with half of them

struct GemvParams {
  const __nv_bfloat16* x;
  const int32_t* packed;
  const __nv_bfloat16* scale;
  const int32_t* expert_ids;  // null: expert 0 for every row
  __nv_bfloat16* out;
  int64_t x_stride;
  int32_t rows, n, k, num_experts, top_k, expert_base;
  bool wide_x;  // rows of x on 16-byte boundaries
};

// The packed word is the A fragment of mma.m16n8k16 (16 weight rows x 16 K of a lane): 16 bytes of a lane
// are the operands of four products.  Operands are the codes themselves, (code - 8) / 512, exact in BF16: one
// mask and one multiply-add for every two.  (By 512 so that 32 products of any finite inputs are finite.)  A group's sum of 32 products is exact in FP32 up to its
// additions and is then multiplied by the group's scale, so that no weight is rounded.  (Masked codes as
// they stand, with their offset taken off the sums by one more product, save those multiply-adds; one row
// of 14336 x 14336 took 30.6 us like that and 31.2 like this, eight rows 34.4 and 30.5.)
__device__ __forceinline__ void operand(uint32_t word, uint32_t (&a)[4]) {
  constexpr uint32_t kOffset = 0xBC80BC80u;                          // -8 / 512, twice
  constexpr uint32_t kTwo124 = 0x7D807D80u, kTwo120 = 0x7B807B80u;  // 2^124 and 2^120, twice
  const uint32_t high = word >> 8;
  a[0] = bf16x2_fma(word & 0x000F000Fu, kTwo124, kOffset);
  a[1] = bf16x2_fma(high & 0x000F000Fu, kTwo124, kOffset);
  a[2] = bf16x2_fma(word & 0x00F000F0u, kTwo120, kOffset);
  a[3] = bf16x2_fma(high & 0x00F000F0u, kTwo120, kOffset);
}

// The product has eight columns, so fewer rows than eight leave columns idle: column n holds row n / kSlots,
// but only the K groups g with g % kSlots == n % kSlots (its other operands are zero).  The scales of
// kSlots groups are then applied at once, with a kSlots-th of the multiplications.
//
// The K axis is split over the warps of a CTA and over a cluster of CTAs; their sums are joined through
// shared memory, always in the same order.

// Joins what the warps, and the CTAs of a cluster, have of kTokens x 64 results.  `sums`: room for
// kWarps + 1 times that many; a lane's are v(token, row) for its rows.
template <int kTokens, int kWarps>
__device__ __forceinline__ void join_and_store(const GemvParams& p, float* sums, int64_t out_row, int rows, int block) {
  const int cluster = gridDim.x, rank = blockIdx.x;
  float* const part = sums + kWarps * kTokens * 64;
  __syncthreads();
  for (int i = threadIdx.x; i < kTokens * 64; i += kWarps * 32) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < kWarps; ++j) v += sums[j * (kTokens * 64) + i];
    const int token = i / 64;
    if (cluster > 1) {
      part[i] = v;
    } else if (token < rows) {
      p.out[(out_row + token) * p.n + block * 64 + i % 64] = __float2bfloat16(512.0f * v);
    }
  }
  if (cluster > 1) {
    __syncwarp();
    ptx::cluster_sync();
    for (int i = threadIdx.x * cluster + rank; i < rows * 64; i += kWarps * 32 * cluster) {
      const uint32_t addr = ptx::smem_u32(part + i);
      float v = 0.0f;
      for (int j = 0; j < cluster; ++j) v += ld_cluster_f32(ptx::map_to_cta(addr, j));
      p.out[(out_row + i / 64) * p.n + block * 64 + i % 64] = __float2bfloat16(512.0f * v);
    }
    __syncwarp();
    ptx::cluster_sync();  // the others have read this CTA's sums
  }
}

// The row's expert; false: one that another GPU holds, whose row is stored as zeros.
__device__ __forceinline__ bool find_expert(const GemvParams& p, int64_t out_row, int block, int32_t* expert) {
  const int64_t local = static_cast<int64_t>(load_arg(p.expert_ids + out_row)) - p.expert_base;
  *expert = static_cast<int32_t>(local);
  if (local >= 0 && local < p.num_experts) return true;
  if (blockIdx.x == 0 && threadIdx.x < 64) p.out[out_row * p.n + block * 64 + threadIdx.x] = __float2bfloat16(0.0f);
  return false;
}

struct GemvPlace {
  const int32_t* words;
  const __nv_bfloat16* scales;
  int64_t out_row;
  int32_t x_row, rows;
};

// Up to four rows: words go straight into the registers that the products read, those of kBatch scale
// groups at a time, all in flight at once.  A warp's loads and products take turns, and instructions (14.6 for a
// word) fill half of an SM's issue slots: eight experts of 4096 x 7168, 132 MB, 27.5 us = 4.8 TB/s, 74 % of a plain
// copy's rate (29.6 us on the slowest of six GPUs, 69 %); one row of 14336 x 14336, whose 224 CTAs are two on some SMs and one on others, 26.5 us = 4.4 TB/s.  One
// row of 4096 x 7168, 16.5 MB, 5.6 us: a launch, one turn and the join of a cluster.
template <int kTokens, int kSlots, int kBatch, int kWarps>
__device__ __forceinline__ void gemv_few(const GemvParams& p, const GemvPlace& at, float (&acc)[4][2]) {
  constexpr int kSets = kBatch / kSlots;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = lane & 3, r = lane >> 2;
  const int groups = p.k / 32;
  const int64_t line = 2 * static_cast<int64_t>(p.n);
  const int token = r / kSlots;  // of the lane's column
  const __nv_bfloat16* const x = p.x + (at.x_row + (token < at.rows ? token : 0)) * p.x_stride + 2 * q;
#pragma unroll
  for (int s = 0; s < 4; ++s) acc[s][0] = acc[s][1] = 0.0f;

  // Groups past the last are read as the last one, with zero inputs and a zero scale.
  for (int first = (blockIdx.x * kWarps + warp) * kBatch; first < groups; first += gridDim.x * kWarps * kBatch) {
    uint4 w[2 * kBatch], sc[kSets][2];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int32_t* const from = at.words + 2 * min(first + i, groups - 1) * line;
      w[2 * i] = load_once(from);
      w[2 * i + 1] = load_once(from + line);
    }
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      // of the groups whose sums this lane will hold: columns 2 q and 2 q + 1
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int g = first + set * kSlots + (2 * q + j) % kSlots;
        sc[set][j] = load_once(at.scales + static_cast<int64_t>(min(g, groups - 1)) * p.n);
        if (g >= groups) sc[set][j] = make_uint4(0, 0, 0, 0);
      }
    }
    // The column's row and groups: 32 inputs of each in fragment order.
    uint32_t xr[kSets][4];
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      const int g = first + set * kSlots + r % kSlots;
      const bool there = token < at.rows && g < groups;
      const uint32_t* const from = reinterpret_cast<const uint32_t*>(x + (there ? 32 * g : 0));
#pragma unroll
      for (int i = 0; i < 4; ++i) xr[set][i] = there ? load_arg(from + 4 * i) : 0u;
    }
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      float c[4][4] = {};
#pragma unroll
      for (int slot = 0; slot < kSlots; ++slot) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4& v = w[2 * (set * kSlots + slot) + h];
          const uint32_t word[4] = {v.x, v.y, v.z, v.w};
          const bool mine = r % kSlots == slot;
          const uint32_t b0 = mine ? xr[set][2 * h] : 0u, b1 = mine ? xr[set][2 * h + 1] : 0u;
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            uint32_t a[4];
            operand(word[s], a);
            ptx::mma_m16n8k16(c[s], a, b0, b1);
          }
        }
      }
      const uint32_t low[4] = {sc[set][0].x, sc[set][0].y, sc[set][0].z, sc[set][0].w};
      const uint32_t high[4] = {sc[set][1].x, sc[set][1].y, sc[set][1].z, sc[set][1].w};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        acc[s][0] = fmaf(c[s][0], bf16_lo(low[s]), fmaf(c[s][1], bf16_lo(high[s]), acc[s][0]));
        acc[s][1] = fmaf(c[s][2], bf16_hi(low[s]), fmaf(c[s][3], bf16_hi(high[s]), acc[s][1]));
      }
    }
  }
}

template <int kTokens, int kSlots, int kBatch, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 16 / kWarps)
gemv_few_kernel(const GemvParams p) {
  static_assert(kSlots > 1 && kBatch % kSlots == 0 && kTokens * kSlots <= 8, "a batch holds whole sets");
  __shared__ float sums[(kWarps + 1) * kTokens * 64];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = lane & 3, r = lane >> 2;
  const int block = blockIdx.y;
  ptx::grid_dependency_wait();
  int32_t expert = 0;
  GemvPlace at = {nullptr, nullptr, 0, 0, p.rows};
  if (p.expert_ids != nullptr) {
    at.out_row = blockIdx.z;
    at.x_row = blockIdx.z / static_cast<uint32_t>(p.top_k);
    at.rows = 1;
    if (!find_expert(p, at.out_row, block, &expert)) return;  // (the same in every CTA of the cluster)
  }
  at.words = p.packed + static_cast<int64_t>(expert) * (p.k / 16) * 2 * p.n + block * 128 + lane * 4;
  at.scales = p.scale + static_cast<int64_t>(expert) * (p.k / 32) * p.n + block * 64 + r * 8;

  float acc[4][2];  // [16-row tile][upper half]
  gemv_few<kTokens, kSlots, kBatch, kWarps>(p, at, acc);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      float v = acc[s][rh];
#pragma unroll
      for (int d = 1; d < kSlots / 2; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
      if (2 * q % kSlots == 0 && 2 * q / kSlots < kTokens) sums[(warp * kTokens + 2 * q / kSlots) * 64 + 16 * s + 8 * rh + r] = v;
    }
  }
  join_and_store<kTokens, kWarps>(p, sums, at.out_row, at.rows, block);
}

// More rows, up to sixteen: a ring of cp.async stages for each warp, 64 K of 64 weight rows: 2 KB of words, their
// scales and the rows' inputs, which ldmatrix then reads as operands (with loads of four bytes straight
// into registers they took most of the time: 16 rows of 14336 x 7168 39.7 us, 23.1 like this).  Instructions bound it,
// 18 for a word with one product and 26 with two, 83 and 72 % of the busiest SM's issue slots: eight rows of 14336 x
// 14336 28.0 us = 4.1 TB/s, 16 of 14336 x 7168 23.1 us = 2.5 TB/s.
template <int kTokens>
struct GemvLayout {
  static constexpr int kTiles = kTokens > 8 ? 2 : 1;  // products of eight columns
  static constexpr int kXPitch = 144;                 // of 64 inputs: an odd number of 16-byte pieces
  static constexpr int kScales = 2048, kX = 2048 + 256;  // offsets
  static constexpr int kStageBytes = kX + kTokens * kXPitch;
  static constexpr int kStages = kTokens <= 8 ? 4 : 3;
  static constexpr int kSmem = kGemvWarps * kStages * kStageBytes;
  static_assert(kSmem >= (kGemvWarps + 1) * kTokens * 64 * 4, "the warps' sums take the ring's place");
};

template <int kTokens>
__device__ __forceinline__ void gemv_rows(const GemvParams& p, uint32_t ring, float (&acc)[GemvLayout<kTokens>::kTiles][4][4]) {
  using L = GemvLayout<kTokens>;
  constexpr int kTiles = L::kTiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = lane >> 2, block = blockIdx.y, rows = p.rows;
  const int pairs = p.k / 64;
  const int64_t line = 2 * static_cast<int64_t>(p.n);
#pragma unroll
  for (int t = 0; t < kTiles; ++t) {
#pragma unroll
    for (int s = 0; s < 4; ++s) acc[t][s][0] = acc[t][s][1] = acc[t][s][2] = acc[t][s][3] = 0.0f;
  }

  // The warp's pairs of scale groups are blockIdx.x * kGemvWarps + warp and every step-th from there.
  const int step = gridDim.x * kGemvWarps;
  int to_load = blockIdx.x * kGemvWarps + warp;
  const int32_t* words = p.packed + block * 128 + lane * 4 + 4 * to_load * line;
  const __nv_bfloat16* scales = p.scale + block * 64 + (lane & 7) * 8 + (2 * to_load + (lane >> 3)) * static_cast<int64_t>(p.n);
  const __nv_bfloat16* x = p.x + 64 * to_load;
  auto load = [&](uint32_t stage) {
    if (to_load < pairs) {
#pragma unroll
      for (int i = 0; i < 4; ++i) ptx::cp_async_16(stage + i * 512 + lane * 16, words + i * line, true);
      if (lane < 16) ptx::cp_async_16(stage + L::kScales + lane * 16, scales, true);
      // (rows on 16-byte boundaries or, one word at a time, on others)
      if (p.wide_x) {
#pragma unroll
        for (int i = 0; i < kTokens / 4; ++i) {
          const int row = 4 * i + (lane >> 3);
          ptx::cp_async_16(stage + L::kX + row * L::kXPitch + (lane & 7) * 16, x + (row < rows ? row * p.x_stride + (lane & 7) * 8 : 0), row < rows);
        }
      } else {
#pragma unroll
        for (int row = 0; row < kTokens; ++row) {
          cp_async_4(stage + L::kX + row * L::kXPitch + lane * 4, x + (row < rows ? row * p.x_stride + lane * 2 : 0), row < rows);
        }
      }
      to_load += step;
      words += 4 * step * line;
      scales += 2 * step * static_cast<int64_t>(p.n);
      x += 64 * step;
    }
    ptx::cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < L::kStages - 1; ++i) load(ring + i * L::kStageBytes);

  for (int pair = blockIdx.x * kGemvWarps + warp; pair < pairs;) {
#pragma unroll
    for (int turn = 0; turn < L::kStages; ++turn) {
      if (pair >= pairs) break;
      ptx::cp_async_wait_group<L::kStages - 2>();
      __syncwarp();
      load(ring + (turn + L::kStages - 1) % L::kStages * L::kStageBytes);
      pair += step;
      const uint32_t stage = ring + turn * L::kStageBytes;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        uint32_t xr[kTiles][4];
        float c[kTiles][4][4] = {};
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          ptx::ldmatrix_x4<0>(stage + L::kX + (8 * t + (lane & 7)) * L::kXPitch + g * 64 + (lane >> 3) * 16, xr[t]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = lds128(stage + (2 * g + h) * 512 + lane * 16);
          const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            uint32_t a[4];
            operand(word[s], a);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) ptx::mma_m16n8k16(c[t][s], a, xr[t][2 * h], xr[t][2 * h + 1]);
          }
        }
        const uint4 sc = lds128(stage + L::kScales + g * 128 + r * 16);
        const uint32_t both[4] = {sc.x, sc.y, sc.z, sc.w};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const float low = bf16_lo(both[s]), high = bf16_hi(both[s]);
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
            acc[t][s][0] = fmaf(c[t][s][0], low, acc[t][s][0]);
            acc[t][s][1] = fmaf(c[t][s][1], low, acc[t][s][1]);
            acc[t][s][2] = fmaf(c[t][s][2], high, acc[t][s][2]);
            acc[t][s][3] = fmaf(c[t][s][3], high, acc[t][s][3]);
          }
        }
      }
    }
  }
  ptx::cp_async_wait_group<0>();
  __syncwarp();
}

template <int kTokens>
__global__ void __launch_bounds__(kGemvWarps * 32, 2)
gemv_rows_kernel(const GemvParams p) {
  using L = GemvLayout<kTokens>;
  extern __shared__ __align__(16) uint8_t gemv_smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = lane & 3, r = lane >> 2;
  const uint32_t ring = ptx::smem_u32(gemv_smem) + warp * (L::kStages * L::kStageBytes);
  ptx::grid_dependency_wait();
  float acc[L::kTiles][4][4];
  gemv_rows<kTokens>(p, ring, acc);
  __syncthreads();  // (the ring's place is the sums')
  float* const sums = reinterpret_cast<float*>(gemv_smem);
#pragma unroll
  for (int t = 0; t < L::kTiles; ++t) {
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      float* const to = sums + (warp * kTokens + 8 * t + 2 * q) * 64 + 16 * s + r;
      to[0] = acc[t][s][0];
      to[64] = acc[t][s][1];
      to[8] = acc[t][s][2];
      to[72] = acc[t][s][3];
    }
  }
  join_and_store<kTokens, kGemvWarps>(p, sums, 0, p.rows, blockIdx.y);
}

struct GemvVariant {
  void (*kernel)(GemvParams);
  int smem, groups, ctas, index, warps;  // groups: that a warp takes at a time; ctas: of an SM
};

template <int kTokens, int kSlots, int kBatch>
GemvVariant few(bool half) {
  if (half) return {gemv_few_kernel<kTokens, kSlots, kBatch, kGemvWarps / 2>, 0, kBatch, 4, kTokens, kGemvWarps / 2};
  return {gemv_few_kernel<kTokens, kSlots, kBatch, kGemvWarps>, 0, kBatch, 2, kTokens, kGemvWarps};
}

template <int kTokens>
GemvVariant many_rows() {
  return {gemv_rows_kernel<kTokens>, GemvLayout<kTokens>::kSmem, 2, 1, kTokens, kGemvWarps};
}

// Allows a kernel its shared memory, once per device.
int allow_smem(const GemvVariant& v, int device) {
  static std::atomic<bool> done[64][17];
  std::atomic<bool>& known = done[device & 63][v.index];
  if (v.smem <= 48 * 1024 || known.load(std::memory_order_acquire)) return kOk;
  CHORD_CUDA(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem));
  known.store(true, std::memory_order_release);
  return kOk;
}

}  // namespace
}  // namespace chord

extern "C" {

int chord_b200_gemv(const void* x, int64_t x_stride, const int32_t* packed, const void* scale, const int32_t* expert_ids,
                    void* out, int64_t rows, int64_t n, int64_t k, int64_t num_experts, int64_t top_k,
                    int64_t expert_base, void* stream) {
  using namespace chord;
  CHORD_REQUIRE(x != nullptr && packed != nullptr && scale != nullptr && out != nullptr, "null tensor pointer");
  CHORD_REQUIRE(n > 0 && n % 128 == 0 && n <= 65535ll * 64, "n must be a positive multiple of 128 up to %lld, got %lld",
                65535ll * 64 / 128 * 128, static_cast<long long>(n));
  CHORD_REQUIRE(k > 0 && k % 64 == 0 && k < (1ll << 30), "k must be a positive multiple of 64, got %lld",
                static_cast<long long>(k));
  CHORD_REQUIRE(num_experts > 0 && num_experts < (1ll << 31), "num_experts must be positive");
  CHORD_REQUIRE(top_k > 0 && top_k < (1ll << 31), "top_k must be positive");
  CHORD_REQUIRE(expert_base >= 0 && expert_base < (1ll << 31), "expert_base out of range");
  CHORD_REQUIRE(x_stride >= k && x_stride % 2 == 0, "rows of x must be k elements or more apart, an even number");
  CHORD_REQUIRE(((reinterpret_cast<uintptr_t>(packed) | reinterpret_cast<uintptr_t>(scale)) & 15u) == 0 &&
                    (reinterpret_cast<uintptr_t>(x) & 3u) == 0 && (reinterpret_cast<uintptr_t>(out) & 1u) == 0,
                "the weight must be 16-byte aligned, x 4-byte and out 2-byte aligned");
  const int64_t limit = expert_ids != nullptr ? 65535 : 16;
  CHORD_REQUIRE(rows >= 0 && rows <= limit, "rows must be in [0, %lld], got %lld", static_cast<long long>(limit),
                static_cast<long long>(rows));
  if (rows == 0) return kOk;
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;

  const int64_t shared = expert_ids != nullptr ? 1 : rows;
  const int64_t blocks = n / 64 * (expert_ids != nullptr ? rows : 1);
  // CTAs of four warps where there are more of them than are resident with eight.  Eight experts of 4096 x 7168
  // 29.3 us with eight warps, 27.5 with four, of 7168 x 2048 16.5 and 15.1; one row of 28416 x 4096 16.2 and
  // 14.2; where all are resident eight are better, 14336 x 14336 26.5 and 27.6, 7168 x 2048 3.1 and 3.6.
  const bool half = blocks > 2ll * device.sm_count;
  // Three and four rows take the ring where a warp has a long way to go: 4096 x 7168 7.0 us without and 6.8 with it,
  // 8192 x 8192 11.4 and 10.1, 14336 x 14336 30.6 and 27.2; 28416 x 4096 16.7 and 18.2, 14336 x 2048 5.9 and 6.2, 1024 x 512
  // 1.9 and 2.3.  Two rows 4096 x 7168 6.4 and 6.9.
  const GemvVariant v = shared == 1 ? few<1, 8, 8>(half) : shared == 2 ? few<2, 4, 8>(half) :
                        shared <= 4 && k <= 4096 ? few<4, 2, 4>(half) :
                        shared <= 8 ? many_rows<8>() : many_rows<16>();
  if (int rc = allow_smem(v, device.device)) return rc;
  // CTAs of a cluster: the fewest with which a warp has the least to do, where all CTAs are resident at once.
  // One row of 4096 x 7168: one CTA for 64 rows of the weight 10.7 us, two 7.5, four 6.2, eight (more than are
  // resident) 11.3; 7168 x 2048, whose batches of K are as many as the warps of one CTA, 3.1 with one, 5.3 with
  // two; 14336 x 14336 26.5 with one, 32.0 with two.  13 rows of 7168 x 2048, whose CTAs are best one to an
  // SM: 5.6 with one, 8.0 with two.
  const int64_t batches = (k / 32 + v.groups - 1) / v.groups;
  int cluster = 1;
  for (int c = 2; c <= 8 && blocks * c <= static_cast<int64_t>(v.ctas) * device.sm_count; c *= 2) {
    const auto turns = [&](int ctas) { return (batches + ctas * v.warps - 1) / (ctas * v.warps); };
    if (turns(c) < turns(cluster)) cluster = c;
  }
  const GemvParams params = {static_cast<const __nv_bfloat16*>(x), packed, static_cast<const __nv_bfloat16*>(scale),
                             expert_ids, static_cast<__nv_bfloat16*>(out), x_stride, static_cast<int32_t>(rows),
                             static_cast<int32_t>(n), static_cast<int32_t>(k), static_cast<int32_t>(num_experts),
                             static_cast<int32_t>(top_k), static_cast<int32_t>(expert_base),
                             x_stride % 8 == 0 && (reinterpret_cast<uintptr_t>(x) & 15u) == 0};
  const dim3 grid(cluster, static_cast<unsigned>(n / 64), static_cast<unsigned>(expert_ids != nullptr ? rows : 1));
  CHORD_CUDA(launch_kernel_clusters(v.kernel, cluster, grid, dim3(v.warps * 32), v.smem, static_cast<cudaStream_t>(stream),
                                    kEarlyLaunch, params));
  return kOk;
}

}  // extern "C"
