// Products of a few rows with packed 4-bit weights, without routing blocks: one weight for up to 16
// rows, or an expert of its own for every row.
#include <cuda_bf16.h>

#include "../../include/chord_b200.h"
#include "common.h"
#include "warp_ops.cuh"

namespace chord {
namespace {

constexpr int kGemvWarps = 8;

struct GemvParams {
  const __nv_bfloat16* x;
  const int32_t* packed;
  const __nv_bfloat16* scale;
  const int32_t* expert_ids;  // null: expert 0 for every row
  __nv_bfloat16* out;
  int64_t x_stride;
  int32_t rows, n, k, num_experts, top_k, expert_base;
};

// The packed word is the A fragment of mma.m16n8k16 (16 weight rows x 16 K of a lane), so a 16-byte
// load per lane brings the operands of four products, and nothing is staged in shared memory: a warp's
// loads of a whole batch of scale groups are in flight at once.  Operands are the codes themselves,
// (code - 8) / 64, exact in BF16; a group's sum of 32 products is exact in FP32 up to its additions and
// is then multiplied by the group's scale, so that no weight is rounded.
//
// kTokens rows share the weight (a power of two; the last ones may be absent).  The product has eight
// columns, so fewer rows than eight leave columns idle: column n holds row n / kSlots, but only the
// K groups g with g % kSlots == n % kSlots (its other operands are zero).  The scales of kSlots groups
// are then applied at once, with a kSlots-th of the multiplications.
template <int kTokens, int kBatch>
__global__ void __launch_bounds__(kGemvWarps * 32, 2)
gemv_kernel(const GemvParams p) {
  constexpr int kTiles = kTokens > 8 ? 2 : 1;             // products of eight columns
  constexpr int kSlots = kTokens > 8 ? 1 : 8 / kTokens;   // scale groups side by side in a product
  constexpr int kSets = kBatch / kSlots;
  static_assert(kSets >= 1 && kBatch % kSlots == 0, "a batch holds whole sets");
  __shared__ float sums[kGemvWarps][kTokens][64];
  __shared__ float part[kTokens][64];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int q = lane & 3, r = lane >> 2;
  const int block = blockIdx.y, cluster = gridDim.x, rank = blockIdx.x;
  ptx::grid_dependency_wait();
  int32_t expert = 0;
  int64_t out_row = 0, x_row = 0;
  int rows = p.rows;
  if (p.expert_ids != nullptr) {
    out_row = blockIdx.z;
    x_row = out_row / p.top_k;
    rows = 1;
    const int64_t local = static_cast<int64_t>(__ldg(p.expert_ids + out_row)) - p.expert_base;
    if (local < 0 || local >= p.num_experts) {  // (the same in every CTA of the cluster)
      if (rank == 0 && threadIdx.x < 64) p.out[out_row * p.n + block * 64 + threadIdx.x] = __float2bfloat16(0.0f);
      return;
    }
    expert = static_cast<int32_t>(local);
  }
  const int groups = p.k / 32;
  const int32_t* words = p.packed + static_cast<int64_t>(expert) * (p.k / 16) * 2 * p.n + block * 128 + lane * 4;
  const __nv_bfloat16* scales = p.scale + static_cast<int64_t>(expert) * groups * p.n + block * 64 + r * 8;
  const int64_t line = 2 * static_cast<int64_t>(p.n);

  // Groups past the last are read as the last one, with zero inputs and a zero scale.
  // Sums of the lane: kSlots > 1: [16-row tile][upper half]; else [tile][product fragment].
  float acc[kTiles][4][4] = {};
  for (int first = (rank * kGemvWarps + warp) * kBatch; first < groups; first += cluster * kGemvWarps * kBatch) {
    uint4 w[2 * kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int32_t* at = words + 2 * min(first + i, groups - 1) * line;
      w[2 * i] = load_once(at);
      w[2 * i + 1] = load_once(at + line);
    }
    // Scales of the groups whose sums this lane will hold: columns 2 q and 2 q + 1.
    constexpr int kScales = kSlots > 1 ? 2 : 1;
    uint4 sc[kSets][kScales];
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
#pragma unroll
      for (int j = 0; j < kScales; ++j) {
        const int g = first + set * kSlots + (kSlots > 1 ? (2 * q + j) % kSlots : 0);
        sc[set][j] = load_once(scales + static_cast<int64_t>(min(g, groups - 1)) * p.n);
        if (g >= groups) sc[set][j] = make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int set = 0; set < kSets; ++set) {
      // The column's row and group: its 32 inputs in fragment order.
      uint32_t xr[kTiles][4];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int token = 8 * t + r / kSlots, g = first + set * kSlots + r % kSlots;
        const bool there = token < rows && g < groups;
        const uint32_t* x = reinterpret_cast<const uint32_t*>(p.x + (x_row + token) * p.x_stride + 32 * g + 2 * q);
#pragma unroll
        for (int i = 0; i < 4; ++i) xr[t][i] = there ? __ldg(x + 4 * i) : 0u;
      }
      float c[kTiles][4][4] = {};
#pragma unroll
      for (int slot = 0; slot < kSlots; ++slot) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4& v = w[2 * (set * kSlots + slot) + h];
          const uint32_t word[4] = {v.x, v.y, v.z, v.w};
          uint32_t b[kTiles][2];
#pragma unroll
          for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int i = 0; i < 2; ++i) b[t][i] = kSlots == 1 || r % kSlots == slot ? xr[t][2 * h + i] : 0u;
          }
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const uint32_t high = word[s] >> 8;
            constexpr uint32_t kOffset = 0xBE00BE00u;  // -8 / 64, twice
            const uint32_t a[4] = {bf16x2_fma(word[s] & 0x000F000Fu, kTwo127, kOffset),
                                   bf16x2_fma(high & 0x000F000Fu, kTwo127, kOffset),
                                   bf16x2_fma(word[s] & 0x00F000F0u, kTwo123, kOffset),
                                   bf16x2_fma(high & 0x00F000F0u, kTwo123, kOffset)};
#pragma unroll
            for (int t = 0; t < kTiles; ++t) ptx::mma_m16n8k16(c[t][s], a, b[t][0], b[t][1]);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t pair[kScales];
#pragma unroll
        for (int j = 0; j < kScales; ++j) {
          const uint4& v = sc[set][j];
          pair[j] = s == 0 ? v.x : s == 1 ? v.y : s == 2 ? v.z : v.w;
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          if constexpr (kSlots > 1) {
            acc[t][s][0] = fmaf(c[t][s][0], bf16_lo(pair[0]), fmaf(c[t][s][1], bf16_lo(pair[1]), acc[t][s][0]));
            acc[t][s][2] = fmaf(c[t][s][2], bf16_hi(pair[0]), fmaf(c[t][s][3], bf16_hi(pair[1]), acc[t][s][2]));
          } else {
            acc[t][s][0] = fmaf(c[t][s][0], bf16_lo(pair[0]), acc[t][s][0]);
            acc[t][s][1] = fmaf(c[t][s][1], bf16_lo(pair[0]), acc[t][s][1]);
            acc[t][s][2] = fmaf(c[t][s][2], bf16_hi(pair[0]), acc[t][s][2]);
            acc[t][s][3] = fmaf(c[t][s][3], bf16_hi(pair[0]), acc[t][s][3]);
          }
        }
      }
    }
  }

  // Sums over the lanes that hold the same row, over the warps, and over the cluster: always in the
  // same order.
#pragma unroll
  for (int s = 0; s < 4; ++s) {
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      if constexpr (kSlots > 1) {
        float v = acc[0][s][2 * rh];
#pragma unroll
        for (int d = 1; d < kSlots / 2; d <<= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
        if (2 * q % kSlots == 0) sums[warp][2 * q / kSlots][16 * s + 8 * rh + r] = v;
      } else {
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          sums[warp][8 * t + 2 * q][16 * s + 8 * rh + r] = acc[t][s][2 * rh];
          sums[warp][8 * t + 2 * q + 1][16 * s + 8 * rh + r] = acc[t][s][2 * rh + 1];
        }
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < kTokens * 64; i += kGemvWarps * 32) {
    float v = 0.0f;
#pragma unroll
    for (int j = 0; j < kGemvWarps; ++j) v += (&sums[j][0][0])[i];
    const int token = i / 64;
    if (cluster > 1) {
      (&part[0][0])[i] = v;
    } else if (token < rows) {
      p.out[(out_row + token) * p.n + block * 64 + i % 64] = __float2bfloat16(64.0f * v);
    }
  }
  if (cluster > 1) {
    __syncwarp();
    ptx::cluster_sync();
    for (int i = threadIdx.x * cluster + rank; i < rows * 64; i += kGemvWarps * 32 * cluster) {
      const uint32_t addr = ptx::smem_u32(&part[0][0] + i);
      float v = 0.0f;
      for (int j = 0; j < cluster; ++j) v += ld_cluster_f32(ptx::map_to_cta(addr, j));
      p.out[(out_row + i / 64) * p.n + block * 64 + i % 64] = __float2bfloat16(64.0f * v);
    }
    __syncwarp();
    ptx::cluster_sync();  // the others have read this CTA's sums
  }
}

using GemvFn = void (*)(GemvParams);

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
  GemvFn kernel;
  int batch = 8;
  if (shared == 1) kernel = gemv_kernel<1, 8>;
  else if (shared == 2) kernel = gemv_kernel<2, 8>;
  else if (shared <= 4) kernel = gemv_kernel<4, 4>, batch = 4;
  else if (shared <= 8) kernel = gemv_kernel<8, 4>, batch = 4;
  else kernel = gemv_kernel<16, 4>, batch = 4;
  const int64_t blocks = n / 64 * (expert_ids != nullptr ? rows : 1);
  const int64_t batches = (k / 32 + batch - 1) / batch;
  int cluster = 1;
  while (cluster < 8 && blocks * cluster < 2 * device.sm_count && cluster * kGemvWarps < batches) cluster *= 2;
  const GemvParams params = {static_cast<const __nv_bfloat16*>(x), packed, static_cast<const __nv_bfloat16*>(scale),
                             expert_ids, static_cast<__nv_bfloat16*>(out), x_stride, static_cast<int32_t>(rows),
                             static_cast<int32_t>(n), static_cast<int32_t>(k), static_cast<int32_t>(num_experts),
                             static_cast<int32_t>(top_k), static_cast<int32_t>(expert_base)};
  const dim3 grid(cluster, static_cast<unsigned>(n / 64), static_cast<unsigned>(expert_ids != nullptr ? rows : 1));
  OptionsReadLock guard(options_mutex());
  CHORD_CUDA(launch_kernel_clusters(kernel, cluster, grid, dim3(kGemvWarps * 32), 0, static_cast<cudaStream_t>(stream),
                                    options().pdl != 0, params));
  return kOk;
}

}  // extern "C"
