// How the work of prompt.cuh is dealt out, and the entry points.
#include <mutex>

#include "../../include/chord_b200.h"
#include "attention.h"
#include "common.h"
#include "prompt_kernels.cuh"
#include "register_split.h"
#include "tensor_map.h"

namespace chord {
namespace {

constexpr int kPlanThreads = 1024;

// The plan by one CTA, for more items or sequences than the main kernel's CTAs go through on their own.
__global__ void __launch_bounds__(kPlanThreads, 1) prompt_plan_kernel(const __grid_constant__ PromptParams p, int32_t log_rows, int32_t log_tokens) {
  __shared__ PromptPlanScratch scratch;
  ptx::grid_dependency_wait();
  PromptPlanner<kPlanThreads> planner(p, scratch, log_rows, log_tokens);
  planner.items([&](int32_t item, const PromptItem& it) { p.items[item] = it; });
  const PromptPlan plan = planner.plan();
  if (threadIdx.x == 0) *p.plan = plan;
#pragma unroll 1
  for (int32_t cta = threadIdx.x; cta < p.ctas; cta += kPlanThreads) {
    p.cta_starts[cta] = planner.start(plan, cta, [&](int32_t item) { return p.items[item].first; }, [&](int32_t item) { return p.items[item].steps; });
  }
}

bool prompt_variant_of(int64_t dim, bool codes, bool bent, PromptVariant* out) {
  if (codes) return bent ? prompt_codes_bent(dim, out) : prompt_codes(dim, out);
  return bent ? prompt_bf16_bent(dim, out) : prompt_bf16(dim, out);
}

// Allows a kernel its shared memory and checks that its warps can divide its registers, once per device.
int allow_prompt(const PromptVariant& v, int64_t dim, bool codes, bool bent, int device) {
  static std::mutex mutex;
  static bool done[64][5][2][2];
  std::lock_guard<std::mutex> guard(mutex);
  bool& known = done[device & 63][dim == 64 ? 0 : dim == 96 ? 1 : dim == 128 ? 2 : dim == 192 ? 3 : 4][codes][bent];
  if (known) return kOk;
  cudaFuncAttributes attributes;
  CHORD_CUDA(cudaFuncGetAttributes(&attributes, v.kernel));
  if (!register_split_fits(attributes.numRegs, v.threads / 32 - kLoadWarp, v.other_regs, kLoadWarp, v.row_regs)) {
    return fail(kUnsupportedDevice, "the attention kernel was compiled to %d registers, too few for its warps", attributes.numRegs);
  }
  CHORD_CUDA(cudaFuncSetAttribute(v.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, v.smem));
  known = true;
  return kOk;
}

constexpr int64_t aligned(int64_t bytes) { return (bytes + 255) / 256 * 256; }

int64_t most_items(int64_t batch, int64_t tokens, int64_t group, int64_t tiles) {
  return tokens * group / (tiles * kPromptTile) + batch;
}

// Where things lie in the workspace.
struct PromptScratch {
  int64_t starts, items, before, parts, end;
  PromptScratch(int64_t max_items, int64_t batch, int64_t ctas, int64_t part_floats) {
    starts = aligned(sizeof(PromptPlan));
    items = starts + aligned(ctas * sizeof(PromptStart));
    before = items + aligned(max_items * sizeof(PromptItem));
    parts = before + aligned(batch * 4);
    end = parts + ctas * 2 * part_floats * 4;
  }
};

struct PromptCall {
  const void* q;
  int64_t q_token, q_head;
  const chord_b200_kv_cache* cache;
  const int32_t* tables;
  int64_t table_stride, max_pages;
  const int32_t *lengths, *offsets, *starts, *prefixes, *own;
  int64_t own_capacity;
  const float *extra, *extra_lse;
  void* out;
  float* lse;
  void* workspace;
  int64_t workspace_bytes;
  int32_t* status;
  int64_t batch, tokens, heads;
  const chord_b200_scores* scores;
  void* stream;
};

int64_t token_capacity(int64_t max_pages, const chord_b200_kv_cache* cache) {
  // (token numbers, those of a step behind the last too, fit 32 bits)
  const int64_t capacity = max_pages * cache->page_size;
  return capacity > (1ll << 31) - 65536 ? (1ll << 31) - 65536 : capacity;
}

// The checks that the entry points share.
int check_prompt(const PromptCall& c) {
  CHORD_REQUIRE(c.q != nullptr && c.tables != nullptr && c.lengths != nullptr && c.offsets != nullptr && c.out != nullptr &&
                    c.workspace != nullptr && c.scores != nullptr,
                "null pointer");
  CHORD_REQUIRE(c.heads > 0 && c.heads <= 65535 && c.heads % c.cache->heads == 0,
                "the number of query heads (%lld) must be a multiple of the cache's (%lld)", static_cast<long long>(c.heads),
                static_cast<long long>(c.cache->heads));
  CHORD_REQUIRE(c.q_token >= 0 && c.q_head >= 0 && c.q_token % 8 == 0 && c.q_head % 8 == 0 &&
                    ((reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.out) | reinterpret_cast<uintptr_t>(c.workspace)) & 15u) == 0,
                "q's rows, out and the workspace must lie on 16-byte boundaries");
  CHORD_REQUIRE(c.max_pages > 0 && c.table_stride >= 0 && c.max_pages < (1ll << 31), "a block table has a page or more");
  CHORD_REQUIRE(c.scores->window >= 0 && c.scores->window < (1ll << 31), "window out of range");
  CHORD_REQUIRE(c.scores->scale - c.scores->scale == 0.0, "scale must be finite");
  CHORD_REQUIRE(cap_fits(*c.scores), "the cap must be zero or from 1e-30 to 1e30, and the scale no more than 1e36 of it");
  PromptVariant v;
  CHORD_REQUIRE(prompt_bf16(c.cache->head_dim, &v), "head_dim must be 64, 96, 128, 192 or 256, got %lld", static_cast<long long>(c.cache->head_dim));
  // (rows of a sequence are numbered in 32 bits)
  CHORD_REQUIRE(c.tokens * (c.heads / c.cache->heads) < (1ll << 31) - 65536, "too many query tokens and heads: %lld x %lld",
                static_cast<long long>(c.tokens), static_cast<long long>(c.heads));
  return kOk;
}

// A descriptor of rows of `dim` elements in up to three further dimensions (sizes, strides in bytes): BF16 in boxes of 64
// elements, swizzled as the products read them, or codes in whole rows.  False where there is none (strides of zero, for one).
bool make_rows_map(CUtensorMap* out, const void* base, bool codes, int64_t dim, int rank, const int64_t* sizes, const int64_t* strides,
                   const uint32_t* box) {
  const EncodeTiledFn encode = encode_tiled_fn();
  if (encode == nullptr) return false;
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim)}, steps[3];
  cuuint32_t boxes[4] = {codes ? static_cast<cuuint32_t>(dim) : 64}, ones[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank - 1; ++i) {
    dims[i + 1] = static_cast<cuuint64_t>(sizes[i]);
    steps[i] = static_cast<cuuint64_t>(sizes[i] == 1 ? 16 : strides[i]);  // (of one only, no stride counts)
    boxes[i + 1] = box[i];
    if (steps[i] == 0 || steps[i] % 16 != 0 || steps[i] >= (1ull << 40)) return false;
  }
  return encode(out, codes ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, static_cast<cuuint32_t>(rank),
                const_cast<void*>(base), dims, steps, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int launch_prompt(const PromptCall& c, const Cache& cache, const DeviceInfo& device) {
  PromptParams p = {};
  p.cache = cache;
  const int64_t group = c.heads / c.cache->heads;
  const bool codes = c.cache->k_scale != nullptr;
  constexpr double kLog2E = 1.4426950408889634074;
  p.scale = static_cast<float>(c.scores->scale * kLog2E);
  // (the plain kernels find the largest score before they scale it, so what they multiply with is above zero, in FP32 too)
  const bool bent = c.scores->cap > 0.0 || c.scores->slopes != nullptr || p.scale <= 0.0f;
  PromptVariant v;
  CHORD_REQUIRE(prompt_variant_of(c.cache->head_dim, codes, bent, &v), "head_dim must be 64, 96, 128, 192 or 256, got %lld",
                static_cast<long long>(c.cache->head_dim));
  if (int rc = allow_prompt(v, c.cache->head_dim, codes, bent, device.device)) return rc;
  const int64_t max_items = most_items(c.batch, c.tokens, group, v.tiles);
  const int64_t ctas = device.sm_count;
  const PromptScratch at(max_items, c.batch, ctas, v.part_floats);
  CHORD_REQUIRE(c.workspace_bytes >= at.end, "the workspace has %lld bytes, this launch needs %lld",
                static_cast<long long>(c.workspace_bytes), static_cast<long long>(at.end));
  uint8_t* const w = static_cast<uint8_t*>(c.workspace);
  p.plan = reinterpret_cast<PromptPlan*>(w);
  p.cta_starts = reinterpret_cast<PromptStart*>(w + at.starts);
  p.items = reinterpret_cast<PromptItem*>(w + at.items);
  p.tiles_before = reinterpret_cast<int32_t*>(w + at.before);
  p.parts = reinterpret_cast<float*>(w + at.parts);
  p.q = static_cast<const __nv_bfloat16*>(c.q);
  p.q_token = c.q_token;
  p.q_head = c.q_head;
  p.tables = c.tables;
  p.table_stride = c.table_stride;
  p.lengths = c.lengths;
  p.offsets = c.offsets;
  p.starts = c.starts;
  p.prefixes = c.prefixes;
  p.own = c.own;
  p.slopes = c.scores->slopes;
  p.extra = c.extra;
  p.extra_lse = c.extra_lse;
  p.out = static_cast<__nv_bfloat16*>(c.out);
  p.out_32 = (reinterpret_cast<uintptr_t>(c.out) & 31u) == 0;
  p.lse = c.lse;
  p.status = c.status;
  p.cap = static_cast<float>(c.scores->cap * kLog2E);
  p.cap_scale = c.scores->cap > 0.0 ? static_cast<float>(c.scores->scale / c.scores->cap) : 0.0f;
  p.batch = static_cast<int32_t>(c.batch);
  p.tokens = static_cast<int32_t>(c.tokens);
  p.heads = static_cast<int32_t>(c.heads);
  p.kv_heads = static_cast<int32_t>(c.cache->heads);
  p.capacity = static_cast<int32_t>(token_capacity(c.max_pages, c.cache));
  p.own_capacity = static_cast<int32_t>(c.own_capacity);
  p.window = static_cast<int32_t>(c.scores->window);
  p.max_items = static_cast<int32_t>(max_items);
  p.ctas = static_cast<int32_t>(ctas);
  p.group = Divisor(static_cast<uint32_t>(group));
  {
    const int64_t page = c.cache->page_size;
    int32_t box = 1;
    while (box < v.step_tokens && page % (2 * box) == 0) box *= 2;
    // (heads or pages that are all one: views with a stride of zero)
    p.head_step = cache.head != 0;
    p.page_step = cache.page != 0;
    const int64_t sizes[3] = {page, p.head_step ? c.cache->heads : 1, p.page_step ? c.cache->num_pages : 1};
    const int64_t strides[3] = {cache.token, cache.head, cache.page};
    const uint32_t boxes[3] = {static_cast<uint32_t>(box), 1, 1};
    // a box starts on 128 bytes of shared memory
    if (!codes || box * c.cache->head_dim % 128 == 0) {
      if (make_rows_map(&p.k_map, c.cache->k, codes, c.cache->head_dim, 4, sizes, strides, boxes) &&
          make_rows_map(&p.v_map, c.cache->v, codes, c.cache->head_dim, 4, sizes, strides, boxes)) {
        p.box = box;
      }
    }
    CHORD_REQUIRE(codes || p.box != 0, "the cache's strides must be from 16 to 2^40 - 16 bytes (those of heads and pages may be zero)");
  }
  if (kPromptTile % group == 0) {
    const int64_t sizes[2] = {c.heads, c.tokens}, strides[2] = {2 * c.q_head, 2 * c.q_token};
    const uint32_t boxes[2] = {static_cast<uint32_t>(group), static_cast<uint32_t>(kPromptTile / group)};
    p.q_boxes = make_rows_map(&p.q_map, c.q, false, c.cache->head_dim, 3, sizes, strides, boxes);
  }
  const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
  p.self = max_items <= kPlanHeld && c.batch <= kPlanHeld;
  if (!p.self) {
    CHORD_CUDA(launch_kernel(prompt_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, kEarlyLaunch, p, v.tiles == 2 ? 8 : 7,
                             v.step_tokens == 128 ? 7 : 6));
  }
  CHORD_CUDA(launch_kernel(v.kernel, dim3(static_cast<unsigned>(ctas)), dim3(static_cast<unsigned>(v.threads)), v.smem, stream, kEarlyLaunch, p));
  // Nothing is cut, whatever the lengths, where there are CTAs for all items and no table holds more than a few steps.
  const bool whole = max_items * c.cache->heads <= ctas && (token_capacity(c.max_pages, c.cache) + v.step_tokens - 1) / v.step_tokens <= kPromptAlone;
  if (ctas > 1 && !whole) {
    CHORD_CUDA(launch_kernel(v.join, dim3(static_cast<unsigned>(ctas - 1), static_cast<unsigned>(v.tiles * c.cache->head_dim / 8)),
                             dim3(kPromptTile), 0, stream, kEarlyLaunch, p));
  }
  return kOk;
}

int64_t prompt_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, const DeviceInfo& device) {
  PromptVariant v, w;
  if (kv_heads <= 0 || heads <= 0 || batch < 0 || tokens < 0 || !prompt_bf16(head_dim, &v) || !prompt_codes(head_dim, &w)) {
    return fail(kInvalidArgument, "head_dim must be 64, 96, 128, 192 or 256, and no size negative"), -1;
  }
  const int64_t floats = v.part_floats > w.part_floats ? v.part_floats : w.part_floats;
  return PromptScratch(most_items(batch, tokens, heads / kv_heads, v.tiles), batch, device.sm_count, floats).end;
}

}  // namespace
}  // namespace chord

extern "C" {

int64_t chord_b200_prompt_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim) {
  using namespace chord;
  DeviceInfo device;
  if (current_device_info(&device)) return -1;
  return prompt_bytes(batch, tokens, heads, kv_heads, head_dim, device);
}

int chord_b200_prompt_attention(const void* q, int64_t q_token, int64_t q_head, const chord_b200_kv_cache* cache,
                                const int32_t* tables, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
                                const int32_t* offsets, const int32_t* starts, const int32_t* prefixes, void* out, float* lse,
                                void* workspace, int64_t workspace_bytes, int32_t* status, int64_t batch, int64_t tokens,
                                int64_t heads, const chord_b200_scores* scores, void* stream) {
  using namespace chord;
  Cache pages;
  if (int rc = make_cache(cache, &pages)) return rc;
  CHORD_REQUIRE(batch >= 0 && batch < (1ll << 31) && tokens >= 0 && tokens < (1ll << 31), "sizes out of range");
  if (batch == 0 || tokens == 0) return kOk;
  const PromptCall c = {q, q_token, q_head, cache, tables, table_stride, max_pages, lengths, offsets, starts, prefixes, nullptr,
                        0, nullptr, nullptr, out, lse, workspace, workspace_bytes, status, batch, tokens, heads, scores, stream};
  if (int rc = check_prompt(c)) return rc;
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  return launch_prompt(c, pages, device);
}

int64_t chord_b200_shared_prefix_attention_workspace_bytes(int64_t groups, int64_t batch, int64_t heads, int64_t kv_heads,
                                                           int64_t head_dim) {
  using namespace chord;
  DeviceInfo device;
  if (current_device_info(&device)) return -1;
  const int64_t prompt = prompt_bytes(groups, batch, heads, kv_heads, head_dim, device);
  if (prompt < 0) return -1;
  const int64_t token = chord_b200_paged_attention_workspace_bytes(head_dim, heads / kv_heads);
  if (token < 0) return -1;
  // the tokens' own parts, their sums, and room for either kernel
  return aligned(batch * heads * head_dim * 4) + aligned(batch * heads * 4) + (prompt > token ? prompt : token);
}

int chord_b200_shared_prefix_attention(const void* q, int64_t q_batch, int64_t q_head, const chord_b200_kv_cache* cache,
                                       const int32_t* prefix_tables, int64_t prefix_stride, int64_t prefix_pages,
                                       const int32_t* prefix_lengths, const int32_t* group_offsets, int64_t groups,
                                       const int32_t* tables, int64_t table_stride, int64_t max_pages, const int32_t* lengths,
                                       void* out, float* lse, int32_t* locks, int64_t num_locks, void* workspace,
                                       int64_t workspace_bytes, int32_t* status, int64_t batch, int64_t heads,
                                       const chord_b200_scores* scores, void* stream) {
  using namespace chord;
  Cache pages;
  if (int rc = make_cache(cache, &pages)) return rc;
  CHORD_REQUIRE(batch >= 0 && batch < (1ll << 31) && groups >= 0 && groups < (1ll << 31), "sizes out of range");
  if (batch == 0 || groups == 0) return kOk;
  const int64_t own_bytes = aligned(batch * heads * cache->head_dim * 4), sum_bytes = aligned(batch * heads * 4);
  uint8_t* const w = static_cast<uint8_t*>(workspace);
  CHORD_REQUIRE(workspace != nullptr && workspace_bytes >= own_bytes + sum_bytes, "the workspace has %lld bytes, this launch needs more",
                static_cast<long long>(workspace_bytes));
  float* const own = reinterpret_cast<float*>(w);
  float* const own_lse = reinterpret_cast<float*>(w + own_bytes);
  void* const rest = w + own_bytes + sum_bytes;
  const int64_t rest_bytes = workspace_bytes - own_bytes - sum_bytes;
  const PromptCall c = {q, q_batch, q_head, cache, prefix_tables, prefix_stride, prefix_pages, prefix_lengths, group_offsets, nullptr,
                        nullptr, lengths, max_pages > 0 ? token_capacity(max_pages, cache) : 0, own, own_lse, out, lse, rest, rest_bytes,
                        status, groups, batch, heads, scores, stream};
  CHORD_REQUIRE(lengths != nullptr && tables != nullptr && locks != nullptr, "null pointer");
  CHORD_REQUIRE(max_pages > 0 && table_stride >= 0 && max_pages < (1ll << 31), "a block table has a page or more");
  if (int rc = check_prompt(c)) return rc;
  DeviceInfo device;
  if (int rc = current_device_info(&device)) return rc;
  if (int rc = require_blackwell(device)) return rc;
  // Each token's own part first, left in FP32; the kernel over the prefixes adds it.
  if (int rc = paged_attention(q, q_batch, q_head, cache, tables, table_stride, max_pages, lengths, nullptr, own, own_lse, locks, num_locks,
                               rest, rest_bytes, status, batch, heads, *scores, true, stream)) {
    return rc;
  }
  return launch_prompt(c, pages, device);
}

}  // extern "C"
