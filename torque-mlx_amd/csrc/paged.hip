// paged.hip -- the paged 8-bit KV cache: kernels and C ABI.  Declarations are in
// include/torque_hip.h.
//
// Kernels
//   paged_append_kernel  new keys and values into their pages, turned to their
//                        positions and into the rotated basis on the way; the
//                        queries of the same tokens beside them
//   paged_read_kernel    pages -> the values they stand for
//   paged_split_kernel   attention of few rows over long contexts
//   paged_merge_kernel   the parts of rows whose keys were cut, as one

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>

#include "paged_append.hpp"
#include "paged_attention.hpp"
#include "torque_hip.h"
#include "tq_host.hpp"

using namespace tq;

namespace {

int check_pages(int num_pages, int page_size, int kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(TQ_ERR_UNSUPPORTED, "Unsupported head dimension: " + std::to_string(head_dim));
  if (page_size != 16 && page_size != 32 && page_size != 64)
    return fail(TQ_ERR_UNSUPPORTED, "Unsupported page size: " + std::to_string(page_size));
  if (num_pages <= 0 || kv_heads <= 0) return fail(TQ_ERR_BAD_ARG, "num_pages and kv_heads must be positive");
  if (kv_heads > 65535) return fail(TQ_ERR_BAD_ARG, "kv_heads must be at most 65535");
  return TQ_OK;
}

int check_batch(int64_t tokens, int batch, int max_pages, int64_t table_stride, const int32_t* starts) {
  if (tokens < 0 || batch < 0 || max_pages < 0) return fail(TQ_ERR_BAD_ARG, "tokens, batch and max_pages must be non-negative");
  if (tokens > INT_MAX) return fail(TQ_ERR_BAD_ARG, "tokens must be at most 2^31 - 1 per call");
  if (table_stride < max_pages) return fail(TQ_ERR_BAD_ARG, "page table rows must not overlap");
  if (starts == nullptr && tokens != batch)
    return fail(TQ_ERR_BAD_ARG, "without token_starts there is one token per sequence: " + std::to_string(tokens) +
                                    " tokens, " + std::to_string(batch) + " sequences");
  return TQ_OK;
}

bool type_ok(int t) { return t == TQ_F32 || t == TQ_F16 || t == TQ_BF16; }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

PagedBatch batch_of(const int32_t* table, int64_t table_stride, int max_pages, const int32_t* lens, const int32_t* starts,
                    int batch, int64_t tokens, int num_pages, int page_size, int kv_heads) {
  PagedBatch p{};
  p.table = table;
  p.table_stride = table_stride;
  p.max_pages = max_pages;
  p.lens = lens;
  p.starts = starts;
  p.batch = batch;
  p.tokens = static_cast<int>(tokens);
  p.log_page = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  p.num_pages = num_pages;
  p.kv_heads = kv_heads;
  return p;
}

template <int D, int T>
int launch_append(PagedAppendArgs a, int64_t blocks, hipStream_t stream) {
  for (a.block0 = 0; a.block0 < blocks; a.block0 += kMaxLaunchBlocks) {
    const unsigned n = static_cast<unsigned>(std::min(blocks - a.block0, kMaxLaunchBlocks));
    hipLaunchKernelGGL((paged_append_kernel<D, T>), dim3(n), dim3(kBlock), 0, stream, a);
    const int rc = launch_status("paged_append_kernel");
    if (rc) return rc;
  }
  return TQ_OK;
}

template <int D>
int launch_append_d(const PagedAppendArgs& a, int64_t blocks, hipStream_t stream) {
  switch (a.batch.log_page) {
    case 4:
      return launch_append<D, 16>(a, blocks, stream);
    case 5:
      return launch_append<D, 32>(a, blocks, stream);
    default:
      return launch_append<D, 64>(a, blocks, stream);
  }
}

// How a call's attention is cut: `items` units of R rows, `workgroups` to a KV
// head (0: a workgroup to an item and no merge).
struct PagedPlan {
  int64_t items;
  int workgroups;
  size_t acc_bytes, ml_bytes, cut_bytes;
};

constexpr int kSplitRows = 16;
constexpr int kLeastTiles = 8;  // tiles of 64 keys that a workgroup takes at least

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

PagedPlan plan_attention(int64_t tokens, int batch, bool ragged, int group, int kv_heads, int head_dim, int max_pages,
                         int page_size, int num_cus) {
  PagedPlan p{};
  p.items = ragged ? tokens * group / kSplitRows + batch : static_cast<int64_t>(batch) * ((group + kSplitRows - 1) / kSplitRows);
  const int64_t tiles = (static_cast<int64_t>(max_pages) * page_size + kTile - 1) / kTile;  // of one sequence, at most
  const int64_t units = p.items * kv_heads;
  if (tiles <= kLeastTiles || units >= 16 * static_cast<int64_t>(num_cus)) return p;
  const int64_t fill = std::max<int64_t>(1, 2 * static_cast<int64_t>(num_cus) / kv_heads);
  const int64_t most = std::max<int64_t>(1, (p.items * std::max<int64_t>(tiles, 1) + kLeastTiles - 1) / kLeastTiles);
  p.workgroups = static_cast<int>(std::min(fill, most));
  const size_t slots = static_cast<size_t>(p.workgroups) * kv_heads * 2 * kSplitRows;
  p.acc_bytes = align256(slots * head_dim * sizeof(float));
  p.ml_bytes = align256(slots * 2 * sizeof(float));
  p.cut_bytes = align256(static_cast<size_t>(p.items) * kv_heads * sizeof(int2));
  return p;
}

template <int D, int PLANES>
int launch_split(const PagedAttentionArgs& a, const PagedPlan& plan, hipStream_t stream) {
  const unsigned heads = static_cast<unsigned>(a.batch.kv_heads);
  if (plan.workgroups == 0) {
    hipLaunchKernelGGL((paged_split_kernel<D, PLANES, false>), dim3(static_cast<unsigned>(plan.items), heads), dim3(kBlock), 0, stream, a);
    return launch_status("paged_split_kernel");
  }
  hipLaunchKernelGGL((paged_split_kernel<D, PLANES, true>), dim3(static_cast<unsigned>(plan.workgroups), heads), dim3(kBlock), 0, stream, a);
  const int rc = launch_status("paged_split_kernel");
  if (rc) return rc;
  const int64_t rows = static_cast<int64_t>(a.batch.tokens) * heads * a.group;
  hipLaunchKernelGGL((paged_merge_kernel<D, kSplitRows>), dim3(static_cast<unsigned>((rows + kWavesPerBlock - 1) / kWavesPerBlock)),
                     dim3(kBlock), 0, stream, a);
  return launch_status("paged_merge_kernel");
}

template <int D>
int launch_attention_d(const PagedAttentionArgs& a, const PagedPlan& plan, hipStream_t stream) {
  return a.query_type == TQ_F32 ? launch_split<D, 3>(a, plan, stream) : launch_split<D, 2>(a, plan, stream);
}

int check_heads(int64_t tokens, int query_heads, int kv_heads) {
  if (query_heads <= 0 || query_heads % kv_heads != 0)
    return fail(TQ_ERR_BAD_ARG, "query head count " + std::to_string(query_heads) + " must be divisible by kv_heads " +
                                    std::to_string(kv_heads));
  if (tokens * query_heads > INT_MAX) return fail(TQ_ERR_BAD_ARG, "tokens x query heads must be at most 2^31 - 1 per call");
  return TQ_OK;
}

}  // namespace

extern "C" {

int tq_paged_append(const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
                    int64_t value_token_stride, int64_t value_head_stride, int kv_dtype, const void* query,
                    int64_t query_token_stride, int64_t query_head_stride, int query_dtype, int query_heads,
                    void* query_out, int64_t tokens, int kv_heads, int head_dim, int8_t* key_pages, int8_t* value_pages,
                    float* key_scales, float* value_scales, int num_pages, int page_size, const int32_t* page_table,
                    int64_t table_stride, int max_pages, const int32_t* context_lens, const int32_t* token_starts,
                    int batch, const void* cos, int64_t cos_stride, const void* sin, int64_t sin_stride, int table_dtype,
                    int64_t table_rows, int rotary_dim, const void* positions, int positions_wide,
                    int64_t positions_stride, int axes, const uint8_t* pair_axes, const float* signs_left,
                    const float* signs_right, int flags, hipStream_t stream) {
  int rc = check_pages(num_pages, page_size, kv_heads, head_dim);
  if (rc) return rc;
  rc = check_batch(tokens, batch, max_pages, table_stride, token_starts);
  if (rc) return rc;
  if (!type_ok(kv_dtype)) return fail(TQ_ERR_BAD_ARG, "dtypes must be F32, F16 or BF16");
  if (query != nullptr) {
    rc = check_heads(tokens, query_heads, kv_heads);
    if (rc) return rc;
    if (!type_ok(query_dtype)) return fail(TQ_ERR_BAD_ARG, "dtypes must be F32, F16 or BF16");
  }
  if (rotary_dim < 0 || rotary_dim % 2 != 0 || rotary_dim > head_dim)
    return fail(TQ_ERR_BAD_ARG, "rotary_dim must be even and at most head_dim");
  if (rotary_dim > 0) {
    if (!type_ok(table_dtype)) return fail(TQ_ERR_BAD_ARG, "dtypes must be F32, F16 or BF16");
    if (table_rows < 0) return fail(TQ_ERR_BAD_ARG, "table_rows must be non-negative");
    if (axes < 1 || axes > 4) return fail(TQ_ERR_BAD_ARG, "positions have 1 to 4 axes, got " + std::to_string(axes));
    if (axes > 1 && (positions == nullptr || pair_axes == nullptr))
      return fail(TQ_ERR_BAD_ARG, "several axes need positions and the axis of each pair");
    if (positions != nullptr && (flags & TQ_TABLES_BY_TOKEN))
      return fail(TQ_ERR_BAD_ARG, "positions and TQ_TABLES_BY_TOKEN exclude each other");
    if ((flags & TQ_TABLES_BY_TOKEN) && table_rows < tokens)
      return fail(TQ_ERR_BAD_ARG, "tables by token need a row for each token");
  }
  if (flags & ~(TQ_ROTATE_VALUES | TQ_TABLES_BY_TOKEN)) return fail(TQ_ERR_BAD_ARG, "unknown flags");
  if ((signs_left == nullptr) != (signs_right == nullptr)) return fail(TQ_ERR_BAD_ARG, "signs come in pairs");
  if ((flags & TQ_ROTATE_VALUES) && signs_left == nullptr) return fail(TQ_ERR_BAD_ARG, "TQ_ROTATE_VALUES needs signs");
  PagedAppendArgs a{};
  for (int i = 0; pair_axes != nullptr && i < rotary_dim / 2; ++i) {
    if (pair_axes[i] >= axes) return fail(TQ_ERR_BAD_ARG, "a pair's axis is not among the positions'");
    a.rotary.pair_axis[i >> 4] |= static_cast<uint32_t>(pair_axes[i]) << (2 * (i & 15));
  }
  if (tokens == 0 || batch == 0) return TQ_OK;
  if (!key || !value || !key_pages || !value_pages || !key_scales || !value_scales || !context_lens ||
      (max_pages > 0 && !page_table) || (query && !query_out) || (rotary_dim > 0 && table_rows > 0 && (!cos || !sin)))
    return fail(TQ_ERR_BAD_ARG, "null pointer argument");
  if (!aligned16(key_pages) || !aligned16(value_pages)) return fail(TQ_ERR_BAD_ARG, "pages must be 16-byte aligned");

  a.batch = batch_of(page_table, table_stride, max_pages, context_lens, token_starts, batch, tokens, num_pages, page_size, kv_heads);
  a.key = {key, kv_dtype, key_token_stride, key_head_stride};
  a.value = {value, kv_dtype, value_token_stride, value_head_stride};
  a.query = {query, query_dtype, query_token_stride, query_head_stride};
  a.query_heads = query_heads;
  a.query_out = query_out;
  a.pages[0] = key_pages;
  a.pages[1] = value_pages;
  a.scales[0] = key_scales;
  a.scales[1] = value_scales;
  a.rotary.cos = cos;
  a.rotary.sin = sin;
  a.rotary.table_type = table_dtype;
  a.rotary.cos_stride = cos_stride;
  a.rotary.sin_stride = sin_stride;
  a.rotary.table_rows = table_rows;
  a.rotary.rotary_dim = rotary_dim;
  a.rotary.positions = positions;
  a.rotary.positions_wide = positions_wide;
  a.rotary.positions_stride = positions_stride;
  a.rotary.axes = axes;
  a.rotary.by_token = (flags & TQ_TABLES_BY_TOKEN) != 0;
  a.signs_left = signs_left;
  a.signs_right = signs_right;
  a.rotate_values = (flags & TQ_ROTATE_VALUES) != 0;
  a.sqrt_d = static_cast<float>(std::sqrt(static_cast<double>(head_dim)));
  const int64_t units = token_starts == nullptr ? batch : tokens / page_size + 2 * static_cast<int64_t>(batch);
  a.kv_blocks = units * kv_heads * 2;
  const int64_t q_rows = query != nullptr ? tokens * query_heads : 0;
  const int64_t blocks = a.kv_blocks + (q_rows + kWavesPerBlock - 1) / kWavesPerBlock;
  switch (head_dim) {
    case 64:
      return launch_append_d<64>(a, blocks, stream);
    case 128:
      return launch_append_d<128>(a, blocks, stream);
    default:
      return launch_append_d<256>(a, blocks, stream);
  }
}

int tq_paged_dequantize(const int32_t* page_ids, int64_t count, const int8_t* key_pages, const int8_t* value_pages,
                        const float* key_scales, const float* value_scales, int num_pages, int page_size, int kv_heads,
                        int head_dim, void* keys_out, void* values_out, int out_dtype, hipStream_t stream) {
  const int rc = check_pages(num_pages, page_size, kv_heads, head_dim);
  if (rc) return rc;
  if (!type_ok(out_dtype)) return fail(TQ_ERR_BAD_ARG, "dtypes must be F32, F16 or BF16");
  if (count < 0) return fail(TQ_ERR_BAD_ARG, "count must be non-negative");
  if (count == 0) return TQ_OK;
  if (!page_ids || !key_pages || !value_pages || !key_scales || !value_scales || !keys_out || !values_out)
    return fail(TQ_ERR_BAD_ARG, "null pointer argument");
  if (!aligned16(key_pages) || !aligned16(value_pages) || !aligned16(keys_out) || !aligned16(values_out))
    return fail(TQ_ERR_BAD_ARG, "pages and outputs must be 16-byte aligned");
  PagedReadArgs a{};
  a.ids = page_ids;
  a.count = count;
  a.pages[0] = key_pages;
  a.pages[1] = value_pages;
  a.scales[0] = key_scales;
  a.scales[1] = value_scales;
  a.out[0] = keys_out;
  a.out[1] = values_out;
  a.out_type = out_dtype;
  a.num_pages = num_pages;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.log_page = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  const int64_t blocks = count * kv_heads * 2;
  for (a.block0 = 0; a.block0 < blocks; a.block0 += kMaxLaunchBlocks) {
    const unsigned n = static_cast<unsigned>(std::min(blocks - a.block0, kMaxLaunchBlocks));
    hipLaunchKernelGGL(paged_read_kernel, dim3(n), dim3(kBlock), 0, stream, a);
    const int rc_launch = launch_status("paged_read_kernel");
    if (rc_launch) return rc_launch;
  }
  return TQ_OK;
}

size_t tq_paged_attention_workspace_bytes(int64_t tokens, int batch, int ragged, int query_heads, int kv_heads,
                                          int head_dim, int max_pages, int page_size, int64_t max_tokens, int num_cus) {
  if (tokens <= 0 || batch <= 0 || kv_heads <= 0 || query_heads <= 0 || query_heads % kv_heads != 0 || max_pages < 0 ||
      check_pages(1, page_size, kv_heads, head_dim) != TQ_OK)
    return 0;
  if (num_cus <= 0) num_cus = device_cu_count();
  (void)max_tokens;
  const PagedPlan p = plan_attention(tokens, batch, ragged != 0, query_heads / kv_heads, kv_heads, head_dim, max_pages, page_size, num_cus);
  return p.acc_bytes + p.ml_bytes + p.cut_bytes;
}

int tq_paged_attention(const void* query, int64_t query_token_stride, int64_t query_head_stride, int query_dtype,
                       int64_t tokens, int query_heads, int kv_heads, int head_dim, const int8_t* key_pages,
                       const int8_t* value_pages, const float* key_scales, const float* value_scales, int num_pages,
                       int page_size, const int32_t* page_table, int64_t table_stride, int max_pages,
                       const int32_t* context_lens, const int32_t* token_starts, int batch, int64_t max_tokens,
                       float scale, void* workspace, size_t workspace_bytes, void* out, int64_t out_token_stride,
                       int64_t out_head_stride, hipStream_t stream) {
  int rc = check_pages(num_pages, page_size, kv_heads, head_dim);
  if (rc) return rc;
  rc = check_batch(tokens, batch, max_pages, table_stride, token_starts);
  if (rc) return rc;
  rc = check_heads(tokens, query_heads, kv_heads);
  if (rc) return rc;
  if (!type_ok(query_dtype)) return fail(TQ_ERR_BAD_ARG, "dtypes must be F32, F16 or BF16");
  if (!std::isfinite(scale)) return fail(TQ_ERR_BAD_ARG, "scale must be finite");
  if (tokens == 0 || batch == 0) return TQ_OK;
  if (!query || !key_pages || !value_pages || !key_scales || !value_scales || !context_lens || (max_pages > 0 && !page_table) || !out)
    return fail(TQ_ERR_BAD_ARG, "null pointer argument");
  if (!aligned16(key_pages) || !aligned16(value_pages)) return fail(TQ_ERR_BAD_ARG, "pages must be 16-byte aligned");
  const int group = query_heads / kv_heads;
  const PagedPlan plan = plan_attention(tokens, batch, token_starts != nullptr, group, kv_heads, head_dim, max_pages, page_size, device_cu_count());
  if (plan.items > INT_MAX) return fail(TQ_ERR_BAD_ARG, "tokens x group exceeds one launch");
  const size_t need = plan.acc_bytes + plan.ml_bytes + plan.cut_bytes;
  if (need > 0 && (workspace == nullptr || workspace_bytes < need))
    return fail(TQ_ERR_BAD_ARG, "workspace too small: " + std::to_string(workspace_bytes) + " bytes, the call needs " + std::to_string(need));
  if (need > 0 && !aligned16(workspace)) return fail(TQ_ERR_BAD_ARG, "the workspace must be 16-byte aligned");
  PagedAttentionArgs a{};
  a.batch = batch_of(page_table, table_stride, max_pages, context_lens, token_starts, batch, tokens, num_pages, page_size, kv_heads);
  a.query = query;
  a.query_type = query_dtype;
  a.q_token_stride = query_token_stride;
  a.q_head_stride = query_head_stride;
  a.out = out;
  a.o_token_stride = out_token_stride;
  a.o_head_stride = out_head_stride;
  a.group = group;
  a.key_pages = key_pages;
  a.value_pages = value_pages;
  a.key_scales = key_scales;
  a.value_scales = value_scales;
  a.score_scale = scale * 1.4426950408889634f;
  a.items = static_cast<int>(plan.items);
  a.workgroups = plan.workgroups;
  a.least_tiles = kLeastTiles;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.acc = reinterpret_cast<float*>(ws);
  a.ml = reinterpret_cast<float*>(ws + plan.acc_bytes);
  a.cut = reinterpret_cast<int2*>(ws + plan.acc_bytes + plan.ml_bytes);
  switch (head_dim) {
    case 64:
      return launch_attention_d<64>(a, plan, stream);
    case 128:
      return launch_attention_d<128>(a, plan, stream);
    default:
      return launch_attention_d<256>(a, plan, stream);
  }
}

}  // extern "C"
