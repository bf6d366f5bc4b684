// paged_append.hip -- appending to the paged 8-bit KV cache and reading it back:
// kernels' launches and C ABI.  Declarations are in include/torque_hip.h.
//
// Kernels
//   paged_append_kernel  new keys and values into their pages, turned to their
//                        positions and into the rotated basis on the way; the
//                        queries of the same tokens beside them
//   paged_read_kernel    pages -> the values they stand for

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "paged_append.hpp"
#include "paged_host.hpp"

using namespace tq;

namespace {

// Heads to a workgroup of an append, which share their tokens' table entries and
// fetch one head's rows while another's are worked on: as many (8 at most) as leave
// this many threads, half of what the GPU holds at once at 128 registers.  8192 tokens
// (1024 elements of the cache to each, bfloat16) in us with 2^17 / 2^18 / 2^19 / 2^20 and
// with 1024 workgroups of whatever size: head_dim 256, pages of 64 54 / 53 / 64 / 85 / 85,
// pages of 16 45 / 45 / 49 / 64 / 45; 128, pages of 64 42 / 46 / 53 / 61 / 53; 64, pages of
// 16 39 / 41 / 42 / 48 / 39.
constexpr int64_t kAppendThreads = int64_t(1) << 17;
int heads_to_block(int64_t rows, int heads, int threads) {
  return static_cast<int>(std::min<int64_t>(8, std::max<int64_t>(1, rows * heads * threads / kAppendThreads)));
}

template <int D, int SIZE>
int launch_append(PagedAppendArgs a, hipStream_t stream) {
  constexpr int kThreads = append_threads(D, SIZE), kRows = kThreads / (D / 16);
  const int64_t batch = a.batch.batch, tokens = a.batch.tokens;
  const int64_t units = SIZE == 0 ? batch : (tokens >> a.batch.log_page) + 2 * batch;
  a.kv_step = heads_to_block(2 * units, a.batch.kv_heads, kThreads);
  a.kv_parts = (a.batch.kv_heads + a.kv_step - 1) / a.kv_step;
  a.kv_blocks = units * a.kv_parts * 2;
  int64_t blocks = a.kv_blocks;
  const bool plain = a.key.vec && a.value.vec && (a.query.data == nullptr || (a.query.vec && a.query.type == a.key.type)) &&
                     (a.rotary.rotary_dim == 0 || (a.rotary.vec && a.rotary.table_type == TQ_F32 && a.rotary.rotary_dim % 16 == 0));
  if (a.query.data != nullptr) {
    const int64_t rows = (tokens + kRows - 1) / kRows;
    a.query_step = heads_to_block(rows, a.query_heads, kThreads);
    a.query_parts = (a.query_heads + a.query_step - 1) / a.query_step;
    blocks += rows * a.query_parts;
  }
  for (a.block0 = 0; a.block0 < blocks; a.block0 += kMaxLaunchBlocks) {
    const unsigned n = static_cast<unsigned>(std::min(blocks - a.block0, kMaxLaunchBlocks));
    const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(n), dim3(kThreads), 0, stream, a); };
    if (!plain)
      launch(paged_append_kernel<D, SIZE, kAnyRows>);
    else if (a.key.type == TQ_F32)
      launch(paged_append_kernel<D, SIZE, kTypeF32>);
    else if (a.key.type == TQ_F16)
      launch(paged_append_kernel<D, SIZE, kTypeF16>);
    else
      launch(paged_append_kernel<D, SIZE, kTypeBF16>);
    const int rc = launch_status("paged_append_kernel");
    if (rc) return rc;
  }
  return TQ_OK;
}

template <int D>
int launch_append_d(const PagedAppendArgs& a, hipStream_t stream) {
  if (a.batch.starts == nullptr) return launch_append<D, 0>(a, stream);
  switch (a.batch.log_page) {
    case 4:
      return launch_append<D, 16>(a, stream);
    case 5:
      return launch_append<D, 32>(a, stream);
    default:
      return launch_append<D, 64>(a, stream);
  }
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
  if (query_out != nullptr && !aligned16(query_out)) return fail(TQ_ERR_BAD_ARG, "query_out must be 16-byte aligned");
  PagedAppendArgs a{};
  a.rotary.axes_used = pair_axes == nullptr && rotary_dim > 0 ? 1 : 0;
  for (int i = 0; pair_axes != nullptr && i < rotary_dim / 2; ++i) {
    if (pair_axes[i] >= axes) return fail(TQ_ERR_BAD_ARG, "a pair's axis is not among the positions'");
    a.rotary.axes_used |= 1u << pair_axes[i];
    a.rotary.pair_axis[i >> 4] |= static_cast<uint32_t>(pair_axes[i]) << (2 * (i & 15));
  }
  if (tokens == 0 || batch == 0) return TQ_OK;
  if (!key || !value || !key_pages || !value_pages || !key_scales || !value_scales || !context_lens ||
      (max_pages > 0 && !page_table) || (query && !query_out) || (rotary_dim > 0 && table_rows > 0 && (!cos || !sin)))
    return fail(TQ_ERR_BAD_ARG, "null pointer argument");
  if (!aligned16(key_pages) || !aligned16(value_pages)) return fail(TQ_ERR_BAD_ARG, "pages must be 16-byte aligned");

  a.batch = batch_of(page_table, table_stride, max_pages, context_lens, token_starts, batch, tokens, num_pages, page_size, kv_heads);
  a.key = {key, kv_dtype, key_token_stride, key_head_stride, vectors(key, kv_dtype, key_token_stride, key_head_stride)};
  a.value = {value, kv_dtype, value_token_stride, value_head_stride, vectors(value, kv_dtype, value_token_stride, value_head_stride)};
  a.query = {query, query_dtype, query_token_stride, query_head_stride, vectors(query, query_dtype, query_token_stride, query_head_stride)};
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
  a.rotary.vec = vectors(cos, table_dtype, cos_stride, 0) && vectors(sin, table_dtype, sin_stride, 0);
  a.rotary.by_token = (flags & TQ_TABLES_BY_TOKEN) != 0;
  a.signs_left = signs_left;
  a.signs_right = signs_right;
  a.rotate_values = (flags & TQ_ROTATE_VALUES) != 0;
  switch (head_dim) {
    case 64:
      return launch_append_d<64>(a, stream);
    case 128:
      return launch_append_d<128>(a, stream);
    default:
      return launch_append_d<256>(a, stream);
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
  a.num_pages = num_pages;
  a.kv_heads = kv_heads;
  a.head_dim = head_dim;
  a.log_page = page_size == 16 ? 4 : page_size == 32 ? 5 : 6;
  const int64_t blocks = count * kv_heads * 2;
  for (a.block0 = 0; a.block0 < blocks; a.block0 += kMaxLaunchBlocks) {
    const unsigned n = static_cast<unsigned>(std::min(blocks - a.block0, kMaxLaunchBlocks));
    if (out_dtype == TQ_F32)
      hipLaunchKernelGGL(paged_read_kernel<kTypeF32>, dim3(n), dim3(kBlock), 0, stream, a);
    else if (out_dtype == TQ_F16)
      hipLaunchKernelGGL(paged_read_kernel<kTypeF16>, dim3(n), dim3(kBlock), 0, stream, a);
    else
      hipLaunchKernelGGL(paged_read_kernel<kTypeBF16>, dim3(n), dim3(kBlock), 0, stream, a);
    const int rc_launch = launch_status("paged_read_kernel");
    if (rc_launch) return rc_launch;
  }
  return TQ_OK;
}

}  // extern "C"
