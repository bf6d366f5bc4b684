// paged_attention.hip -- attention over the paged 8-bit KV cache: kernels' launches
// and C ABI.  Declarations are in include/torque_hip.h.
//
// Kernels
//   paged_split_kernel   attention of few rows over long contexts
//   paged_chunk_kernel   attention of many rows
//   paged_merge_kernel   the parts of rows whose keys were cut, as one

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "paged_chunk.hpp"
#include "paged_host.hpp"

using namespace tq;

namespace {

// How a call's attention is cut: `items` units of R rows, `workgroups` to a KV
// head (0: a workgroup to an item and no merge).
struct PagedPlan {
  bool chunk;  // paged_chunk_kernel
  int rows;    // R
  int64_t items;
  int workgroups;
  size_t acc_bytes, ml_bytes, cut_bytes;
};

constexpr int kSplitRows = 16;
constexpr int64_t kMostUnits = int64_t(1) << 22;  // workgroups of up to 768 threads: a launch holds 2^32 - 1 work-items
constexpr int kLeastTiles = 8;  // tiles of 64 keys that a workgroup takes at least

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

// Which kernel runs.  The chunk kernel reads a tile of keys once for 128 rows and
// the split kernel once for 16, but a tile costs a chunk workgroup 2 to 3 us however
// few of its rows are there, and fewer workgroups share the keys.  Measured, split /
// chunk in us (16-bit queries, 8 heads of the cache; 4 at head_dim 256):
//   head_dim 128, one sequence: 128 rows over 2000 keys 17.9 / 32.1, over 8000 33 /
//   36, over 32000 65 / 50; 512 rows over 8000 64 / 58; 2048 rows over 512 31 / 28,
//   over 2000 93 / 68
//   eight sequences: 128 rows over 4000 58 / 57, 256 over 1000 72 / 60, 512 over 128 52 / 21
//   head_dim 256: 64 rows over 32000 59 / 53, 512 over 8000 85 / 70, 2048 over 2000 104 / 77
//   head_dim 64: 128 rows over 32000 40 / 39, 1024 over 8000 64 / 57
// so a sequence has to bring half a unit of rows, and the call either enough units
// or enough rows x tiles x heads.  Lengths lie on the device: the page table's
// width stands for them, so a table wider than its sequences favours the chunk kernel.
constexpr int64_t kChunkRowsLeast = kChunkRows / 2;
constexpr int64_t kChunkUnits = 128;
constexpr double kChunkWork = 1 << 18;

// The most tiles of a sequence that one workgroup walks alone, with no merge.  A tile
// takes a workgroup of the split kernel 0.16, 0.34 and 1.04 us at head_dim 64, 128 and
// 256, and cutting costs 4 to 8.  Uncut / cut in us, 16-bit queries, 8 heads (4 at 256):
//   head_dim 64: one sequence of 1500 tokens 9.0 / 11.9, of 4000 15.5 / 11.7; eight of
//   1500 9.2 / 12.3, of 4000 15.8 / 17.2
//   head_dim 128: one of 1500 13.7 / 14.0, of 2000 16.3 / 14.7; eight of 1500 14.2 / 14.7,
//   of 2000 16.6 / 15.6
//   head_dim 256: eight of 600 18.5 / 26.7, of 1000 23.7 / 20.5
// and where the sequences are enough for the GPU, some longer ones: of up to 2000 tokens
// each, 32 at head_dim 64 11.3 / 23.6, at 128 19.3 / 31.2, 64 33.7 / 39.7, 256 129 / 125; of
// up to 8000, 64 at 128 110 / 97, 128 at 256 306 / 204.
int64_t whole_tiles(bool chunk, int64_t units, int num_cus, int head_dim) {
  return chunk ? kLeastTiles : (units >= num_cus ? 64 : 48) * 64 / head_dim;
}

PagedPlan plan_attention(int64_t tokens, int batch, bool ragged, int group, int kv_heads, int head_dim, int max_pages,
                         int page_size, int64_t max_tokens, int num_cus) {
  PagedPlan p{};
  if (!ragged) max_tokens = 1;
  if (max_tokens <= 0) max_tokens = (tokens + batch - 1) / batch;  // unknown: as if all had as many
  const int64_t tiles = (static_cast<int64_t>(max_pages) * page_size + kTile - 1) / kTile;  // of one sequence, at most
  const int64_t rows = tokens * group;
  p.chunk = std::min(max_tokens, tokens) * group >= kChunkRowsLeast &&
            ((rows + kChunkRows - 1) / kChunkRows * kv_heads >= kChunkUnits || static_cast<double>(rows) * tiles * kv_heads >= kChunkWork);
  p.rows = p.chunk ? kChunkRows : kSplitRows;
  p.items = ragged ? tokens * group / p.rows + batch : static_cast<int64_t>(batch) * ((group + p.rows - 1) / p.rows);
  const int64_t units = p.items * kv_heads;
  if (tiles <= whole_tiles(p.chunk, units, num_cus, head_dim) || units >= (p.chunk ? 1 : 16) * static_cast<int64_t>(num_cus) || p.items * tiles >= INT_MAX) return p;
  const int64_t fill = std::max<int64_t>(1, (p.chunk ? (head_dim == 256 ? 1 : 2) : 1) * static_cast<int64_t>(num_cus) / kv_heads);
  const int64_t most = std::max<int64_t>(1, (p.items * tiles + kLeastTiles - 1) / kLeastTiles);
  p.workgroups = static_cast<int>(std::min(fill, most));
  const size_t slots = static_cast<size_t>(p.workgroups) * kv_heads * 2 * p.rows;
  p.acc_bytes = align256(slots * head_dim * sizeof(float));
  p.ml_bytes = align256(slots * 2 * sizeof(float));
  p.cut_bytes = align256(static_cast<size_t>(p.items) * kv_heads * sizeof(int2));
  return p;
}

// The attention kernel over the plan's workgroups, and the merge where keys are cut.
template <int D, int PLANES>
int launch_planned(const PagedAttentionArgs& a, const PagedPlan& plan, hipStream_t stream) {
  const unsigned heads = static_cast<unsigned>(a.batch.kv_heads);
  const char* name = plan.chunk ? "paged_chunk_kernel" : "paged_split_kernel";
  const dim3 grid(static_cast<unsigned>(plan.workgroups == 0 ? plan.items : plan.workgroups), heads);
  const auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(plan.chunk ? chunk_threads(D) : split_waves(D) * kWave), 0, stream, a); };
  if (plan.workgroups == 0) {
    if (plan.chunk)
      launch(paged_chunk_kernel<D, PLANES - 1, false>);
    else
      launch(paged_split_kernel<D, PLANES, false>);
    return launch_status(name);
  }
  if (plan.chunk)
    launch(paged_chunk_kernel<D, PLANES - 1, true>);
  else
    launch(paged_split_kernel<D, PLANES, true>);
  const int rc = launch_status(name);
  if (rc) return rc;
  const int64_t rows = static_cast<int64_t>(a.batch.tokens) * heads * a.group;
  const dim3 merge(static_cast<unsigned>((rows + kWavesPerBlock - 1) / kWavesPerBlock));
  if (plan.chunk)
    hipLaunchKernelGGL((paged_merge_kernel<D, kChunkRows, 1>), merge, dim3(kBlock), 0, stream, a);
  else if (plan.workgroups < 8 * plan.items)  // fewer than 8 parts to a row, by and large
    hipLaunchKernelGGL((paged_merge_kernel<D, kSplitRows, 1>), merge, dim3(kBlock), 0, stream, a);
  else if (plan.workgroups < 64 * plan.items)
    hipLaunchKernelGGL((paged_merge_kernel<D, kSplitRows, 4>), dim3(static_cast<unsigned>(rows)), dim3(4 * kWave), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<D, kSplitRows, 16>), dim3(static_cast<unsigned>(rows)), dim3(16 * kWave), 0, stream, a);
  return launch_status("paged_merge_kernel");
}

template <int D>
int launch_attention_d(const PagedAttentionArgs& a, const PagedPlan& plan, hipStream_t stream) {
  return a.query_type == TQ_F32 ? launch_planned<D, 3>(a, plan, stream) : launch_planned<D, 2>(a, plan, stream);
}

// A call's plan as the host queries ask for it.
int plan_for(int64_t tokens, int batch, int ragged, int query_heads, int kv_heads, int head_dim, int max_pages, int page_size,
             int64_t max_tokens, int num_cus, PagedPlan* p) {
  int rc = check_pages(1, page_size, kv_heads, head_dim);
  if (rc) return rc;
  if (max_pages < 0 || tokens > INT_MAX) return fail(TQ_ERR_BAD_ARG, "tokens, batch and max_pages must be non-negative");
  rc = check_heads(tokens, query_heads, kv_heads);
  if (rc) return rc;
  *p = plan_attention(tokens, batch, ragged != 0, query_heads / kv_heads, kv_heads, head_dim, max_pages, page_size, max_tokens,
                      num_cus > 0 ? num_cus : device_cu_count());
  return TQ_OK;
}

}  // namespace

extern "C" {

size_t tq_paged_attention_workspace_bytes(int64_t tokens, int batch, int ragged, int query_heads, int kv_heads,
                                          int head_dim, int max_pages, int page_size, int64_t max_tokens, int num_cus) {
  PagedPlan p{};
  if (tokens <= 0 || batch <= 0 ||
      plan_for(tokens, batch, ragged, query_heads, kv_heads, head_dim, max_pages, page_size, max_tokens, num_cus, &p) != TQ_OK)
    return 0;
  return p.acc_bytes + p.ml_bytes + p.cut_bytes;
}

const char* tq_paged_attention_kernel(int64_t tokens, int batch, int ragged, int query_heads, int kv_heads, int head_dim,
                                      int max_pages, int page_size, int64_t max_tokens, int num_cus) {
  PagedPlan p{};
  if (tokens <= 0 || batch <= 0) {
    fail(TQ_ERR_BAD_ARG, "tokens and batch must be positive");
    return nullptr;
  }
  if (plan_for(tokens, batch, ragged, query_heads, kv_heads, head_dim, max_pages, page_size, max_tokens, num_cus, &p) != TQ_OK) return nullptr;
  const int d = head_dim == 64 ? 0 : head_dim == 128 ? 1 : 2;
  static const char* const names[2][3] = {{"paged_split_kernel<64>", "paged_split_kernel<128>", "paged_split_kernel<256>"},
                                          {"paged_chunk_kernel<64>", "paged_chunk_kernel<128>", "paged_chunk_kernel<256>"}};
  return names[p.chunk ? 1 : 0][d];
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
  const PagedPlan plan = plan_attention(tokens, batch, token_starts != nullptr, group, kv_heads, head_dim, max_pages, page_size, max_tokens, device_cu_count());
  if (plan.items > INT_MAX || (plan.workgroups == 0 && plan.items * kv_heads > kMostUnits))
    return fail(TQ_ERR_BAD_ARG, "tokens x heads exceed one launch; attend with fewer sequences per call");
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
  a.o_vec = vectors(out, query_dtype, out_token_stride, out_head_stride);
  a.q_vec = vectors(query, query_dtype, query_token_stride, query_head_stride);
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
