// Checks of arguments that the paged cache's entry points share, and the batch as
// the kernels take it.
#pragma once

#include <climits>

#include "paged_common.hpp"
#include "torque_hip.h"
#include "tq_host.hpp"

namespace tq {

inline int check_pages(int num_pages, int page_size, int kv_heads, int head_dim) {
  if (head_dim != 64 && head_dim != 128 && head_dim != 256)
    return fail(TQ_ERR_UNSUPPORTED, "Unsupported head dimension: " + std::to_string(head_dim));
  if (page_size != 16 && page_size != 32 && page_size != 64)
    return fail(TQ_ERR_UNSUPPORTED, "Unsupported page size: " + std::to_string(page_size));
  if (num_pages <= 0 || kv_heads <= 0) return fail(TQ_ERR_BAD_ARG, "num_pages and kv_heads must be positive");
  if (kv_heads > 65535) return fail(TQ_ERR_BAD_ARG, "kv_heads must be at most 65535");
  return TQ_OK;
}

inline int check_batch(int64_t tokens, int batch, int max_pages, int64_t table_stride, const int32_t* starts) {
  if (tokens < 0 || batch < 0 || max_pages < 0) return fail(TQ_ERR_BAD_ARG, "tokens, batch and max_pages must be non-negative");
  if (tokens > INT_MAX) return fail(TQ_ERR_BAD_ARG, "tokens must be at most 2^31 - 1 per call");
  if (table_stride < max_pages) return fail(TQ_ERR_BAD_ARG, "page table rows must not overlap");
  if (starts == nullptr && tokens != batch)
    return fail(TQ_ERR_BAD_ARG, "without token_starts there is one token per sequence: " + std::to_string(tokens) +
                                    " tokens, " + std::to_string(batch) + " sequences");
  return TQ_OK;
}

inline bool type_ok(int t) { return t == TQ_F32 || t == TQ_F16 || t == TQ_BF16; }
inline bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

inline PagedBatch batch_of(const int32_t* table, int64_t table_stride, int max_pages, const int32_t* lens, const int32_t* starts,
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

inline int check_heads(int64_t tokens, int query_heads, int kv_heads) {
  if (query_heads <= 0 || query_heads % kv_heads != 0)
    return fail(TQ_ERR_BAD_ARG, "query head count " + std::to_string(query_heads) + " must be divisible by kv_heads " +
                                    std::to_string(kv_heads));
  if (tokens * query_heads > INT_MAX) return fail(TQ_ERR_BAD_ARG, "tokens x query heads must be at most 2^31 - 1 per call");
  return TQ_OK;
}


// Whether rows of 8 elements from `p`, strides apart, are 16-byte aligned.
inline bool vectors(const void* p, int type, int64_t s0, int64_t s1) {
  const int64_t size = type == TQ_F32 ? 4 : 2;
  return aligned16(p) && s0 * size % 16 == 0 && s1 * size % 16 == 0;
}

}  // namespace tq
