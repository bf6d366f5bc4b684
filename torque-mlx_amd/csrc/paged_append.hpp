// Appending to the paged 8-bit cache, and reading pages back.
#pragma once

#include "paged_common.hpp"

namespace tq {

// Rotary positions: row r of the tables turns a token; with several axes each
// pair of dimensions (d, d + rotary_dim / 2) has an axis whose position it is
// turned by (time, height and width of an image's patch).
struct PagedRotary {
  const void* cos;  // [table_rows, rotary_dim]
  const void* sin;
  int table_type;
  int64_t cos_stride, sin_stride, table_rows;
  int rotary_dim;         // 0: no rotation
  const void* positions;  // [axes, tokens] int32 or int64; null: the cache position, or the token's row
  int positions_wide;     // int64
  int64_t positions_stride;
  int axes;
  int by_token;         // table row = row of the call
  uint32_t pair_axis[8];  // 2 bits for each of up to 128 pairs
};

struct PagedRows {
  const void* data;  // [tokens, heads, D], unit stride along D
  int type;
  int64_t token_stride, head_stride;
};

struct PagedAppendArgs {
  PagedBatch batch;
  PagedRows key, value, query;
  int query_heads;
  void* query_out;  // [tokens, query_heads, D] of the query's type
  int8_t* pages[2];   // keys, values
  float* scales[2];
  PagedRotary rotary;
  const float* signs_left;  // null: no rotated basis
  const float* signs_right;
  int rotate_values;
  float sqrt_d;
  int64_t kv_blocks;  // workgroups that hold pages; queries follow
  int64_t block0;     // first workgroup of this launch
};

// This lane's elements of row `token`, turned to its position; false where a
// position is outside the tables.
template <int D>
__device__ __forceinline__ bool paged_turn(const PagedAppendArgs& a, const PagedRows& x, int64_t base, int64_t token,
                                           int64_t position, const int (&axis)[D / kWave], float (&v)[D / kWave]) {
  constexpr int E = D / kWave;
  const PagedRotary& r = a.rotary;
  const int d0 = lane_id() * E, half = r.rotary_dim / 2;
  bool good = true;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int d = d0 + i;
    v[i] = load_as_f32(x.data, base + d, x.type);
    if (d >= r.rotary_dim) continue;
    int64_t row = r.by_token ? token : position;
    if (r.positions != nullptr) {
      const int64_t at = axis[i] * r.positions_stride + token;
      row = r.positions_wide ? static_cast<const int64_t*>(r.positions)[at] : static_cast<const int32_t*>(r.positions)[at];
    }
    if (row < 0 || row >= r.table_rows) {
      good = false;
      continue;
    }
    const float w = d < half ? -load_as_f32(x.data, base + d + half, x.type) : load_as_f32(x.data, base + d - half, x.type);
    const float c = load_as_f32(r.cos, row * r.cos_stride + d, r.table_type);
    const float s = load_as_f32(r.sin, row * r.sin_stride + d, r.table_type);
    v[i] = __fadd_rn(__fmul_rn(v[i], c), __fmul_rn(w, s));
  }
  return __ballot(!good) == 0;
}

template <int D>
__device__ __forceinline__ void paged_axes(const PagedRotary& r, int (&axis)[D / kWave]) {
  constexpr int E = D / kWave;
  const int half = max(r.rotary_dim / 2, 1);
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int d = lane_id() * E + i, pair = d < half ? d : d - half;
    uint32_t word = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) word = (pair >> 4) == k ? r.pair_axis[k] : word;
    axis[i] = (word >> (2 * (pair & 15))) & 3;
  }
}

__device__ __forceinline__ int paged_code(float x, float inv) {
  const float y = __fmul_rn(x, inv);
  return y != y ? 0 : static_cast<int>(fminf(fmaxf(rintf(y), -127.f), 127.f));
}

// One workgroup for each page that the call writes, head and stream (keys or
// values): its new rows are turned, taken into the rotated basis, held against
// the largest of them and written; where that makes the page's scale grow, the
// codes that it held before are rounded anew at the larger scale.  No other
// workgroup touches the page's head.  Slots past the sequence's end keep what
// they held.  The workgroups behind those turn the queries, a wavefront to a row.
//
// Units of work: sequence b owns the units from starts[b] / T + 2 b on, one to a
// page, which is room enough wherever in a page it begins (n rows touch at most
// n / T + 2 pages); a unit without a page ends at once.
//
// Each element is read once and written once, 2 to 4 bytes against 1: memory is
// the bound at prompt sizes, the launch at single tokens.
template <int D, int T>
__global__ __launch_bounds__(kBlock) void paged_append_kernel(const PagedAppendArgs a) {
  constexpr int E = D / kWave;
  constexpr int Q = T / 16;  // quads of slots to a wavefront
  __shared__ float s_top[kWavesPerBlock];
  const PagedBatch& p = a.batch;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int64_t block = a.block0 + blockIdx.x;
  int axis[E];
  paged_axes<D>(a.rotary, axis);

  if (block >= a.kv_blocks) {  // queries
    const int64_t row = (block - a.kv_blocks) * kWavesPerBlock + wave;
    if (row >= static_cast<int64_t>(p.tokens) * a.query_heads) return;
    const int token = static_cast<int>(row / a.query_heads), h = static_cast<int>(row - static_cast<int64_t>(token) * a.query_heads);
    int64_t position;
    if (p.starts == nullptr) {
      position = static_cast<int64_t>(p.lens[token]) - 1;
    } else {
      const int b = wave_last(p.batch, token, [&](int i) { return static_cast<int64_t>(paged_start(p, i)); });
      const PagedSequence s = paged_sequence(p, b);
      if (token < s.row0 || token >= s.row0 + s.rows) {
#pragma unroll
        for (int i = 0; i < E; ++i) store_as(a.query_out, row * D + lane * E + i, 0.f, a.query.type);
        return;
      }
      position = s.first + token - s.row0;
    }
    float v[E];
    const bool good = paged_turn<D>(a, a.query, token * a.query.token_stride + h * a.query.head_stride, token, position, axis, v);
    if (a.signs_left != nullptr) wave_rotate<D>(v, a.signs_right, a.signs_left, a.sqrt_d);
#pragma unroll
    for (int i = 0; i < E; ++i) store_as(a.query_out, row * D + lane * E + i, good ? v[i] : NAN, a.query.type);
    return;
  }

  const int is_v = static_cast<int>(block & 1);
  const int64_t hu = block >> 1, unit = hu / p.kv_heads;
  const int h = static_cast<int>(hu - unit * p.kv_heads);
  int b = static_cast<int>(unit);
  int64_t place = 0;
  if (p.starts != nullptr) {
    auto base = [&](int i) { return static_cast<int64_t>(paged_start(p, i) / T + 2 * i); };
    b = wave_last(p.batch, unit, base);
    place = unit - base(b);
  }
  const PagedSequence s = paged_sequence(p, b);
  const int64_t c0 = max(s.first, int64_t(0));
  const int64_t page = c0 / T + place;
  const int64_t lo = max(c0, page * T), hi = min(static_cast<int64_t>(s.len), page * T + T);
  if (place < 0 || lo >= hi) return;
  const int id = paged_page(p, b, page);
  if (id < 0) return;
  const int kept = static_cast<int>(lo - page * T), end = static_cast<int>(hi - page * T);  // slots [kept, end) are new
  const int64_t token0 = s.row0 + (page * T - s.first);  // row of slot 0, were it new

  const PagedRows& x = is_v ? a.value : a.key;
  const bool rotate = a.signs_left != nullptr && (!is_v || a.rotate_values);
  float v[4 * Q][E];
  uint32_t mine = 0;  // slots of this wavefront that are written
  float top = -1.f;
#pragma unroll
  for (int k = 0; k < 4 * Q; ++k) {
    const int slot = 4 * (wave + kWavesPerBlock * (k >> 2)) + (k & 3);
#pragma unroll
    for (int i = 0; i < E; ++i) v[k][i] = 0.f;
    if (slot < kept || slot >= end) continue;
    const int64_t token = token0 + slot, at = token * x.token_stride + h * x.head_stride;
    bool good = true;
    if (is_v) {
#pragma unroll
      for (int i = 0; i < E; ++i) v[k][i] = load_as_f32(x.data, at + lane * E + i, x.type);
    } else {
      good = paged_turn<D>(a, x, at, token, page * T + slot, axis, v[k]);
    }
    if (rotate) wave_rotate<D>(v[k], a.signs_right, a.signs_left, a.sqrt_d);
    if (!good) continue;
    mine |= 1u << k;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const float m = fabsf(v[k][i]);
      top = fmaxf(top, m < INFINITY ? m : 0.f);
    }
  }
  top = group_reduce<kWave, OpMax>(top);
  if (lane == 0) s_top[wave] = top;
  float* scales = a.scales[is_v] + static_cast<int64_t>(id) * p.kv_heads + h;
  const float held = kept > 0 ? *scales : 0.f;
  __syncthreads();
  top = fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3]));
  if (top < 0.f) return;  // no row had a position
  const float scale = fmaxf(held, paged_scale(top));
  if (threadIdx.x == 0) *scales = scale;
  int8_t* out = a.pages[is_v] + (static_cast<int64_t>(id) * p.kv_heads + h) * (D * T);

  if (kept > 0 && scale != held) {  // the older codes at the grown scale
    const float ratio = __fdiv_rn(held, scale);
    uint32_t* words = reinterpret_cast<uint32_t*>(out);
    for (int w = threadIdx.x; w < D * T / 4; w += kBlock) {
      const int slot0 = is_v ? 4 * (w % (T / 4)) : w / (D / 4);
      if (slot0 >= kept) continue;
      uint32_t old = words[w], made = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int code = static_cast<int8_t>(old >> (8 * i));
        const bool again = is_v ? slot0 + i < kept : true;
        made |= static_cast<uint32_t>((again ? paged_code(static_cast<float>(code), ratio) : code) & 0xff) << (8 * i);
      }
      words[w] = made;
    }
    __syncthreads();  // a word may hold new slots as well
  }

  const float inv = __fdiv_rn(1.f, scale);
#pragma unroll
  for (int m = 0; m < Q; ++m) {
    const int quad = wave + kWavesPerBlock * m;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int d = lane * E + i;
      uint32_t word = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) word |= static_cast<uint32_t>(paged_code(v[4 * m + k][i], inv) & 0xff) << (8 * k);
      if (is_v && ((mine >> (4 * m)) & 15u) == 15u) {
        *reinterpret_cast<uint32_t*>(out + d * T + 4 * quad) = word;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (!((mine >> (4 * m + k)) & 1u)) continue;
          const int slot = 4 * quad + k;
          out[is_v ? d * T + slot : slot * D + d] = static_cast<int8_t>(word >> (8 * k));
        }
      }
    }
  }
}

struct PagedReadArgs {
  const int32_t* ids;  // [count]
  int64_t count;
  const int8_t* pages[2];
  const float* scales[2];
  void* out[2];  // [count, kv_heads, T, D]
  int out_type;
  int num_pages, kv_heads, head_dim, log_page;
  int64_t block0;
};

// Pages as the values they stand for: one workgroup to a page, head and stream;
// values go through LDS, which turns them back.
__global__ __launch_bounds__(kBlock) void paged_read_kernel(const PagedReadArgs a) {
  __shared__ int8_t s_codes[256 * 68];
  const int T = 1 << a.log_page, D = a.head_dim;
  const int64_t block = a.block0 + blockIdx.x;
  const int is_v = static_cast<int>(block & 1);
  const int64_t hn = block >> 1, n = hn / a.kv_heads;
  const int h = static_cast<int>(hn - n * a.kv_heads);
  const int id = a.ids[n];
  const bool there = id >= 0 && id < a.num_pages;
  const int64_t from = there ? static_cast<int64_t>(id) * a.kv_heads + h : 0;
  const float scale = there ? a.scales[is_v][from] : 0.f;
  const uint32_t* words = reinterpret_cast<const uint32_t*>(a.pages[is_v] + from * D * T);
  const int64_t to = hn * D * T;
  if (is_v) {
    for (int w = threadIdx.x; w < D * T / 4; w += kBlock) {
      const int d = w >> (a.log_page - 2), t = 4 * (w & (T / 4 - 1));
      *reinterpret_cast<uint32_t*>(s_codes + d * (T + 4) + t) = there ? words[w] : 0u;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < D * T; i += kBlock)
      store_as(a.out[1], to + i, scale * static_cast<float>(s_codes[(i & (D - 1)) * (T + 4) + i / D]), a.out_type);
  } else {
    for (int w = threadIdx.x; w < D * T / 4; w += kBlock) {
      const uint32_t word = there ? words[w] : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        store_as(a.out[0], to + 4 * w + k, scale * static_cast<float>(static_cast<int8_t>(word >> (8 * k))), a.out_type);
    }
  }
}

}  // namespace tq
