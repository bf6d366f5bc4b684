// Attention over the paged 8-bit cache.
//
//   o = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q . k_j),  j up to the query's position
//
// Query rows of one KV head are taken in order (token, head of the group), so
// that all query heads of a group, and neighbouring tokens, share the keys that
// a unit of work loads.  Both products run with the keys' (values') codes as the
// left operand and the query rows as the columns of the right one: column j of
// the scores, its weights and its output stay in the lanes l with l mod 16 = j
// from the first product to the last, so the softmax needs no exchange but the
// maximum over four lanes.
#pragma once

#include "paged_common.hpp"

namespace tq {

typedef int PagedI4 __attribute__((ext_vector_type(4)));

struct PagedAttentionArgs {
  PagedBatch batch;
  const void* query;  // [tokens, query_heads, D], unit stride along D
  int query_type;
  int64_t q_token_stride, q_head_stride;
  int q_vec;  // eight elements are 16-byte aligned
  void* out;  // the query's type
  int64_t o_token_stride, o_head_stride;
  int o_vec;
  int group;  // query heads to a KV head
  const int8_t* key_pages;
  const int8_t* value_pages;
  const float* key_scales;
  const float* value_scales;
  float score_scale;  // softmax scale times log2(e)
  int items;          // units of R rows, room for all
  int workgroups;     // to a KV head, where the work is cut
  int least_tiles;    // tiles that a workgroup takes at least, where the work is cut
  float* acc;         // [workgroups, kv_heads, 2][R][D] partial sums
  float* ml;          // [workgroups, kv_heads, 2][R][2] their maximum and weight
  int2* cut;          // [items, kv_heads]: first workgroup and number of parts (0: the rows are whole)
};

constexpr int kTile = 64;  // tokens to a step

// R rows of the call that one workgroup holds, and the keys they see.
struct PagedItem {
  int b;
  PagedSequence s;
  int row0, rows;  // rows of the sequence, counted (token, head of the group)
  int tiles;       // tiles of keys that its last token sees
};

template <int R>
__device__ __forceinline__ int64_t paged_item_base(const PagedAttentionArgs& a, int b) {
  if (a.batch.starts == nullptr) return static_cast<int64_t>(b) * ((a.group + R - 1) / R);
  return static_cast<int64_t>(paged_start(a.batch, b)) * a.group / R + b;
}

template <int R>
__device__ __forceinline__ PagedItem paged_item_of(const PagedAttentionArgs& a, int b, int64_t unit) {
  PagedItem it;
  it.b = b;
  it.s = paged_sequence(a.batch, b);
  const int64_t all = static_cast<int64_t>(it.s.rows) * a.group, row0 = unit * R;
  it.rows = unit < 0 ? 0 : static_cast<int>(min(max(all - row0, int64_t(0)), int64_t(R)));
  it.row0 = static_cast<int>(row0);
  const int64_t last = it.rows == 0 ? 0 : (row0 + it.rows - 1) / a.group;
  const int64_t keys = min(max(it.s.first + last + 1, int64_t(0)), static_cast<int64_t>(it.s.len));
  it.tiles = static_cast<int>((keys + kTile - 1) / kTile);
  return it;
}

// Item `index`, found by one lane alone (each lane may ask for another).
template <int R>
__device__ __forceinline__ PagedItem paged_item(const PagedAttentionArgs& a, int index) {
  int lo = 0, hi = a.batch.batch - 1;
  if (a.batch.starts == nullptr) {
    lo = index / ((a.group + R - 1) / R);
  } else {
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (paged_item_base<R>(a, mid) <= index)
        lo = mid;
      else
        hi = mid - 1;
    }
  }
  return paged_item_of<R>(a, lo, index - paged_item_base<R>(a, lo));
}

// What an item counts for where the work is cut: its tiles, and one where it
// sees nothing, so that somebody writes its zeros.
__device__ __forceinline__ int paged_cost(const PagedItem& it) { return it.rows == 0 ? 0 : max(it.tiles, 1); }

// Sum over the workgroup, the same in every thread; `before` is the sum of the
// threads before this one.
template <int WAVES>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* before, int64_t* s_wave) {
  int64_t sum = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t other = __shfl_up(sum, d);
    if (lane_id() >= d) sum += other;
  }
  const int wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane_id() == kWave - 1) s_wave[wave] = sum;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) base += s_wave[w];
    total += s_wave[w];
  }
  *before = base + sum - v;
  return total;
}

// Runs work(item, index, from, to, whole, slot) for each part of an item that
// falls to this workgroup.
//
// CUT: the tiles of all items, one after another, are dealt out in equal runs, a
// run to a workgroup, whatever sequence they belong to: a batch of very
// different lengths, one long sequence and a chunk over a long context fill the
// GPU alike, and the host need not know a length.  A part that is not a whole
// item leaves its sums in the workgroup's slot 0 (an item begun before) or 1 (an
// item that it begins), for the merge.
// Otherwise workgroup x has item x.
template <int R, bool CUT, int WAVES, class Work>
__device__ __forceinline__ void paged_schedule(const PagedAttentionArgs& a, int h, Work work) {
  if constexpr (!CUT) {
    const int index = a.items - 1 - static_cast<int>(blockIdx.x);  // a sequence's last rows see the most keys
    const PagedItem it = paged_item<R>(a, index);
    if (it.rows > 0) work(it, 0, it.tiles, true, 0);
  } else {
    __shared__ int64_t s_wave[WAVES];
    __shared__ int s_index;
    __shared__ int64_t s_offset;
    constexpr int N = WAVES * kWave;
    const int workgroups = gridDim.x, tid = threadIdx.x;
    int64_t total = 0, before = 0;
    int64_t mine = 0;
    for (int i0 = 0; i0 < a.items; i0 += N)
      if (i0 + tid < a.items) mine += paged_cost(paged_item<R>(a, i0 + tid));
    total = block_scan<WAVES>(mine, &before, s_wave);
    const int64_t run = max((total + workgroups - 1) / workgroups, static_cast<int64_t>(a.least_tiles));
    int64_t at = run * blockIdx.x;
    const int64_t end = min(at + run, total);
    if (at >= end) return;
    if (tid == 0) s_index = a.items;  // nothing to do, were no item found
    int64_t base = 0;
    for (int i0 = 0; i0 < a.items; i0 += N) {
      const int64_t cost = i0 + tid < a.items ? paged_cost(paged_item<R>(a, i0 + tid)) : 0;
      const int64_t all = block_scan<WAVES>(cost, &before, s_wave);
      if (at < base + all) {  // the same in every thread
        if (at >= base + before && at < base + before + cost) {
          s_index = i0 + tid;
          s_offset = at - base - before;
        }
        break;
      }
      base += all;
    }
    __syncthreads();
    int index = s_index;
    int64_t offset = s_offset;
    while (at < end && index < a.items) {
      const PagedItem it = paged_item<R>(a, index);
      const int cost = paged_cost(it);
      if (cost > 0) {
        const int64_t take = min(cost - offset, end - at);
        if (offset == 0 && tid == 0) {
          const int64_t first = at / run, last = (at + cost - 1) / run;
          a.cut[static_cast<int64_t>(index) * a.batch.kv_heads + h] =
              make_int2(static_cast<int>(first), last > first ? static_cast<int>(last - first + 1) : 0);
        }
        const bool whole = take == cost;
        const int from = static_cast<int>(min(offset, static_cast<int64_t>(it.tiles)));
        const int to = static_cast<int>(min(offset + take, static_cast<int64_t>(it.tiles)));
        work(it, from, to, whole, offset == 0 ? 1 : 0);
        at += take;
      }
      offset = 0;
      ++index;
    }
  }
}

// Row r (token, head of the group) of an item: where it lies in the call.
struct PagedRowAt {
  int token, head;  // row of the call, query head
  int64_t keys;     // keys that it sees
};
__device__ __forceinline__ PagedRowAt paged_row(const PagedAttentionArgs& a, const PagedItem& it, int h, int r) {
  const int row = it.row0 + r, token = row / a.group;
  PagedRowAt at;
  at.token = it.s.row0 + token;
  at.head = h * a.group + row - token * a.group;
  at.keys = min(max(it.s.first + token + 1, int64_t(0)), static_cast<int64_t>(it.s.len));
  return at;
}

// The bytes k of four words as one word.
__device__ __forceinline__ uint32_t byte_of_each(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int k) {
  const uint32_t pick = 0x0C0C0400u + 0x00000101u * k;  // (second operand's byte k, first operand's byte k)
  return __builtin_amdgcn_perm(b, a, pick) | (__builtin_amdgcn_perm(d, c, pick) << 16);
}

// 16 consecutive elements of a query row (zeros where there is none).
__device__ __forceinline__ void paged_query16(const PagedAttentionArgs& a, int64_t at, bool live, float (&x)[16]) {
  if (live) {
    load8<kAnyRows>(a.query, at, a.query_type, a.q_vec, x);
    load8<kAnyRows>(a.query, at + 8, a.query_type, a.q_vec, x + 8);
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
  }
}
// Four consecutive elements of the output, at a multiple of 4 of a row.
__device__ __forceinline__ void paged_store4(const PagedAttentionArgs& a, int64_t at, const float (&v)[4]) {
  if (!a.o_vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) store_as(a.out, at + i, v[i], a.query_type);
  } else if (a.query_type == kTypeF32) {
    *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + at) =
        make_uint2(two_halves(v[0], v[1], a.query_type), two_halves(v[2], v[3], a.query_type));
  }
}
__device__ __forceinline__ void paged_extent(const float (&x)[16], float* top, bool* fine) {
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    *top = fmaxf(*top, fabsf(x[i]));
    *fine = *fine && fabsf(x[i]) < INFINITY;
  }
}
// Their products with f, rounded, in PLANES balanced base-256 digits, the highest first.
template <int PLANES>
__device__ __forceinline__ void paged_digits(const float (&x)[16], float f, bool bad, PagedI4 (&q)[PLANES]) {
  constexpr float kUnit = PLANES == 3 ? 8323072.f : 32512.f;  // 127 x 256^(PLANES-1)
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t digit[PLANES] = {};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      int n = bad ? 0 : static_cast<int>(fminf(fmaxf(rintf(x[4 * w + e] * f), -kUnit), kUnit));
#pragma unroll
      for (int k = PLANES - 1; k >= 0; --k) {
        const int d = k == 0 ? n : static_cast<int8_t>(n);
        digit[k] |= static_cast<uint32_t>(d & 0xff) << (8 * e);
        n = (n - d) >> 8;
      }
    }
#pragma unroll
    for (int k = 0; k < PLANES; ++k) q[k][w] = static_cast<int>(digit[k]);
  }
}

// paged_split_kernel<D, PLANES>: few rows (single tokens, drafts) over long
// contexts; one wavefront takes every fourth tile of 64 keys by itself, straight
// from memory to the matrix instructions' operands.
//
// The codes are multiplied as they are, in v_mfma_i32_16x16x64_i8.  A query row
// is an integer in PLANES balanced base-256 digits (|q| <= 127 x 256^(PLANES-1),
// relative to the row's largest element): digits times codes sum exactly in 32
// bits, so a score is as good as the query's rounding, 2^-16 of its largest
// element with two digits (float16 and bfloat16 queries) and 2^-24 with three
// (float32).  The weights of a tile, relative to the tile's own largest, are
// held the same way; the sums over tokens are exact integers and enter the
// running float32 sums once a tile.  A value page's scale vs goes into the
// weight's exponent: w = exp2(s + log2 vs - max), and w / vs sums to the
// denominator, so one integer product serves pages of different scales.
//
// A-operand rows: tokens 16 (i / 4) + 4 s + i mod 4 for product s of 4.  Lane
// (column j, g = lane / 16) then holds the scores of tokens 16 g .. 16 g + 15,
// which is what it needs as the second product's right operand: 16 bytes of
// weights for 16 bytes of values that lie side by side in the transposed page.
template <int D, int PLANES, bool CUT>
__global__ __launch_bounds__(kBlock, 2) void paged_split_kernel(const PagedAttentionArgs a) {
  constexpr int R = 16, C = D / 64, DT = D / 16;
  constexpr int P = D + 4;  // LDS pitch of a row of sums
  constexpr float kUnit = PLANES == 3 ? 8323072.f : 32512.f;  // 127 x 256^(PLANES-1)
  __shared__ float s_acc[kWavesPerBlock][R][P];
  __shared__ float s_ml[kWavesPerBlock][R][2];
  const PagedBatch& p = a.batch;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int j = lane & 15, g = lane >> 4;
  const int h = blockIdx.y;
  const int T = 1 << p.log_page;

  paged_schedule<R, CUT, kWavesPerBlock>(a, h, [&](const PagedItem& it, int from, int to, bool whole, int slot) {
    // ---- this lane's query row, 16 dimensions of each chunk of 64
    const bool live = j < it.rows;
    const PagedRowAt at = paged_row(a, it, h, live ? j : 0);
    PagedI4 q[PLANES][C];
    float unit;  // a score is the digits' product times this and the key page's scale
    {
      const int64_t base = at.token * a.q_token_stride + at.head * a.q_head_stride;
      float x[C][16];
      float top = 0.f;
      bool fine = true;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        paged_query16(a, base + 64 * c + 16 * g, live, x[c]);
        paged_extent(x[c], &top, &fine);
      }
      top = xor_reduce<32, OpMax>(xor_reduce<16, OpMax>(top));
      const bool bad = xor_reduce<32, OpMax>(xor_reduce<16, OpMax>(fine ? 0.f : 1.f)) > 0.f;
      const float f = top > 1e-30f ? kUnit / top : 0.f;
      unit = bad ? NAN : (top > 1e-30f ? top / kUnit : 0.f) * a.score_scale;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        PagedI4 d[PLANES];
        paged_digits<PLANES>(x[c], f, bad, d);
#pragma unroll
        for (int k = 0; k < PLANES; ++k) q[k][c] = d[k];
      }
    }
    const int64_t keys = live ? at.keys : 0;

    float m = -INFINITY, l = 0.f;
    float acc[DT][4];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[t][r] = 0.f;

    for (int tile = from + wave; tile < to; tile += kWavesPerBlock) {
      const int64_t tok0 = static_cast<int64_t>(tile) * kTile;
      // key rows of this lane: group i / 4 of 16 tokens; values and scores: group g
      const int64_t kt = tok0 + 16 * (j >> 2), vt = tok0 + 16 * g;
      const int kid = kt < it.s.len ? paged_page(p, it.b, kt >> p.log_page) : -1;
      const int vid = vt < it.s.len ? paged_page(p, it.b, vt >> p.log_page) : -1;
      const int64_t kpage = static_cast<int64_t>(max(kid, 0)) * p.kv_heads + h;
      const int64_t vpage = static_cast<int64_t>(max(vid, 0)) * p.kv_heads + h;
      const int8_t* kp = a.key_pages + kpage * (D << p.log_page) + ((kt & (T - 1)) + (j & 3)) * D + 16 * g;
      const int8_t* vp = a.value_pages + vpage * (D << p.log_page) + (vt & (T - 1)) + static_cast<int64_t>(j) * T;
      PagedI4 kv[4][C], vv[DT];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int c = 0; c < C; ++c) kv[s][c] = *reinterpret_cast<const PagedI4*>(kp + 4 * s * D + 64 * c);
#pragma unroll
      for (int t = 0; t < DT; ++t) vv[t] = *reinterpret_cast<const PagedI4*>(vp + 16 * t * T);
      const float ks = a.key_scales[vpage] * unit;
      const float vs = a.value_scales[vpage];
      const float shift = __log2f(vs);

      float w[16];
      float top = -INFINITY;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        PagedI4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < C; ++c) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[s][c], q[0][c], hi, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) hi[r] <<= 8;
#pragma unroll
        for (int c = 0; c < C; ++c) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[s][c], q[1][c], hi, 0, 0, 0);
        if constexpr (PLANES == 3) {
#pragma unroll
          for (int c = 0; c < C; ++c) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(kv[s][c], q[2][c], lo, 0, 0, 0);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float f = static_cast<float>(hi[r]);
          if constexpr (PLANES == 3) f = fmaf(f, 256.f, static_cast<float>(lo[r]));
          const bool seen = vid >= 0 && vt + 4 * s + r < keys;
          w[4 * s + r] = seen ? fmaf(f, ks, shift) : -INFINITY;
          top = fmaxf(top, w[4 * s + r]);
        }
      }
      top = xor_reduce<32, OpMax>(xor_reduce<16, OpMax>(top));
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      uint32_t n[16];
      constexpr float kMagic = 8388608.f + (PLANES == 3 ? 32896.f : 128.f);  // 2^23 and 128 for each lower digit
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float e = fast_exp2(w[i] - base);
        sum += e;
        n[i] = __float_as_uint(fmaf(e, kUnit, kMagic));  // the integer in the mantissa's low bits
      }
      const float next = fmaxf(m, top);
      const float keep = m == next ? 1.f : fast_exp2(m - next), part = top == -INFINITY ? 0.f : fast_exp2(top - next);
      l = l * keep + (vid >= 0 ? sum * part / vs : 0.f);
      m = next;

      PagedI4 wq[PLANES];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < PLANES; ++k) {
          const uint32_t word = byte_of_each(n[4 * i], n[4 * i + 1], n[4 * i + 2], n[4 * i + 3], PLANES - 1 - k);
          wq[k][i] = static_cast<int>(k == 0 ? word : word ^ 0x80808080u);
        }
#pragma unroll
      for (int t = 0; t < DT; ++t) {
        PagedI4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
        hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[t], wq[0], hi, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) hi[r] <<= 8;
        hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[t], wq[1], hi, 0, 0, 0);
        if constexpr (PLANES == 3) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(vv[t], wq[2], lo, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float f = static_cast<float>(hi[r]);
          if constexpr (PLANES == 3) f = fmaf(f, 256.f, static_cast<float>(lo[r]));
          acc[t][r] = fmaf(f, part, acc[t][r] * keep);
        }
      }
    }

    // ---- the four wavefronts' sums as one
    l = xor_reduce<32, OpSum>(xor_reduce<16, OpSum>(l));
    __syncthreads();  // the item before is written out
    if (g == 0) {
      s_ml[wave][j][0] = m;
      s_ml[wave][j][1] = l;
    }
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) s_acc[wave][j][16 * t + 4 * g + r] = acc[t][r];
    __syncthreads();
    for (int i = threadIdx.x; i < R * D; i += kBlock) {
      const int row = i / D, d = i & (D - 1);
      if (row >= it.rows) break;
      float top = -INFINITY, sum = 0.f, weight = 0.f;
#pragma unroll
      for (int v = 0; v < kWavesPerBlock; ++v) top = fmaxf(top, s_ml[v][row][0]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int v = 0; v < kWavesPerBlock; ++v) {
        const float f = fast_exp2(s_ml[v][row][0] - base);
        sum = fmaf(s_acc[v][row][d], f, sum);
        weight = fmaf(s_ml[v][row][1], f, weight);
      }
      sum *= 1.f / kUnit;
      if (whole) {
        const PagedRowAt o = paged_row(a, it, h, row);
        store_as(a.out, o.token * a.o_token_stride + o.head * a.o_head_stride + d, weight == 0.f ? 0.f : sum / weight, a.query_type);
      } else {
        const int64_t at_slot = (static_cast<int64_t>(blockIdx.x) * p.kv_heads + h) * 2 + slot;
        a.acc[(at_slot * R + row) * D + d] = sum;
        if (d == 0) {
          a.ml[(at_slot * R + row) * 2] = top;
          a.ml[(at_slot * R + row) * 2 + 1] = weight;
        }
      }
    }
  });
}

// Rows whose keys were cut: the parts' sums, brought to the largest maximum and
// added in the order of the keys.  One wavefront to a row.
template <int D, int R>
__global__ __launch_bounds__(kBlock) void paged_merge_kernel(const PagedAttentionArgs a) {
  constexpr int E = D / kWave;
  const PagedBatch& p = a.batch;
  const int heads = p.kv_heads * a.group;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kWavesPerBlock + (threadIdx.x >> 6);
  if (row >= static_cast<int64_t>(p.tokens) * heads) return;
  const int token = static_cast<int>(row / heads), head = static_cast<int>(row - static_cast<int64_t>(token) * heads);
  const int h = head / a.group;
  int b = token;
  if (p.starts != nullptr) b = wave_last(p.batch, token, [&](int i) { return static_cast<int64_t>(paged_start(p, i)); });
  const PagedSequence s = paged_sequence(p, b);
  if (token < s.row0 || token >= s.row0 + s.rows) return;
  const int64_t local = static_cast<int64_t>(token - s.row0) * a.group + head - h * a.group;
  const int64_t item = paged_item_base<R>(a, b) + local / R;
  const int r = static_cast<int>(local % R);
  const int2 cut = a.cut[item * p.kv_heads + h];
  if (cut.x < 0 || cut.y <= 0 || cut.y > a.workgroups - cut.x) return;  // whole, or (row offsets that decrease) not dealt out
  const int lane = lane_id();
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  auto slot = [&](int k) { return (static_cast<int64_t>(cut.x + k) * p.kv_heads + h) * 2 + (k == 0 ? 1 : 0); };
  for (int k = lane; k < cut.y; k += kWave) m = fmaxf(m, a.ml[(slot(k) * R + r) * 2]);
  m = group_reduce<kWave, OpMax>(m);
  if (m == -INFINITY) m = 0.f;
#pragma unroll 4
  for (int k = 0; k < cut.y; ++k) {
    const int64_t at = slot(k) * R + r;
    const float f = fast_exp2(a.ml[at * 2] - m);
    l = fmaf(a.ml[at * 2 + 1], f, l);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(a.acc[at * D + lane * E + i], f, o[i]);
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    store_as(a.out, token * a.o_token_stride + head * a.o_head_stride + lane * E + i, l == 0.f ? 0.f : o[i] / l, a.query_type);
}

}  // namespace tq
