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

// Counts of rows (tokens x group), items and tiles of a call stay below 2^31 (the
// host sees to it), so that nothing here divides 64 bits.
template <int R>
__device__ __forceinline__ int paged_item_base(const PagedAttentionArgs& a, int b) {
  if (a.batch.starts == nullptr) return b * ((a.group + R - 1) / R);
  return paged_start(a.batch, b) * a.group / R + b;
}

template <int R>
__device__ __forceinline__ PagedItem paged_item_of(const PagedAttentionArgs& a, int b, int unit) {
  PagedItem it;
  it.b = b;
  it.s = paged_sequence(a.batch, b);
  const int all = it.s.rows * a.group;
  const bool some = unit >= 0 && unit <= all / R;
  it.row0 = some ? unit * R : 0;
  it.rows = some ? min(all - it.row0, R) : 0;
  const int last = it.rows == 0 ? 0 : (it.row0 + it.rows - 1) / a.group;
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

// Sum of the lanes up to and with this one, of the first `lanes`.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lanes) {
  for (int d = 1; d < lanes; d <<= 1) {
    const uint32_t other = static_cast<uint32_t>(__shfl_up(static_cast<int>(v), d));
    if (lane_id() >= d) v += other;
  }
  return v;
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
//
// Every wavefront finds its workgroup's run by itself, 64 items at a time, without
// a barrier: the lengths are the first load of the call, and all else waits for them.
template <int R, bool CUT, class Work>
__device__ __forceinline__ void paged_schedule(const PagedAttentionArgs& a, int h, Work work) {
  if constexpr (!CUT) {
    const int index = a.items - 1 - static_cast<int>(blockIdx.x);  // a sequence's last rows see the most keys
    const PagedItem it = paged_item<R>(a, index);
    if (it.rows > 0) work(it, 0, it.tiles, true, 0);
  } else {
    const uint32_t workgroups = gridDim.x;
    const int lane = lane_id();
    auto cost_of = [&](int index) { return index < a.items ? static_cast<uint32_t>(paged_cost(paged_item<R>(a, index))) : 0u; };
    auto lanes_of = [&](int i0) { return min(a.items - i0, kWave); };
    auto lane_of = [](uint32_t v, int k) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), k)); };
    uint32_t mine = cost_of(lane), sum = wave_scan(mine, lanes_of(0));
    uint32_t total = lane_of(sum, lanes_of(0) - 1);
    for (int i0 = kWave; i0 < a.items; i0 += kWave)
      total += lane_of(wave_scan(cost_of(i0 + lane), lanes_of(i0)), lanes_of(i0) - 1);
    const uint32_t run = max((total + workgroups - 1) / workgroups, static_cast<uint32_t>(a.least_tiles));
    uint32_t at = run * blockIdx.x;  // below 2^32: a run more than the total at most, and least_tiles for each workgroup
    const uint32_t end = min(at + run, total);
    if (at >= end) return;
    int index = a.items;  // nothing to do, were no item found
    uint32_t offset = 0, base = 0;
    for (int i0 = 0; i0 < a.items; i0 += kWave) {
      if (i0 > 0) {
        mine = cost_of(i0 + lane);
        sum = wave_scan(mine, lanes_of(i0));
      }
      const uint32_t all = lane_of(sum, lanes_of(i0) - 1);
      if (at < base + all) {  // the item that holds tile `at`: the first whose sum passes it
        const int k = __ffsll(__ballot(lane < lanes_of(i0) && base + sum > at)) - 1;
        index = i0 + k;
        offset = at - base - lane_of(sum - mine, k);
        break;
      }
      base += all;
    }
    while (at < end && index < a.items) {
      const PagedItem it = paged_item<R>(a, index);
      const uint32_t cost = paged_cost(it);
      if (cost > 0) {
        const uint32_t take = min(cost - offset, end - at);
        if (offset == 0 && threadIdx.x == 0) {
          const uint32_t last = (at + cost - 1) / run;  // at / run is this workgroup
          a.cut[static_cast<int64_t>(index) * a.batch.kv_heads + h] =
              make_int2(static_cast<int>(blockIdx.x), last > blockIdx.x ? static_cast<int>(last - blockIdx.x + 1) : 0);
        }
        const int from = min(static_cast<int>(offset), it.tiles), to = min(static_cast<int>(offset + take), it.tiles);
        work(it, from, to, take == cost, offset == 0 ? 1 : 0);
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
// Bits of the largest of |x| and `top` (an infinity, a NaN above all).
__device__ __forceinline__ uint32_t paged_extent(const float (&x)[16], uint32_t top) {
#pragma unroll
  for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
  return top;
}

// The bytes k of four words as one word.
__device__ __forceinline__ uint32_t byte_of_each(uint32_t a, uint32_t b, uint32_t c, uint32_t d, int k) {
  const uint32_t pick = 0x0C0C0400u + 0x00000101u * k;  // (second operand's byte k, first operand's byte k)
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, pick), __builtin_amdgcn_perm(b, a, pick), 0x05040100u);
}

// Integers n = x f, rounded, |n| <= kQueryUnit, in PLANES balanced base-256 digits,
// the highest first.  The sum with 2^23 and an offset rounds them and leaves
// n + offset in the mantissa's low bits, whose bytes are the digits, each off by
// what the offset has there: 128, and 64 at the top of three (2^22 + 32896 in all).
template <int PLANES>
constexpr float kQueryUnit = PLANES == 3 ? 4161280.f : 32512.f;  // with the offset below 2^23, and below 2^16
template <int PLANES>
__device__ __forceinline__ void paged_digits(const float (&x)[16], float f, PagedI4 (&q)[PLANES]) {
  constexpr float kMagic = 8388608.f + (PLANES == 3 ? 4194304.f + 32896.f : 32768.f + 128.f);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    uint32_t n[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) n[e] = __float_as_uint(fmaf(x[4 * w + e], f, kMagic));
#pragma unroll
    for (int k = 0; k < PLANES; ++k) {
      const uint32_t bytes = byte_of_each(n[0], n[1], n[2], n[3], PLANES - 1 - k);
      if (PLANES == 3 && k == 0)  // less 64: bytes below 128 with the sign bit set leave no borrow
        q[k][w] = static_cast<int>(((bytes | 0x80808080u) - 0x40404040u) ^ 0x80808080u);
      else
        q[k][w] = static_cast<int>(bytes ^ 0x80808080u);
    }
  }
}
// What digits are multiplied back by, and what elements are multiplied with: NaN
// for a row with an element that is not finite, 0 for one (of almost) nothing.
template <int PLANES>
__device__ __forceinline__ float paged_unit(uint32_t top, float* f) {
  const float t = __uint_as_float(top);
  *f = t > 1e-30f && t < INFINITY ? kQueryUnit<PLANES> / t : 0.f;
  return !(t < INFINITY) ? NAN : t > 1e-30f ? t / kQueryUnit<PLANES> : 0.f;
}

// paged_split_kernel<D, PLANES>: few rows (single tokens, drafts) over long
// contexts; one wavefront takes every eighth tile of 64 keys by itself, straight
// from memory to the matrix instructions' operands.
//
// The codes are multiplied as they are, in v_mfma_i32_16x16x64_i8.  A query row
// is integers in PLANES balanced base-256 digits, relative to the row's largest
// element: digits times codes sum exactly in 32 bits, so a score is as good as the
// query's rounding, 2^-16 of its largest element with two digits (float16 and
// bfloat16 queries) and 2^-23 with three (float32).  The weights of a tile, relative to the tile's own largest, are
// held the same way; the sums over tokens are exact integers and enter the
// running float32 sums once a tile.  A value page's scale vs goes into the
// weight's exponent: w = exp2(s + log2 vs - max), and w / vs sums to the
// denominator, so one integer product serves pages of different scales.
//
// A-operand rows: tokens 16 (i / 4) + 4 s + i mod 4 for product s of 4.  Lane
// (column j, g = lane / 16) then holds the scores of tokens 16 g .. 16 g + 15,
// which is what it needs as the second product's right operand: 16 bytes of
// weights for 16 bytes of values that lie side by side in the transposed page.
//
// Memory bounds it where a unit's 16 rows are few for the bytes of a key: 48 ragged
// sequences of up to 8000 tokens (4 heads of 128, 189 MB) take 44.7 us, 4.2 TB/s,
// 131072 tokens of 2 heads of 256 (float32 queries, 134 MB) 34 us.  A call of one
// sequence first waits 4.5 us for the launch, its length, page numbers and first
// keys (32768 tokens of 8 heads of 128: 16.8 us for 67 MB).  With 64 dimensions to
// a score the vector instructions count more (about 280 a tile and wavefront).
// A wavefront's next keys are on their way from the moment the current ones are
// multiplied, its next values likewise, and page numbers a tile before that.
constexpr int split_waves(int d) { return d == 256 ? 4 : d == 128 ? 8 : 12; }

template <int D, int PLANES, bool CUT>
__global__ __launch_bounds__(split_waves(D) * kWave, split_waves(D) / 4) void paged_split_kernel(const PagedAttentionArgs a) {
  constexpr int R = 16, C = D / 64, DT = D / 16, kSplitWaves = split_waves(D);
  constexpr int P = D + 4;  // LDS pitch of a row of sums
  constexpr float kUnit = 127.f * (PLANES == 3 ? 65536.f : 256.f);  // 127 x 256^(PLANES-1)
  __shared__ __align__(16) float s_acc[kSplitWaves][R][P];
  __shared__ float s_ml[kSplitWaves][R][2];
  const PagedBatch& p = a.batch;
  const int lane = lane_id(), wave = threadIdx.x >> 6;
  const int j = lane & 15, g = lane >> 4;
  const int h = blockIdx.y;
  const int T = 1 << p.log_page;

  paged_schedule<R, CUT>(a, h, [&](const PagedItem& it, int from, int to, bool whole, int slot) {
    // ---- page numbers: this lane's key rows are in group j / 4 of a tile's 16 tokens, its values and scores in group g
    const int32_t* list = p.table + it.b * p.table_stride;
    auto page_of = [&](int tile, int group) {  // a length is at most what the list holds
      const int t = tile * kTile + 16 * group;
      const int id = tile < to && t < it.s.len ? list[t >> p.log_page] : -1;
      return id < p.num_pages ? id : -1;  // below 0: none either
    };
    struct Tile {  // a tile's keys, values and scales, as this lane multiplies them
      PagedI4 kv[4][C], vv[DT];
      float ks, vs;
    };
    auto load_keys = [&](Tile& x, int tile, int id) {
      const int64_t page = static_cast<int64_t>(max(id, 0)) * p.kv_heads + h;
      const int first = (tile * kTile + 16 * (j >> 2)) & (T - 1);
      const int8_t* kp = a.key_pages + page * (D << p.log_page) + (first + (j & 3)) * D + 16 * g;
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int c = 0; c < C; ++c) x.kv[s][c] = *reinterpret_cast<const PagedI4*>(kp + 4 * s * D + 64 * c);
    };
    auto load_values = [&](Tile& x, int tile, int id) {
      const int64_t page = static_cast<int64_t>(max(id, 0)) * p.kv_heads + h;
      const int8_t* vp = a.value_pages + page * (D << p.log_page) + ((tile * kTile + 16 * g) & (T - 1)) + j * T;
#pragma unroll
      for (int t = 0; t < DT; ++t) x.vv[t] = *reinterpret_cast<const PagedI4*>(vp + 16 * t * T);
    };
    auto load_scales = [&](Tile& x, int id) {
      const int64_t page = static_cast<int64_t>(max(id, 0)) * p.kv_heads + h;
      x.ks = a.key_scales[page];
      x.vs = a.value_scales[page];
    };
    // Two sets of registers at head_dim 256, whose wavefronts have 512 each and a SIMD to themselves: the next tile is
    // on its way while one is multiplied.  Elsewhere one set, reloaded as its keys, then its values are done with.
    constexpr bool kAhead = D == 256;
    Tile tiles[kAhead ? 2 : 1];
    // The query row's load goes first: loads return in order, and its digits are made while keys are on their way.
    const bool live = j < it.rows;
    const PagedRowAt at = paged_row(a, it, h, live ? j : 0);
    float x[C][16];
#pragma unroll
    for (int c = 0; c < C; ++c)
      paged_query16(a, at.token * a.q_token_stride + at.head * a.q_head_stride + 64 * c + 16 * g, live, x[c]);
    int tile = from + wave;
    int vid = page_of(tile, g), knext = -1, vnext = -1;
    if (tile < to) {
      const int kid = page_of(tile, j >> 2);
      knext = page_of(tile + kSplitWaves, j >> 2);
      vnext = page_of(tile + kSplitWaves, g);
      load_keys(tiles[0], tile, kid);
      load_scales(tiles[0], vid);
      load_values(tiles[0], tile, vid);
    }
    // ---- this lane's query row, 16 dimensions of each chunk of 64
    PagedI4 q[PLANES][C];
    float unit;  // a score is the digits' product times this and the key page's scale
    {
      uint32_t top = 0;
#pragma unroll
      for (int c = 0; c < C; ++c) top = paged_extent(x[c], top);
      top = __float_as_uint(xor_reduce<32, OpBits>(xor_reduce<16, OpBits>(__uint_as_float(top))));
      float f;
      unit = paged_unit<PLANES>(top, &f) * a.score_scale;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        PagedI4 d[PLANES];
        paged_digits<PLANES>(x[c], f, d);
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

    auto step = [&](Tile& now, Tile& then) {
      const auto& kv = now.kv;
      const auto& vv = now.vv;
      if (kAhead && tile + kSplitWaves < to) {
        load_keys(then, tile + kSplitWaves, knext);
        load_scales(then, vnext);
        load_values(then, tile + kSplitWaves, vnext);
      }
      const int64_t vt = static_cast<int64_t>(tile) * kTile + 16 * g;
      const int kafter = page_of(tile + 2 * kSplitWaves, j >> 2), vafter = page_of(tile + 2 * kSplitWaves, g);
      const float by = now.ks * unit, shift = __log2f(now.vs), back = 1.f / now.vs;
      const int seen = vid >= 0 ? static_cast<int>(min(max(keys - vt, int64_t(0)), int64_t(16))) : 0;  // of its 16 tokens

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
          w[4 * s + r] = fmaf(f, by, shift);
        }
      }
      if (__ballot(seen < 16) != 0) {  // a sequence's last tile, an earlier draft, a page that is none
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = i < seen ? w[i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, w[i]);
      if (!kAhead && tile + kSplitWaves < to) {
        load_keys(then, tile + kSplitWaves, knext);
        load_scales(then, vnext);
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
      // The running maximum moves where a tile exceeds it by 2^8 and more, in few tiles: sums are multiplied then only.
      if (__ballot(top > m + 8.f) != 0) {
        const float next = fmaxf(m, top);
        const float keep = m == next ? 1.f : fast_exp2(m - next);
        m = next;
        l *= keep;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[t][r] *= keep;
      }
      const float part = top == -INFINITY ? 0.f : fast_exp2(top - m);
      l = fmaf(sum, vid >= 0 ? part * back : 0.f, l);

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
          acc[t][r] = fmaf(f, part, acc[t][r]);
        }
      }
      if (!kAhead && tile + kSplitWaves < to) load_values(then, tile + kSplitWaves, vnext);
      vid = vnext;
      knext = kafter;
      vnext = vafter;
      tile += kSplitWaves;
    };
    while (tile < to) {
      step(tiles[0], tiles[kAhead ? 1 : 0]);
      if constexpr (kAhead)
        if (tile < to) step(tiles[1], tiles[0]);
    }

    // ---- the wavefronts' sums as one
    l = xor_reduce<32, OpSum>(xor_reduce<16, OpSum>(l));
    __syncthreads();  // the item before is written out
    if (live) {
      if (g == 0) {
        s_ml[wave][j][0] = m;
        s_ml[wave][j][1] = l;
      }
#pragma unroll
      for (int t = 0; t < DT; ++t)
        *reinterpret_cast<float4*>(&s_acc[wave][j][16 * t + 4 * g]) = make_float4(acc[t][0], acc[t][1], acc[t][2], acc[t][3]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < it.rows * (D / 4); i += kSplitWaves * kWave) {
      const int row = i / (D / 4), d = 4 * (i & (D / 4 - 1));
      float top = -INFINITY, weight = 0.f;
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int v = 0; v < kSplitWaves; ++v) top = fmaxf(top, s_ml[v][row][0]);
      const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
      for (int v = 0; v < kSplitWaves; ++v) {
        const float f = fast_exp2(s_ml[v][row][0] - base);
        const float4 x = *reinterpret_cast<const float4*>(&s_acc[v][row][d]);
        sum.x = fmaf(x.x, f, sum.x), sum.y = fmaf(x.y, f, sum.y), sum.z = fmaf(x.z, f, sum.z), sum.w = fmaf(x.w, f, sum.w);
        weight = fmaf(s_ml[v][row][1], f, weight);
      }
      if (whole) {
        const PagedRowAt o = paged_row(a, it, h, row);
        const float f = weight == 0.f ? 0.f : 1.f / (weight * kUnit);
        const float out[4] = {sum.x * f, sum.y * f, sum.z * f, sum.w * f};
        paged_store4(a, o.token * a.o_token_stride + o.head * a.o_head_stride + d, out);
      } else {
        constexpr float f = 1.f / kUnit;
        const int64_t at_slot = ((static_cast<int64_t>(blockIdx.x) * p.kv_heads + h) * 2 + slot) * R + row;
        *reinterpret_cast<float4*>(a.acc + at_slot * D + d) = make_float4(sum.x * f, sum.y * f, sum.z * f, sum.w * f);
        if (d == 0) {
          a.ml[at_slot * 2] = top;
          a.ml[at_slot * 2 + 1] = weight;
        }
      }
    }
  });
}

// Rows whose keys were cut: the parts' sums, brought to the largest maximum and
// added in a fixed order.  WAVES wavefronts to a row deal its parts out: one below
// 8 parts, 4, and 16 from 64 parts on (128 parts of head_dim 256: 27 us with one
// wavefront, 6.5 with 4, 5.9 with 16; 32 parts of 128: 8.6 with one, 3.9 with 4, 4.7 with 16).
template <int D, int R, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? kBlock : WAVES * kWave) void paged_merge_kernel(const PagedAttentionArgs a) {
  constexpr int E = D / kWave;
  __shared__ float s_sum[WAVES][D + 2];
  const PagedBatch& p = a.batch;
  const int heads = p.kv_heads * a.group, wave = threadIdx.x >> 6, lane = lane_id();
  const uint32_t row = WAVES == 1 ? blockIdx.x * kWavesPerBlock + wave : blockIdx.x;
  if (row >= static_cast<uint32_t>(p.tokens) * heads) return;
  const int token = row / heads, head = row - token * heads;
  const int h = head / a.group;
  int b = token;
  if (p.starts != nullptr) b = wave_last(p.batch, token, [&](int i) { return static_cast<int64_t>(paged_start(p, i)); });
  const PagedSequence s = paged_sequence(p, b);
  if (token < s.row0 || token >= s.row0 + s.rows) return;
  const int local = (token - s.row0) * a.group + head - h * a.group;
  const int64_t item = paged_item_base<R>(a, b) + local / R;
  const int r = local % R;
  const int2 cut = a.cut[item * p.kv_heads + h];
  if (cut.x < 0 || cut.y <= 0 || cut.y > a.workgroups - cut.x) return;  // whole, or (row offsets that decrease) not dealt out
  auto slot = [&](int k) { return ((static_cast<int64_t>(cut.x + k) * p.kv_heads + h) * 2 + (k == 0 ? 1 : 0)) * R + r; };
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int i = 0; i < E; ++i) o[i] = 0.f;
  for (int k = lane; k < cut.y; k += kWave) m = fmaxf(m, a.ml[slot(k) * 2]);
  m = group_reduce<kWave, OpMax>(m);
  if (m == -INFINITY) m = 0.f;
#pragma unroll 8
  for (int k = WAVES == 1 ? 0 : wave; k < cut.y; k += WAVES) {
    const int64_t at = slot(k);
    const float2 ml = *reinterpret_cast<const float2*>(a.ml + at * 2);
    const float f = fast_exp2(ml.x - m);
    const float* x = a.acc + at * D + lane * E;
    l = fmaf(ml.y, f, l);
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = fmaf(x[i], f, o[i]);
  }
  if constexpr (WAVES > 1) {
#pragma unroll
    for (int i = 0; i < E; ++i) s_sum[wave][lane * E + i] = o[i];
    if (lane == 0) s_sum[wave][D] = l;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) {
      l += s_sum[w][D];
#pragma unroll
      for (int i = 0; i < E; ++i) o[i] += s_sum[w][lane * E + i];
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
    store_as(a.out, token * a.o_token_stride + head * a.o_head_stride + lane * E + i, l == 0.f ? 0.f : o[i] / l, a.query_type);
}

}  // namespace tq
