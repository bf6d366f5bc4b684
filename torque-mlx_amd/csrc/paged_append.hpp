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
  uint32_t axes_used;   // bit a: some pair is turned by axis a
  int by_token;         // table row = row of the call
  int vec;              // eight entries are 16-byte aligned
  uint32_t pair_axis[8];  // 2 bits for each of up to 128 pairs
};

struct PagedRows {
  const void* data;  // [tokens, heads, D], unit stride along D
  int type;
  int64_t token_stride, head_stride;
  int vec;  // eight elements are 16-byte aligned
};

struct PagedAppendArgs {
  PagedBatch batch;
  PagedRows key, value, query;
  int query_heads;
  int query_step, query_parts;  // heads to a workgroup, workgroups to a token's heads
  void* query_out;  // [tokens, query_heads, D] of the query's type
  int8_t* pages[2];   // keys, values
  float* scales[2];
  PagedRotary rotary;
  const float* signs_left;  // null: no rotated basis
  const float* signs_right;
  int rotate_values;
  int kv_step, kv_parts;  // heads to a workgroup, workgroups to a page's heads
  int64_t kv_blocks;      // workgroups that hold pages; queries follow
  int64_t block0;     // first workgroup of this launch
};

// ---- rows with 16 elements to a lane, as append_kernel holds them: lane l of a
// row's D / 16 has the elements 8 l .. 8 l + 7 and D / 2 + 8 l ..

// Place of lane `pl` among its row's lanes: the upper half of eight is mirrored,
// so that row_half_mirror pairs places 4 apart.
template <int D>
__device__ __forceinline__ int row_place(int pl) {
  return D >= 128 && (pl & 4) ? (pl & 8) + 11 - (pl & 7) : pl;
}

// The table entries that turn this lane's 16 elements of row `token`; false where
// a position is outside the tables (nothing is read then).
template <int D, int KIND>
__device__ __forceinline__ bool paged_angles(const PagedRotary& r, int l, int64_t token, int64_t position, float (&c)[16],
                                             float (&s)[16]) {
  constexpr bool PLAIN = KIND != kAnyRows;
  constexpr int TABLE = PLAIN ? static_cast<int>(kTypeF32) : kAnyRows;
  const int half = r.rotary_dim / 2;
  int64_t row[4] = {r.by_token ? token : position, 0, 0, 0};
  bool good = true;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k > 0 && r.axes == 1) continue;
    if (r.positions != nullptr && k < r.axes) {
      const int64_t at = k * r.positions_stride + token;
      row[k] = r.positions_wide ? static_cast<const int64_t*>(r.positions)[at] : static_cast<const int32_t*>(r.positions)[at];
    }
    if ((r.axes_used >> k) & 1) good = good && row[k] >= 0 && row[k] < r.table_rows;
  }
  if (!good) return false;
  if (PLAIN && r.axes > 1) {  // eight pairs: the rows of the axes among them, each taken where it is the pair's
    uint32_t bits[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int d0 = h * (D / 2) + 8 * l, pair0 = d0 < half ? d0 : d0 - half;
      uint32_t word = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) word = (pair0 >> 4) == k ? r.pair_axis[k] : word;
      bits[h] = d0 < r.rotary_dim ? (word >> (2 * (pair0 & 8))) & 0xffffu : 0x10000u;  // bit 16: no pairs here
    }
#pragma unroll 1  // one axis's entries in registers at a time
    for (int k = 0; k < r.axes; ++k) {
      const int64_t at = k == 0 ? row[0] : k == 1 ? row[1] : k == 2 ? row[2] : row[3];
      // pairs of axis k: two zero bits where the pair's axis and k agree
      const uint32_t other = k * 0x5555u;
      float ck[2][8], sk[2][8];
      uint32_t same[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t x = (bits[h] & 0xffffu) ^ other;
        same[h] = bits[h] >> 16 ? 0u : ~(x | (x >> 1)) & 0x5555u;
        if (same[h] == 0) continue;
        const int d0 = h * (D / 2) + 8 * l;
        load8<TABLE>(r.cos, at * r.cos_stride + d0, r.table_type, true, ck[h]);
        load8<TABLE>(r.sin, at * r.sin_stride + d0, r.table_type, true, sk[h]);
      }
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool here = (same[h] >> (2 * i)) & 1;
          c[8 * h + i] = here ? ck[h][i] : c[8 * h + i];
          s[8 * h + i] = here ? sk[h][i] : s[8 * h + i];
        }
    }
    return true;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d0 = h * (D / 2) + 8 * l;
    if (d0 >= r.rotary_dim) continue;
    if (PLAIN || (r.axes == 1 && d0 + 8 <= r.rotary_dim)) {
      load8<TABLE>(r.cos, row[0] * r.cos_stride + d0, r.table_type, r.vec, c + 8 * h);
      load8<TABLE>(r.sin, row[0] * r.sin_stride + d0, r.table_type, r.vec, s + 8 * h);
      continue;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + i;
      if (d >= r.rotary_dim) continue;
      const int pair = d < half ? d : d - half;
      uint32_t word = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) word = (pair >> 4) == k ? r.pair_axis[k] : word;
      const int axis = (word >> (2 * (pair & 15))) & 3;
      const int64_t at = axis == 0 ? row[0] : axis == 1 ? row[1] : axis == 2 ? row[2] : row[3];
      c[8 * h + i] = load_as_f32(r.cos, at * r.cos_stride + d, r.table_type);
      s[8 * h + i] = load_as_f32(r.sin, at * r.sin_stride + d, r.table_type);
    }
  }
  return true;
}

// This lane's 16 elements of a row, turned.  Every operation is rounded by itself,
// as the torch operations of apply_rotary round it in float32 (one more per
// element than with a fused multiply-add: keys next to a code's border then have
// the codes that the composition of torch operations gives them).
template <int D, int KIND>
__device__ __forceinline__ void paged_turn(const PagedRotary& r, const PagedRows& x, int64_t base, int l, const float (&c)[16],
                                           const float (&s)[16], float (&v)[16]) {
#pragma clang fp contract(off)
  constexpr bool PLAIN = KIND != kAnyRows;
  const int half = r.rotary_dim / 2;
  if (r.rotary_dim == D) {  // an element's partner lies in the same lane
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = v[i], b = v[8 + i];
      v[i] = a * c[i] - b * s[i];
      v[8 + i] = b * c[8 + i] + a * s[8 + i];
    }
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d0 = h * (D / 2) + 8 * l;
    if (d0 >= r.rotary_dim) continue;
    float w[8];
    if (PLAIN || half % 8 == 0) {  // eight elements have their partners side by side
      load8<KIND>(x.data, base + (d0 < half ? d0 + half : d0 - half), x.type, x.vec, w);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = d0 + i;
        w[i] = d < r.rotary_dim ? load_as_f32(x.data, base + (d < half ? d + half : d - half), x.type) : 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int d = d0 + (PLAIN ? 0 : i);
      if (!PLAIN && d >= r.rotary_dim) continue;
      v[8 * h + i] = v[8 * h + i] * c[8 * h + i] + (d < half ? -w[i] : w[i]) * s[8 * h + i];
    }
  }
}

template <int D>
constexpr float kInverseRoot = D == 64 ? 0.125f : D == 256 ? 0.0625f : 0.0883883476483184405501f;

// x / sqrt(D), rounded once.  For 128, whose root is no power of two: the
// quotient by the rounded reciprocal, corrected by its exact remainder
// (Markstein's division step); infinities and NaN as they come.
template <int D>
__device__ __forceinline__ float over_root(float x) {
  const float q = __fmul_rn(x, kInverseRoot<D>);
  if constexpr (D != 128) return q;
  constexpr float kRoot = 11.3137084989847603904f;
  const float y = fmaf(fmaf(-q, kRoot, x), kInverseRoot<D>, q);
  return fabsf(q) < INFINITY ? y : q;
}

// This lane's signs after the transform as bits (1: negative), with the sign that
// the transform's steps between lanes leave.
template <int D>
__device__ __forceinline__ uint32_t second_signs(const float* left, int l) {
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) bits |= (__float_as_uint(left[(i >> 3) * (D / 2) + 8 * l + (i & 7)]) >> 31) << i;
  return __builtin_popcount(l) & 1 ? ~bits : bits;
}
__device__ __forceinline__ float signed_by(float x, uint32_t bits, int i) {
  return __uint_as_float(__float_as_uint(x) ^ ((bits << (31 - i)) & 0x80000000u));
}

// The Walsh-Hadamard transform of a row, in wave_fwht's order.
template <int D>
__device__ __forceinline__ void transform16(float (&v)[16], int l) {
#pragma unroll
  for (int st = 1; st < 8; st <<= 1)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if ((i & st) == 0) {
        const float x = v[i], y = v[i + st];
        v[i] = __fadd_rn(x, y);
        v[i + st] = __fsub_rn(x, y);
      }
  pair_step<kDppXor1>(v, (l & 1) ? -1.f : 1.f);
  pair_step<kDppXor2>(v, (l & 2) ? -1.f : 1.f);
  if constexpr (D >= 128) pair_step<kDppHalfMirror>(v, (l & 4) ? -1.f : 1.f);
  if constexpr (D >= 256) pair_step<kDppRor8>(v, (l & 8) ? -1.f : 1.f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = v[i], y = v[i + 8];
    v[i] = __fadd_rn(x, y);
    v[i + 8] = __fsub_rn(x, y);
  }
}

__device__ __forceinline__ int paged_code(float x, float inv) {
  const float y = __fmul_rn(x, inv);
  return y != y ? 0 : static_cast<int>(fminf(fmaxf(rintf(y), -127.f), 127.f));
}

// Four codes as one word.  FINE: all are finite and at most 127 steps, so the sum
// with 1.5 x 2^23 rounds them and has their low bytes in its mantissa.
template <bool FINE>
__device__ __forceinline__ uint32_t four_codes(const float* v, float inv) {
  uint32_t n[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) n[i] = FINE ? __float_as_uint(fmaf(v[i], inv, 12582912.f)) : static_cast<uint32_t>(paged_code(v[i], inv));
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(n[3], n[2], 0x0C0C0400u), __builtin_amdgcn_perm(n[1], n[0], 0x0C0C0400u), 0x05040100u);
}

// This lane's 16 elements of a row on their way from memory, as they lie there.
template <int KIND>
struct RowLoad {
  uint4 w[KIND == kTypeF32 ? 4 : 2];
  __device__ __forceinline__ void start(const PagedRows& x, int64_t at, int half) {
    const char* p = static_cast<const char*>(x.data) + at * (KIND == kTypeF32 ? 4 : 2);
    const uint4* lo = reinterpret_cast<const uint4*>(p);
    const uint4* hi = reinterpret_cast<const uint4*>(p + half * (KIND == kTypeF32 ? 4 : 2));
    if constexpr (KIND == kTypeF32)
      w[0] = lo[0], w[1] = lo[1], w[2] = hi[0], w[3] = hi[1];
    else
      w[0] = lo[0], w[1] = hi[0];
  }
  __device__ __forceinline__ void take(float (&v)[16]) const {
    if constexpr (KIND == kTypeF32) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[4 * i] = __uint_as_float(w[i].x), v[4 * i + 1] = __uint_as_float(w[i].y);
        v[4 * i + 2] = __uint_as_float(w[i].z), v[4 * i + 3] = __uint_as_float(w[i].w);
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t u[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) two_floats(u[i], KIND, v + 8 * h + 2 * i);
      }
    }
  }
};
template <>
struct RowLoad<kAnyRows> {
  float w[16];
  __device__ __forceinline__ void start(const PagedRows& x, int64_t at, int half) {
    load8<kAnyRows>(x.data, at, x.type, x.vec, w);
    load8<kAnyRows>(x.data, at + half, x.type, x.vec, w + 8);
  }
  __device__ __forceinline__ void take(float (&v)[16]) const {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = w[i];
  }
};

// What turns this lane's 16 elements of a token's rows, the same for all of its
// heads: table entries, with the first signs in them (exactly: they are +-1), and
// the second signs.  The rotated basis takes wave_rotate's operations on the same
// operands, so its float32 result is the same.
template <int D>
struct RowTurn {
  float c[16], s[16];
  uint32_t second;
  bool turned, based;

  // Whether element i is turned (eight are alike where the rows' kind is known).
  template <int KIND>
  static __device__ __forceinline__ bool in_table(const PagedAppendArgs& a, int l, int i) {
    return (i >> 3) * (D / 2) + 8 * l + (KIND == kAnyRows ? i & 7 : 0) < a.rotary.rotary_dim;
  }

  template <int KIND>
  __device__ __forceinline__ bool set(const PagedAppendArgs& a, bool rotary, bool basis, int l, int64_t token, int64_t position) {
    turned = rotary;
    based = basis;
    const bool good = !rotary || paged_angles<D, KIND>(a.rotary, l, token, position, c, s);
    turned = turned && good;
    if (based) {
      second = second_signs<D>(a.signs_left, l);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float first = a.signs_right[(i >> 3) * (D / 2) + 8 * l + (i & 7)];
        const bool table = turned && in_table<KIND>(a, l, i);
        c[i] = table ? c[i] * first : first;
        s[i] = table ? s[i] * first : 0.f;
      }
    }
    return good;
  }

  // ROUGH: a result that is rounded to 16 bits next is as good with the product
  // by 1 / sqrt(D) as with the quotient, half a step of float32 apart.
  template <int KIND>
  __device__ __forceinline__ void apply(const PagedAppendArgs& a, const PagedRows& x, int64_t base, int l, bool rough, float (&v)[16]) const {
    if (turned) paged_turn<D, KIND>(a.rotary, x, base, l, c, s, v);
    if (!based) return;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (!turned || !in_table<KIND>(a, l, i)) v[i] *= c[i];
    transform16<D>(v, l);
    if (rough) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = signed_by(v[i] * kInverseRoot<D>, second, i);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = signed_by(over_root<D>(v[i]), second, i);
    }
  }
};

// One workgroup for each page that the call writes, stream (keys or values) and
// few heads, D / 16 lanes to a slot: the new rows are turned, taken into the
// rotated basis, held against the largest of them and written; where that makes
// the page's scale grow, the codes that it held before are rounded anew at the
// larger scale.  No other workgroup touches the page's head.  Slots past the
// sequence's end keep what they held.  The workgroups behind those turn the
// queries, T tokens and a few heads each.  A workgroup's heads share their tokens'
// table entries, which are twice to four times as many bytes as a row, and the
// next head's rows are on their way while one is worked on.
//
// Units of work: sequence b owns the units from starts[b] / T + 2 b on, one to a
// page, which is room enough wherever in a page it begins (n rows touch at most
// n / T + 2 pages); a unit without a page ends at once.
//
// Each element is read once and written once, 2 to 4 bytes against 1: memory is
// the bound at prompt sizes, the launch and three dependent loads (length, page
// number, scale) at single tokens.
//
// 32768 tokens of 8 heads (and 32 query heads) of 128 in float16 take 175 us, 4.2
// TB/s over the 738 MB read and written; one token of one sequence 5.3 us.
//
// KIND: the type of all rows, which are 16-byte aligned, as are float32 tables,
// and rotary_dim a multiple of 16; or kAnyRows, which looks each of these up and
// fetches elements one by one where it must, in twice the registers.
//
// SIZE: the page size T; or 0 for a call with one token to a sequence, which one
// wavefront to a page holds without waiting for others (T is looked up).
constexpr int append_threads(int d, int size) { return size == 0 ? kWave : d * size / 16; }

template <int D, int SIZE, int KIND>
__global__ __launch_bounds__(append_threads(D, SIZE)) __attribute__((amdgpu_waves_per_eu(KIND == kAnyRows ? 2 : KIND == kTypeF32 && append_threads(D, SIZE) <= 256 ? 3 : 4)))
void paged_append_kernel(const PagedAppendArgs a) {
  constexpr int NT = append_threads(D, SIZE), WAVES = NT / kWave;
  constexpr int LPR = D / 16;  // lanes to a row
  constexpr int P = D + 4;     // LDS pitch of a value row's codes
  __shared__ uint32_t s_top[2][WAVES];
  __shared__ uint32_t s_rows[SIZE * P / 4 + 1];
  const PagedBatch& p = a.batch;
  const int log_page = SIZE == 0 ? p.log_page : SIZE == 16 ? 4 : SIZE == 32 ? 5 : 6, T = 1 << log_page;
  const int tid = threadIdx.x, wave = tid >> 6, lane = lane_id();
  const int l = row_place<D>(tid & (LPR - 1)), mine = tid / LPR;
  const int64_t block = a.block0 + blockIdx.x;
  RowTurn<D> turn;

  if (block >= a.kv_blocks) {  // queries
    const int64_t qb = block - a.kv_blocks, tb = qb / a.query_parts;
    const int part = static_cast<int>(qb - tb * a.query_parts);
    const int64_t token = tb * (NT / LPR) + mine;
    if (token >= p.tokens) return;
    int64_t position;
    bool ours = true;
    if (p.starts == nullptr) {
      position = static_cast<int64_t>(p.lens[token]) - 1;
    } else {
      int lo = 0, hi = p.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (paged_start(p, mid) <= token)
          lo = mid;
        else
          hi = mid - 1;
      }
      const PagedSequence q = paged_sequence(p, lo);
      ours = token >= q.row0 && token < q.row0 + q.rows;
      position = q.first + token - q.row0;
    }
    const int h0 = part * a.query_step, h1 = min(h0 + a.query_step, a.query_heads);
    const int64_t row = token * a.query.token_stride + 8 * l;
    RowLoad<KIND> next;
    next.start(a.query, row + h0 * a.query.head_stride, D / 2);
    const bool good = turn.template set<KIND>(a, ours && a.rotary.rotary_dim > 0, a.signs_left != nullptr, l, token, position);
    const bool rough = (KIND == kAnyRows ? a.query.type : KIND) != kTypeF32;
    for (int h = h0; h < h1; ++h) {
      float v[16];
      next.take(v);
      if (h + 1 < h1) next.start(a.query, row + (h + 1) * a.query.head_stride, D / 2);
      turn.template apply<KIND>(a, a.query, token * a.query.token_stride + h * a.query.head_stride, l, rough, v);
      if (!ours || !good) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = ours ? NAN : 0.f;
      }
      const int64_t to = (token * a.query_heads + h) * D + 8 * l;
      store8<KIND>(a.query_out, to, a.query.type, v);
      store8<KIND>(a.query_out, to + D / 2, a.query.type, v + 8);
    }
    return;
  }

  const int is_v = static_cast<int>(block & 1);
  const int64_t pu = block >> 1, unit = pu / a.kv_parts;
  const int h0 = static_cast<int>(pu - unit * a.kv_parts) * a.kv_step, h1 = min(h0 + a.kv_step, p.kv_heads);
  int b = static_cast<int>(unit);
  int64_t place = 0;
  if (p.starts != nullptr) {
    auto base = [&](int i) { return static_cast<int64_t>((paged_start(p, i) >> log_page) + 2 * i); };
    b = wave_last(p.batch, unit, base);
    place = unit - base(b);
  }
  const PagedSequence q = paged_sequence(p, b);
  const int64_t c0 = max(q.first, int64_t(0));
  const int64_t page = (c0 >> log_page) + place;
  const int64_t lo = max(c0, page * T), hi = min(static_cast<int64_t>(q.len), page * T + T);
  if (place < 0 || lo >= hi) return;
  const int id = paged_page(p, b, page);
  if (id < 0) return;
  const int kept = static_cast<int>(lo - page * T), count = static_cast<int>(hi - lo);  // slots kept .. kept + count are new
  const int64_t token = q.row0 + (lo - q.first) + mine;  // this lane's, if there are so many
  const int slot = kept + mine;
  const bool whole = SIZE != 0 && is_v && count == SIZE;  // value rows of a whole page go through LDS, which turns them

  const PagedRows& x = is_v ? a.value : a.key;
  const int64_t row = token * x.token_stride + 8 * l;
  float* scales = a.scales[is_v] + static_cast<int64_t>(id) * p.kv_heads;
  RowLoad<KIND> next;
  bool ours = mine < count;
  if (ours) next.start(x, row + h0 * x.head_stride, D / 2);
  ours = turn.template set<KIND>(a, ours && !is_v && a.rotary.rotary_dim > 0, a.signs_left != nullptr && (!is_v || a.rotate_values), l,
                                 token, lo + mine) && ours;
  if (__syncthreads_or(ours) == 0) return;  // no row has a position

  for (int h = h0; h < h1; ++h) {
    const float held = kept > 0 ? scales[h] : 0.f;
    float v[16];
    if (ours) {
      next.take(v);
      if (h + 1 < h1) next.start(x, row + (h + 1) * x.head_stride, D / 2);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = 0.f;
    }
    turn.template apply<KIND>(a, x, token * x.token_stride + h * x.head_stride, l, false, v);
    uint32_t top = 0;  // bits of the largest |x|: an infinity, a NaN above all
    if (ours) {
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
    }
    auto reduce = [&](uint32_t t, int at) {
      t = __float_as_uint(group_reduce<kWave, OpBits>(__uint_as_float(t)));
      if constexpr (WAVES > 1) {
        if (lane == 0) s_top[at][wave] = t;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) t = max(t, s_top[at][w]);
      }
      return t;
    };
    top = reduce(top, h & 1);
    const bool fine = top < 0x7f800000u;
    if (!fine) {  // the largest finite element
      top = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const uint32_t m = __float_as_uint(v[i]) & 0x7fffffffu;
        if (ours && m < 0x7f800000u) top = max(top, m);
      }
      __syncthreads();
      top = reduce(top, h & 1);
    }
    const float scale = fmaxf(held, paged_scale(__uint_as_float(top)));
    if (tid == 0) scales[h] = scale;
    int8_t* out = a.pages[is_v] + (static_cast<int64_t>(id) * p.kv_heads + h) * (D * T);

    if (kept > 0 && scale != held) {  // the older codes at the grown scale
      const float ratio = __fdiv_rn(held, scale);
      uint32_t* words = reinterpret_cast<uint32_t*>(out);
#pragma unroll 1
      for (int w = tid; w < D * T / 4; w += NT) {
        const int slot0 = is_v ? 4 * (w & (T / 4 - 1)) : w / (D / 4);
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
    uint32_t word[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) word[i] = fine ? four_codes<true>(v + 4 * i, inv) : four_codes<false>(v + 4 * i, inv);
    if constexpr (SIZE != 0) {
      if (whole) {
        uint32_t* to = s_rows + slot * (P / 4) + 2 * l;
        to[0] = word[0], to[1] = word[1];
        to[D / 8] = word[2], to[D / 8 + 1] = word[3];
        __syncthreads();
        const int tq = tid % (SIZE / 4), dq = tid / (SIZE / 4);  // four tokens by four dimensions
        uint32_t r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = s_rows[(4 * tq + i) * (P / 4) + dq];
        const uint32_t ab = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), cd = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u);
        const uint32_t ef = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u), gh = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
        uint32_t* put = reinterpret_cast<uint32_t*>(out + 4 * dq * SIZE + 4 * tq);
        put[0] = __builtin_amdgcn_perm(cd, ab, 0x05040100u);
        put[SIZE / 4] = __builtin_amdgcn_perm(cd, ab, 0x07060302u);
        put[SIZE / 2] = __builtin_amdgcn_perm(gh, ef, 0x05040100u);
        put[3 * SIZE / 4] = __builtin_amdgcn_perm(gh, ef, 0x07060302u);
        if constexpr (WAVES == 1) __syncthreads();  // the next head's rows overwrite these (with more waves its maximum waits)
        continue;
      }
    }
    if (ours && !is_v) {
      *reinterpret_cast<uint2*>(out + slot * D + 8 * l) = make_uint2(word[0], word[1]);
      *reinterpret_cast<uint2*>(out + slot * D + D / 2 + 8 * l) = make_uint2(word[2], word[3]);
    } else if (ours) {
      int8_t* put = out + 8 * l * T + slot;
#pragma unroll
      for (int i = 0; i < 16; ++i) put[((i >> 3) * (D / 2) + (i & 7)) * T] = static_cast<int8_t>(word[i >> 2] >> (8 * (i & 3)));
    }
  }
}

struct PagedReadArgs {
  const int32_t* ids;  // [count]
  int64_t count;
  const int8_t* pages[2];
  const float* scales[2];
  void* out[2];  // [count, kv_heads, T, D]
  int num_pages, kv_heads, head_dim, log_page;
  int64_t block0;
};

// Pages as the values they stand for: one workgroup to a page, head and stream.
// A thread has 16 codes of a key row, or 4 dimensions by 8 tokens of the
// transposed values, which it turns in registers.
template <int TYPE>
__global__ __launch_bounds__(kBlock) void paged_read_kernel(const PagedReadArgs a) {
  const int T = 1 << a.log_page, D = a.head_dim;
  const int64_t block = a.block0 + blockIdx.x;
  const int is_v = static_cast<int>(block & 1);
  const int64_t hn = block >> 1, n = hn / a.kv_heads;
  const int h = static_cast<int>(hn - n * a.kv_heads);
  const int id = a.ids[n];
  const bool there = id >= 0 && id < a.num_pages;
  const int64_t from = there ? static_cast<int64_t>(id) * a.kv_heads + h : 0;
  const float scale = there ? a.scales[is_v][from] : 0.f;
  const int8_t* codes = a.pages[is_v] + from * D * T;
  const int64_t to = hn * D * T;
  auto value = [&](uint32_t word, int k) { return there ? scale * static_cast<float>(static_cast<int8_t>(word >> (8 * k))) : 0.f; };
  if (!is_v) {
    for (int u = threadIdx.x; u < D * T / 16; u += kBlock) {
      const uint4 x = reinterpret_cast<const uint4*>(codes)[u];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
      float v[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = value(w[i >> 2], i & 3);
      store8<TYPE>(a.out[0], to + 16 * u, TYPE, v);
      store8<TYPE>(a.out[0], to + 16 * u + 8, TYPE, v + 8);
    }
    return;
  }
  for (int u = threadIdx.x; u < D * T / 32; u += kBlock) {
    const int dq = u & (D / 4 - 1), to8 = u / (D / 4);  // dimensions 4 dq .., tokens 8 to8 ..
    uint2 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint2*>(codes + (4 * dq + i) * T + 8 * to8);
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = value(t < 4 ? x[i].x : x[i].y, t & 3);
      const int64_t at = to + static_cast<int64_t>(8 * to8 + t) * D + 4 * dq;
      if constexpr (TYPE == kTypeF32)
        *reinterpret_cast<float4*>(static_cast<float*>(a.out[1]) + at) = make_float4(v[0], v[1], v[2], v[3]);
      else
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out[1]) + at) = make_uint2(two_halves(v[0], v[1], TYPE), two_halves(v[2], v[3], TYPE));
    }
  }
}

}  // namespace tq
