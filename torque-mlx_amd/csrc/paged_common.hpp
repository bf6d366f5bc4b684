// What the kernels over the paged 8-bit cache share: the pages, the batch of
// sequences that a call serves, and the search for the sequence of a unit of
// work.
//
// Pages (T = page_size slots, 16, 32 or 64):
//   key_pages    int8  [num_pages, kv_heads, T, D]
//   value_pages  int8  [num_pages, kv_heads, D, T]   transposed, see below
//   key_scales, value_scales  float32 [num_pages, kv_heads]
// A held value is code * scale; appends write scales that are powers of two,
// so rescaling a page's older codes rounds once, at the halved code, and the
// product of code and scale is exact in bfloat16 and in float32.
//
// Values are held transposed because the attention's second product sums over
// tokens: with a head's tokens contiguous for each dimension, a lane's 16-byte
// load is a whole operand of the 8-bit matrix instruction and nothing moves
// between lanes or through LDS.
//
// Nothing that lies on the device is trusted for addresses: lengths are cut to
// the page table, page numbers outside the pool are passed over, row offsets
// are cut to the rows there are.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "tq_device.hpp"

namespace tq {

struct PagedBatch {
  const int32_t* table;  // [batch, max_pages], rows table_stride apart
  int64_t table_stride;
  int max_pages;
  const int32_t* lens;    // [batch]: tokens of each sequence, the call's own included
  const int32_t* starts;  // [batch + 1] rows of each sequence in the call, or null: one row each
  int batch;
  int tokens;  // rows of the call
  int log_page;
  int num_pages;
  int kv_heads;
};

// Tokens of a sequence, at most: a tile's last token is counted in 32 bits too.
constexpr int64_t kMostTokens = 0x7fffff00;

struct PagedSequence {
  int row0, rows;  // its rows of the call
  int len;         // its tokens, at most what the page table holds and at least 0
  int64_t first;   // position of its first row (negative where there are more rows than tokens)
};

__device__ __forceinline__ int paged_start(const PagedBatch& p, int b) {
  return min(max(p.starts[b], 0), p.tokens);
}

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch& p, int b) {
  PagedSequence s;
  if (p.starts == nullptr) {
    s.row0 = b;
    s.rows = 1;
  } else {
    s.row0 = paged_start(p, b);
    s.rows = max(paged_start(p, b + 1) - s.row0, 0);
  }
  const int64_t len = p.lens[b];
  s.first = len - s.rows;
  s.len = static_cast<int>(min(min(max(len, int64_t(0)), kMostTokens), static_cast<int64_t>(p.max_pages) << p.log_page));
  return s;
}

// The page number at place j of sequence b, or -1.
__device__ __forceinline__ int paged_page(const PagedBatch& p, int b, int64_t j) {
  if (j < 0 || j >= p.max_pages) return -1;
  const int id = p.table[b * p.table_stride + j];
  return id >= 0 && id < p.num_pages ? id : -1;
}

// The last b in [0, batch) with base(b) <= u, for base not decreasing (0 where
// it is not): 64 places are looked at at once, so a batch of up to 64
// sequences costs one load.
template <class Base>
__device__ __forceinline__ int wave_last(int batch, int64_t u, Base base) {
  int lo = 0, count = batch;
  while (count > 1) {
    const int step = (count + kWave - 1) / kWave;
    const int at = lane_id() * step;
    const bool here = at < count && base(lo + at) <= u;
    const unsigned long long mask = __ballot(here);
    const int k = mask == 0 ? 0 : 63 - __clzll(mask);
    lo += k * step;
    count = min(step, count - k * step);
  }
  return lo;
}

// The least power of two s, 2^-40 or more, with |x| <= 127 s.
__device__ __forceinline__ float paged_scale(float largest) {
  if (!(largest > 0.f)) return 0x1p-40f;
  int e;
  const float m = frexpf(largest, &e);
  return fmaxf(ldexpf(1.f, e - 7 + (m > 127.f / 128.f ? 1 : 0)), 0x1p-40f);
}

// ---- rows of a model's tensors

// What a kernel knows of its rows when it is compiled: their type (16-byte
// aligned, float32 tables, eight elements' partners side by side), or nothing.
constexpr int kAnyRows = 3;

__device__ __forceinline__ void two_floats(uint32_t w, int type, float* v) {
  if (type == kTypeF16) {
    v[0] = __half2float(__ushort_as_half(static_cast<uint16_t>(w)));
    v[1] = __half2float(__ushort_as_half(static_cast<uint16_t>(w >> 16)));
  } else {
    v[0] = __uint_as_float(w << 16);
    v[1] = __uint_as_float(w & 0xffff0000u);
  }
}

// Eight consecutive elements; `vec`: they are 16-byte aligned.
template <int KIND>
__device__ __forceinline__ void load8(const void* p, int64_t at, int type, bool vec, float* v) {
  if constexpr (KIND != kAnyRows) type = KIND, vec = true;
  if (vec && type == kTypeF32) {
    const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 a = q[0], b = q[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else if (vec) {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) two_floats(w[i], type, v + 2 * i);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = load_as_f32(p, at + i, type);
  }
}

typedef float PagedF2 __attribute__((ext_vector_type(2)));
typedef _Float16 PagedH2 __attribute__((ext_vector_type(2)));
typedef __bf16 PagedB2 __attribute__((ext_vector_type(2)));

// Two values in 16 bits each, rounded to nearest even (one instruction either way).
__device__ __forceinline__ uint32_t two_halves(float lo, float hi, int type) {
  const PagedF2 v = {lo, hi};
  return type == kTypeF16 ? __builtin_bit_cast(uint32_t, __builtin_convertvector(v, PagedH2))
                          : __builtin_bit_cast(uint32_t, __builtin_convertvector(v, PagedB2));
}

template <int KIND>
__device__ __forceinline__ void store8(void* p, int64_t at, int type, const float* v) {  // 16-byte aligned
  if constexpr (KIND != kAnyRows) type = KIND;
  if (type == kTypeF32) {
    float4* q = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    q[0] = make_float4(v[0], v[1], v[2], v[3]);
    q[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = two_halves(v[2 * i], v[2 * i + 1], type);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + at) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

}  // namespace tq
