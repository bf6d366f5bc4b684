// Attention of many rows: chunks of prompts over the paged 8-bit cache.
#pragma once

#include <type_traits>

#include "paged_attention.hpp"

namespace tq {

typedef int PagedI16 __attribute__((ext_vector_type(16)));
typedef float PagedF16 __attribute__((ext_vector_type(16)));
typedef _Float16 PagedH8 __attribute__((ext_vector_type(8)));

constexpr int kChunkRows = 128;  // 32 to a wavefront
constexpr int chunk_threads(int d) { return d == 256 ? 512 : 256; }

// Four codes as float16, exactly: with the sign bit turned they are 0..255, which
// the low byte of the float16 1024 holds; 1152 = 1024 + 128 comes off again.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t* out) {
  const uint32_t u = w ^ 0x80808080u;
  const PagedH2 off = {static_cast<_Float16>(-1152.f), static_cast<_Float16>(-1152.f)};
  out[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(PagedH2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
  out[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(PagedH2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
}
__device__ __forceinline__ void codes_to_half(uint4 w, uint16_t* to) {  // 16 codes to 32 bytes
  uint32_t x[8];
  codes_to_half(w.x, x), codes_to_half(w.y, x + 2), codes_to_half(w.z, x + 4), codes_to_half(w.w, x + 6);
  reinterpret_cast<uint4*>(to)[0] = make_uint4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<uint4*>(to)[1] = make_uint4(x[4], x[5], x[6], x[7]);
}

// The query rows of 32 columns as right operands of the score product, and the
// product.  `unit` times a product (of codes) is the score over the page's scale.

// float16 (head_dim 64 and 128): a row is brought to [2^13, 2^14) by a power of
// two, which keeps 16-bit queries as they are; float32 ones are two float16,
// together good to 2^-22.  The codes are float16 in LDS.
template <int D, int TERMS>
struct HalfScores {
  static constexpr int kPitch = 2 * (D + 8);  // bytes of a key in LDS
  PagedH8 q[TERMS][D / 16];

  __device__ __forceinline__ float set(const PagedAttentionArgs& a, int64_t base, bool live, int g) {
    uint32_t bits = 0;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float x[16];
      paged_query16(a, base + 32 * c + 16 * g, live, x);
      bits = paged_extent(x, bits);
    }
    const float top = xor_reduce<32, OpBits>(__uint_as_float(bits));
    const bool bad = !(top < INFINITY);
    int e;
    frexpf(top, &e);
    const float f = top > 1e-30f && !bad ? ldexpf(1.f, 14 - e) : 0.f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float x[16];
      paged_query16(a, base + 32 * c + 16 * g, live, x);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float y = bad ? 0.f : x[i] * f;
        const _Float16 hi = static_cast<_Float16>(y);
        q[0][2 * c + (i >> 3)][i & 7] = hi;
        if constexpr (TERMS == 2) q[1][2 * c + (i >> 3)][i & 7] = static_cast<_Float16>(y - static_cast<float>(hi));
      }
    }
    return bad ? NAN : (f > 0.f ? 1.f / f : 0.f) * a.score_scale;
  }
  static __device__ __forceinline__ void put(int8_t* to, int row, int piece, uint4 codes) {
    codes_to_half(codes, reinterpret_cast<uint16_t*>(to + row * kPitch + 32 * piece));
  }
  // Lane group g has dimensions 32 c + 16 g .. of chunk c, in the keys as in the query.
  __device__ __forceinline__ void run(const int8_t* keys, int row, int g, float (&out)[16]) const {
    PagedF16 sum = {};
    const int8_t* kp = keys + row * kPitch + 32 * g;
#pragma unroll
    for (int c = 0; c < D / 16; ++c) {
      const PagedH8 k = *reinterpret_cast<const PagedH8*>(kp + 64 * (c >> 1) + 16 * (c & 1));
      sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[0][c], sum, 0, 0, 0);
      if constexpr (TERMS == 2) sum = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, q[1][c], sum, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) out[r] = sum[r];
  }
};

// 8 bits (head_dim 256): digits as in paged_split_kernel; the keys take half the
// bytes of LDS, which is what this width has least of.
template <int D, int TERMS>
struct DigitScores {
  static constexpr int kPitch = D + 16, PLANES = TERMS + 1;
  PagedI4 q[PLANES][D / 32];

  __device__ __forceinline__ float set(const PagedAttentionArgs& a, int64_t base, bool live, int g) {
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float x[16];
      paged_query16(a, base + 32 * c + 16 * g, live, x);
      top = paged_extent(x, top);
    }
    top = __float_as_uint(xor_reduce<32, OpBits>(__uint_as_float(top)));
    float f;
    const float unit = paged_unit<PLANES>(top, &f) * a.score_scale;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      float x[16];
      paged_query16(a, base + 32 * c + 16 * g, live, x);
      PagedI4 d[PLANES];
      paged_digits<PLANES>(x, f, d);
#pragma unroll
      for (int k = 0; k < PLANES; ++k) q[k][c] = d[k];
    }
    return unit;
  }
  static __device__ __forceinline__ void put(int8_t* to, int row, int piece, uint4 codes) {
    *reinterpret_cast<uint4*>(to + row * kPitch + 16 * piece) = codes;
  }
  __device__ __forceinline__ void run(const int8_t* keys, int row, int g, float (&out)[16]) const {
    const int8_t* kp = keys + row * kPitch + 16 * g;
    PagedI4 kv[D / 32];
#pragma unroll
    for (int c = 0; c < D / 32; ++c) kv[c] = *reinterpret_cast<const PagedI4*>(kp + 32 * c);
    PagedI16 hi = {}, lo = {};
#pragma unroll
    for (int c = 0; c < D / 32; ++c) hi = __builtin_amdgcn_mfma_i32_32x32x32_i8(kv[c], q[0][c], hi, 0, 0, 0);
#pragma unroll
    for (int r = 0; r < 16; ++r) hi[r] <<= 8;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) hi = __builtin_amdgcn_mfma_i32_32x32x32_i8(kv[c], q[1][c], hi, 0, 0, 0);
    if constexpr (PLANES == 3) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) lo = __builtin_amdgcn_mfma_i32_32x32x32_i8(kv[c], q[2][c], lo, 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      out[r] = static_cast<float>(hi[r]);
      if constexpr (PLANES == 3) out[r] = fmaf(out[r], 256.f, static_cast<float>(lo[r]));
    }
  }
};

// paged_chunk_kernel<D, TERMS>: 128 rows to a workgroup, 32 to a wavefront; the
// wavefronts share each tile of 64 keys through LDS.  At head_dim 256 a second
// four wavefronts take the same rows: either four score half of a tile's keys and
// sum half of the value dimensions, the weights going through LDS between, so that
// a wavefront's sums fit its registers beside the query and two run on a SIMD.
//
// The weights are rounded to float16, 2^-12 of themselves at most, an error of the
// size of a 16-bit result's own; for float32 queries (TERMS 2) a second product
// takes their remainders.  Values become float16 exactly on their way into LDS, so
// the sums of v_mfma_f32_32x32x16_f16 stay in their float32 registers from tile to
// tile.  The running maximum moves only when a tile exceeds it by 2^8; weights
// carry 2^7, so that they stay below float16's largest and a weight of 2^-31 of
// the largest still counts.
//
// Measured: 2048 tokens of 32 query heads after 6000, head_dim 128, bfloat16: 369 us,
// 638 TFLOP/s; 2000 tokens of 16 after 6001 at 256: 354 us, 646 TFLOP/s without the
// merge, the matrix pipe 31 % busy: the wavefronts of a SIMD come to the exponentials
// together, after the same barriers.
//
// Score register r of lane (column j, g = lane / 32) is the 32x32 product's row
// 8 (r / 4) + 4 g + r mod 4; the key at that row is token 16 (r / 8) + 8 g +
// r mod 8, so eight registers are the eight tokens of a 16-deep right operand
// of the second product, and 16 tokens, which share a page, are eight registers of
// every lane: page scales are scalars.
template <int D, int TERMS, bool CUT>
__global__ __launch_bounds__(chunk_threads(D), 2) void paged_chunk_kernel(const PagedAttentionArgs a) {
  using Scores = std::conditional_t<D == 256, DigitScores<D, TERMS>, HalfScores<D, TERMS>>;
  constexpr int NT = chunk_threads(D), R = kChunkRows, HALVES = NT / 256;
  constexpr int DH = D / HALVES, DT = DH / 32, SUBS = 2 / HALVES;  // halves of a tile that a wavefront scores
  constexpr int KP = Scores::kPitch, VP = kTile + 8;  // LDS pitches: bytes of a key, float16 of a value dimension
  constexpr int UNITS = 4 * D / NT;                   // 16-byte pieces of a tile's keys (values) to a thread
  constexpr float kLift = 7.f;
  __shared__ __align__(16) int8_t s_k[2][kTile * KP];
  __shared__ __align__(16) uint16_t s_v[2][D * VP];
  // of a tile's four groups of 16 tokens: the next tile's page numbers, this one's
  // key scales, log2 of the value scales and their inverses (0: no page)
  __shared__ __align__(16) int s_next[2][4];
  __shared__ __align__(16) float s_scale[2][3][4];
  // HALVES 2: the rows' maxima over either half of a tile, and the weights of a tile
  __shared__ float s_top[HALVES][HALVES == 2 ? R : 1];
  __shared__ __align__(16) PagedH8 s_w[HALVES == 2 ? 4 : 1][4][TERMS][kWave];
  const PagedBatch& p = a.batch;
  const int tid = threadIdx.x, lane = lane_id(), wave = tid >> 6;
  const int j = lane & 31, g = lane >> 5;
  const int h = blockIdx.y;
  const int T = 1 << p.log_page;

  paged_schedule<R, CUT>(a, h, [&](const PagedItem& it, int from, int to, bool whole, int slot) {
    const int half = wave >> 2, r0 = 32 * (wave & 3), d0 = DH * half;
    const bool live = r0 + j < it.rows;
    const PagedRowAt at = paged_row(a, it, h, live ? r0 + j : 0);
    const int64_t keys = live ? at.keys : 0;
    Scores scores;
    const float unit = scores.set(a, at.token * a.q_token_stride + at.head * a.q_head_stride, live, g);
    // keys that every row of the workgroup sees, and that any row of this wavefront sees
    const int64_t all_see = paged_row(a, it, h, 0).keys;
    const int64_t some_see = r0 < it.rows ? paged_row(a, it, h, min(r0 + 31, it.rows - 1)).keys : 0;

    float m = -INFINITY, l = 0.f;
    PagedF16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) acc[t] = PagedF16{};

    // Thread i below 4 looks up group i of the tiles to come: page numbers two tiles ahead, scales one, so that
    // neither load is waited for.
    auto page_of = [&](int tile) {
      const int64_t t = static_cast<int64_t>(tile) * kTile + 16 * tid;
      return tid < 4 && tile < to && t < it.s.len ? paged_page(p, it.b, t >> p.log_page) : -1;
    };
    int ahead, now;
    float ks_of, vs_of;
    auto scales_of = [&](int id) {
      const int64_t page = static_cast<int64_t>(max(id, 0)) * p.kv_heads + h;
      ks_of = a.key_scales[page];
      vs_of = a.value_scales[page];
      now = id;
    };
    uint4 kr[UNITS], vr[UNITS];
    auto fetch = [&](const int4 id, int tile) {
#pragma unroll
      for (int n = 0; n < UNITS; ++n) {
        const int u = tid + n * NT;
        const int row = u / (D / 16), piece = u % (D / 16);  // key rows
        const int kgroup = row >> 4, vgroup = u & 3, d = u >> 2;  // value dimensions
        const int kid = kgroup < 2 ? (kgroup == 0 ? id.x : id.y) : (kgroup == 2 ? id.z : id.w);
        const int vid = vgroup < 2 ? (vgroup == 0 ? id.x : id.y) : (vgroup == 2 ? id.z : id.w);
        const int64_t kpage = static_cast<int64_t>(max(kid, 0)) * p.kv_heads + h;
        const int64_t vpage = static_cast<int64_t>(max(vid, 0)) * p.kv_heads + h;
        const int kslot = (tile * kTile + row) & (T - 1), vslot = (tile * kTile + 16 * vgroup) & (T - 1);
        kr[n] = *reinterpret_cast<const uint4*>(a.key_pages + kpage * (D << p.log_page) + kslot * D + 16 * piece);
        vr[n] = *reinterpret_cast<const uint4*>(a.value_pages + vpage * (D << p.log_page) + d * T + vslot);
      }
    };
    auto put = [&](int buffer) {
#pragma unroll
      for (int n = 0; n < UNITS; ++n) {
        const int u = tid + n * NT;
        Scores::put(s_k[buffer], u / (D / 16), u % (D / 16), kr[n]);
        codes_to_half(vr[n], s_v[buffer] + (u >> 2) * VP + 16 * (u & 3));
      }
      if (tid < 4) {
        s_next[buffer][tid] = ahead;
        s_scale[buffer][0][tid] = ks_of;
        s_scale[buffer][1][tid] = __log2f(vs_of);
        s_scale[buffer][2][tid] = now < 0 ? 0.f : 1.f / vs_of;
      }
    };

    __syncthreads();  // the item before has done with LDS
    if (from < to) {
      ahead = page_of(from);
      if (tid < 4) {
        scales_of(ahead);
        s_next[1][tid] = ahead;
        ahead = page_of(from + 1);
      }
      __syncthreads();
      fetch(*reinterpret_cast<const int4*>(s_next[1]), from);
    }
    for (int tile = from; tile < to; ++tile) {
      const int buffer = (tile - from) & 1;
      put(buffer);
      lds_barrier();
      if (tile + 1 < to) {
        fetch(*reinterpret_cast<const int4*>(s_next[buffer]), tile + 1);
        if (tid < 4) {
          scales_of(ahead);
          ahead = page_of(tile + 2);
        }
      }
      const int64_t tok0 = static_cast<int64_t>(tile) * kTile;
      if (HALVES == 2 || tok0 < some_see) {
        const float4 k4 = *reinterpret_cast<const float4*>(s_scale[buffer][0]), s4 = *reinterpret_cast<const float4*>(s_scale[buffer][1]);
        const float4 b4 = *reinterpret_cast<const float4*>(s_scale[buffer][2]);
        const float ks[4] = {k4.x, k4.y, k4.z, k4.w}, shift[4] = {s4.x, s4.y, s4.z, s4.w}, back[4] = {b4.x, b4.y, b4.z, b4.w};
        const bool here = tok0 + kTile <= all_see && b4.x != 0.f && b4.y != 0.f && b4.z != 0.f && b4.w != 0.f;
        float w[SUBS][16];
        float top = -INFINITY;
#pragma unroll
        for (int n = 0; n < SUBS; ++n) {
          const int s = HALVES == 2 ? half : n;
          // row i of the product is token 16 (i / 16) + 8 (i / 4 mod 2) + 4 (i / 8 mod 2) + i mod 4
          const int row = 32 * s + 16 * (j >> 4) + 8 * ((j >> 2) & 1) + 4 * ((j >> 3) & 1) + (j & 3);
          scores.run(s_k[buffer], row, g, w[n]);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float by = s == 0 ? (r < 8 ? ks[0] : ks[1]) : (r < 8 ? ks[2] : ks[3]);
            const float up = s == 0 ? (r < 8 ? shift[0] : shift[1]) : (r < 8 ? shift[2] : shift[3]);
            w[n][r] = fmaf(w[n][r], by * unit, up);
          }
          if (!here) {
            const int64_t left = keys - (tok0 + 32 * s + 8 * g);  // keys seen from this lane's first on
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float b = s == 0 ? (r < 8 ? back[0] : back[1]) : (r < 8 ? back[2] : back[3]);
              w[n][r] = b != 0.f && 16 * (r >> 3) + (r & 7) < left ? w[n][r] : -INFINITY;
            }
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, w[n][r]);
        }
        top = xor_reduce<32, OpMax>(top);
        if constexpr (HALVES == 2) {  // the other half's maximum: both halves' weights are relative to the same
          if (g == 0) s_top[half][r0 + j] = top;
          lds_barrier();
          top = fmaxf(top, s_top[1 - half][r0 + j]);
        }
        if (__ballot(top > m + 8.f) != 0) {
          const float next = fmaxf(m, top);
          const float keep = m == next ? 1.f : fast_exp2(m - next);
          m = next;
          l *= keep;
#pragma unroll
          for (int t = 0; t < DT; ++t) acc[t] *= keep;
        }
        const float base = m == -INFINITY ? 0.f : m - kLift;
        auto weigh = [&](const float* x, PagedH8* p16) {  // of 16 tokens, one page; their sum
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float e = fast_exp2(x[i] - base);
            sum += e;
            p16[0][i] = static_cast<_Float16>(e);
            if constexpr (TERMS == 2) p16[TERMS - 1][i] = static_cast<_Float16>(e - static_cast<float>(p16[0][i]));
          }
          return sum;
        };
        auto gather = [&](int kc, const PagedH8* p16) {
#pragma unroll
          for (int t = 0; t < DT; ++t) {
            const PagedH8 v = *reinterpret_cast<const PagedH8*>(s_v[buffer] + (d0 + 32 * t + j) * VP + 16 * kc + 8 * g);
#pragma unroll
            for (int n = 0; n < TERMS; ++n) acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p16[n], acc[t], 0, 0, 0);
          }
        };
        if constexpr (HALVES == 2) {
          PagedH8 own[2][TERMS];
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float sum = weigh(w[0] + 8 * n, own[n]);
            l = fmaf(sum, half == 0 ? (n == 0 ? back[0] : back[1]) : (n == 0 ? back[2] : back[3]), l);
#pragma unroll
            for (int k = 0; k < TERMS; ++k) s_w[wave & 3][2 * half + n][k][lane] = own[n][k];
          }
          lds_barrier();
#pragma unroll
          for (int kc = 0; kc < 4; ++kc) {
            PagedH8 p16[TERMS];
#pragma unroll
            for (int k = 0; k < TERMS; ++k) p16[k] = s_w[wave & 3][kc][k][lane];
            gather(kc, p16);
          }
        } else {
#pragma unroll
          for (int kc = 0; kc < 4; ++kc) {
            PagedH8 p16[TERMS];
            l = fmaf(weigh(w[kc >> 1] + 8 * (kc & 1), p16), back[kc], l);
            gather(kc, p16);
          }
        }
      }
    }

    l = xor_reduce<32, OpSum>(l);
    if constexpr (HALVES == 2) {  // either half has summed its own tokens' weights
      __syncthreads();
      if (g == 0) s_top[half][r0 + j] = l;
      __syncthreads();
      l += s_top[1 - half][r0 + j];
    }
    if (!live) return;
    if (whole) {
      const int64_t o = at.token * a.o_token_stride + at.head * a.o_head_stride + d0 + 4 * g;
      const float f = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v[4] = {acc[t][4 * r] * f, acc[t][4 * r + 1] * f, acc[t][4 * r + 2] * f, acc[t][4 * r + 3] * f};
          paged_store4(a, o + 32 * t + 8 * r, v);
        }
    } else {
      const int64_t at_slot = ((static_cast<int64_t>(blockIdx.x) * p.kv_heads + h) * 2 + slot) * R + r0 + j;
#pragma unroll
      for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          *reinterpret_cast<float4*>(a.acc + at_slot * D + d0 + 32 * t + 8 * r + 4 * g) =
              make_float4(acc[t][4 * r], acc[t][4 * r + 1], acc[t][4 * r + 2], acc[t][4 * r + 3]);
      if (g == 0 && d0 == 0) {
        a.ml[at_slot * 2] = m;
        a.ml[at_slot * 2 + 1] = l;
      }
    }
  });
}

}  // namespace tq
