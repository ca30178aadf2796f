// Pieces that the attention kernels over the 4-bit cache share (kv4_attn.hip, kv4_prompt.hip).
#pragma once
#include "kv4.h"

namespace w4a8 {

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ v4f mfma16(const v4w& a, const v4w& b, const v4f& c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, a), __builtin_bit_cast(v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// 8 codes of a word -> 16 + code, register r holding codes r and r + 4
template <int DT>
__device__ __forceinline__ v4w widen(uint32_t w) {
  constexpr int pos = DT == kBF16 ? 3 : 6;  // 16 in a mantissa of 7 (10) bits: a code's unit is bit 3 (6)
  constexpr uint32_t mask = 0x000f000fu << pos, one = DT == kBF16 ? 0x41804180u : 0x4c004c00u;
  v4w o;
  o[0] = ((w << pos) & mask) | one;
  o[1] = ((DT == kBF16 ? w >> 1 : w << 2) & mask) | one;
  o[2] = ((DT == kBF16 ? w >> 5 : w >> 2) & mask) | one;
  o[3] = ((w >> (12 - pos)) & mask) | one;
  return o;
}

// the same value over the four lanes that hold a column (xor 16 and xor 32)
__device__ __forceinline__ float col_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float col_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N == 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + 4 * i);
      w[i] = u.x; w[i + 1] = u.y; w[i + 2] = u.z; w[i + 3] = u.w;
    }
  }
}

// The page numbers of a tile, wave-uniform: those of its tokens 0..15 and 16..31 (a page holds at least 16),
// as the table has them, -1 where it has none. Looked up a tile before they are used: the scalar loads
// then have nobody waiting. (Nothing writes the table during a launch: constant address space.)
typedef const int32_t __attribute__((address_space(4))) * Table;
struct Pages {
  int a, b;
};
__device__ __forceinline__ Pages look_up(const Kv4Attn& p, Table table, int t, int len) {
  Pages r = {-1, -1};
  const int i = t >> p.c.shift, j = (t + 16) >> p.c.shift;
  if (t < len && i < p.s.width) r.a = table[i];
  if (t + 16 < len && j < p.s.width) r.b = table[j];
  return r;
}
__device__ __forceinline__ bool exists(const Kv4Attn& p, int page) { return (uint32_t)page < (uint32_t)p.c.pages; }
// block `i` of 4 of the tile at t: this lane's; a missing page reads block 0, which is there, and its values
// are not used
__device__ __forceinline__ uint32_t pick(const Kv4Attn& p, const Pages& pg, int h, int t, int i) {
  const int a = exists(p, pg.a) ? kv4_block(p.c, pg.a, h, t) : 0, b = exists(p, pg.b) ? kv4_block(p.c, pg.b, h, t + 16) : 0;
  return (uint32_t)((i < 2 ? a : b) + (i & 1));
}

template <int DT>
__device__ __forceinline__ float lo16(uint32_t w) {
  return DT == kBF16 ? __uint_as_float(w << 16) : f16_to_f32((uint16_t)(w & 0xffffu));
}
template <int DT>
__device__ __forceinline__ float hi16(uint32_t w) {
  return DT == kBF16 ? __uint_as_float(w & 0xffff0000u) : f16_to_f32((uint16_t)(w >> 16));
}

typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
}

// A sequence of the call: its rows and its length. Columns are its queries in order, G heads each.
struct Span {
  int64_t start;
  int n, cols, len, first_pos;  // new tokens, columns, length, position of the first new token
};
__device__ __forceinline__ Span kv4_span(const Kv4Attn& p, int b) {
  Span s;
  kv4_rows(p.s, b, s.start, s.n);
  s.cols = s.n * p.G;
  const int64_t cap = (int64_t)p.s.width << p.c.shift;
  const int len = p.s.lens[b];
  // one token past the table's end stands for all of them: its page is missing
  s.len = len > cap ? (int)(cap + 1 < 0x7fffffff ? cap + 1 : 0x7fffffff) : len < 0 ? 0 : len;
  s.first_pos = len - s.n;
  return s;
}
// the keys [from, upto) that query i of the span sees
__device__ __forceinline__ int seen_from(const Kv4Attn& p, const Span& s, int i) {
  return p.window ? min(max(s.first_pos + i - p.window + 1, 0), s.len) : 0;
}
__device__ __forceinline__ int seen_upto(const Kv4Attn& p, const Span& s, int i) {
  return p.causal ? min(max(s.first_pos + i + 1, 0), s.len) : s.len;
}
// The keys that some, [lo, hi), and that all, [lo_all, hi_all), of columns c0 .. c1 - 1 see: columns are queries
// in order, so the first and the last one tell.
struct Keys {
  int lo, hi, lo_all, hi_all;
};
__device__ __forceinline__ Keys kv4_keys(const Kv4Attn& p, const Span& s, int c0, int c1) {
  if (c0 >= c1) return {0, 0, 0, 0};
  const int i0 = c0 / p.G, i1 = (c1 - 1) / p.G;
  return {seen_from(p, s, i0), seen_upto(p, s, i1), seen_from(p, s, i1), seen_upto(p, s, i0)};
}
// Of the wave's columns c0 .. : the query, from its first column's i0 = c0 / G, r0 = c0 % G, and its head
__device__ __forceinline__ int kv4_query(const Kv4Attn& p, int i0, int r0, int x, int& head) {
  const int c = r0 + x, i = (int)__umulhi((uint32_t)c << 1, p.gmul);
  head = c - i * p.G;
  return i0 + i;
}

// 32 channels of a query as the operand that meets codes in their words' order (elements 0 4, 1 5, 2 6, 3 7 of
// each 8), and their sum
__device__ __forceinline__ v4w query_operand(const uint4& u) {
  return v4w{(u.x & 0xffffu) | (u.z << 16), (u.x >> 16) | (u.z & 0xffff0000u), (u.y & 0xffffu) | (u.w << 16),
             (u.y >> 16) | (u.w & 0xffff0000u)};
}
template <int DT>
__device__ __forceinline__ float sum8(const uint4& u) {
  return ((lo16<DT>(u.x) + hi16<DT>(u.x)) + (lo16<DT>(u.y) + hi16<DT>(u.y))) +
         ((lo16<DT>(u.z) + hi16<DT>(u.z)) + (lo16<DT>(u.w) + hi16<DT>(u.w)));
}

// One lane's DB neighbouring channels of a column, from channel `d0` of (row, head): the output, or the split's
// part for kv4_join_kernel. m: the maximum in powers of two; first: this lane writes the column's statistics.
template <int D, int DT>
__device__ __forceinline__ void kv4_store(const Kv4Attn& p, int split, int64_t row, int head, int d0, const float (&v)[D / 16],
                                          float m, float sum, bool first) {
  constexpr int DB = D / 16;
  const int Hq = p.c.H * p.G;
  if (p.splits > 1) {
    const int64_t at = ((int64_t)split * p.s.T + row) * Hq + head;
    float* op = p.po + at * D + d0;
#pragma unroll
    for (int d = 0; d < DB; d += 4) *reinterpret_cast<v4f*>(op + d) = v4f{v[d], v[d + 1], v[d + 2], v[d + 3]};
    if (first) {
      p.pml[at * 2] = m;
      p.pml[at * 2 + 1] = sum;
    }
    return;
  }
  // no key seen: the sum is 0, the output 0
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* op = p.out + row * p.ldo + head * p.ho + d0;
#pragma unroll
  for (int d = 0; d < DB; d += 4) {
    uint2 u;
    u.x = (uint32_t)to_dtype(v[d] * inv, DT) | ((uint32_t)to_dtype(v[d + 1] * inv, DT) << 16);
    u.y = (uint32_t)to_dtype(v[d + 2] * inv, DT) | ((uint32_t)to_dtype(v[d + 3] * inv, DT) << 16);
    *reinterpret_cast<uint2*>(op + d) = u;
  }
  if (p.lse && first) p.lse[row * Hq + head] = sum == 0.f ? -__builtin_inff() : m * 0.69314718055994531f + logf(sum);
}

}  // namespace w4a8
