// Attention over the paged 4-bit cache (layout: kv4.h), for decode and for prompts.
//
// Per key/value head, the queries that share it are the columns of the matrix products: column c is
// query c / G, query head h * G + c % G. A wave takes 16 NQ columns and walks tiles of 32 tokens, with
// one pass over the cache and the running maximum and sum of the softmax in f32:
//   S = U Q^T      U = 16 + c: the codes as bf16/fp16 numbers 16..31, made by a shift and an and-or for
//                  two codes, exact in either type. The accumulators start at -16 sum(q), so S is q c;
//   x = s S + m sum(q)                       the score, with nothing rounded but f32 sums;
//   O += (p s)^T U, C += p (m - 16 s)        out = (O + C) / sum p.
// p s enters its product as the sum of two bf16 terms (rounded by at most 2^-18 of itself: one term would
// cost as much accuracy as the output's own rounding), with U in bf16 whatever the model's type, so that
// a small V step does not fall below fp16's range.
// The row of S that a lane of group g = lane / 16 holds is chosen to be the token whose V codes that
// lane holds (tokens 8 g + r in the first 16 rows' register r, 8 g + 4 + r in the second's), so p goes
// from one product into the next in its lane, and nothing passes through LDS.
// The running maximum is raised only when a score passes it by 8 (in powers of two): p stays below 2^8,
// and most tiles need no exchange between lanes and no rescaling.
//
// Split: WKV waves of a workgroup (and the splits of the grid) walk the same columns over different
// tiles; their (O, C, sum, max) are joined through LDS, and those of the splits through the workspace
// by kv4_join_kernel.
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

// what one lane reads of a tile: its two rows of K, its 8 tokens of V's channels, and those tokens' scales
template <int D>
struct Tile {
  uint32_t k[2][D / 32], v[D / 16], ks[8], vs[8];
};

// of a tile's blocks: the one with this lane's K rows, and the one of its group (-1: no such page)
struct Blocks {
  int k, g;
};

template <int D>
__device__ __forceinline__ Blocks find_blocks(const Kv4Attn& p, int b, int h, int64_t t0, int len, int lane) {
  const int gk = (lane & 15) >> 2, g = lane >> 4;
  const int64_t tk = t0 + 8 * gk, tg = t0 + 8 * g;
  const int pk = tk < len ? kv4_page(p.c, p.s, b, tk) : -1;
  const int pg = tg < len ? kv4_page(p.c, p.s, b, tg) : -1;
  return {pk < 0 ? 0 : kv4_block(p.c, pk, h, (int)(tk & 0x7fffffff)), pg < 0 ? -1 : kv4_block(p.c, pg, h, (int)(tg & 0x7fffffff))};
}

template <int D>
__device__ __forceinline__ void load_tile(const Kv4Attn& p, const Blocks& at, int lane, Tile<D>& t) {
  const int g = lane >> 4, r = lane & 3;
  const int bg = at.g < 0 ? 0 : at.g;  // block 0 is there to be read; what it gives is not used
  const uint8_t* kp = p.c.k + (int64_t)at.k * (4 * D) + r * (D / 2) + g * (D / 8);
  load_words(kp, t.k[0]);
  load_words(kp + 4 * (D / 2), t.k[1]);
  load_words(p.c.v + (int64_t)bg * (4 * D) + (lane & 15) * (D / 4), t.v);
  load_words(reinterpret_cast<const uint8_t*>(p.c.ks + (int64_t)bg * 8), t.ks);
  load_words(reinterpret_cast<const uint8_t*>(p.c.vs + (int64_t)bg * 8), t.vs);
}

template <int DT>
__device__ __forceinline__ float lo16(uint32_t w) {
  return DT == kBF16 ? __uint_as_float(w << 16) : f16_to_f32((uint16_t)(w & 0xffffu));
}
template <int DT>
__device__ __forceinline__ float hi16(uint32_t w) {
  return DT == kBF16 ? __uint_as_float(w & 0xffff0000u) : f16_to_f32((uint16_t)(w >> 16));
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}

// D: channels; DT: the model's type; NQ: blocks of 16 columns per wave; WKV: 4 waves over the tokens, or 1:
// 4 waves over the columns
template <int D, int DT, int NQ, int WKV>
__global__ void __launch_bounds__(256)
kv4_attn_kernel(const Kv4Attn p) {
  constexpr int KS = D / 32, DB = D / 16;  // products per S tile, blocks of 16 channels
  constexpr int kCols = 16 * NQ * (WKV == 1 ? 4 : 1);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, col = lane & 15;
  const int h = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % p.splits;
  const int Hq = p.c.H * p.G;
  int64_t start;
  int n;
  kv4_rows(p.s, b, start, n);
  const int64_t cols = (int64_t)n * p.G;
  const int64_t cap = (int64_t)p.s.width << p.c.shift;
  // one token past the table's end stands for all of them: its page is missing
  const int len0 = p.s.lens[b];
  const int len = len0 > cap ? (int)(cap + 1 < 0x7fffffff ? cap + 1 : 0x7fffffff) : len0 < 0 ? 0 : len0;
  const int first_pos = len0 - n;  // position of the first new token

  __shared__ float red_o[WKV == 1 ? 1 : 3 * 16 * NQ * D];
  __shared__ float red_ml[WKV == 1 ? 1 : 4 * 16 * NQ * 2];

  // the last tiles of columns have the most keys: first
  const int64_t qtiles = (cols + kCols - 1) / kCols;
  const int64_t gq = gridDim.x / p.splits;
  for (int64_t qi = blockIdx.x / p.splits; qi < qtiles; qi += gq) {
    const int64_t c0 = (qtiles - 1 - qi) * kCols + (WKV == 1 ? wave * 16 * NQ : 0);
    // per block of columns: the query's token and head, and the keys [klo, khi) that it sees
    int klo[NQ], khi[NQ];
    v4w qf[NQ][KS];
    float qs[NQ];
    int64_t row[NQ];
    int head[NQ];
    int lo = 0x7fffffff, hi = 0, lo_all = 0, hi_all = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int64_t c = c0 + 16 * j + col;
      const bool on = c < cols;
      const int64_t i = on ? c / p.G : 0;
      head[j] = h * p.G + (int)(on ? c - i * p.G : 0);
      row[j] = on ? start + i : -1;
      const int64_t pos = first_pos + i;
      const int64_t e = p.causal ? pos + 1 : len, a = p.window ? pos - p.window + 1 : 0;
      khi[j] = on ? (int)(e < 0 ? 0 : e < len ? e : len) : 0;
      klo[j] = (int)(a < 0 ? 0 : a < len ? a : len);
      if (on && klo[j] < khi[j]) {
        lo = klo[j] < lo ? klo[j] : lo;
        hi = khi[j] > hi ? khi[j] : hi;
      }
      if (on) {
        lo_all = klo[j] > lo_all ? klo[j] : lo_all;
        hi_all = khi[j] < hi_all ? khi[j] : hi_all;
      }
      const uint16_t* qp = p.q + (on ? start + i : start) * p.ldq + head[j] * p.hq + g * (D / 4);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const uint4 u = on ? *reinterpret_cast<const uint4*>(qp + 8 * w) : make_uint4(0, 0, 0, 0);
        // the codes' order: elements 0 4, 1 5, 2 6, 3 7
        qf[j][w][0] = (u.x & 0xffffu) | (u.z << 16);
        qf[j][w][1] = (u.x >> 16) | (u.z & 0xffff0000u);
        qf[j][w][2] = (u.y & 0xffffu) | (u.w << 16);
        qf[j][w][3] = (u.y >> 16) | (u.w & 0xffff0000u);
        const uint32_t x[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e2 = 0; e2 < 4; ++e2) sum += lo16<DT>(x[e2]) + hi16<DT>(x[e2]);
      }
      qs[j] = col_sum(sum);
    }
    // over the wave
#pragma unroll
    for (int s = 1; s < 16; s <<= 1) {
      lo = min(lo, __shfl_xor(lo, s));
      hi = max(hi, __shfl_xor(hi, s));
      lo_all = max(lo_all, __shfl_xor(lo_all, s));
      hi_all = min(hi_all, __shfl_xor(hi_all, s));
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    lo_all = __builtin_amdgcn_readfirstlane(lo_all);
    hi_all = __builtin_amdgcn_readfirstlane(hi_all);

    v4f o[NQ][DB];
    float m[NQ], l[NQ], cc[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      m[j] = -__builtin_inff();
      l[j] = cc[j] = 0.f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[j][d] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    const int t_first = lo < hi ? lo >> 5 : 0;
    const int nt = lo < hi ? ((hi + 31) >> 5) - t_first : 0;
    const int hop = (p.splits - 1) * p.ct;
    auto next = [&](int t) {
      t += WKV;
      return (t & (p.ct - 1)) < WKV ? t + hop : t;
    };
    int t = split * p.ct + (WKV == 1 ? 0 : wave);
    Tile<D> cur;
    Blocks at = {0, -1};
    if (t < nt) {
      at = find_blocks<D>(p, b, h, (int64_t)(t_first + t) * 32, hi, lane);
      load_tile<D>(p, at, lane, cur);
    }
    int tn = next(t);
    Blocks nat = {0, -1};
    if (tn < nt) nat = find_blocks<D>(p, b, h, (int64_t)(t_first + tn) * 32, hi, lane);
    while (t < nt) {
      const Tile<D> x = cur;
      const bool missing = at.g < 0;
      const int t0 = (t_first + t) * 32;
      at = nat;
      if (tn < nt) load_tile<D>(p, at, lane, cur);
      const int tnn = next(tn);
      if (tnn < nt) nat = find_blocks<D>(p, b, h, (int64_t)(t_first + tnn) * 32, hi, lane);

      v4f s[NQ][2];
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[j][0][r] = s[j][1][r] = -16.f * qs[j];
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const v4w a0 = widen<DT>(x.k[0][w]), a1 = widen<DT>(x.k[1][w]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          s[j][0] = mfma16<DT>(a0, qf[j][w], s[j][0]);
          s[j][1] = mfma16<DT>(a1, qf[j][w], s[j][1]);
        }
      }
      const int tb = t0 + 8 * g;  // this lane's first token
      const bool whole = t0 >= lo_all && t0 + 32 <= hi_all;
      v4w ph[NQ], pl[NQ];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float y[8], top = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = __builtin_fmaf(lo16<DT>(x.ks[i]), s[j][i >> 2][i & 3], hi16<DT>(x.ks[i]) * qs[j]) * p.scale;
          if (missing) y[i] = __builtin_nanf("");
          if (!whole && !(tb + i >= klo[j] && tb + i < khi[j])) y[i] = -__builtin_inff();
          top = fmaxf(top, y[i]);
        }
        if (__ballot(top > m[j] + 8.f)) {
          const float mn = fmaxf(m[j], col_max(top));
          const float f = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m[j] - mn);
          m[j] = mn;
          l[j] *= f;
          cc[j] *= f;
#pragma unroll
          for (int d = 0; d < DB; ++d) o[j][d] *= f;
        }
        const float mu = m[j] == -__builtin_inff() ? 0.f : m[j];
        float ps[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float pr = __builtin_amdgcn_exp2f(y[i] - mu);
          const float sv = lo16<DT>(x.vs[i]), mv = hi16<DT>(x.vs[i]);
          l[j] += pr;
          // an unseen token's scale may be anything: 0 times it is not 0
          const bool off = !whole && y[i] == -__builtin_inff();
          ps[i] = off ? 0.f : pr * sv;
          cc[j] = off ? cc[j] : __builtin_fmaf(pr, __builtin_fmaf(-16.f, sv, mv), cc[j]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ph[j][r] = pack_bf16(ps[r], ps[r + 4]);
          pl[j][r] = pack_bf16(ps[r] - __uint_as_float(ph[j][r] << 16), ps[r + 4] - __uint_as_float(ph[j][r] & 0xffff0000u));
        }
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const v4w a = widen<kBF16>(x.v[d]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          o[j][d] = mfma16<kBF16>(a, ph[j], o[j][d]);
          o[j][d] = mfma16<kBF16>(a, pl[j], o[j][d]);
        }
      }
      t = tn;
      tn = tnn;
    }

#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      l[j] = col_sum(l[j]);
      cc[j] = col_sum(cc[j]);
#pragma unroll
      for (int d = 0; d < DB; ++d) o[j][d] += cc[j];
    }
    if (WKV > 1) {
      // join the waves: all to the common maximum, waves 1 to 3 through LDS to wave 0
#pragma unroll
      for (int j = 0; j < NQ; ++j)
        if (g == 0) {
          red_ml[((wave * NQ + j) * 16 + col) * 2] = m[j];
          red_ml[((wave * NQ + j) * 16 + col) * 2 + 1] = l[j];
        }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float mn = -__builtin_inff(), sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) mn = fmaxf(mn, red_ml[((w * NQ + j) * 16 + col) * 2]);
        const float mu = mn == -__builtin_inff() ? 0.f : mn;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          sum += red_ml[((w * NQ + j) * 16 + col) * 2 + 1] * __builtin_amdgcn_exp2f(red_ml[((w * NQ + j) * 16 + col) * 2] - mu);
        const float f = __builtin_amdgcn_exp2f(m[j] - mu);
        m[j] = mn;
        l[j] = sum;
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          o[j][d] *= f;
          if (wave)
            *reinterpret_cast<v4f*>(&red_o[((((wave - 1) * NQ + j) * DB + d) * 64 + lane) * 4]) = o[j][d];
        }
      }
      __syncthreads();
      if (wave == 0)
#pragma unroll
        for (int j = 0; j < NQ; ++j)
#pragma unroll
          for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int w = 0; w < 3; ++w)
              o[j][d] += *reinterpret_cast<const v4f*>(&red_o[(((w * NQ + j) * DB + d) * 64 + lane) * 4]);
    }
    // lane: channels DB * 4 g + DB r + d of its column
    if (WKV == 1 || wave == 0)
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        if (row[j] < 0) continue;
        if (p.splits > 1) {
          const int64_t at_o = ((int64_t)split * p.s.T + row[j]) * Hq + head[j];
          float* op = p.po + at_o * D + g * (DB * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DB; d += 4)
              *reinterpret_cast<v4f*>(op + r * DB + d) = v4f{o[j][d][r], o[j][d + 1][r], o[j][d + 2][r], o[j][d + 3][r]};
          if (g == 0) {
            p.pml[at_o * 2] = m[j];
            p.pml[at_o * 2 + 1] = l[j];
          }
        } else {
          // no key seen: the sum is 0, the output 0
          const float inv = l[j] == 0.f ? 0.f : 1.f / l[j];
          uint16_t* op = p.out + row[j] * p.ldo + head[j] * p.ho + g * (DB * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int d = 0; d < DB; d += 4) {
              uint2 u;
              u.x = (uint32_t)to_dtype(o[j][d][r] * inv, DT) | ((uint32_t)to_dtype(o[j][d + 1][r] * inv, DT) << 16);
              u.y = (uint32_t)to_dtype(o[j][d + 2][r] * inv, DT) | ((uint32_t)to_dtype(o[j][d + 3][r] * inv, DT) << 16);
              *reinterpret_cast<uint2*>(op + r * DB + d) = u;
            }
          if (p.lse && g == 0)
            p.lse[row[j] * Hq + head[j]] = l[j] == 0.f ? -__builtin_inff() : m[j] * 0.69314718055994531f + logf(l[j]);
        }
      }
    if (WKV > 1) __syncthreads();  // before the next tile of columns writes LDS
  }
}

// The splits of one row and head: 64 lanes, D / 64 channels each, a wave per (row, head).
template <int D, int DT>
__global__ void __launch_bounds__(256)
kv4_join_kernel(const Kv4Attn p) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int Hq = p.c.H * p.G;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= p.s.T * Hq) return;
  const int64_t row = id / Hq, head = id - row * Hq, step = p.s.T * Hq;
  if (row >= p.s.cu[p.s.B] || row < p.s.cu[0]) return;  // rows of no sequence stay as they are
  float mn = -__builtin_inff();
  for (int s = 0; s < p.splits; ++s) mn = fmaxf(mn, p.pml[(s * step + id) * 2]);
  const float mu = mn == -__builtin_inff() ? 0.f : mn;
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int s = 0; s < p.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(p.pml[(s * step + id) * 2] - mu);
    l += f * p.pml[(s * step + id) * 2 + 1];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += f * p.po[(s * step + id) * D + lane * E + e];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* op = p.out + row * p.ldo + head * p.ho + lane * E;
#pragma unroll
  for (int e = 0; e < E; ++e) op[e] = to_dtype(o[e] * inv, DT);
  if (p.lse && lane == 0) p.lse[id] = l == 0.f ? -__builtin_inff() : mn * 0.69314718055994531f + logf(l);
}

Kv4Plan kv4_plan(int64_t T, int B, int H, int G, int D, int64_t max_q, int64_t max_kv) {
  Kv4Plan pl;
  const int64_t cols = max_q * G;
  const bool few = cols <= 16;
  pl.wkv = few ? 4 : 1;
  pl.nq = few || D == 256 ? 1 : 2;
  const int64_t per = few ? 16 : 64 * pl.nq;
  pl.qgrid = (cols + per - 1) / per;
  const int64_t tiles = (max_kv + 31) / 32;
  // enough workgroups for the card (256 CUs, several each), steps of at least 128 tokens
  int64_t want = 2048 / (pl.qgrid * H * B > 0 ? pl.qgrid * H * B : 1);
  if (!few && want > 8) want = 8;
  pl.ct = 4;
  while (pl.ct * want < tiles && pl.ct < 1024) pl.ct *= 2;
  pl.splits = (int)((tiles + pl.ct - 1) / pl.ct);
  if (pl.splits > want) pl.splits = (int)want;
  if (pl.splits < 1) pl.splits = 1;
  if (pl.splits > 64) pl.splits = 64;
  return pl;
}

int64_t kv4_workspace(int64_t T, int Hq, int D, int splits) {
  return splits <= 1 ? 0 : (int64_t)splits * T * Hq * (D + 2) * 4;
}

template <int D, int DT>
static int launch_dt(Kv4Attn& p, const Kv4Plan& pl, hipStream_t st) {
  const dim3 g((unsigned)(pl.qgrid * pl.splits), (unsigned)p.c.H, (unsigned)p.s.B), b(256);
  if (pl.wkv == 4) hipLaunchKernelGGL((kv4_attn_kernel<D, DT, 1, 4>), g, b, 0, st, p);
  else hipLaunchKernelGGL((kv4_attn_kernel<D, DT, D == 256 ? 1 : 2, 1>), g, b, 0, st, p);
  if (hipGetLastError() != hipSuccess) return kErrHip;
  if (pl.splits > 1) {
    const int64_t rows = p.s.T * p.c.H * p.G;
    hipLaunchKernelGGL((kv4_join_kernel<D, DT>), dim3((unsigned)((rows + 3) / 4)), b, 0, st, p);
  }
  return hipGetLastError() == hipSuccess ? kOk : kErrHip;
}

int launch_kv4_attention(Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, void* ws, hipStream_t st) {
  p.splits = pl.splits;
  p.ct = pl.ct;
  p.po = reinterpret_cast<float*>(ws);
  p.pml = p.po + (int64_t)pl.splits * p.s.T * p.c.H * p.G * D;
  if (dtype == kBF16)
    return D == 64 ? launch_dt<64, kBF16>(p, pl, st) : D == 128 ? launch_dt<128, kBF16>(p, pl, st) : launch_dt<256, kBF16>(p, pl, st);
  return D == 64 ? launch_dt<64, kF16>(p, pl, st) : D == 128 ? launch_dt<128, kF16>(p, pl, st) : launch_dt<256, kF16>(p, pl, st);
}

}  // namespace w4a8
