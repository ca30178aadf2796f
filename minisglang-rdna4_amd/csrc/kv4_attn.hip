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

typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2bf));
}

// D: channels; DT: the model's type; NQ: blocks of 16 columns per wave; WKV: 4 waves over the tokens, or 1:
// 4 waves over the columns
template <int D, int DT, int NQ, int WKV>
__global__ void __launch_bounds__(256, WKV == 1 ? 1 : D == 256 ? 2 : 3)
kv4_attn_kernel(const Kv4Attn p) {
  constexpr int KS = D / 32, DB = D / 16;  // products per S tile, blocks of 16 channels
  constexpr int kCols = 16 * NQ * (WKV == 1 ? 4 : 1);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int h = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % p.splits;
  const int Hq = p.c.H * p.G;
  int64_t start;
  int n;
  kv4_rows(p.s, b, start, n);
  const int cols = n * p.G;
  const int64_t cap = (int64_t)p.s.width << p.c.shift;
  // one token past the table's end stands for all of them: its page is missing
  const int len0 = p.s.lens[b];
  const int len = len0 > cap ? (int)(cap + 1 < 0x7fffffff ? cap + 1 : 0x7fffffff) : len0 < 0 ? 0 : len0;
  const int first_pos = len0 - n;  // position of the first new token

  const float slack = 8.f / p.scale;
  __shared__ float red_o[WKV == 1 ? 1 : 4 * 16 * D];
  __shared__ float red_ml[WKV == 1 ? 1 : 4 * 16 * 2];

  // the last tiles of columns have the most keys: first
  const int qtiles = (cols + kCols - 1) / kCols;
  const int gq = gridDim.x / p.splits;
  for (int qi = blockIdx.x / p.splits; qi < qtiles; qi += gq) {
    const int c0 = (qtiles - 1 - qi) * kCols + (WKV == 1 ? wave * 16 * NQ : 0);
    // Columns are queries in order, so the keys that all of them and that any of them sees, [lo_all, hi_all) and
    // [lo, hi), follow from the first and the last one.
    const int cend = c0 + 16 * NQ < cols ? c0 + 16 * NQ : cols;
    const int i0 = c0 / p.G, r0 = c0 - i0 * p.G, i1 = (cend - 1) / p.G;
    auto upto = [&](int i) { return p.causal ? min(max(first_pos + i + 1, 0), len) : len; };
    auto from = [&](int i) { return p.window ? min(max(first_pos + i - p.window + 1, 0), len) : 0; };
    const int lo = from(i0), lo_all = from(i1), hi_all = upto(i0), hi = c0 < cols ? upto(i1) : 0;
    const int t_first = lo < hi ? lo >> 5 : 0;
    const int nt = lo < hi ? ((hi + 31) >> 5) - t_first : 0;
    const int hop = (p.splits - 1) * p.ct;
    auto next = [&](int t) {
      t += WKV;
      return (t & (p.ct - 1)) < WKV ? t + hop : t;
    };
    const Table table = (Table)(uintptr_t)(p.s.table + b * p.s.ldt);
    // Each part of the next tile is loaded into the registers of this one's as soon as they are free.
    uint32_t kw[2][KS], vw[DB], ksw[8], vsw[8];
    auto load_k = [&](const Pages& pg, int t) {
      const uint8_t* kp = p.c.k + (uint64_t)pick(p, pg, h, t, (lane & 15) >> 2) * (4 * D) + ((lane & 3) * (D / 2) + g * (D / 8));
      load_words(kp, kw[0]);
      load_words(kp + 4 * (D / 2), kw[1]);
    };
    auto load_v = [&](const Pages& pg, int t) {
      load_words(p.c.v + (uint64_t)pick(p, pg, h, t, g) * (4 * D) + (lane & 15) * (D / 4), vw);
    };
    auto load_s = [&](const Pages& pg, int t) {
      const uint64_t o = (uint64_t)pick(p, pg, h, t, g) * 32;
      load_words(reinterpret_cast<const uint8_t*>(p.c.ks) + o, ksw);
      load_words(reinterpret_cast<const uint8_t*>(p.c.vs) + o, vsw);
    };
    int t = split * p.ct + (WKV == 1 ? 0 : wave);
    int tn = next(t);
    auto token = [&](int t) { return (t_first + t) * 32; };
    Pages at = {-1, -1}, nat = {-1, -1};
    if (t < nt) at = look_up(p, table, token(t), hi);
    if (tn < nt) nat = look_up(p, table, token(tn), hi);

    // this lane's query of column 16 j + col
    auto query = [&](int j, int& head) {
      const int x = r0 + 16 * j + col, i = (int)__umulhi((uint32_t)x << 1, p.gmul);
      head = h * p.G + x - i * p.G;
      return i0 + i;
    };
    uint4 qr[NQ][KS];
    int klo[NQ], khi[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      int head;
      const int i = query(j, head);
      const bool on = c0 + 16 * j + col < cols;
      khi[j] = on ? upto(i) : 0;
      klo[j] = from(i);
      const uint16_t* qp = p.q + (start + (on ? i : 0)) * p.ldq + (on ? head : 0) * p.hq + g * (D / 4);
#pragma unroll
      for (int w = 0; w < KS; ++w) qr[j][w] = on ? *reinterpret_cast<const uint4*>(qp + 8 * w) : make_uint4(0, 0, 0, 0);
    }
    if (t < nt) {
      load_k(at, token(t));
      load_s(at, token(t));
      load_v(at, token(t));
    }
    v4w qf[NQ][KS];
    float qs[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const uint4 u = qr[j][w];
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

    v4f o[NQ][DB];
    float m[NQ], mu[NQ], l[NQ], cc[NQ];  // mu: m in powers of two, 0 while no key was seen
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      m[j] = -__builtin_inff();
      mu[j] = l[j] = cc[j] = 0.f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[j][d] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    while (t < nt) {
      const int t0 = token(t);
      const int tnn = next(tn);
      Pages nnat = {-1, -1};
      if (tnn < nt) nnat = look_up(p, table, token(tnn), hi);

      v4f s[NQ][2];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        const float q16 = -16.f * qs[j];
        s[j][0] = s[j][1] = v4f{q16, q16, q16, q16};
      }
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const v4w a0 = widen<DT>(kw[0][w]), a1 = widen<DT>(kw[1][w]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          s[j][0] = mfma16<DT>(a0, qf[j][w], s[j][0]);
          s[j][1] = mfma16<DT>(a1, qf[j][w], s[j][1]);
        }
      }
      if (tn < nt) load_k(nat, token(tn));

      const bool whole = t0 >= lo_all && t0 + 32 <= hi_all && exists(p, at.a) && exists(p, at.b);
      v4w ph[NQ], pl[NQ];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float y[8], sv[8], mv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          y[i] = __builtin_fmaf(lo16<DT>(ksw[i]), s[j][i >> 2][i & 3], hi16<DT>(ksw[i]) * qs[j]);
          sv[i] = lo16<DT>(vsw[i]);
          mv[i] = __builtin_fmaf(-16.f, sv[i], hi16<DT>(vsw[i]));
        }
        if (!whole) {
          // an unseen token's scale may be anything, and 0 times it is not 0; a missing page is NaN to whoever sees it
          const int a = klo[j] - (t0 + 8 * g), e = khi[j] - (t0 + 8 * g);
          const bool missing = !exists(p, g < 2 ? at.a : at.b);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool see = i >= a && i < e;
            y[i] = !see ? -__builtin_inff() : missing ? __builtin_nanf("") : y[i];
            sv[i] = see ? sv[i] : 0.f;
            mv[i] = see ? mv[i] : 0.f;
          }
        }
        const float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
        if (__ballot(top > m[j] + slack)) {
          const float mn = fmaxf(m[j], col_max(top));
          const float f = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m[j] - mn) * p.scale);
          m[j] = mn;
          mu[j] = mn == -__builtin_inff() ? 0.f : mn * p.scale;
          l[j] *= f;
          cc[j] *= f;
#pragma unroll
          for (int d = 0; d < DB; ++d) o[j][d] *= f;
        }
        float ps[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(y[i], p.scale, -mu[j]));
          l[j] += pr;
          ps[i] = pr * sv[i];
          cc[j] = __builtin_fmaf(pr, mv[i], cc[j]);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ph[j][r] = pack_bf16(ps[r], ps[r + 4]);
          pl[j][r] = pack_bf16(ps[r] - __uint_as_float(ph[j][r] << 16), ps[r + 4] - __uint_as_float(ph[j][r] & 0xffff0000u));
        }
      }
      if (tn < nt) load_s(nat, token(tn));
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const v4w a = widen<kBF16>(vw[d]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          o[j][d] = mfma16<kBF16>(a, ph[j], o[j][d]);
          o[j][d] = mfma16<kBF16>(a, pl[j], o[j][d]);
        }
      }
      if (tn < nt) load_v(nat, token(tn));
      at = nat;
      nat = nnat;
      t = tn;
      tn = tnn;
    }

#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      m[j] *= p.scale;
      l[j] = col_sum(l[j]);
      cc[j] = col_sum(cc[j]);
#pragma unroll
      for (int d = 0; d < DB; ++d) o[j][d] += cc[j];
    }
    // a lane's channels: DB (4 g + r) + d of its column, r = 0..3
    auto store = [&](int j, int r, const float (&v)[DB], float mx, float sum) {
      if (c0 + 16 * j + col >= cols) return;
      int head;
      const int64_t row = start + query(j, head);
      const bool first = g == 0 && r == 0;
      if (p.splits > 1) {
        const int64_t at_o = ((int64_t)split * p.s.T + row) * Hq + head;
        float* op = p.po + at_o * D + (4 * g + r) * DB;
#pragma unroll
        for (int d = 0; d < DB; d += 4) *reinterpret_cast<v4f*>(op + d) = v4f{v[d], v[d + 1], v[d + 2], v[d + 3]};
        if (first) {
          p.pml[at_o * 2] = mx;
          p.pml[at_o * 2 + 1] = sum;
        }
      } else {
        // no key seen: the sum is 0, the output 0
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        uint16_t* op = p.out + row * p.ldo + head * p.ho + (4 * g + r) * DB;
#pragma unroll
        for (int d = 0; d < DB; d += 4) {
          uint2 u;
          u.x = (uint32_t)to_dtype(v[d] * inv, DT) | ((uint32_t)to_dtype(v[d + 1] * inv, DT) << 16);
          u.y = (uint32_t)to_dtype(v[d + 2] * inv, DT) | ((uint32_t)to_dtype(v[d + 3] * inv, DT) << 16);
          *reinterpret_cast<uint2*>(op + d) = u;
        }
        if (p.lse && first) p.lse[row * Hq + head] = sum == 0.f ? -__builtin_inff() : mx * 0.69314718055994531f + logf(sum);
      }
    };
    if constexpr (WKV == 1) {
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[DB];
#pragma unroll
          for (int d = 0; d < DB; ++d) v[d] = o[j][d][r];
          store(j, r, v, m[j], l[j]);
        }
    } else {
      // join the waves through LDS, each to the common maximum; wave r then sums and writes the channels of r
      static_assert(NQ == 1, "one block of columns");
      if (g == 0) {
        red_ml[(wave * 16 + col) * 2] = m[0];
        red_ml[(wave * 16 + col) * 2 + 1] = l[0];
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) *reinterpret_cast<v4f*>(&red_o[((wave * DB + d) * 64 + lane) * 4]) = o[0][d];
      __syncthreads();
      float mw[4], mx = -__builtin_inff(), sum = 0.f, v[DB];
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, mw[w] = red_ml[(w * 16 + col) * 2]);
#pragma unroll
      for (int d = 0; d < DB; ++d) v[d] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = mx == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(mw[w] - mx);
        sum += f * red_ml[(w * 16 + col) * 2 + 1];
#pragma unroll
        for (int d = 0; d < DB; ++d) v[d] += f * red_o[((w * DB + d) * 64 + lane) * 4 + wave];
      }
      store(0, wave, v, mx, sum);
      __syncthreads();  // before the next tile of columns writes LDS
    }
  }
}

// The splits of one row and head: a wave, first a lane per split (at most 64) for the maxima and sums, then
// D / 64 channels per lane. Splits that saw no key are not read.
template <int D, int DT>
__global__ void __launch_bounds__(256)
kv4_join_kernel(const Kv4Attn p) {
  constexpr int E = D / 64;
  const int lane = threadIdx.x & 63;
  const int Hq = p.c.H * p.G;
  const int rows = (int)p.s.T * Hq;
  const int id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (id >= rows) return;
  const int row = id / Hq, head = id - row * Hq;
  if (row >= p.s.cu[p.s.B] || row < p.s.cu[0]) return;  // rows of no sequence stay as they are
  float ms = -__builtin_inff(), ls = 0.f;
  if (lane < p.splits) {
    const v2f ml = *reinterpret_cast<const v2f*>(p.pml + ((int64_t)lane * rows + id) * 2);
    ms = ml.x;
    ls = ml.y;
  }
  const float mn = wave_max(ms);
  const float f = mn == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(ms - mn);
  const float l = wave_sum(ls == 0.f ? 0.f : ls * f);
  uint64_t todo = __ballot(!(ls == 0.f));
  float o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  const float* po = p.po + (int64_t)id * D + lane * E;
  while (todo) {
    // four at a time, all loaded before the first is used
    float v[4][E], w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = todo ? __builtin_ctzll(todo) : 0;
      w[u] = todo ? lane_f(f, s) : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) v[u][e] = todo ? po[(int64_t)s * rows * D + e] : 0.f;
      todo &= todo - 1;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(w[u], v[u][e], o[e]);
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
