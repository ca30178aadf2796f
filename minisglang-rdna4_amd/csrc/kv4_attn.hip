// Attention over the paged 4-bit cache (layout: kv4.h), for decode and for prompts.
//
// Per key/value head, the queries that share it are the columns of the matrix products: column c is
// query c / G, query head h * G + c % G. A wave takes 16 NQ columns and walks tiles of 32 tokens, with
// one pass over the cache and the running maximum and sum of the softmax in f32:
//   S = c Q^T,   x = s S + m sum(q),   p = 2^(x scale - M),   O += (p s)^T c,   C += p m,   out = (O + C) / sum p.
// Codes. A code in bits 2 .. 5 of an fp16 number is the subnormal c 2^-22, in bits 6 .. 9 c 2^-18: two shifts
// and four ands turn the 8 codes of a word into an fp16 operand, with no offset and no rounding (the matrix
// units keep subnormals). The other operand carries the 2^-4 of the higher codes, the sums the 2^22.
// The matrix units line a subnormal's products up by the exponent of the least normal number, and cut what is then
// below f32's last place of the largest: a code in the lowest bits, one shift less, loses 7 bits and more. Sums
// over weights exp(1.5 N(0, 1)) then came out low by 22 units in the last place, and come out low by 2 (by 0.01 with
// all codes in bits 6 .. 9, which takes four shifts), where outputs of long contexts are a hundredth of what is summed.
// Queries enter in fp16 for either model type: a power of two per row puts their largest value at 2^14, so
// values down to 2^-27 of it (bf16 models) or 2^-24 (fp16) are exact.
// p s enters in fp16, w: for fp16 models as two terms (22 bits), for bf16 models as one, rounded by at most 2^-11 of
// itself. So that errors meet c - 7.5, and not the whole of c, what is summed is
// O - 7.5 sum w + sum p (m + 7.5 s), sum w by one more product with a row of ones: bf16 models' error is within 2^-11
// of half a V vector's range, an eighth of the output's own rounding. A wave subtracts 7.5 sum w from O every kFresh
// tiles, since f32 sums of uncentred codes lose what the output is made of: one wave over 131072 tokens was off by
// 2.7e-3 of the output's norm (D = 64, equal weights, fp16), where the rounding is 2.3e-4. So that p s stays in fp16's
// range whatever V's steps are, p carries 2^-e, 2^e about the largest step so far over 64: it moves with the running
// maximum, column by column, and drops out of the quotient.
// The row of S that a lane of group g = lane / 16 holds is chosen to be the token whose V codes that
// lane holds (tokens 8 g + r in the first 16 rows' register r, 8 g + 4 + r in the second's), so p goes
// from one product into the next in its lane, and nothing passes through LDS.
// The running maximum is raised only when a score passes it by 8 (in powers of two): p stays below 2^8,
// and most tiles need no exchange between lanes and no rescaling. M is x's rounded to f32, the same for every p of
// the column and for its join with other waves, so the rounding drops out as long as it is within 1: to 2^24. From
// there on (far_off) every tile passes the check, and the maximum is subtracted there, before the scale is applied.
//
// WKV = 4 (decode): the waves of a workgroup walk the same 16 columns over different tiles and join through
// LDS. WKV = 1 (more than 16 columns): each wave has columns of its own; the waves read the same tiles at about
// the same time, and share them in the caches. Where that leaves the card empty the grid splits the tokens
// too, and kv4_join_kernel joins the parts.
//
// Measured. Decode is bound by HBM: two sequences of 131072 tokens x 8 heads of 128 (280 MB) 64 us, 4.4 TB/s, with
// cold caches, at 3 waves per SIMD (warm 59; at 4 waves, whose 128 registers spill, 87). Prompts by the vector unit:
// 8192 + 5690 + 3190 tokens, 32 heads of 128 (898 GFLOP) 1.56 ms, 574 TFLOP/s: 354 vector instructions a tile and
// wave, 96 of them to widen codes and 180 for the softmax of 32 columns, beside 34 MFMA of 16 cycles; 2 waves per
// SIMD (16 columns a wave, 3 waves: 1.66 ms). Of that, codes in bits 2 and up instead of 0 and up take 2%, and so does
// centring O every 32 tiles (every 8: 3%); fp16 models' sum w takes a tenth of their 150 us for chunks at 64 channels.
#include "kv4.h"

namespace w4a8 {

int launch_kv4_tree_attn(const Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, hipStream_t st);

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v4f mfma16(const v4w& a, const v4w& b, const v4f& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

// The codes of a word as fp16 subnormals: register r holds codes r and r + 4, times 2^-22 for even r, 2^-18 for odd
__device__ __forceinline__ v4w widen(uint32_t w) {
  const uint32_t u = w << 2, x = w >> 6;
  return v4w{u & 0x003c003cu, u & 0x03c003c0u, x & 0x003c003cu, x & 0x03c003c0u};
}
constexpr int kUnit = 22;          // sums of codes are in 2^-kUnit
constexpr float kOne = 4194304.f;  // 2^kUnit
constexpr int kFresh = 32;         // tiles that a wave sums before it takes the codes' mean out

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

// The page numbers of a tile, wave-uniform: those of its tokens 0..15 and 16..31 (a page holds at least 16), as
// the table has them, -1 past its end. Looked up a tile before they are used: the scalar loads then have
// nobody waiting. (Nothing writes the table during a launch: constant address space.)
typedef const int32_t __attribute__((address_space(4))) * Table;
struct Pages {
  int a, b;
};
__device__ __forceinline__ Pages look_up(const Kv4Attn& p, Table table, int t, int len) {
  const int i = t >> p.c.shift;
  Pages r;
  r.a = r.b = i < p.s.width ? table[i] : -1;
  // a tile of longer pages lies in one; slots past the sequence's end may be read there, not used
  if (p.c.shift == 4) r.b = t + 16 < len && i + 1 < p.s.width ? table[i + 1] : -1;
  return r;
}
// The tile's blocks: of tokens 0..15 and of 16..31, each with the next one. A missing page reads block 0, which is
// there, and its values are not used.
struct Blocks {
  uint32_t a, b;
  bool has_a, has_b;
};
__device__ __forceinline__ Blocks blocks_of(const Kv4Attn& p, const Pages& pg, int h, int t) {
  Blocks r;
  r.has_a = (uint32_t)pg.a < (uint32_t)p.c.pages;
  r.has_b = (uint32_t)pg.b < (uint32_t)p.c.pages;
  r.a = r.has_a ? (uint32_t)kv4_block(p.c, pg.a, h, t) : 0;
  r.b = r.has_b ? (p.c.shift == 4 ? (uint32_t)kv4_block(p.c, pg.b, h, t + 16) : r.a + 2) : 0;
  return r;
}
// block `i` of 4 of the tile: this lane's
// (values, not b's members: a choice of members is one of addresses, which the compiler would make in LDS)
__device__ __forceinline__ uint32_t pick(const Blocks& b, int i) {
  const uint32_t x = b.a, y = b.b;
  return (i < 2 ? x : y) + (i & 1);
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
__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2h));
}

// the keys [from, upto) that query i of the span sees: a window past the table's end still has the missing token
__device__ __forceinline__ int seen_from(const Kv4Attn& p, const Span& s, int i) {
  const int n = s.first_pos + i + 1;  // keys up to the query's own
  return p.window && n > p.window ? min(n - p.window, s.len - 1) : 0;
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

// over the wave
__device__ __forceinline__ int wave_min_i(int v) {
  v = min(v, dpp_i<kDppXor1>(v));
  v = min(v, dpp_i<kDppXor2>(v));
  v = min(v, dpp_i<kDppHalfMirror>(v));
  v = min(v, dpp_i<kDppRowMirror>(v));
  return min(min(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
             min(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}

// the maximum m itself where m times its factor is past what M holds to within 1, else 0
__device__ __forceinline__ float far_off(float m, float sc) {
  return fabsf(m) * sc >= 16777216.f && m != -__builtin_inff() ? m : 0.f;
}

template <int DT>
__device__ __forceinline__ void unpack_query(const uint4& u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = lo16<DT>(w[i]);
    f[2 * i + 1] = hi16<DT>(w[i]);
  }
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

// D: channels; DT: the model's type; NQ: blocks of 16 columns per wave; WKV: waves of a workgroup that share
// their columns; TREE: new tokens are seen as the bits tell, and not up to the query's own
template <int D, int DT, int NQ, int WKV, bool TREE>
__global__ void __launch_bounds__(256, D == 256 || (NQ == 2 && D == 128) ? 2 : 3)
kv4_attn_kernel(const Kv4Attn p) {
  static_assert(WKV == 1 || (WKV == 4 && NQ == 1), "side by side, or one block of columns");
  constexpr int KS = D / 32, DB = D / 16;  // products per S tile, blocks of 16 channels
  constexpr int W = DT == kF16 ? 2 : 1;    // fp16 terms of p s
  constexpr int kCols = 16 * NQ * (WKV == 1 ? 4 : 1);
  constexpr float kInf = __builtin_inff();
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int h = blockIdx.y, b = TREE ? kv4_longest(p.s, blockIdx.z) : (int)blockIdx.z;
  const int split = blockIdx.x % p.splits;
  const Span sp = kv4_span<TREE>(p, b);
  const Table table = (Table)(uintptr_t)(p.s.table + b * p.s.ldt);
  __shared__ float red_o[WKV == 1 ? 1 : 4 * 16 * D];
  __shared__ float red_ml[WKV == 1 ? 1 : 4 * 16 * 2];

  const int qtiles = (sp.cols + kCols - 1) / kCols;
  const int gq = gridDim.x / p.splits;
  for (int qi = blockIdx.x / p.splits; qi < qtiles; qi += gq) {
    // the last columns have the most keys: first
    const int c0 = (qtiles - 1 - qi) * kCols + (WKV == 1 ? wave * 16 * NQ : 0);
    Keys ks = kv4_keys(p, sp, c0, min(c0 + 16 * NQ, sp.cols));
    // this lane's queries: columns 16 j + col
    const int i0 = c0 / p.G, r0 = c0 - i0 * p.G;
    int tree_lo[NQ];
    if constexpr (TREE) {
      // the cached keys come before the new ones; which of those a query sees, its bits tell
      const int first = min(max(sp.first_pos, 0), sp.len);
      int lo = first, lo_all = 0;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        int head;
        const int i = kv4_query(p, i0, r0, 16 * j + col, head);
        const bool on = c0 + 16 * j + col < sp.cols;
        tree_lo[j] = on ? tree_from(p, sp, i) : first;
        lo = min(lo, tree_lo[j]);
        lo_all = max(lo_all, on ? tree_lo[j] : 0);
      }
      ks.lo = wave_min_i(lo);
      ks.lo_all = -wave_min_i(-lo_all);
      ks.hi = c0 < sp.cols ? sp.len : ks.lo;
      ks.hi_all = first;
    }
    const int t_first = ks.lo >> 5, nt = ks.lo < ks.hi ? ((ks.hi + 31) >> 5) - t_first : 0;
    auto token = [&](int t) { return (t_first + t) * 32; };
    // Each part of the next tile is loaded into the registers of this one's as soon as they are free.
    uint32_t kw[2][KS], vw[DB], ksw[8], vsw[8];
    auto load_k = [&](const Blocks& bl) {
      const uint8_t* kp = p.c.k + (uint64_t)pick(bl, (lane & 15) >> 2) * (4 * D) + ((lane & 3) * (D / 2) + g * (D / 8));
      load_words(kp, kw[0]);
      load_words(kp + 4 * (D / 2), kw[1]);
    };
    auto load_v = [&](const Blocks& bl) { load_words(p.c.v + (uint64_t)pick(bl, g) * (4 * D) + (lane & 15) * (D / 4), vw); };
    auto load_s = [&](const Blocks& bl) {
      const uint64_t o = (uint64_t)pick(bl, g) * 32;
      load_words(reinterpret_cast<const uint8_t*>(p.c.ks) + o, ksw);
      load_words(reinterpret_cast<const uint8_t*>(p.c.vs) + o, vsw);
    };
    // tiles are dealt out one by one, over the splits and their waves: all have the same share of a sequence
    const int step = p.splits * WKV;
    int t = split * WKV + (WKV == 1 ? 0 : wave);
    int tn = t + step;
    Pages first = {-1, -1}, nat = {-1, -1};
    if (t < nt) first = look_up(p, table, token(t), ks.hi);
    if (tn < nt) nat = look_up(p, table, token(tn), ks.hi);

    uint4 qr[NQ][KS];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      int head;
      const int i = kv4_query(p, i0, r0, 16 * j + col, head);
      const bool on = c0 + 16 * j + col < sp.cols;
      const uint16_t* qp = p.q + (sp.start + (on ? i : 0)) * p.ldq + (h * p.G + (on ? head : 0)) * p.hq + g * (D / 4);
#pragma unroll
      for (int w = 0; w < KS; ++w) qr[j][w] = on ? *reinterpret_cast<const uint4*>(qp + 8 * w) : make_uint4(0, 0, 0, 0);
    }
    Blocks at = blocks_of(p, first, h, token(t));
    if (t < nt) {
      load_k(at);
      load_s(at);
      load_v(at);
    }
    v4w qf[NQ][KS];
    float qs[NQ], sc[NQ];  // sum(q) and x's factor, in the products' units
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      float sum = 0.f, top = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        float f[8];
        unpack_query<DT>(qr[j][w], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += f[e];
          top = fmaxf(top, fabsf(f[e]));
        }
      }
      top = col_max(top);
      // 2^eq puts the largest value into [2^14, 2^15), where that is above 2^-106: below it, and for scales that small,
      // scores are zero for any keys, and x's factor has to have a reciprocal and to leave -inf what it is
      const int eq = min(max(141 - (int)(__float_as_uint(top) >> 23), -100), 120);
      qs[j] = __builtin_ldexpf(col_sum(sum), eq - kUnit);
      sc[j] = fmaxf(__builtin_ldexpf(p.scale, kUnit - eq), 0x1p-120f);
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        float f[8];
        unpack_query<DT>(qr[j][w], f);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int er = r & 1 ? eq - 4 : eq;
          qf[j][w][r] = pack_f16(__builtin_ldexpf(f[r], er), __builtin_ldexpf(f[r + 4], er));
        }
      }
    }

    v4f o[NQ][DB], ws[NQ];                // ws: sum w since O was last centred, in every register
    float thr[NQ];                        // scores up to here leave the maximum as it is: m and 8 powers of two, or none
    float m[NQ], mu[NQ], l[NQ], cc[NQ];   // mu: M, the maximum in powers of two (0 while no key was seen, or far_off) plus e
    float lim[NQ];                        // 2^(e + 6): steps up to here are in its range; 0: none was seen yet
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      lim[j] = 0.f;
      m[j] = thr[j] = -kInf;
      mu[j] = l[j] = cc[j] = 0.f;
      ws[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DB; ++d) o[j][d] = v4f{0.f, 0.f, 0.f, 0.f};
    }

    int fresh = kFresh;
    while (t < nt) {
      const int t0 = token(t);
      const int tnn = tn + step;
      const bool more = tn < nt;
      const Blocks next = blocks_of(p, nat, h, token(tn));
      if (tnn < nt) nat = look_up(p, table, token(tnn), ks.hi);

      v4f s[NQ][2];
#pragma unroll
      for (int j = 0; j < NQ; ++j) s[j][0] = s[j][1] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < KS; ++w)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const v4w a = widen(kw[z][w]);
#pragma unroll
          for (int j = 0; j < NQ; ++j) s[j][z] = mfma16(a, qf[j][w], s[j][z]);
        }
      if (more) load_k(next);

      float y[NQ][8], sv[8], mv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float sk = lo16<DT>(ksw[i]), mk = hi16<DT>(ksw[i]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) y[j][i] = __builtin_fmaf(sk, s[j][i >> 2][i & 3], mk * qs[j]);
        sv[i] = lo16<DT>(vsw[i]);
        mv[i] = __builtin_fmaf(7.5f, sv[i], hi16<DT>(vsw[i]));
      }
      auto top8 = [](const float (&v)[8]) {
        return fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), fmaxf(fmaxf(v[4], v[5]), fmaxf(v[6], v[7])));
      };
      float ts[NQ];  // the largest V step that the column sees
#pragma unroll
      for (int j = 0; j < NQ; ++j) ts[j] = top8(sv);
      if (!(t0 >= ks.lo_all && t0 + 32 <= ks.hi_all && at.has_a && at.has_b)) {
        // An unseen token's scale may be anything, and 0 times it is not 0: what is not finite, and a missing page,
        // is NaN in the score of whoever sees it, and 0 here.
        const bool ha = at.has_a, hb = at.has_b, missing = !(g < 2 ? ha : hb);
        int klo[NQ], khi[NQ];  // the column's keys, from this lane's first token
        uint32_t tree[NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          int head;
          const int i = kv4_query(p, i0, r0, 16 * j + col, head);
          const bool on = c0 + 16 * j + col < sp.cols;
          if constexpr (TREE) {
            klo[j] = tree_lo[j] - (t0 + 8 * g);
            khi[j] = (on ? ks.hi_all : 0) - (t0 + 8 * g);
            tree[j] = on ? tree_bits(p, sp, i, t0 + 8 * g - sp.first_pos) : 0;
          } else {
            khi[j] = (on ? seen_upto(p, sp, i) : 0) - (t0 + 8 * g);
            klo[j] = seen_from(p, sp, i) - (t0 + 8 * g);
          }
          ts[j] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool bad = missing || !__builtin_isfinite(sv[i]) || !__builtin_isfinite(mv[i]);
          sv[i] = bad ? 0.f : sv[i];
          mv[i] = bad ? 0.f : mv[i];
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            const bool see = (i >= klo[j] && i < khi[j]) || (TREE && (tree[j] >> i & 1));
            y[j][i] = see ? (bad ? __builtin_nanf("") : y[j][i]) : -kInf;
            ts[j] = see ? fmaxf(ts[j], sv[i]) : ts[j];
          }
        }
      }
      float top[NQ];
      bool up = false;
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        top[j] = top8(y[j]);
        up = up || top[j] > thr[j] || ts[j] > lim[j];
      }
      if (__ballot(up)) {
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          // a column that has no need keeps its bits, whatever its neighbours do
          const float tt = col_max(ts[j]), tp = col_max(top[j]);
          const bool need = tp > thr[j] || tt > lim[j];
          // 2^-e takes the column's largest step to [2^5, 2^6); steps that 2^-40 bounds stay below
          const int old = (int)(__float_as_uint(lim[j]) >> 23), le = (int)((__float_as_uint(tt) >> 23) & 255u) + 1;
          const int nl = need ? min(max(max(le, old), 87), 227) : old;  // lim's exponent
          lim[j] = __uint_as_float((uint32_t)nl << 23);
          const float mn = need ? fmaxf(m[j], tp) : m[j];
          const float was = far_off(m[j], sc[j]), is = far_off(mn, sc[j]);
          const float mun = need ? (mn == -kInf || is != 0.f ? 0.f : mn * sc[j]) + (float)(nl - 133) : mu[j];
          // nothing summed yet: any
          const float f = m[j] == -kInf ? 1.f : __builtin_amdgcn_exp2f(__builtin_fmaf(was - is, sc[j], mu[j] - mun));
          m[j] = mn;
          mu[j] = mun;
          thr[j] = is != 0.f ? -kInf : mn + 8.f / sc[j];
          l[j] *= f;
          cc[j] *= f;
          ws[j] *= f;
#pragma unroll
          for (int d = 0; d < DB; ++d) o[j][d] *= f;
#pragma unroll
          for (int i = 0; i < 8; ++i) y[j][i] -= is;
        }
      }
#pragma unroll
      for (int i = 1; i < 8; i += 2) sv[i] *= 0.0625f;  // the higher codes
      v4w ph[NQ], pl[NQ];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float ps[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(y[j][i], sc[j], -mu[j]));
          l[j] += pr;
          cc[j] = __builtin_fmaf(pr, mv[i], cc[j]);
          ps[i] = pr * sv[i];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          ph[j][r] = pack_f16(ps[r], ps[r + 4]);
          if (W == 2)
            pl[j][r] = pack_f16(ps[r] - f16_to_f32((uint16_t)(ph[j][r] & 0xffffu)), ps[r + 4] - f16_to_f32((uint16_t)(ph[j][r] >> 16)));
        }
        // sum w: ones, sixteens against the higher codes' 1/16
        const v4w ones = {0x3c003c00u, 0x4c004c00u, 0x3c003c00u, 0x4c004c00u};
        ws[j] = mfma16(ones, ph[j], ws[j]);
        if (W == 2) ws[j] = mfma16(ones, pl[j], ws[j]);
      }
      if (more) load_s(next);
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const v4w a = widen(vw[d]);
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          o[j][d] = mfma16(a, ph[j], o[j][d]);
          if (W == 2) o[j][d] = mfma16(a, pl[j], o[j][d]);
        }
      }
      if (more) load_v(next);
      if (--fresh == 0) {
        fresh = kFresh;
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
#pragma unroll
          for (int d = 0; d < DB; ++d) o[j][d] -= (7.5f / kOne) * ws[j];
          ws[j] = v4f{0.f, 0.f, 0.f, 0.f};
        }
      }
      at = next;
      t = tn;
      tn = tnn;
    }

    // O in the codes' units is kOne times the products' sum
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      l[j] = col_sum(l[j]);
      cc[j] = col_sum(cc[j]) - 7.5f * ws[j][0];
      // beside a far_off maximum e would be lost: it goes into the sums
      const float is = far_off(m[j], sc[j]), fe = is != 0.f ? __builtin_amdgcn_exp2f(mu[j]) : 1.f;
      mu[j] = m[j] == -kInf ? -kInf : is != 0.f ? is * sc[j] : mu[j];
      l[j] *= fe;
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[j][d][r] = fe * __builtin_fmaf(o[j][d][r], kOne, cc[j]);
    }
    auto store = [&](int j, int r, const float (&v)[DB], float mx, float sum) {
      int head;
      const int i = kv4_query(p, i0, r0, 16 * j + col, head);
      // a lane's channels: DB (4 g + r) + d of its column
      if (c0 + 16 * j + col < sp.cols)
        kv4_store<D, DT>(p, split, sp.start + i, h * p.G + head, (4 * g + r) * DB, v, mx, sum, g == 0 && r == 0);
    };
    if constexpr (WKV == 1) {
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[DB];
#pragma unroll
          for (int d = 0; d < DB; ++d) v[d] = o[j][d][r];
          store(j, r, v, mu[j], l[j]);
        }
    } else {
      // join the waves through LDS, each to the common maximum; wave r then sums and writes the channels of r
      if (g == 0) {
        red_ml[(wave * 16 + col) * 2] = mu[0];
        red_ml[(wave * 16 + col) * 2 + 1] = l[0];
      }
#pragma unroll
      for (int d = 0; d < DB; ++d) *reinterpret_cast<v4f*>(&red_o[((wave * DB + d) * 64 + lane) * 4]) = o[0][d];
      __syncthreads();
      float mw[4], mx = -kInf, sum = 0.f, v[DB];
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, mw[w] = red_ml[(w * 16 + col) * 2]);
#pragma unroll
      for (int d = 0; d < DB; ++d) v[d] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = mx == -kInf ? 0.f : __builtin_amdgcn_exp2f(mw[w] - mx);
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
  if (p.lse && lane == 0) p.lse[id] = l == 0.f ? -__builtin_inff() : mn * 0.69314718055994531f + logf(l) + p.lse_more;
}

// Splits of the tokens. Decode (3 workgroups of 4 waves per CU, 768 on the card): one round of the card, and up to
// four per sequence and head where that many more workgroups even out sequences of different lengths; a split has
// 8 tiles, two for each wave, and the first 8 are not worth the join's launch. us, with the splits that
// this gives / without: 64 sequences of up to 8192 tokens x 8 heads 76 / 84, 16 of 4000 22 / 39, one of 8000
// 14 / 62, two of 131072 59 / 1050; 48 of 500 12 (unsplit) / 15 in two. No more than 16 splits, or one per 64 tiles,
// up to the 64 that kv4_join_kernel has lanes for: the join's time grows with them, which short contexts do not earn
// back. us, at most 16 / this / at most 64, one sequence on 8 heads: 8192 tokens 13.7 / 13.7 / 15.0, 32768
// 27.6 / 28.0 / 24.3, 131072 78 / 39.7 / 39.5; on one head 8192 13.4 / 13.1 / 14.0, 32768 25.1 / 25.2 / 20.3, 131072
// 72 / 32 / 32.
// More columns (2 workgroups of 32-column waves per CU, 512; 16-column waves 1024): as many rounds, up to four
// splits below one round. us: 512 new tokens on 8192 141 / 352, 7 chunks of 257 on up to 6001 155 / 205, 16 x 8 new
// tokens on 4096 38 / 122; one prompt of 2048 fills the card, 121 (unsplit) / 130 in two.
Kv4Plan kv4_plan(int64_t T, int B, int H, int G, int D, int64_t max_q, int64_t max_kv) {
  Kv4Plan pl = {};
  // a bound below the mean or past all rows is wrong: the workspace or the grid would grow with it
  if (max_q < (T + B - 1) / B) max_q = (T + B - 1) / B;
  if (max_q > T) max_q = T;
  const int64_t cols = max_q * G;
  pl.few = cols <= 16;
  // 32 columns a wave, or 16 where those of a workgroup cover a sequence's, and for 256 channels, whose 32 would
  // not fit the registers of two waves per SIMD
  pl.nq = pl.few || D == 256 || cols <= 64 ? 1 : 2;
  const int64_t per = pl.few ? 16 : 64 * pl.nq;
  pl.qgrid = (cols + per - 1) / per;
  const int64_t pairs = pl.qgrid * H * B, tiles = (max_kv + 31) / 32;
  auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
  auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  const int64_t round = pl.few ? 768 : pl.nq == 2 ? 512 : 1024;
  int64_t s = round / pairs;
  if (pl.few || pairs < round) s = most(s, least(4, 2048 / pairs));
  s = least(s, pl.few ? tiles / 8 - 1 : tiles / 8);
  s = least(s, least(64, most(16, tiles / 64)));
  pl.splits = (int)most(s, 1);
  return pl;
}

// A tree's. More than 64 columns, without a window and with a context that is worth its tables, go to kv4_tree_attn_kernel: a
// workgroup of 8 waves per CU, or two of 4 for up to 128 columns; one round of the card, or two splits where the sequences
// fill less than that. us, there / in kv4_attn_kernel (8 heads of 4 queries, 128 channels, bf16), 64 and 72 columns: 32 users on
// 4000 107 / 97 and 115 / 136, 8 on 16000 103 / 93 and 110 / 122, 8 on 512 22 / 18 and 23 / 22, 8 on 300 19 / 16 and 20 / 20. One
// user breaks even at 16000 only: 72 columns on 512 20 / 16, on 4000 26 / 24, on 16000 39 / 39. The others are
// kv4_attn_kernel's, and more than 16 columns of few sequences get splits for all of the CUs, of at least 4 tiles: the join is
// cheap then. us, with it / as above: 13 tokens of 4 heads a group on 2000 16.1 / 17.9, on 30000 46 / 74.
Kv4Plan kv4_tree_plan(int64_t T, int B, int H, int G, int D, int64_t window, int64_t max_q, int64_t max_kv) {
  Kv4Plan pl = kv4_plan(T, B, H, G, D, max_q, max_kv);
  if (max_q < (T + B - 1) / B) max_q = (T + B - 1) / B;
  const int64_t cols = (max_q < T ? max_q : T) * G;
  if (window || pl.few) return pl;
  auto most = [](int64_t a, int64_t b) { return a > b ? a : b; };
  auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  const int64_t cus = 256;
  if (D > 128 || cols <= 64 || max_kv < 512) {
    pl.splits = (int)most(pl.splits, least(least(cus / (pl.qgrid * H * B), (max_kv + 31) / 32 / 4), 32));
    return pl;
  }
  pl.wide = cols > 128 ? 8 : 4;
  pl.qgrid = (cols + 32 * pl.wide - 1) / (32 * pl.wide);
  const int64_t pairs = pl.qgrid * H * B, tiles = (max_kv + 63) / 64, round = cus * 8 / pl.wide;
  const int64_t s = pairs < round ? most(round / pairs, 2) : 1;
  pl.splits = (int)most(least(least(s, tiles / 4), 64), 1);
  return pl;
}

int64_t kv4_workspace(int64_t T, int Hq, int D, int splits) {
  return splits <= 1 ? 0 : (int64_t)splits * T * Hq * (D + 2) * 4;
}

template <int D, int DT, bool TREE>
static int launch_dt(Kv4Attn& p, const Kv4Plan& pl, hipStream_t st) {
  const int64_t rows = p.s.T * p.c.H * p.G;
  if (pl.qgrid * pl.splits > kMaxGrid || (pl.splits > 1 && rows / 4 >= kMaxGrid)) return kErrUnsupported;
  const dim3 g((unsigned)(pl.qgrid * pl.splits), (unsigned)p.c.H, (unsigned)p.s.B), b(256);
  if (pl.wide) {
    p.lse_more = kWideLse;
    const int rc = launch_kv4_tree_attn(p, D, DT, pl, st);
    if (rc) return rc;
  } else if (pl.few) hipLaunchKernelGGL((kv4_attn_kernel<D, DT, 1, 4, TREE>), g, b, 0, st, p);
  else if (pl.nq == 1) hipLaunchKernelGGL((kv4_attn_kernel<D, DT, 1, 1, TREE>), g, b, 0, st, p);
  else hipLaunchKernelGGL((kv4_attn_kernel<D, DT, D == 256 ? 1 : 2, 1, TREE>), g, b, 0, st, p);
  if (hipPeekAtLastError() != hipSuccess) return kErrHip;
  if (pl.splits > 1) hipLaunchKernelGGL((kv4_join_kernel<D, DT>), dim3((unsigned)((rows + 3) / 4)), b, 0, st, p);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

template <int DT, bool TREE>
static int launch_d(Kv4Attn& p, int D, const Kv4Plan& pl, hipStream_t st) {
  return D == 64 ? launch_dt<64, DT, TREE>(p, pl, st) : D == 128 ? launch_dt<128, DT, TREE>(p, pl, st) : launch_dt<256, DT, TREE>(p, pl, st);
}

int launch_kv4_attention(Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, void* ws, hipStream_t st) {
  p.splits = pl.splits;
  p.po = reinterpret_cast<float*>(ws);
  p.pml = p.po + (int64_t)pl.splits * p.s.T * p.c.H * p.G * D;
  if (dtype == kBF16) return p.bits ? launch_d<kBF16, true>(p, D, pl, st) : launch_d<kBF16, false>(p, D, pl, st);
  return p.bits ? launch_d<kF16, true>(p, D, pl, st) : launch_d<kF16, false>(p, D, pl, st);
}

}  // namespace w4a8
