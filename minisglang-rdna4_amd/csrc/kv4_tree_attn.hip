// Attention of many drafted tokens, more than 64 columns of them, over the 4-bit cache (layout: kv4.h). All of a sequence's
// drafted tokens see the same context and all of it, so all but the last tiles have no masks, and what a tile's keys share
// need not be kept apart by column. (Fewer columns, and windows, are kv4_attn_kernel's.)
//
// The queries that share a key/value head are columns (column c: query c / G, head h G + c % G), 32 a wave, and the 4 or 8
// waves of a workgroup share tiles of 64 tokens that are widened to fp16 once, in LDS:
//   S = b sum(q) + K' Q^T,  p = 2^(S scale - M),  O += V'^T p   (32x32x16 products; tokens, then channels are rows).
// K' = s (c - 7.5) as s/2 (2 c - 15), b = m + 7.5 s. bf16 models: s comes as s 2^-e, e one for the tile, so that it fits fp16 (one
// for each token, and S times their difference, where steps of a tile are more than 2^20 apart): 8 bits times the code's 4 lose
// one bit at most, 2^-11 of what is left once the middle of the vector's range is taken out; fp16 models, whose scores ought to
// be better than that, have K' = 2 c - 15, exactly, b = 2 m / s + 15, and S times s/2 afterwards.
// V' = s c + m, rounded once to fp16 (2^-11), times 2^-e with e the largest so far. fp16 models have the codes, exactly, p s
// rounded instead (times 2^-e, e of the largest step so far) and sum p (m + 7.5 s) beside the product, in f32: their
// output would show the rounding of V' (norm of the error over the output's 3.5e-4, so 3.0e-4; rounding the output 2.1e-4).
// p is rounded to fp16, and its sum is of the rounded ones: 2^7 and more for the largest score, so that what is lost below
// fp16's least, 2^-32 of that a token, is nothing over any context. Powers of two change no bits, unless values of a bf16
// model's context and drafts are more than 2^29 apart: the small ones are then lost.
// Queries enter in fp16 with a power of two per row, as in kv4_attn_kernel.
//
// Codes become fp16 by an or into the lowest bits of 1024 and a packed subtraction. A word of K codes is 8 channels of a
// token, one of V codes 8 tokens of a channel: in either case 16 bytes that one lane of a product wants, in the order of the
// nibbles 0, 4, 1, 5, 2, 6, 3, 7. Q's channels, and which token each row of S is, follow that order, and p goes from one product
// into the next in its lane.
// Codes of the next tile and scales of the one after the next are loaded while a tile is worked on, and widened behind it.
// The scales are unpacked by two of the waves, by turns, a token a lane, into tables. What is read from LDS is read a product
// or more ahead, exponentials run behind the products of the 16 tokens before them, and the next tile's widening behind the
// last products: in the compiler's own order each product waited for its operands (14 us more in either case below).
// us, this launch alone, under the profiler: 48 users' 26 tokens and less on up to 8192 (8 heads of 4 queries, bf16) 184, with
// kv4_attn_kernel 216; two users' 60 tokens on 65536 and less, fp16, 205 (with V' rounded as bf16 models have it 187) / 279.
// Waves without columns only widen: 6 us of the second. No unit is full: of the second's busy cycles vector instructions take
// 58 %, matrix products 31 %, LDS 43 % (the first's 53, 24, 35); two waves a SIMD, which the accumulators leave room for, do not
// cover each other's latencies. Tried: the waves of a SIMD half a tile apart, so that one has products while the other has
// exponentials (no faster).
#include "kv4.h"
#include "tile32.h"

namespace w4a8 {

constexpr int kStep = 64;  // tokens of a tile

typedef float v8f __attribute__((ext_vector_type(8)));

struct alignas(32) ScaleTable {
  float b[kStep];        // in the order of S's rows: [32 tokens][half][16 registers]
  float s[kStep];        // what S is multiplied by, in that order: half of K's steps, of bf16 models, if `apart`, 2^(the token's e - e)
  uint32_t ks[kStep];    // bf16 models: half of K's step, twice, by token
  uint32_t v[8][8];      // bf16 models: V's steps of tokens j and j + 4 of the block (j < 4), and their least values
  float sv[kStep];       // fp16 models: V's steps, in the order of S's rows,
  float bv[kStep];       // and the middles m + 7.5 s, which may be past fp16's end
  int ek, ev, apart;
};

// A word's codes of nibbles j and j + 4 as fp16 numbers, c and 2 c - 15: 1024 with a code in its lowest bits, or a bit higher.
// The masks and 1024 are in registers, which takes one instruction for the and and the or.
struct Masks {
  uint32_t code, twice, magic;
};
__device__ __forceinline__ Masks masks() {
  Masks m = {0x000f000fu, 0x001e001eu, 0x64006400u};
  asm volatile("" : "+s"(m.code), "+s"(m.twice), "+v"(m.magic));
  return m;
}
__device__ __forceinline__ v2h codes_of(uint32_t w, int j, const Masks& m) {
  return __builtin_bit_cast(v2h, ((w >> (4 * j)) & m.code) | m.magic) - v2h{(_Float16)1024.f, (_Float16)1024.f};
}
__device__ __forceinline__ v2h centred(uint32_t w, int j, const Masks& m) {
  const uint32_t x = j == 0 ? w << 1 : w >> (4 * j - 1);
  return __builtin_bit_cast(v2h, (x & m.twice) | m.magic) - v2h{(_Float16)1039.f, (_Float16)1039.f};
}

template <int D, int DT, int NW>
__global__ void __launch_bounds__(64 * NW, 2)
kv4_tree_attn_kernel(const Kv4Attn p) {
  using P = Place<D>;
  static_assert(P::kTile == kStep, "a tile of K lies as a prompt's does");
  constexpr int KS = D / 16, CT = D / 32, kCols = 32 * NW, NT = 64 * NW;
  constexpr int U = 8 * D / NT;     // words of K, and of V, of a thread and tile
  constexpr bool kFold = DT == kBF16;
  constexpr int kLeastEv = -100;
  constexpr float kMost = 7.f;  // p is 2^7 and up to 2^15 (what may come before M follows) for the largest score
  constexpr float kInf = __builtin_inff();
  __shared__ __align__(16) unsigned char kt[2][P::kBytes];
  __shared__ __align__(16) unsigned char vt[2][kStep * D * 2];
  __shared__ __align__(32) ScaleTable tab[3];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int h = blockIdx.y, b = kv4_longest(p.s, blockIdx.z);
  const int splits = p.splits, split = blockIdx.x % splits;
  const Span sp = kv4_span<true>(p, b);
  if (sp.cols == 0) return;
  const int first = min(max(sp.first_pos, 0), sp.len);  // the context's tokens, seen by all; the new ones as their bits tell
  const int nt = (sp.len + kStep - 1) / kStep;
  const int count = split < nt ? (nt - split + splits - 1) / splits : 0;
  // Pages of 16 tiles, a lane for each 16 tokens: looked up 16 tiles before the first of them is loaded
  const int32_t* table = p.s.table + b * p.s.ldt;
  auto look_up = [&](int group) {
    const int k = group * 16 + (lane >> 2), t = (split + k * splits) * kStep + 16 * (lane & 3), i = t >> p.c.shift;
    return k < count && t < sp.len && i < p.s.width ? table[i] : -1;
  };
  int pages = 0, ahead = 0, group = 0;  // of tiles 16 group .. and of the 16 after them
  // block of the 16 tokens `u` of tile k, or -1: for all lanes, or a lane's own
  auto block_of = [&](int page, int k, int u) {
    return (uint32_t)page < (uint32_t)p.c.pages ? kv4_block(p.c, page, h, (split + k * splits) * kStep + 16 * u) : -1;
  };
  auto unit_of = [&](int k, int u) {
    return block_of(__builtin_amdgcn_readlane((k >> 4) == group ? pages : ahead, (k & 15) * 4 + u), k, u);
  };
  // K's words in the order of Place, 16 bytes of a row at a time
  auto row_of = [](int at) {
    return D == 64 ? ((at >> 6) & 1) * 8 + ((at >> 5) & 1) * 4 + ((at >> 2) & 3) : (at >> 6) * 4 + ((at >> 2) & 3);
  };
  auto chunk_of = [](int at) {
    return D == 64 ? ((at >> 4) & 1) * 4 + ((at & 3) ^ ((at >> 5) & 1)) : ((at >> 4) & 3) * 4 + (at & 3);
  };
  uint32_t kw[U], vw[U];
  const Masks ms = masks();
  auto load_codes = [&](int k) {
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int unit = (i * NT + wave * 64) / (2 * D), at = (i * NT + (int)threadIdx.x) & (2 * D - 1);
      const int x = unit_of(k, unit);
      const uint64_t base = (uint64_t)(x < 0 ? 0 : x) * (4 * D);  // block 0 is there; its values are not used
      kw[i] = *reinterpret_cast<const uint32_t*>(p.c.k + base + (row_of(at) * (D / 8) + chunk_of(at)) * 4);
      vw[i] = *reinterpret_cast<const uint32_t*>(p.c.v + base + at * 4);
    }
  };
  // piece j of 2 U of the next tile: a word of K, or one of V
  struct Steps {
    v4w s, m;
  };
  auto steps_of = [&](const ScaleTable& tb, int j) {
    const int i = j >> 1, unit = (i * NT + wave * 64) / (2 * D), at = (i * NT + (int)threadIdx.x) & (2 * D - 1);
    Steps r = {};
    if (j & 1) {
      if (!kFold) return r;
      const int blk = unit * 2 + at / D;
      r.s = *reinterpret_cast<const v4w*>(&tb.v[blk][0]);
      r.m = *reinterpret_cast<const v4w*>(&tb.v[blk][4]);
    } else if (kFold) {
      r.s[0] = tb.ks[unit * 16 + row_of(at)];
    }
    return r;
  };
  auto widen = [&](const Steps& sm, int j, unsigned char* kd, unsigned char* vd) {
    const int i = j >> 1, unit = (i * NT + wave * 64) / (2 * D), at = (i * NT + (int)threadIdx.x) & (2 * D - 1);
    v4w x;
    if (j & 1) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t s2 = sm.s[e], m2 = sm.m[e];
        if (!kFold) x[e] = __builtin_bit_cast(uint32_t, centred(vw[i], e, ms));
        else x[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(codes_of(vw[i], e, ms), __builtin_bit_cast(v2h, s2),
                                                                      __builtin_bit_cast(v2h, m2)));
      }
      *reinterpret_cast<v4w*>(vd + unit * (32 * D) + at * 16) = x;
    } else {
      const uint32_t s2 = sm.s[0];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const v2h c = centred(kw[i], e, ms);
        x[e] = __builtin_bit_cast(uint32_t, kFold ? c * __builtin_bit_cast(v2h, s2) : c);
      }
      *reinterpret_cast<v4w*>(kd + P::at(unit * 16 + row_of(at), chunk_of(at))) = x;
    }
  };
  // two of the waves, others in the next tile: a token's scales, of K and of V
  uint32_t sk = 0, sv = 0;
  bool there = false;
  auto turn = [&](int k) { return (wave ^ (2 * k)) & (NW - 1); };
  auto load_scales = [&](int k) {
    if (turn(k) > 1) return;
    const int x = block_of(__shfl((k >> 4) == group ? pages : ahead, (k & 15) * 4 + (lane >> 4)), k, lane >> 4);
    const int64_t at = (int64_t)(x < 0 ? 0 : x) * 8 + (lane & 15);
    there = x >= 0;
    sk = p.c.ks[at];
    sv = p.c.vs[at];
  };
  auto unpack_scales = [&](int k, ScaleTable& tb, const ScaleTable& last) {
    if (turn(k) > 1 || k >= count) return;
    const bool in = (split + k * splits) * kStep + lane < sp.len;
    auto lo = [](uint32_t w) { return from_dtype((uint16_t)(w & 0xffffu), DT); };
    auto hi = [](uint32_t w) { return from_dtype((uint16_t)(w >> 16), DT); };
    const float s0 = lo(sk), m0 = hi(sk), s1 = lo(sv), m1 = hi(sv);
    const bool bad_v = !there || !__builtin_isfinite(s1) || !__builtin_isfinite(__builtin_fmaf(15.f, s1, m1)) || !__builtin_isfinite(m1);
    const float c0 = __builtin_fmaf(7.5f, s0, m0);
    const bool bad = bad_v || !__builtin_isfinite(s0) || !__builtin_isfinite(c0);
    const int nib = lane & 7;
    const int r = (lane >> 5) * 32 + ((lane >> 3) & 1) * 16 + ((lane >> 4) & 1) * 8 + (nib < 4 ? 2 * nib : 2 * nib - 7);
    if (turn(k) == 0) {
      const float s = in && !bad ? s0 : 0.f;
      int e = 0;
      if (kFold) {
        // the largest step into [2^11, 2^12): times 7.5 it stays in fp16
        // (and least values that no kv4_append gives such a step stay in f32)
        const float size = in && !bad ? fmaxf(s, fabsf(m0) * 0x1p-14f) : 0.f;
        auto power = [](float x) { return min(max((int)(__float_as_uint(x) >> 23) - 138, -100), 120); };
        e = power(wave_max(size));
        // with one e, fp16 has fewer than a step's 8 bits for those 2^24 below the largest: the tokens have an e each then
        const bool apart = __ballot(size > 0x1p-120f && power(size) < e - 20) != 0;
        const int own = apart ? power(size) : e;
        const uint32_t x = (uint32_t)f32_to_f16(__builtin_ldexpf(s, -own - 1));
        tb.ks[lane] = x | (x << 16);
        tb.b[r] = !in ? 0.f : bad ? __builtin_nanf("") : __builtin_ldexpf(c0, -own);
        if (apart) tb.s[r] = __builtin_ldexpf(1.f, own - e);
        if (lane == 0) tb.apart = apart;
      } else {
        // a vector of equal values has no step, and codes of 0: any small one does
        const float s2 = fmaxf(0.5f * s, fmaxf(fabsf(m0) * 0x1p-30f, 0x1p-60f));
        tb.b[r] = !in ? 0.f : bad ? __builtin_nanf("") : m0 / s2 + 15.f;
        tb.s[r] = s2;
      }
      if (lane == 0) tb.ek = e;
    } else {
      const bool use = in && !bad;
      const float s = use ? s1 : 0.f, m = use ? m1 : 0.f;
      // bf16 models: the largest value into [2^14, 2^15); fp16 models: the largest step into [1/2, 1)
      const float most = wave_max(kFold ? fmaxf(fabsf(m), fabsf(__builtin_fmaf(15.f, s, m))) : s);
      const int ev_run = max(k == 0 ? kLeastEv : last.ev, min((int)(__float_as_uint(most) >> 23) - (kFold ? 141 : 126), 120));
      if (kFold) {
        uint16_t* v = reinterpret_cast<uint16_t*>(&tb.v[lane >> 3][0]) + (nib & 3) * 2 + (nib >> 2);
        v[0] = f32_to_f16(__builtin_ldexpf(s, -ev_run));
        v[8] = f32_to_f16(__builtin_ldexpf(m, -ev_run));
      } else {
        tb.sv[r] = __builtin_ldexpf(s, -ev_run);
        tb.bv[r] = __builtin_fmaf(7.5f, s, m);
      }
      if (lane == 0) tb.ev = ev_run;
    }
  };

  // a lane's part of the addresses
  const int rho = col, token = ((rho >> 4) & 1) * 16 + ((rho >> 2) & 1) * 8 + (((rho >> 3) & 1) * 2 + ((rho & 3) >> 1)) + 4 * (rho & 1);
  const int k_lane = P::at(token, half), v_lane = (half * D + col) * 16;

  const int qtiles = (sp.cols + kCols - 1) / kCols, gq = gridDim.x / splits;
  for (int qi = blockIdx.x / splits; qi < qtiles; qi += gq) {
    const int c = qi * kCols + wave * 32 + col;
    const bool on = c < sp.cols;
    const int i = on ? c / p.G : 0, head = h * p.G + (on ? c - i * p.G : 0);
    const uint16_t* qp = p.q + (sp.start + i) * p.ldq + head * p.hq + half * 8;
    uint4 qr[KS];
#pragma unroll
    for (int w = 0; w < KS; ++w) qr[w] = on ? *reinterpret_cast<const uint4*>(qp + 16 * w) : make_uint4(0, 0, 0, 0);
    group = 0;
    pages = look_up(0);
    ahead = look_up(1);
    load_codes(0);
    load_scales(0);
    unpack_scales(0, tab[0], tab[0]);
    load_scales(1);

    v4w qf[KS];
    float qs, sc;
    {
      float sum = 0.f, top = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        float f[8];
        unpack8(qr[w], DT, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          sum += f[e];
          top = fmaxf(top, fabsf(f[e]));
        }
      }
      top = pair_max(top);
      // 2^eq puts the largest value into [2^14, 2^15), where that is above 2^-106
      const int eq = min(max(141 - (int)(__float_as_uint(top) >> 23), -100), 120);
      qs = __builtin_ldexpf(pair_sum(sum), eq);
      sc = fmaxf(__builtin_ldexpf(p.scale, -eq), 0x1p-120f);
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        float f[8];
        unpack8(qr[w], DT, f);
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[w][j] = pack16<kF16>(__builtin_ldexpf(f[j], eq), __builtin_ldexpf(f[j + 4], eq));
      }
    }
    v16f o[CT];
#pragma unroll
    for (int d = 0; d < CT; ++d) o[d] = v16f{};
    float bo = 0.f;  // fp16 models: sum of p (m + 7.5 s)
    float m = -kInf, thr = -kInf, mu = 0.f, l = 0.f;  // m: the maximum as a score over scale, times the query's power of two
    int ev = kLeastEv;
    auto in_order = [] { __builtin_amdgcn_sched_barrier(0); };  // the compiler would have each read of LDS wait where it is used
    // S starts as b sum(q)
    v16f s[2];
    auto start = [&](const ScaleTable& tb) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const float* tbl = &tb.b[kb * 32 + half * 16];
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = tbl[r];
      }
      in_order();
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) s[kb] *= qs;
    };
    // of 8 of a lane's 32 values of S
    struct Weights {
      v8f s, b;
    };
    auto weights = [&](const ScaleTable& tb, int g) {
      const int at = (g >> 1) * 32 + half * 16 + (g & 1) * 8;
      return Weights{*reinterpret_cast<const v8f*>(&tb.sv[at]), *reinterpret_cast<const v8f*>(&tb.bv[at])};
    };
    auto v_operand = [&](const unsigned char* vc, int f, int d) { return lds_read(vc + v_lane + (2 * f * D + 32 * d) * 16); };
    __syncthreads();
    unpack_scales(1, tab[1], tab[0]);
    load_scales(2);
#pragma unroll
    for (int j = 0; j < 2 * U; ++j) widen(steps_of(tab[0], j), j, kt[0], vt[0]);
    start(tab[0]);
    __syncthreads();

    auto fetch = [&](int k) {  // of the tiles after k
      load_codes(k + 1);  // behind the last tile: of block 0, for nobody
      unpack_scales(k + 2, tab[(k + 2) % 3], tab[(k + 1) % 3]);
      load_scales(k + 3);
      if (((k + 2) & 15) == 0) {  // the next iteration's codes are the next group's first
        pages = ahead;
        ahead = look_up(++group + 1);
      }
    };
    if (qi * kCols + wave * 32 >= sp.cols) {  // no columns: only the wave's part of the tiles
      for (int k = 0; k < count; ++k) {
        fetch(k);
#pragma unroll
        for (int j = 0; j < 2 * U; ++j) widen(steps_of(tab[(k + 1) % 3], j), j, kt[(k + 1) & 1], vt[(k + 1) & 1]);
        __syncthreads();
      }
      continue;
    }
    for (int k = 0; k < count; ++k) {
      const ScaleTable& tb = tab[k % 3];
      const unsigned char* kc = kt[k & 1];
      const unsigned char* vc = vt[k & 1];
      const int t0 = (split + k * splits) * kStep;
      v4w ka[KS], va[CT];
      Weights ws[2];
#pragma unroll
      for (int w = 0; w < KS; ++w) ka[w] = lds_read(kc + k_lane + P::at(0, 2 * w));
      in_order();
      fetch(k);

      const int now = __builtin_amdgcn_readfirstlane(tb.ev);
      if (now != ev) {
        const float f = __builtin_ldexpf(1.f, ev - now);
#pragma unroll
        for (int d = 0; d < CT; ++d) o[d] *= f;
        ev = now;
      }
      const float fe = kFold ? __builtin_ldexpf(1.f, __builtin_amdgcn_readfirstlane(tb.ek)) : 1.f;
      // f32 holds either factor, but not each product of them. Below 2^-120, where scores of the tile are as good as zero, it
      // has to leave -inf what it is, as sc has; past f32's end it has to leave a score of 0 at that. (Two instructions with a
      // constant in each: one with both wants them in registers, and spills those of the 4-wave form: 336 us as 367.)
      const float sct = kFold ? fmaxf(fminf(sc * fe, 0x1.fffffep+127f), 0x1p-120f) : sc;
      in_order();
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        s[0] = mfma32<kF16>(ka[w], qf[w], s[0]);
        ka[w] = lds_read(kc + k_lane + P::at(32, 2 * w));
        in_order();
      }
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        s[1] = mfma32<kF16>(ka[w], qf[w], s[1]);
        if (w < CT) va[w] = v_operand(vc, 0, w);
        if (!kFold && w >= KS - 2) ws[w & 1] = weights(tb, w & 1);
        in_order();
      }
      if (!kFold || __builtin_amdgcn_readfirstlane(tb.apart)) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const float* tsl = &tb.s[kb * 32 + half * 16];
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] *= tsl[r];
        }
      }
      if (t0 + kStep > first) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            const int at = t0 + 32 * kb + 16 * s2 + 8 * half, old = first - at;  // tokens of the context among the 8
            const uint32_t see = (on ? tree_bits(p, sp, i, at - sp.first_pos) : 0u) | (old <= 0 ? 0u : old >= 8 ? 255u : (1u << old) - 1);
#pragma unroll
            for (int e = 0; e < 8; ++e) s[kb][8 * s2 + e] = see >> ((e >> 1) + 4 * (e & 1)) & 1 ? s[kb][8 * s2 + e] : -kInf;
          }
      }
      float top = -kInf;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fmaxf(s[0][r], s[1][r]));
      top *= fe;
      if (__ballot(top > thr)) {
        const float tp = pair_max(top);
        // a column that has no need keeps its bits, whatever its neighbours do
        const bool need = tp > thr;
        const float mn = need ? fmaxf(m, tp) : m;
        const float was = far_off(m, sc), is = far_off(mn, sc);
        const float mun = need ? (mn == -kInf || is != 0.f ? 0.f : __builtin_fmaf(mn, sc, -kMost)) : mu;
        const float f = m == -kInf ? 1.f : __builtin_amdgcn_exp2f(__builtin_fmaf(was - is, sc, mu - mun));
        m = mn;
        mu = mun;
        thr = is != 0.f ? -kInf : mn + 8.f / sc;
        l *= f;
        bo *= f;
#pragma unroll
        for (int d = 0; d < CT; ++d) o[d] *= f;
        // not -inf: where the tile's unit is far below a negative maximum, a masked score less that would be NaN
        const float back = kFold ? fmaxf(is / fe, -0x1.fffffep+127f) : is;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          s[0][r] -= back;
          s[1][r] -= back;
        }
      }
      // Exponentials run behind products of the ones before them, and the next tile is widened behind the last ones.
      v4w pf[4];
      auto two = [&](int x) {  // p of values 2 x and 2 x + 1 of the 32
        const v16f& sv = s[x >> 3];
        const int e = (2 * x) & 15;
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e], sct, -mu));
        const float z = __builtin_amdgcn_exp2f(__builtin_fmaf(sv[e + 1], sct, -mu));
        const uint32_t w = pack16<kF16>(a, z);
        l = add_pair<kF16>(w, l);
        const Weights& ww = ws[(x >> 2) & 1];
        if (!kFold) {
          bo = __builtin_fmaf(a, ww.b[(2 * x) & 7], bo);
          bo = __builtin_fmaf(z, ww.b[(2 * x + 1) & 7], bo);
        }
        pf[x >> 2][x & 3] = kFold ? w : pack16<kF16>(a * ww.s[(2 * x) & 7], z * ww.s[(2 * x + 1) & 7]);
      };
#pragma unroll
      for (int x = 0; x < 4; ++x) two(x);
      const ScaleTable& tn = tab[(k + 1) % 3];
      Steps sm[2];
#pragma unroll
      for (int f = 0; f < 4; ++f)
#pragma unroll
        for (int d = 0; d < CT; ++d) {
          in_order();
          o[d] = mfma32<kF16>(va[d], pf[f], o[d]);
          if (f < 3) {
            va[d] = v_operand(vc, f + 1, d);
#pragma unroll
            for (int x = 0; x < 4 / CT; ++x) two(4 * f + 4 + d * (4 / CT) + x);
          }
          if (!kFold && f < 2 && d == 0) ws[f] = weights(tb, f + 2);
          if (f == 2 && d < 2) sm[d] = steps_of(tn, d);
          if (f == 3 && d < 2 * U) {
            widen(sm[d & 1], d, kt[(k + 1) & 1], vt[(k + 1) & 1]);
            if (d + 2 < 2 * U) sm[d & 1] = steps_of(tn, d + 2);
          }
        }
      in_order();
#pragma unroll
      for (int j = CT; j < 2 * U; ++j) {
        widen(sm[j & 1], j, kt[(k + 1) & 1], vt[(k + 1) & 1]);
        if (j + 2 < 2 * U) sm[j & 1] = steps_of(tn, j + 2);
      }
      start(tn);
      __syncthreads();
    }

    l = pair_sum(l);
    bo = pair_sum(bo);
    if (on) {
      const int Hq = p.c.H * p.G;
      const float back = __builtin_ldexpf(1.f, kFold ? ev : ev - 1), is = far_off(m, sc);
      const float most = m == -kInf ? -kInf : is != 0.f ? is * sc : mu;
      if (splits > 1) {
        const int64_t at = ((int64_t)split * p.s.T + sp.start + i) * Hq + head;
        float* op = p.po + at * D + half * 4;
        const float part = back * kWidePart, more = bo * kWidePart;
#pragma unroll
        for (int d = 0; d < CT; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<v4f*>(op + d * 32 + 2 * r) = v4f{__builtin_fmaf(o[d][r], part, more), __builtin_fmaf(o[d][r + 1], part, more),
                                                              __builtin_fmaf(o[d][r + 2], part, more), __builtin_fmaf(o[d][r + 3], part, more)};
        if (half == 0) {
          p.pml[at * 2] = most;
          p.pml[at * 2 + 1] = l * kWidePart;
        }
      } else {
        const float inv = l == 0.f ? 0.f : back / l, more = l == 0.f ? 0.f : bo / l;  // no key seen: 0
        uint16_t* op = p.out + (sp.start + i) * p.ldo + head * p.ho + half * 4;
#pragma unroll
        for (int d = 0; d < CT; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<v2w*>(op + d * 32 + 2 * r) =
                v2w{pack16<DT>(__builtin_fmaf(o[d][r], inv, more), __builtin_fmaf(o[d][r + 1], inv, more)),
                    pack16<DT>(__builtin_fmaf(o[d][r + 2], inv, more), __builtin_fmaf(o[d][r + 3], inv, more))};
        if (p.lse && half == 0)
          p.lse[(sp.start + i) * Hq + head] = l == 0.f ? -kInf : most * 0.69314718055994531f + logf(l);
      }
    }
  }
}

template <int D, int DT>
static int launch_dt(const Kv4Attn& p, const Kv4Plan& pl, hipStream_t st) {
  if (pl.qgrid * p.splits > kMaxGrid / 2) return kErrUnsupported;
  const dim3 g((unsigned)(pl.qgrid * p.splits), (unsigned)p.c.H, (unsigned)p.s.B);
  if (pl.wide == 4) hipLaunchKernelGGL((kv4_tree_attn_kernel<D, DT, 4>), g, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((kv4_tree_attn_kernel<D, DT, 8>), g, dim3(512), 0, st, p);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

// pl: that of a tree (kv4_tree_plan), its workgroups of 4 or 8 waves
int launch_kv4_tree_attn(const Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, hipStream_t st) {
  if (dtype == kBF16) return D == 64 ? launch_dt<64, kBF16>(p, pl, st) : launch_dt<128, kBF16>(p, pl, st);
  return D == 64 ? launch_dt<64, kF16>(p, pl, st) : launch_dt<128, kF16>(p, pl, st);
}

}  // namespace w4a8
