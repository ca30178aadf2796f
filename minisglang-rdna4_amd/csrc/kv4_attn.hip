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
#include "kv4_attn.h"

namespace w4a8 {

void launch_kv4_prompt(const Kv4Attn& p, int D, int dtype, int nq, dim3 grid, hipStream_t st);

// Decode: 16 columns, the 4 waves of a workgroup (and the splits of the grid) over the tokens.
template <int D, int DT>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 3)
kv4_decode_kernel(const Kv4Attn p) {
  constexpr int KS = D / 32, DB = D / 16;  // products per S tile, blocks of 16 channels
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int h = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % p.splits;
  const Span sp = kv4_span(p, b);
  const float slack = 8.f / p.scale;
  __shared__ float red_o[4 * 16 * D];
  __shared__ float red_ml[4 * 16 * 2];

  const int qtiles = (sp.cols + 15) / 16;
  const int gq = gridDim.x / p.splits;
  for (int qi = blockIdx.x / p.splits; qi < qtiles; qi += gq) {
    const int c0 = qi * 16;
    const Keys ks = kv4_keys(p, sp, c0, min(c0 + 16, sp.cols));
    const int t_first = ks.lo >> 5, nt = ks.lo < ks.hi ? ((ks.hi + 31) >> 5) - t_first : 0;
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
    // tiles are dealt out one by one, over the splits and their waves: all have the same share of a sequence
    const int step = p.splits * 4;
    int t = split * 4 + wave;
    int tn = t + step;
    auto token = [&](int t) { return (t_first + t) * 32; };
    Pages at = {-1, -1}, nat = {-1, -1};
    if (t < nt) at = look_up(p, table, token(t), ks.hi);
    if (tn < nt) nat = look_up(p, table, token(tn), ks.hi);

    // this lane's query
    const int i0 = c0 / p.G;
    int head;
    const int qry = kv4_query(p, i0, c0 - i0 * p.G, col, head);
    head += h * p.G;
    const bool on = c0 + col < sp.cols;
    const int klo = seen_from(p, sp, qry), khi = on ? seen_upto(p, sp, qry) : 0;
    uint4 qr[KS];
    {
      const uint16_t* qp = p.q + (sp.start + (on ? qry : 0)) * p.ldq + (on ? head : 0) * p.hq + g * (D / 4);
#pragma unroll
      for (int w = 0; w < KS; ++w) qr[w] = on ? *reinterpret_cast<const uint4*>(qp + 8 * w) : make_uint4(0, 0, 0, 0);
    }
    if (t < nt) {
      load_k(at, token(t));
      load_s(at, token(t));
      load_v(at, token(t));
    }
    v4w qf[KS];
    float qs = 0.f;
#pragma unroll
    for (int w = 0; w < KS; ++w) {
      qf[w] = query_operand(qr[w]);
      qs += sum8<DT>(qr[w]);
    }
    qs = col_sum(qs);

    v4f o[DB];
    float m = -__builtin_inff(), mu = 0.f, l = 0.f, cc = 0.f;  // mu: m in powers of two, 0 while no key was seen
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = v4f{0.f, 0.f, 0.f, 0.f};

    while (t < nt) {
      const int t0 = token(t);
      const int tnn = tn + step;
      Pages nnat = {-1, -1};
      if (tnn < nt) nnat = look_up(p, table, token(tnn), ks.hi);

      const float q16 = -16.f * qs;
      v4f s[2] = {v4f{q16, q16, q16, q16}, v4f{q16, q16, q16, q16}};
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        s[0] = mfma16<DT>(widen<DT>(kw[0][w]), qf[w], s[0]);
        s[1] = mfma16<DT>(widen<DT>(kw[1][w]), qf[w], s[1]);
      }
      if (tn < nt) load_k(nat, token(tn));

      float y[8], sv[8], mv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y[i] = __builtin_fmaf(lo16<DT>(ksw[i]), s[i >> 2][i & 3], hi16<DT>(ksw[i]) * qs);
        sv[i] = lo16<DT>(vsw[i]);
        mv[i] = __builtin_fmaf(-16.f, sv[i], hi16<DT>(vsw[i]));
      }
      if (!(t0 >= ks.lo_all && t0 + 32 <= ks.hi_all && exists(p, at.a) && exists(p, at.b))) {
        // an unseen token's scale may be anything, and 0 times it is not 0; a missing page is NaN to whoever sees it
        const int a = klo - (t0 + 8 * g), e = khi - (t0 + 8 * g);
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
      if (__ballot(top > m + slack)) {
        const float mn = fmaxf(m, col_max(top));
        const float f = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m - mn) * p.scale);
        m = mn;
        mu = mn == -__builtin_inff() ? 0.f : mn * p.scale;
        l *= f;
        cc *= f;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[d] *= f;
      }
      float ps[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(y[i], p.scale, -mu));
        l += pr;
        ps[i] = pr * sv[i];
        cc = __builtin_fmaf(pr, mv[i], cc);
      }
      v4w ph, pl;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ph[r] = pack_bf16(ps[r], ps[r + 4]);
        pl[r] = pack_bf16(ps[r] - __uint_as_float(ph[r] << 16), ps[r + 4] - __uint_as_float(ph[r] & 0xffff0000u));
      }
      if (tn < nt) load_s(nat, token(tn));
#pragma unroll
      for (int d = 0; d < DB; ++d) {
        const v4w a = widen<kBF16>(vw[d]);
        o[d] = mfma16<kBF16>(a, ph, o[d]);
        o[d] = mfma16<kBF16>(a, pl, o[d]);
      }
      if (tn < nt) load_v(nat, token(tn));
      at = nat;
      nat = nnat;
      t = tn;
      tn = tnn;
    }

    l = col_sum(l);
    cc = col_sum(cc);
    // join the waves through LDS, each to the common maximum; wave r then sums and writes the channels of r
    if (g == 0) {
      red_ml[(wave * 16 + col) * 2] = m * p.scale;
      red_ml[(wave * 16 + col) * 2 + 1] = l;
    }
#pragma unroll
    for (int d = 0; d < DB; ++d) *reinterpret_cast<v4f*>(&red_o[((wave * DB + d) * 64 + lane) * 4]) = o[d] + cc;
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
    // a lane's channels: DB (4 g + r) + d of its column
    if (on) kv4_store<D, DT>(p, split, sp.start + qry, head, (4 * g + wave) * DB, v, mx, sum, g == 0 && wave == 0);
    __syncthreads();  // before the next tile of columns writes LDS
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
  // a bound below the mean is wrong; the workspace would grow with it
  if (max_q < (T + B - 1) / B) max_q = (T + B - 1) / B;
  const int64_t cols = max_q * G;
  pl.few = cols <= 16;
  // the prompt kernel's columns per wave: 32, or 16 where those of a workgroup cover a sequence's, and for 256
  // channels, whose 32 would not fit the registers of two waves per SIMD
  pl.nq = D == 256 || cols <= 64 ? 1 : 2;
  const int64_t per = pl.few ? 16 : 64 * pl.nq;
  pl.qgrid = (cols + per - 1) / per;
  const int64_t pairs = pl.qgrid * H * B, tiles = (max_kv + 31) / 32;
  // a tile per wave at least
  const int64_t most = pl.few ? (tiles + 3) / 4 : tiles;
  int64_t s = pl.few ? 2048 / pairs : 512 / pairs;
  if (s > (pl.few ? 48 : 8)) s = pl.few ? 48 : 8;
  if (s > most) s = most;
  pl.splits = s < 1 ? 1 : (int)s;
  return pl;
}

int64_t kv4_workspace(int64_t T, int Hq, int D, int splits) {
  return splits <= 1 ? 0 : (int64_t)splits * T * Hq * (D + 2) * 4;
}

template <int D, int DT>
static int launch_dt(Kv4Attn& p, const Kv4Plan& pl, hipStream_t st) {
  const dim3 g((unsigned)(pl.qgrid * pl.splits), (unsigned)p.c.H, (unsigned)p.s.B), b(256);
  if (pl.few) hipLaunchKernelGGL((kv4_decode_kernel<D, DT>), g, b, 0, st, p);
  else launch_kv4_prompt(p, D, DT, pl.nq, g, st);
  if (hipGetLastError() != hipSuccess) return kErrHip;
  if (pl.splits > 1) {
    const int64_t rows = p.s.T * p.c.H * p.G;
    hipLaunchKernelGGL((kv4_join_kernel<D, DT>), dim3((unsigned)((rows + 3) / 4)), b, 0, st, p);
  }
  return hipGetLastError() == hipSuccess ? kOk : kErrHip;
}

int launch_kv4_attention(Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, void* ws, hipStream_t st) {
  p.splits = pl.splits;
  p.po = reinterpret_cast<float*>(ws);
  p.pml = p.po + (int64_t)pl.splits * p.s.T * p.c.H * p.G * D;
  if (dtype == kBF16)
    return D == 64 ? launch_dt<64, kBF16>(p, pl, st) : D == 128 ? launch_dt<128, kBF16>(p, pl, st) : launch_dt<256, kBF16>(p, pl, st);
  return D == 64 ? launch_dt<64, kF16>(p, pl, st) : D == 128 ? launch_dt<128, kF16>(p, pl, st) : launch_dt<256, kF16>(p, pl, st);
}

}  // namespace w4a8
