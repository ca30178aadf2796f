// Attention over the paged 4-bit cache for more than 16 columns (queries times heads of a group): prompts, their
// chunks, speculated tokens. The mathematics and the operands are kv4_attn.hip's; the differences:
//
// The 4 waves of a workgroup have 16 NQ columns each and walk the same tiles of 32 tokens. A tile's codes are
// widened once per workgroup: each wave loads a quarter of the words, widens them and puts the operands into LDS
// in the order in which every wave reads them (16 bytes a lane, no conflicts), the token scales beside them,
// while the tile before is computed from the other buffer. Widening costs 128 vector instructions a tile of
// D = 128, as much as the softmax of 16 columns, and the vector unit is what bounds this kernel.
//
// p s enters its product in fp16. For fp16 models as two terms; for bf16 models as one, w, rounded by 2^-12 of
// itself. Its error must not meet the codes' offset of 16 and the zero point: the output is summed as
//   O + sum p (m + 7.5 s) - 23.5 sum w,   O = sum w (16 + c),
// where it multiplies c - 7.5, so 2^-12 of half a V vector's range, an eighth of the output's own rounding.
// sum w is one more product, with a row of ones. So that p s stays inside fp16's range whatever V's steps are, p
// carries a power of two, 2^-e with 2^e about the largest step so far: it moves with the running maximum and
// drops out of the quotient.
#include "kv4_attn.h"

namespace w4a8 {

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2h));
}

template <int D, int DT, int NQ>
__global__ void __launch_bounds__(256, 2)
kv4_prompt_kernel(const Kv4Attn p) {
  constexpr int KS = D / 32, DB = D / 16;
  constexpr int W = DT == kF16 ? 2 : 1;  // fp16 terms of p s
  constexpr int kCols = 64 * NQ;
  // of a tile: K operands [half][step][lane], V operands [block][lane], 16 bytes each
  constexpr int kOps = (2 * KS + DB) * 64;
  // words of K and V per lane: each wave stages half of K's rows or half of V's blocks, DB / 2 words a lane
  constexpr int SW = DB / 2;
  static_assert(SW == KS, "K and V have as many words");
  __shared__ v4w ops[2][kOps];
  // token scales by group of 8, two neighbours per 16 bytes: (s, m) of K, (s, m - 16 s or m + 7.5 s) of V
  __shared__ v4f ksc[2][4][4], vsc[2][4][4];
  __shared__ float vtop[2];

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, col = lane & 15;
  const int h = blockIdx.y, b = blockIdx.z;
  const int split = blockIdx.x % p.splits;
  const Span sp = kv4_span(p, b);
  const Table table = (Table)(uintptr_t)(p.s.table + b * p.s.ldt);

  const int qtiles = (sp.cols + kCols - 1) / kCols;
  const int gq = gridDim.x / p.splits;
  for (int qi = blockIdx.x / p.splits; qi < qtiles; qi += gq) {
    // the last columns have the most keys: first
    const int w0 = (qtiles - 1 - qi) * kCols, c0 = w0 + wave * 16 * NQ;
    const Keys all = kv4_keys(p, sp, w0, min(w0 + kCols, sp.cols));       // the workgroup's
    const Keys ks = kv4_keys(p, sp, c0, min(c0 + 16 * NQ, sp.cols));      // the wave's
    const int t_first = all.lo >> 5, nt = all.lo < all.hi ? ((all.hi + 31) >> 5) - t_first : 0;
    auto token = [&](int t) { return (t_first + t) * 32; };

    // the wave's quarter of a tile, and a scale word of one of its 32 tokens (waves 0 and 1, lanes 0 to 31)
    uint32_t raw[SW], rsc = 0;
    auto load = [&](const Pages& pg, int t) {
      if (wave < 2)
        load_words(p.c.k + (uint64_t)pick(p, pg, h, t, (lane & 15) >> 2) * (4 * D) +
                       ((wave * 4 + (lane & 3)) * (D / 2) + g * (D / 8)), raw);
      else
        load_words(p.c.v + (uint64_t)pick(p, pg, h, t, g) * (4 * D) + ((lane & 15) * (D / 4) + (wave - 2) * (D / 8)), raw);
      if (wave < 2 && lane < 32) rsc = (wave ? p.c.vs : p.c.ks)[(uint64_t)pick(p, pg, h, t, lane >> 3) * 8 + (lane & 7)];
    };
    auto stage = [&](const Pages& pg, int t, int buf) {
#pragma unroll
      for (int w = 0; w < SW; ++w)
        ops[buf][(wave * SW + w) * 64 + lane] = wave < 2 ? widen<DT>(raw[w]) : widen<kF16>(raw[w]);
      if (wave < 2) {
        const float s = lo16<DT>(rsc), m = hi16<DT>(rsc);
        float* to = reinterpret_cast<float*>(wave ? &vsc[buf][0][0] : &ksc[buf][0][0]) + 2 * lane;
        // a missing page is NaN to whoever sees it
        const bool missing = !exists(p, (lane & 31) < 16 ? pg.a : pg.b);
        if (lane < 32) {
          to[0] = wave == 0 && missing ? __builtin_nanf("") : s;
          to[1] = wave ? __builtin_fmaf(W == 2 ? -16.f : 7.5f, s, m) : m;
        }
        if (wave) {
          // the largest step among tokens that the workgroup sees
          const bool in = lane < 32 && t + lane >= all.lo && t + lane < all.hi && !missing;
          const float top = wave_max(in ? s : 0.f);
          if (lane == 0) vtop[buf] = top;
        }
      }
    };

    const int i0 = c0 / p.G, r0 = c0 - i0 * p.G;
    int klo[NQ], khi[NQ];
    v4w qf[NQ][KS];
    float qs[NQ];
    const int step = p.splits;
    int t = split;
    Pages at = {-1, -1}, nat = {-1, -1};
    if (t < nt) {
      at = look_up(p, table, token(t), all.hi);
      load(at, token(t));
    }
    if (t + step < nt) nat = look_up(p, table, token(t + step), all.hi);
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      int head;
      const int i = kv4_query(p, i0, r0, 16 * j + col, head);
      const bool on = c0 + 16 * j + col < sp.cols;
      khi[j] = on ? seen_upto(p, sp, i) : 0;
      klo[j] = seen_from(p, sp, i);
      const uint16_t* qp = p.q + (sp.start + (on ? i : 0)) * p.ldq + (h * p.G + (on ? head : 0)) * p.hq + g * (D / 4);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const uint4 u = on ? *reinterpret_cast<const uint4*>(qp + 8 * w) : make_uint4(0, 0, 0, 0);
        qf[j][w] = query_operand(u);
        sum += sum8<DT>(u);
      }
      qs[j] = col_sum(sum);
    }
    v4f o[NQ][DB], ws[NQ];  // ws: sum w (bf16 models), in every register
    float m[NQ], mu[NQ], l[NQ], cc[NQ];  // mu: m in powers of two (0 while no key was seen), plus e
    int ex = -127;                       // the steps' power of two; none yet
    const float slack = 8.f / p.scale;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      m[j] = -__builtin_inff();
      mu[j] = l[j] = cc[j] = 0.f;
      ws[j] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < DB; ++d) o[j][d] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    if (t < nt) stage(at, token(t), 0);
    __syncthreads();

    for (int buf = 0; t < nt; buf ^= 1) {
      const int t0 = token(t), tn = t + step;
      const bool more = tn < nt;
      const Pages cur = at;
      Pages nnat = {-1, -1};
      if (more) load(nat, token(tn));
      if (tn + step < nt) nnat = look_up(p, table, token(tn + step), all.hi);
      if (t0 < ks.hi && t0 + 32 > ks.lo) {
        // the power of two at or above the tile's largest step; steps that small that 2^-40 bounds them stay there
        const int te = max(min((int)((__float_as_uint(vtop[buf]) >> 23) & 255u) - 126, 100), -40);
        if (__builtin_amdgcn_readfirstlane(te) > ex) {
          const int en = __builtin_amdgcn_readfirstlane(te);
          if (ex > -127) {
            const float f = __builtin_amdgcn_exp2f((float)(ex - en));
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
              l[j] *= f;
              cc[j] *= f;
              ws[j] *= f;
#pragma unroll
              for (int d = 0; d < DB; ++d) o[j][d] *= f;
            }
          }
          ex = en;
#pragma unroll
          for (int j = 0; j < NQ; ++j) mu[j] = (m[j] == -__builtin_inff() ? 0.f : m[j] * p.scale) + (float)ex;
        }
        v4f s[NQ][2];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          const float q16 = -16.f * qs[j];
          s[j][0] = s[j][1] = v4f{q16, q16, q16, q16};
        }
#pragma unroll
        for (int w = 0; w < KS; ++w)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const v4w a = ops[buf][(u * KS + w) * 64 + lane];
#pragma unroll
            for (int j = 0; j < NQ; ++j) s[j][u] = mfma16<DT>(a, qf[j][w], s[j][u]);
          }
        const bool whole = t0 >= ks.lo_all && t0 + 32 <= ks.hi_all;
        v4w ph[NQ], pl[NQ];
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          float y[8], sv[8], mv[8];
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            const v4f k2 = ksc[buf][g][i / 2], v2 = vsc[buf][g][i / 2];
            y[i] = __builtin_fmaf(k2[0], s[j][i >> 2][i & 3], k2[1] * qs[j]);
            y[i + 1] = __builtin_fmaf(k2[2], s[j][i >> 2][(i & 3) + 1], k2[3] * qs[j]);
            sv[i] = v2[0];
            mv[i] = v2[1];
            sv[i + 1] = v2[2];
            mv[i + 1] = v2[3];
          }
          if (!whole) {
            // an unseen token's scale may be anything, and 0 times it is not 0
            const int a = klo[j] - (t0 + 8 * g), e = khi[j] - (t0 + 8 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const bool see = i >= a && i < e;
              y[i] = see ? y[i] : -__builtin_inff();
              sv[i] = see ? sv[i] : 0.f;
              mv[i] = see ? mv[i] : 0.f;
            }
          }
          const float top = fmaxf(fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])), fmaxf(fmaxf(y[4], y[5]), fmaxf(y[6], y[7])));
          if (__ballot(top > m[j] + slack)) {
            const float mn = fmaxf(m[j], col_max(top));
            const float f = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((m[j] - mn) * p.scale);
            m[j] = mn;
            mu[j] = (mn == -__builtin_inff() ? 0.f : mn * p.scale) + (float)ex;
            l[j] *= f;
            cc[j] *= f;
            ws[j] *= f;
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
            ph[j][r] = pack_f16(ps[r], ps[r + 4]);
            if (W == 2)
              pl[j][r] = pack_f16(ps[r] - f16_to_f32((uint16_t)(ph[j][r] & 0xffffu)), ps[r + 4] - f16_to_f32((uint16_t)(ph[j][r] >> 16)));
          }
        }
        if (W == 1)
#pragma unroll
          for (int j = 0; j < NQ; ++j)
            ws[j] = mfma16<kF16>(v4w{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}, ph[j], ws[j]);
#pragma unroll
        for (int d = 0; d < DB; ++d) {
          const v4w a = ops[buf][(2 * KS + d) * 64 + lane];
#pragma unroll
          for (int j = 0; j < NQ; ++j) {
            o[j][d] = mfma16<kF16>(a, ph[j], o[j][d]);
            if (W == 2) o[j][d] = mfma16<kF16>(a, pl[j], o[j][d]);
          }
        }
      }
      if (more) stage(nat, token(tn), buf ^ 1);
      __syncthreads();
      at = nat;
      nat = nnat;
      t = tn;
    }
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      // back to the common power of two, for the splits to be joined and the logarithm of the sum
      const float f = ex > -127 ? __builtin_amdgcn_exp2f((float)ex) : 1.f;
      const float sum = col_sum(l[j]) * f, c = (col_sum(cc[j]) - (W == 1 ? 23.5f * ws[j][0] : 0.f)) * f;
      int head;
      const int i = kv4_query(p, i0, r0, 16 * j + col, head);
      if (c0 + 16 * j + col < sp.cols)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          float v[DB];
#pragma unroll
          for (int d = 0; d < DB; ++d) v[d] = __builtin_fmaf(o[j][d][r], f, c);
          kv4_store<D, DT>(p, split, sp.start + i, h * p.G + head, (4 * g + r) * DB, v, m[j] * p.scale, sum, g == 0 && r == 0);
        }
    }
  }
}

template <int D, int DT>
static void launch_prompt(const Kv4Attn& p, int nq, dim3 grid, hipStream_t st) {
  if constexpr (D != 256)
    if (nq == 2) {
      hipLaunchKernelGGL((kv4_prompt_kernel<D, DT, 2>), grid, dim3(256), 0, st, p);
      return;
    }
  hipLaunchKernelGGL((kv4_prompt_kernel<D, DT, 1>), grid, dim3(256), 0, st, p);
}

void launch_kv4_prompt(const Kv4Attn& p, int D, int dtype, int nq, dim3 grid, hipStream_t st) {
  if (dtype == kBF16) {
    if (D == 64) launch_prompt<64, kBF16>(p, nq, grid, st);
    else if (D == 128) launch_prompt<128, kBF16>(p, nq, grid, st);
    else launch_prompt<256, kBF16>(p, nq, grid, st);
  } else {
    if (D == 64) launch_prompt<64, kF16>(p, nq, grid, st);
    else if (D == 128) launch_prompt<128, kF16>(p, nq, grid, st);
    else launch_prompt<256, kF16>(p, nq, grid, st);
  }
}

}  // namespace w4a8
