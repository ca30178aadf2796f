// Attention over whole prompts, packed: every key is a new token's, in 16 bits, in the same call.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q k_j - M),  j over the keys that the row sees.
//
// The queries that share a key/value head are columns: column c of a sequence is its query c / G, head h G + c % G, so the
// 128 columns of a workgroup are 128 / G neighbouring queries, which see almost the same keys. A wave has 32 columns; per
// 32 keys
//   S = K Q^T (32x32x16, keys are rows),  P = exp of S,  O += V^T P (channels are rows).
// A lane's 16 values of S are one column's, and P's operand wants 8 keys of one column in a lane: any 8, as long as V's
// operand has the same. So P stays in its registers; V's operand comes from LDS by transposed reads.
// K and V tiles go from memory straight into LDS (LDS-DMA), the next one while this one is worked on. A DMA lane's 16
// bytes land side by side; which 16 bytes those are is free. They are put so that 4 rows times 64 bytes lie together, and
// groups of 4 rows 16 bytes off a multiple of 256: both kinds of read then meet every bank once, at addresses that are one
// register and a constant.
// The running maximum is raised only when a score passes it by 8 (in powers of two): p stays below 2^8 (fp16 2^15), and most tiles
// need neither an exchange between lanes nor a rescaling of O. Sums and O are f32. p is rounded to the type for its product
// (by at most 2^-8 of itself for bf16, 2^-11 for fp16), as v is, and the sum that divides is of the rounded ones: the
// rounding then weighs values a little differently, and equal values keep their bits. fp16: M is 7 less, so that what is
// lost below fp16's least, 2^-32 a key of the largest, is nothing over any prompt.
//
// Measured: 8192 + 5690 + 3190 tokens, 32 heads on 8 of 128 channels (898 GFLOP), 0.88 ms, 1023 TFLOP/s, bf16; heads of 64
// 904, of 256 925; a window of 1024 802, not causal 1074; 23 prompts of up to 1869 tokens, 24 heads on 8 of 64, 676, fp16 632.
// Heads of 128 are bound by power: the matrix units are busy for half of the cycles (0.53, vector instructions 0.45), whose clock
// falls, under the profiler to 1.75 GHz (1.02 ms), and the same cycles take 0.79 ms at 2.2 GHz where all values are 0;
// products alone, from registers, reach 1.7 PFLOP/s on such values. No exponentials at all would save 6% of the time, no
// reads of K from LDS 5%, no copies of K and V into LDS 12%. Heads of 64, with twice the exponentials for a product, by
// vector instructions and products together: 0.63 and 0.37 of the busy cycles, and a SIMD passes little of one beside the
// other (16 products of a wave take 527 cycles, 128 fma of another 571, both 723).
// Steps, all under the profiler. First version 774 TFLOP/s: S, exponentials and products one after another, 8 waves a workgroup
// (two workgroups of 4 waves on a CU do not wait for each other: 23 prompts of up to 1999 tokens, heads of 64, 281 -> 234 us).
// Other steps: blocks of 32 keys whose S is computed while the block before passes through its exponentials (1161 -> 1055 us, heads of 64 762 -> 653), what
// is not finite dealt with before the products and not beside them, whose outputs then stay in their registers (-> 1016, 193
// us). Tried: tiles of 32 keys for all (three waves per SIMD spill, two are no faster, heads of 64 slower: 660 TFLOP/s); 64
// columns a wave (heads of 64 the same; of 128 take the registers of a SIMD, and half the time goes into moving them).
#include <type_traits>

#include "prompt_attn.h"
#include "tile32.h"

namespace w4a8 {

// D: channels; DT: the type; NW: waves
template <int D, int DT, int NW>
__global__ void __launch_bounds__(64 * NW, D == 64 ? 3 : 2)
prompt_attn_kernel(const PromptAttn p) {
  using P = Place<D>;
  constexpr int kTile = P::kTile;
  constexpr int KS = D / 16, CT = D / 32;       // steps of S, tiles of 32 channels
  constexpr int kDma = P::kDmas / NW;           // DMAs of a wave and tile
  static_assert(P::kDmas % NW == 0 && (D < 256 || kDma % 2 == 0), "every wave has the same, of whole rows");
  constexpr int kCols = 32 * NW;
  // Whether S of the next 32 keys is computed while these pass through their exponentials. Heads of 256 channels have no
  // registers for it, and twice the products per exponential.
  constexpr bool kAhead = D < 256;
  constexpr int kLead = kAhead ? 32 : 0;
  constexpr float kInf = __builtin_inff();
  constexpr float kMost = DT == kF16 ? 7.f : 0.f;  // p is 2^kMost at least for the largest score
  constexpr uint32_t kExp = DT == kBF16 ? 0x7f807f80u : 0x7c007c00u;  // exponents of two values
  constexpr uint32_t kOnes = DT == kBF16 ? 0x3f80u : 0x3c00u;
  __shared__ __align__(16) unsigned char k0[P::kBytes];
  __shared__ __align__(16) unsigned char k1[P::kBytes];
  __shared__ __align__(16) unsigned char v0[P::kBytes];
  __shared__ __align__(16) unsigned char v1[P::kBytes];
  __shared__ int flags[NW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = lane >> 5, col = lane & 31;
  const int h = blockIdx.x % p.H, b = blockIdx.y;

  const int64_t lo = p.cu[b], hi = p.cu[b + 1];
  const int64_t start = lo < 0 ? 0 : lo, end = hi < p.T ? hi : p.T;
  const int n = end > start ? (int)(end - start) : 0;
  const int cols = n * p.G;
  const int qtiles = (cols + kCols - 1) / kCols, gq = gridDim.x / p.H;

  const uint16_t* kbase = p.k + start * p.ldk + h * p.hk;
  const uint16_t* vbase = p.v + start * p.ldv + h * p.hv;
  // a lane's part of the addresses; the rest is constant
  const int k_lane = P::at(col, half);
  const int i16 = lane & 15;
  const int v_lane = P::at(half * 4 + (i16 >> 2), ((lane >> 4) & 1) * 2 + ((i16 & 3) >> 1)) + (i16 & 1) * 8;

  // a lane's offset in its wave's first DMA of a tile; the wave's others are of the next rows, or for 256 channels of the
  // rows' other half
  const int x0 = wave * kDma;
  const uint32_t k_off = (uint32_t)(P::dma_row(x0, lane) * (int)p.ldk * 2 + P::dma_chunk(x0, lane) * 16);
  const uint32_t v_off = (uint32_t)(P::dma_row(x0, lane) * (int)p.ldv * 2 + P::dma_chunk(x0, lane) * 16);
  auto fetch = [&](const uint16_t* base, int64_t ld, uint32_t off, int row0, unsigned char* dst) {
    const int rows = min(kTile, n - row0);  // rows past the end are zeros in LDS
    if (rows <= 0) return;
    const BufRsrc r = make_rsrc(base + (int64_t)row0 * ld, (uint32_t)(((rows - 1) * (int)ld + D) * 2));
    asm volatile("" : "+v"(off));  // offsets of all DMAs, kept over the loop, would take registers
#pragma unroll
    for (int u = 0; u < kDma; ++u) {
      const uint32_t step = D == 256 ? (uint32_t)(u >> 1) * 8 * (uint32_t)ld + (u & 1) * 256 : (uint32_t)u * (2 * P::kRows) * (uint32_t)ld;
      lds_dma16(r, dst + P::dma_at(x0 + u), off + step, 0);
    }
  };
  auto landed = [] { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  for (int qi = blockIdx.x / p.H; qi < qtiles; qi += gq) {
    const int w0 = (qtiles - 1 - qi) * kCols;  // the last columns have the most keys: first
    const int c0 = w0 + wave * 32;
    // the keys [from, upto) that query i sees
    auto from = [&](int i) { return p.window && i >= p.window ? i - p.window + 1 : 0; };
    auto upto = [&](int i) { return p.causal ? i + 1 : n; };
    const int iw0 = w0 / p.G, iw1 = (min(w0 + kCols, cols) - 1) / p.G;
    const int t_first = from(iw0) / kTile, t_end = (upto(iw1) + kTile - 1) / kTile;
    const int wg_lo = from(iw1), wg_hi = upto(iw0);  // what all of the workgroup's columns see
    // of the wave: what some, and what all of its columns see
    const bool any = c0 < cols;
    const int i0 = c0 / p.G, i1 = any ? (min(c0 + 32, cols) - 1) / p.G : i0;
    const int key_lo = from(i0), key_hi = any ? upto(i1) : 0, all_lo = from(i1), all_hi = any ? upto(i0) : 0;
    // of the lane
    const int x = c0 - i0 * p.G + col, dq = (int)__umulhi((uint32_t)x << 1, p.gmul);
    const int query = i0 + dq, head = h * p.G + x - dq * p.G;
    const bool on = c0 + col < cols;
    const int klo = from(query), khi = on ? upto(query) : 0;

    // So that an iteration uses up a tile of each, K's tiles lie kLead keys behind V's.
    if (kAhead) fetch(kbase, p.ldk, k_off, t_first * kTile, k1);
    fetch(kbase, p.ldk, k_off, t_first * kTile + kLead, k0);
    fetch(vbase, p.ldv, v_off, t_first * kTile, v0);
    v4w qf[KS];
    {
      const uint16_t* qp = p.q + (start + (on ? query : 0)) * p.ldq + (on ? head : h * p.G) * p.hq + half * 8;
#pragma unroll
      for (int w = 0; w < KS; ++w) {
        const v4w z = {0, 0, 0, 0};
        qf[w] = on ? *reinterpret_cast<const v4w*>(qp + 16 * w) : z;
      }
    }
    v16f o[CT], s0, s1 = v16f{};
    uint32_t marks[CT];  // channels that saw what is not finite, a bit each
#pragma unroll
    for (int c = 0; c < CT; ++c) {
      o[c] = v16f{};
      marks[c] = 0;
    }
    float m = -kInf, thr = -kInf, mu = 0.f, l = 0.f;
    auto scores = [&](const unsigned char* kc, int kb) {
      v16f r = v16f{};
#pragma unroll
      for (int w = 0; w < KS; ++w) r = mfma32<DT>(lds_read(kc + k_lane + P::at(32 * kb, 2 * w)), qf[w], r);
      return r;
    };
    landed();
    if (kAhead) {
      s0 = scores(k1, 0);
      landed();
    }

    // Edge tiles, that not all of the workgroup's columns see whole, may hold infinities or NaN that some do not see, and
    // 0 times those is not 0. Where a tile has any, they leave it, and who sees them has its channels marked.
    auto seen = [](int r, int rlo, int rhi) {  // key r of the lane's 16, by its column [rlo, rhi)
      const int at = (r >> 2) * 8 + (r & 3);
      return at >= rlo && at < rhi;
    };
    auto gone = [](uint32_t w) {  // the halves that are not finite
      const uint32_t x = ~w & kExp;
      return ((x & 0xffffu) == 0 ? 0xffffu : 0u) | ((x >> 16) == 0 ? 0xffff0000u : 0u);
    };
    auto clean = [&](int t, unsigned char* vc) {
      uint32_t some = 0;
#pragma unroll
      for (int u = 0; u < kDma; ++u) {
        const v4w w = lds_read(vc + P::dma_at(wave * kDma + u) + lane * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) some |= gone(w[e]);
      }
      if (lane == 0) flags[wave] = 0;
      if (some) flags[wave] = 1;
      __syncthreads();
      int f = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) f |= flags[w];
      if (!f) return;
#pragma unroll 1
      for (int k = 0; k < kTile; k += 32) {
        const int rlo = klo - t * kTile - k - 4 * half, rhi = khi - t * kTile - k - 4 * half;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          v16f hit = v16f{};
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) {
            v4w is, who;
            const unsigned char* vp = vc + v_lane + P::at(16 * s2, 4 * c) + (k ? P::at(32, 0) : 0);
            const v2w a = lds_read_tr(vp), d = lds_read_tr(vp + P::at(8, 0));
            const v4w v = {a.x, a.y, d.x, d.y};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              is[e] = gone(v[e]) & (kOnes | (kOnes << 16));
              who[e] = (seen(8 * s2 + 2 * e, rlo, rhi) ? kOnes : 0u) | (seen(8 * s2 + 2 * e + 1, rlo, rhi) ? kOnes << 16 : 0u);
            }
            hit = mfma32<DT>(is, who, hit);
          }
#pragma unroll
          for (int r = 0; r < 16; ++r) marks[c] |= hit[r] > 0.f ? 1u << r : 0u;
        }
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < kDma; ++u) {
        unsigned char* at = vc + P::dma_at(wave * kDma + u) + lane * 16;
        v4w w = lds_read(at);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] &= ~gone(w[e]);
        *reinterpret_cast<v4w*>(at) = w;
      }
      __syncthreads();
    };

    // the 32 keys from key0: values in block kb of vc. Ahead: S in s, and S of the next 32 keys, in block kb of kc, into
    // sn; else their keys are there.
    auto block = [&](int key0, auto kb_, const unsigned char* kc, const unsigned char* vc, v16f& s, v16f& sn) {
      constexpr int kb = decltype(kb_)::value;
      if (key0 >= key_hi) return;
      v4w ka[KS];
      if constexpr (kAhead) {
#pragma unroll
        for (int w = 0; w < KS; ++w) ka[w] = lds_read(kc + k_lane + P::at(32 * kb, 2 * w));
      } else {
        s = scores(kc, kb);
      }
      if (key0 < all_lo || key0 + 32 > all_hi) {
        const int rlo = klo - key0 - 4 * half, rhi = khi - key0 - 4 * half;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = seen(r, rlo, rhi) ? s[r] : -kInf;
      }
      float top = -kInf;
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
      if (__ballot(top > thr)) {
        const float tp = pair_max(top);
        // a column that has no need keeps its bits, whatever its neighbours do
        const bool need = tp > thr;
        const float mn = need ? fmaxf(m, tp) : m;
        const float was = far_off(m, p.scale), is = far_off(mn, p.scale);
        const float mun = need ? (mn == -kInf || is != 0.f ? 0.f : __builtin_fmaf(mn, p.scale, -kMost)) : mu;
        const float f = m == -kInf ? 1.f : __builtin_amdgcn_exp2f(__builtin_fmaf(was - is, p.scale, mu - mun));
        m = mn;
        mu = mun;
        thr = is != 0.f ? -kInf : mn + 8.f / p.scale;
        l *= f;
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c] *= f;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] -= is;
      }
      auto v_operand = [&](int c, int s2) {
        const v2w a = lds_read_tr(vc + v_lane + P::at(32 * kb + 16 * s2, 4 * c));
        const v2w d = lds_read_tr(vc + v_lane + P::at(32 * kb + 16 * s2 + 8, 4 * c));
        return v4w{a.x, a.y, d.x, d.y};
      };
      v4w va[CT];
      if constexpr (kAhead)
#pragma unroll
        for (int c = 0; c < CT; ++c) va[c] = v_operand(c, 0);
      if constexpr (kAhead) {
        sn = v16f{};
#pragma unroll
        for (int w = 0; w < KS; ++w) sn = mfma32<DT>(ka[w], qf[w], sn);  // behind the last keys: of what was there
      }
      v4w pf[2];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], p.scale, -mu));
        const float c = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r + 1], p.scale, -mu));
        const uint32_t w = pack16<DT>(a, c);
        pf[r >> 3][(r & 7) >> 1] = w;
        l = add_pair<DT>(w, l);
      }
      if constexpr (kAhead) {
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c] = mfma32<DT>(va[c], pf[0], o[c]);
#pragma unroll
        for (int c = 0; c < CT; ++c) va[c] = v_operand(c, 1);
#pragma unroll
        for (int c = 0; c < CT; ++c) o[c] = mfma32<DT>(va[c], pf[1], o[c]);
      } else {
#pragma unroll
        for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
          for (int c = 0; c < CT; ++c) o[c] = mfma32<DT>(v_operand(c, s2), pf[s2], o[c]);
      }
    };
    auto tile = [&](int t, const unsigned char* kc, unsigned char* vc, unsigned char* kn, unsigned char* vn) {
      if (t + 1 < t_end) {
        fetch(vbase, p.ldv, v_off, (t + 1) * kTile, vn);
        fetch(kbase, p.ldk, k_off, (t + 1) * kTile + kLead, kn);
      }
      if (t * kTile < wg_lo || (t + 1) * kTile > wg_hi) clean(t, vc);
      block(t * kTile, std::integral_constant<int, 0>{}, kc, vc, s0, s1);
      if constexpr (kTile == 64) block(t * kTile + 32, std::integral_constant<int, 1>{}, kc, vc, s1, s0);
      landed();
    };
    for (int t = t_first; t < t_end; t += 2) {
      tile(t, k0, v0, k1, v1);
      if (t + 1 < t_end) tile(t + 1, k1, v1, k0, v0);
    }

    l = pair_sum(l);
    if (on) {
      const float inv = l == 0.f ? 0.f : 1.f / l;  // no key seen: 0
      uint16_t* op = p.out + (start + query) * p.ldo + head * p.ho + half * 4;
#pragma unroll
      for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
#pragma unroll
          for (int e = r; e < r + 4; ++e) o[c][e] = marks[c] >> e & 1 ? __builtin_nanf("") : o[c][e];
          const v2w u = {pack16<DT>(o[c][r] * inv, o[c][r + 1] * inv), pack16<DT>(o[c][r + 2] * inv, o[c][r + 3] * inv)};
          *reinterpret_cast<v2w*>(op + c * 32 + 2 * r) = u;
        }
      if (p.lse && half == 0) {
        const float is = far_off(m, p.scale);
        p.lse[(start + query) * (int64_t)(p.H * p.G) + head] =
            l == 0.f ? -kInf : (is != 0.f ? is * p.scale : mu) * 0.69314718055994531f + logf(l);
      }
    }
  }
}

template <int D, int DT>
static int launch_dt(const PromptAttn& p, int64_t max_q, hipStream_t st) {
  constexpr int NW = D == 256 ? 8 : 4;
  const int64_t tiles = (max_q * p.G + 32 * NW - 1) / (32 * NW);
  if (tiles * p.H > kMaxGrid / 2) return kErrUnsupported;
  const dim3 g((unsigned)(tiles * p.H), (unsigned)p.B);
  hipLaunchKernelGGL((prompt_attn_kernel<D, DT, NW>), g, dim3(64 * NW), 0, st, p);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

int launch_prompt_attention(const PromptAttn& p, int D, int dtype, int64_t max_q, hipStream_t st) {
  // a bound below the mean or past all rows is wrong: the grid would grow with it
  if (max_q < (p.T + p.B - 1) / p.B) max_q = (p.T + p.B - 1) / p.B;
  if (max_q > p.T) max_q = p.T;
  if (dtype == kBF16)
    return D == 64 ? launch_dt<64, kBF16>(p, max_q, st)
                   : D == 128 ? launch_dt<128, kBF16>(p, max_q, st) : launch_dt<256, kBF16>(p, max_q, st);
  return D == 64 ? launch_dt<64, kF16>(p, max_q, st)
                 : D == 128 ? launch_dt<128, kF16>(p, max_q, st) : launch_dt<256, kF16>(p, max_q, st);
}

}  // namespace w4a8
