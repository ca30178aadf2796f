// Attention over whole prompts, packed: every key is a new token's, in 16 bits, in the same call.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(scale log2(e) q k_j - M),  j over the keys that the row sees.
//
// The queries that share a key/value head are columns: column c of a sequence is its query c / G, head h G + c % G, so
// 256 columns are 256 / G neighbouring queries, which see almost the same keys. A wave has 32 columns; per 32 keys
//   S = K Q^T (32x32x16, keys are rows),  P = exp of S,  O += V^T P (channels are rows).
// A lane's 16 values of S are one column's, and P's operand wants 8 keys of one column in a lane: any 8, as long as V's
// operand has the same. So P stays in its registers; V's operand comes from LDS by transposed reads.
// K and V tiles of 64 keys go from memory straight into LDS (LDS-DMA), the next one while this one is worked on. A
// DMA lane's 16 bytes land side by side; which 16 bytes those are is free. They are put so that 4 rows times 64 bytes
// lie together, and groups of 4 rows 16 bytes off a multiple of 256: both kinds of read then meet every bank once, at
// addresses that are one register and a constant.
// The running maximum is raised only when a score passes it by 8 (in powers of two): p stays below 2^8, and most tiles
// need neither an exchange between lanes nor a rescaling of O. Sums and O are f32; p is rounded to the type for its
// product (by at most 2^-8 of itself for bf16, 2^-11 for fp16; sum p is of the unrounded ones), as v is.
#include "prompt_attn.h"

namespace w4a8 {

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));
typedef uint32_t v2w __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((__vector_size__(8)));

constexpr int kTile = 64;  // keys

template <int DT>
__device__ __forceinline__ v16f mfma32(const v4w& a, const v4w& b, const v16f& c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2b));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2h));
}

// over the two lanes that hold a column (xor 32)
__device__ __forceinline__ float pair_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// the maximum m itself where m times its factor is past what one f32 number holds to within 1, else 0
__device__ __forceinline__ float far_off(float m, float sc) {
  return fabsf(m) * sc >= 16777216.f && m != -__builtin_inff() ? m : 0.f;
}

// Where the 16 bytes `chunk` (8 channels) of row `r` lie in a tile of D channels, for the DMA and both kinds of read
template <int D>
struct Place {
  // rows of 64 channels come 8 to a DMA; the second 4 of them swap neighbouring chunks
  static constexpr int kGroup = D == 64 ? 1024 + 32 : 8 * D + 16;  // bytes from one group of rows to the next
  static constexpr int kRows = D == 64 ? 8 : 4;                    // rows of a group
  static constexpr int kBytes = kTile / kRows * kGroup;
  static constexpr int kDmas = kTile * D / 8 / 64;                 // wave-wide DMAs of a tile
  static __device__ __forceinline__ constexpr int at(int r, int chunk) {
    if (D == 64)
      return (r >> 3) * kGroup + ((r >> 2) & 1) * 512 + (chunk >> 2) * 256 + (r & 3) * 64 + ((chunk & 3) ^ ((r >> 2) & 1)) * 16;
    return (r >> 2) * kGroup + (chunk >> 2) * 256 + (r & 3) * 64 + (chunk & 3) * 16;
  }
  // DMA x's place in LDS, and the row and chunk that its lane brings there
  static __device__ __forceinline__ constexpr int dma_at(int x) {
    return D == 256 ? (x >> 1) * kGroup + (x & 1) * 1024 : x * kGroup;
  }
  static __device__ __forceinline__ int dma_row(int x, int lane) {
    return D == 64 ? x * 8 + ((lane >> 5) << 2) + ((lane >> 2) & 3) : (D == 256 ? x >> 1 : x) * 4 + ((lane >> 2) & 3);
  }
  static __device__ __forceinline__ int dma_chunk(int x, int lane) {
    if (D == 64) return ((lane >> 4) & 1) * 4 + ((lane & 3) ^ (lane >> 5));
    return (D == 256 ? (x & 1) * 16 : 0) + (lane >> 4) * 4 + (lane & 3);
  }
};

__device__ __forceinline__ v4w lds_read(const unsigned char* p) { return *reinterpret_cast<const v4w*>(p); }
// 4 keys of this lane's channel: the 16 lanes of a group give the addresses of 4 rows times 16 channels
__device__ __forceinline__ v2w lds_read_tr(const unsigned char* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(v2w, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p));
#else
  return v2w{0, 0};
#endif
}

// D: channels; DT: the type; NW: waves
template <int D, int DT, int NW>
__global__ void __launch_bounds__(64 * NW, D == 256 ? 1 : 2)
prompt_attn_kernel(const PromptAttn p) {
  using P = Place<D>;
  constexpr int KS = D / 16, CT = D / 32;       // steps of S, tiles of 32 channels
  constexpr int kDma = P::kDmas / NW;           // DMAs of a wave and tile
  static_assert(P::kDmas % NW == 0, "every wave has the same");
  constexpr int kCols = 32 * NW;
  constexpr float kInf = __builtin_inff();
  constexpr uint32_t kExp = DT == kBF16 ? 0x7f807f80u : 0x7c007c00u;  // exponents of two values
  constexpr uint32_t kOnes = DT == kBF16 ? 0x3f80u : 0x3c00u;
  __shared__ __align__(16) unsigned char k0[P::kBytes];
  __shared__ __align__(16) unsigned char k1[P::kBytes];
  __shared__ __align__(16) unsigned char v0[P::kBytes];
  __shared__ __align__(16) unsigned char v1[P::kBytes];
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

  auto fetch = [&](const uint16_t* base, int64_t ld, int t, unsigned char* dst) {
    const int rows = min(kTile, n - t * kTile);  // rows past the end are zeros in LDS
    const BufRsrc r = make_rsrc(base + (int64_t)t * kTile * ld, (uint32_t)(((rows - 1) * (int)ld + D) * 2));
#pragma unroll
    for (int u = 0; u < kDma; ++u) {
      const int x = wave * kDma + u;
      lds_dma16(r, dst + P::dma_at(x), (uint32_t)(P::dma_row(x, lane) * (int)ld * 2 + P::dma_chunk(x, lane) * 16), 0);
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
    // of the wave: what some, and what all of its columns see
    const bool any = c0 < cols;
    const int i0 = c0 / p.G, i1 = any ? (min(c0 + 32, cols) - 1) / p.G : i0;
    const int key_lo = from(i0), key_hi = any ? upto(i1) : 0, all_lo = from(i1), all_hi = any ? upto(i0) : 0;
    // of the lane
    const int x = c0 - i0 * p.G + col, dq = (int)__umulhi((uint32_t)x << 1, p.gmul);
    const int query = i0 + dq, head = h * p.G + x - dq * p.G;
    const bool on = c0 + col < cols;
    const int klo = from(query), khi = on ? upto(query) : 0;

    fetch(kbase, p.ldk, t_first, k0);
    fetch(vbase, p.ldv, t_first, v0);
    v4w qf[KS];
    {
      const uint16_t* qp = p.q + (start + (on ? query : 0)) * p.ldq + (on ? head : h * p.G) * p.hq + half * 8;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const v4w z = {0, 0, 0, 0};
        qf[s] = on ? *reinterpret_cast<const v4w*>(qp + 16 * s) : z;
      }
    }
    v16f o[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) o[c] = v16f{};
    float m = -kInf, thr = -kInf, mu = 0.f, l = 0.f;
    landed();

    auto tile = [&](int t, const unsigned char* kc, const unsigned char* vc, unsigned char* kn, unsigned char* vn) {
      if (t + 1 < t_end) {
        fetch(kbase, p.ldk, t + 1, kn);
        fetch(vbase, p.ldv, t + 1, vn);
      }
      const int key0 = t * kTile;
      if (key0 < key_hi && key0 + kTile > key_lo) {
        v16f s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[kb] = v16f{};
#pragma unroll
          for (int w = 0; w < KS; ++w)
            s[kb] = mfma32<DT>(lds_read(kc + k_lane + P::at(32 * kb, 2 * w)), qf[w], s[kb]);
        }
        const bool full = key0 >= all_lo && key0 + kTile <= all_hi;
        bool bad = false;  // an infinity or a NaN in V that some column may not see
        // key r of the lane's in block kb, seen by its column [rlo, rhi)
        auto seen = [](int kb, int r, int rlo, int rhi) {
          const int at = kb * 32 + (r >> 2) * 8 + (r & 3);
          return at >= rlo && at < rhi;
        };
        if (!full) {
          typedef unsigned short v2us __attribute__((ext_vector_type(2)));
          v2us least = {0xffff, 0xffff};
          for (int i = 0; i < P::kDmas; ++i) {
            const v4w u = lds_read(vc + P::dma_at(i) + lane * 16);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              least = __builtin_elementwise_min(least, __builtin_bit_cast(v2us, ~u[e] & kExp));
          }
          const int rlo = klo - key0 - 4 * half, rhi = khi - key0 - 4 * half;
          bad = __ballot(least[0] == 0 || least[1] == 0) != 0;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] = seen(kb, r, rlo, rhi) ? s[kb][r] : -kInf;
        }
        float top = -kInf;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
        if (__ballot(top > thr)) {
          const float tp = pair_max(top);
          // a column that has no need keeps its bits, whatever its neighbours do
          const bool need = tp > thr;
          const float mn = need ? fmaxf(m, tp) : m;
          const float was = far_off(m, p.scale), is = far_off(mn, p.scale);
          const float mun = need ? (mn == -kInf || is != 0.f ? 0.f : mn * p.scale) : mu;
          const float f = m == -kInf ? 1.f : __builtin_amdgcn_exp2f(__builtin_fmaf(was - is, p.scale, mu - mun));
          m = mn;
          mu = mun;
          thr = is != 0.f ? -kInf : mn + 8.f / p.scale;
          l *= f;
#pragma unroll
          for (int c = 0; c < CT; ++c) o[c] *= f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[kb][r] -= is;
        }
        v4w pf[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; r += 2) {
            const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], p.scale, -mu));
            const float c = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r + 1], p.scale, -mu));
            l += a;
            l += c;
            pf[kb][r >> 3][(r & 7) >> 1] = pack16<DT>(a, c);
          }
        auto v_operand = [&](int c, int kb, int s2) {
          const v2w a = lds_read_tr(vc + v_lane + P::at(32 * kb + 16 * s2, 4 * c));
          const v2w d = lds_read_tr(vc + v_lane + P::at(32 * kb + 16 * s2 + 8, 4 * c));
          return v4w{a.x, a.y, d.x, d.y};
        };
        if (!bad) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
              for (int c = 0; c < CT; ++c) o[c] = mfma32<DT>(v_operand(c, kb, s2), pf[kb][s2], o[c]);
        } else {
          // 0 times what is not finite is not 0: such values leave the product, and a product of where they are with
          // who sees them makes NaN of those channels
          int rlo = klo - key0 - 4 * half, rhi = khi - key0 - 4 * half;
          asm volatile("" : "+v"(rlo), "+v"(rhi));  // worked out again: 64 masks would not fit the scalar registers
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            v16f hit = v16f{};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
              for (int s2 = 0; s2 < 2; ++s2) {
                v4w a = v_operand(c, kb, s2), is, who;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const uint32_t x = ~a[e] & kExp;
                  const uint32_t gone = ((x & 0xffffu) == 0 ? 0xffffu : 0u) | ((x >> 16) == 0 ? 0xffff0000u : 0u);
                  a[e] &= ~gone;
                  is[e] = gone & (kOnes | (kOnes << 16));
                  who[e] = (seen(kb, 8 * s2 + 2 * e, rlo, rhi) ? kOnes : 0u) |
                           (seen(kb, 8 * s2 + 2 * e + 1, rlo, rhi) ? kOnes << 16 : 0u);
                }
                o[c] = mfma32<DT>(a, pf[kb][s2], o[c]);
                hit = mfma32<DT>(is, who, hit);
              }
#pragma unroll
            for (int r = 0; r < 16; ++r) o[c][r] = hit[r] > 0.f ? __builtin_nanf("") : o[c][r];
          }
        }
      }
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
  constexpr int NW = D == 256 ? 4 : 8;
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
