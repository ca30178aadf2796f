// Writing new tokens into the 4-bit cache and reading tokens back (layout and formulas: kv4.h).
//
// A vector of D channels is D / 8 lanes with 8 neighbouring channels each, so a wave has 8, 4 or 2 vectors
// side by side (D = 64, 128, 256) and the minimum and maximum of each are 3 to 5 steps between lanes. Both
// are exact, so the codes do not depend on any order.
//
// Append: a wave per block of 8 tokens and head, V's words hold 8 tokens each, so this wave is the only writer
// of its words; tokens of the block that are not new keep their nibbles. Blocks are found from the rows: a row
// leads its block when it is the first new token in it. A wave looks at `rows` rows, 8 of a prompt, which lead one
// block as a rule, or one of a decode step, which leads its own.
// All loads of a block are in flight before the first is used. 6900 prompt tokens x 4 heads of 128 (14 MB in, 4 MB
// out) 14 us, and 7 us to read them back (a wave per token and head, with wave-wide reductions of one vector at a
// time, 35 and 17); 64 decode tokens x 8 heads 5 and 3.3 us. Bound by the chain row -> sequence -> page -> block,
// one dependent read each, and for prompts by the quantizing, 16 vectors a wave at 3.5 waves per SIMD.
#include "kv4.h"

namespace w4a8 {

// the last sequence b with cu[b] <= i, 64 candidates at a time; i is wave-uniform
__device__ __forceinline__ int kv4_sequence(const Kv4Batch& s, int64_t i, int lane) {
  int lo = 0, n = s.B;
  while (n > 1) {
    const int stride = (n + 63) / 64, at = lane * stride;
    const uint64_t below = __ballot(at < n && s.cu[lo + (at < n ? at : 0)] <= i);
    const int k = below ? 63 - __builtin_clzll(below) : 0;
    lo += k * stride;
    n = n - k * stride < stride ? n - k * stride : stride;
  }
  return lo;
}

// the place of row i (a lane's own), given the wave's first row's sequence: its position, whether it is its
// sequence's first row, and how many rows follow it there, itself included. False: no sequence has it.
struct Place {
  int b;
  int64_t pos;
  bool first;
  int left;
};
__device__ __forceinline__ bool kv4_place(const Kv4Batch& s, int b, int64_t i, Place& p) {
  while (b + 1 < s.B && s.cu[b + 1] <= i) ++b;
  int64_t start;
  int n;
  kv4_rows(s, b, start, n);
  if (i < start || i >= start + n) return false;
  p.b = b;
  p.left = (int)(start + n - i);
  p.pos = (int64_t)s.lens[b] - p.left;
  p.first = i == start;
  return true;
}

// maximum over the L lanes of a vector
template <int L>
__device__ __forceinline__ float vector_max(float v) {
  v = fmaxf(v, dpp_f<kDppXor1>(v));
  v = fmaxf(v, dpp_f<kDppXor2>(v));
  v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
  if (L >= 16) v = fmaxf(v, dpp_f<kDppRowMirror>(v));
  if (L == 32) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  }
  return v;
}
// or over the wave's vectors (lanes L apart)
template <int L>
__device__ __forceinline__ uint32_t vectors_or(uint32_t v) {
  if (L == 8) v |= (uint32_t)dpp_i<0x128>((int)v);  // 8 lanes round in a row of 16
  if (L <= 16) {
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = a[0] | a[1];
  }
  auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return b[0] | b[1];
}

// codes of the lane's 8 channels of its vector, with step and least value as stored
template <int L, int dtype>
__device__ __forceinline__ void quantize(const uint4& u, uint32_t (&c)[8], uint32_t& sm) {
  float f[8];
  unpack8(u, dtype, f);
  float lo = f[0], hi = f[0], far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    lo = fminf(lo, f[i]);
    hi = fmaxf(hi, f[i]);
    far = fmaxf(far, __builtin_isfinite(f[i]) ? 0.f : 1.f);
  }
  lo = -vector_max<L>(-lo);
  hi = vector_max<L>(hi);
  far = vector_max<L>(far);
  // the type's own rounding of the step: codes are chosen for the step that readers see
  const float tiny = dtype == kF16 ? 5.9604644775390625e-08f : 1.1754943508222875e-38f;
  const float raw = fmaxf((hi - lo) / 15.0f, fmaxf(hi, -lo) * 6.103515625e-05f);
  const float s = fmaxf(from_dtype(to_dtype(raw, dtype), dtype), tiny);
  const bool good = far == 0.f && __builtin_isfinite(s) && __builtin_isfinite(raw);
  // rint of the correctly rounded quotient. The product with 1 / s is within 2^-21 of it, so it rounds alike
  // wherever it is not that near to a half; the wave divides where a lane is.
  const float inv = __builtin_amdgcn_rcpf(s);
  float r[8];
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float q = (f[i] - lo) * inv;
    r[i] = __builtin_rintf(q);
    near = near || !(fabsf(q - r[i]) < 0.4999f);
  }
  if (__ballot(near))
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __builtin_rintf((f[i] - lo) / s);
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = good ? (uint32_t)fminf(fmaxf(r[i], 0.0f), 15.0f) : 0u;
  const uint32_t nan = dtype == kF16 ? 0x7e007e00u : 0x7fc07fc0u;
  sm = good ? (uint32_t)to_dtype(s, dtype) | ((uint32_t)to_dtype(lo, dtype) << 16) : nan;
}

template <int D, int DT>
__global__ void __launch_bounds__(256)
kv4_append_kernel(const uint16_t* __restrict__ k, int64_t ldk, int64_t hk, const uint16_t* __restrict__ v, int64_t ldv,
                  int64_t hv, Kv4Cache c, Kv4Batch s, int rows) {
  constexpr int L = D / 8, VP = 64 / L, PASS = 8 / VP;  // lanes per vector, vectors per wave, passes for 8 tokens
  const int lane = threadIdx.x & 63;
  const uint32_t id = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t i0 = (int64_t)(id / (uint32_t)c.H) * rows;
  const int h = (int)(id % (uint32_t)c.H);
  if (i0 >= s.T) return;
  Place pl = {};
  const int64_t i = i0 + lane;
  const int b0 = kv4_sequence(s, i0, lane);
  const bool leads = lane < rows && i < s.T && kv4_place(s, b0, i, pl) && pl.pos >= 0 &&
                     ((pl.pos & 7) == 0 || pl.first);
  const int page = leads ? kv4_page(c, s, pl.b, pl.pos) : -1;
  uint64_t todo = __ballot(leads && page >= 0);
  const int tok0 = lane / L, ch = (lane & (L - 1)) * 8;
  for (; todo; todo &= todo - 1) {
    const int x = __builtin_ctzll(todo);
    const int pos = __builtin_amdgcn_readlane((int)pl.pos, x);
    const int left = __builtin_amdgcn_readlane(pl.left, x);
    const int64_t blk = kv4_block(c, __builtin_amdgcn_readlane(page, x), h, pos & ~7);
    const int j0 = pos & 7, cnt = left < 8 - j0 ? left : 8 - j0;
    const uint16_t* kp = k + (i0 + x) * ldk + h * hk + ch;
    const uint16_t* vp = v + (i0 + x) * ldv + h * hv + ch;
    uint32_t* vd = reinterpret_cast<uint32_t*>(c.v + blk * (4 * D)) + ch;
    uint4 kr[PASS], vr[PASS], old[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
#pragma unroll
    for (int p = 0; p < PASS; ++p) {
      const int tok = p * VP + tok0;  // lanes of tokens that are not there hold the first one's
      kr[p] = *reinterpret_cast<const uint4*>(kp + (tok < cnt ? tok : 0) * ldk);
      vr[p] = *reinterpret_cast<const uint4*>(vp + (tok < cnt ? tok : 0) * ldv);
    }
    if (cnt < 8 && tok0 == 0) {
      old[0] = *reinterpret_cast<const uint4*>(vd);
      old[1] = *reinterpret_cast<const uint4*>(vd + 4);
    }
    uint32_t words[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int p = 0; p < PASS; ++p)
      if (p * VP < cnt) {
        const int tok = p * VP + tok0;
        const bool on = tok < cnt;
        uint32_t cc[8], sm, w = 0;
        quantize<L, DT>(kr[p], cc, sm);
#pragma unroll
        for (int e = 0; e < 8; ++e) w |= cc[e] << (4 * e);
        if (on) {
          *reinterpret_cast<uint32_t*>(c.k + blk * (4 * D) + (j0 + tok) * (D / 2) + ch / 2) = w;
          if (ch == 0) c.ks[blk * 8 + j0 + tok] = sm;
        }
        quantize<L, DT>(vr[p], cc, sm);
        if (on) {
#pragma unroll
          for (int e = 0; e < 8; ++e) words[e] |= cc[e] << (4 * (j0 + tok));
          if (ch == 0) c.vs[blk * 8 + j0 + tok] = sm;
        }
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) words[e] = vectors_or<L>(words[e]);
    if (tok0 == 0) {
      const uint32_t keep = ~((cnt == 8 ? ~0u : (1u << (4 * cnt)) - 1) << (4 * j0));
      const uint32_t o[8] = {old[0].x, old[0].y, old[0].z, old[0].w, old[1].x, old[1].y, old[1].z, old[1].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) words[e] |= o[e] & keep;
      *reinterpret_cast<uint4*>(vd) = make_uint4(words[0], words[1], words[2], words[3]);
      *reinterpret_cast<uint4*>(vd + 4) = make_uint4(words[4], words[5], words[6], words[7]);
    }
  }
}

// Rows of the cache as values in the model's type: s c + m with one rounding to f32 (the product is
// exact) and one to the type. A row without a place in the cache (before the sequence's first token,
// on a page that does not exist) is NaN. A vector per D / 8 lanes, heads of a row side by side.
template <int D, int DT>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4Cache c, Kv4Batch s, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
  constexpr int L = D / 8, VP = 64 / L;
  const int lane = threadIdx.x & 63;
  const uint32_t id0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * VP;
  if (id0 >= s.T * c.H) return;
  const int b0 = kv4_sequence(s, id0 / (uint32_t)c.H, lane);
  const uint32_t id = id0 + lane / L;
  const int64_t i = id / (uint32_t)c.H;
  const int h = (int)(id % (uint32_t)c.H), ch = (lane & (L - 1)) * 8;
  Place pl;
  if (i >= s.T || !kv4_place(s, b0, i, pl)) return;
  const int page = kv4_page(c, s, pl.b, pl.pos);
  uint32_t ks = DT == kF16 ? 0x7e007e00u : 0x7fc07fc0u, vs = ks, kc = 0, vc[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  const int j = (int)(pl.pos & 7);
  if (page >= 0) {
    const int64_t blk = kv4_block(c, page, h, (int)(pl.pos & ~(int64_t)7));
    const uint4* vd = reinterpret_cast<const uint4*>(c.v + blk * (4 * D) + ch * 4);
    kc = *reinterpret_cast<const uint32_t*>(c.k + blk * (4 * D) + j * (D / 2) + ch / 2);
    const uint4 a = vd[0], b = vd[1];
    vc[0] = a.x; vc[1] = a.y; vc[2] = a.z; vc[3] = a.w;
    vc[4] = b.x; vc[5] = b.y; vc[6] = b.z; vc[7] = b.w;
    ks = c.ks[blk * 8 + j];
    vs = c.vs[blk * 8 + j];
  }
  auto value = [&](uint32_t code, uint32_t sm) {
    return (uint32_t)to_dtype(__builtin_fmaf((float)code, from_dtype((uint16_t)(sm & 0xffffu), DT),
                                             from_dtype((uint16_t)(sm >> 16), DT)), DT);
  };
  uint32_t kw[4], vw[4];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    kw[e / 2] = value((kc >> (4 * e)) & 15u, ks) | (value((kc >> (4 * e + 4)) & 15u, ks) << 16);
    vw[e / 2] = value((vc[e] >> (4 * j)) & 15u, vs) | (value((vc[e + 1] >> (4 * j)) & 15u, vs) << 16);
  }
  *reinterpret_cast<uint4*>(k + (int64_t)id * D + ch) = make_uint4(kw[0], kw[1], kw[2], kw[3]);
  *reinterpret_cast<uint4*>(v + (int64_t)id * D + ch) = make_uint4(vw[0], vw[1], vw[2], vw[3]);
}

template <int DT>
static void append(int D, dim3 g, const uint16_t* k, int64_t ldk, int64_t hk, const uint16_t* v, int64_t ldv, int64_t hv,
                   const Kv4Cache& c, const Kv4Batch& s, int rows, hipStream_t st) {
  if (D == 64) hipLaunchKernelGGL((kv4_append_kernel<64, DT>), g, dim3(256), 0, st, k, ldk, hk, v, ldv, hv, c, s, rows);
  else if (D == 128) hipLaunchKernelGGL((kv4_append_kernel<128, DT>), g, dim3(256), 0, st, k, ldk, hk, v, ldv, hv, c, s, rows);
  else hipLaunchKernelGGL((kv4_append_kernel<256, DT>), g, dim3(256), 0, st, k, ldk, hk, v, ldv, hv, c, s, rows);
}

int launch_kv4_append(const void* k, int64_t ldk, int64_t hk, const void* v, int64_t ldv, int64_t hv, int dtype, int D,
                      const Kv4Cache& c, const Kv4Batch& s, hipStream_t st) {
  // one row per wave while that many waves (8192) fill the card no more than once
  const int rows = s.T * c.H <= 8192 ? 1 : 8;
  const int64_t wgs = ((s.T + rows - 1) / rows * c.H + 3) / 4;
  if (wgs > kMaxGrid) return kErrUnsupported;
  const dim3 g((unsigned)wgs);
  auto kp = reinterpret_cast<const uint16_t*>(k), vp = reinterpret_cast<const uint16_t*>(v);
  if (dtype == kBF16) append<kBF16>(D, g, kp, ldk, hk, vp, ldv, hv, c, s, rows, st);
  else append<kF16>(D, g, kp, ldk, hk, vp, ldv, hv, c, s, rows, st);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

template <int DT>
static void read(int D, dim3 g, const Kv4Cache& c, const Kv4Batch& s, uint16_t* k, uint16_t* v, hipStream_t st) {
  if (D == 64) hipLaunchKernelGGL((kv4_read_kernel<64, DT>), g, dim3(256), 0, st, c, s, k, v);
  else if (D == 128) hipLaunchKernelGGL((kv4_read_kernel<128, DT>), g, dim3(256), 0, st, c, s, k, v);
  else hipLaunchKernelGGL((kv4_read_kernel<256, DT>), g, dim3(256), 0, st, c, s, k, v);
}

int launch_kv4_read(const Kv4Cache& c, const Kv4Batch& s, int dtype, int D, void* k, void* v, hipStream_t st) {
  const int per = 4 * 512 / D;  // vectors per workgroup
  const int64_t wgs = (s.T * c.H + per - 1) / per;
  if (wgs > kMaxGrid) return kErrUnsupported;
  const dim3 g((unsigned)wgs);
  auto kp = reinterpret_cast<uint16_t*>(k), vp = reinterpret_cast<uint16_t*>(v);
  if (dtype == kBF16) read<kBF16>(D, g, c, s, kp, vp, st);
  else read<kF16>(D, g, c, s, kp, vp, st);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

}  // namespace w4a8
