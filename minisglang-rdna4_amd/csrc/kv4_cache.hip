// Writing new tokens into the 4-bit cache and reading tokens back (layout and formulas: kv4.h).
//
// A wave per (block of 8 tokens, head), found from the rows: the wave of the first new token in a block
// does that block's new tokens, the waves of the others return. V's words hold 8 tokens each, so this
// wave is the only writer of its words; tokens of the block that are not new keep their nibbles.
// Each lane holds E neighbouring channels of up to 8 tokens, all loaded before the first is used; the
// minimum and the maximum of a vector are wave reductions. Both are exact, so the codes do not depend
// on any order.
#include "kv4.h"

namespace w4a8 {

__device__ __forceinline__ float wave_min(float v) { return -wave_max(-v); }

// the sequence whose rows hold row i: the last b with cu[b] <= i
__device__ __forceinline__ int kv4_sequence(const Kv4Batch& s, int64_t i) {
  int lo = 0, hi = s.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s.cu[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}

template <int E>
__device__ __forceinline__ void load_e(const uint16_t* p, uint32_t (&w)[E / 2]) {
  if constexpr (E == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else { const uint2 u = *reinterpret_cast<const uint2*>(p); w[0] = u.x; w[1] = u.y; }
}

// codes of the wave's vector (x in this lane's channels), step and least value packed as stored
template <int E>
__device__ __forceinline__ void quantize(const uint32_t (&w)[E / 2], int dtype, bool on, uint32_t (&c)[E], uint32_t& sm) {
  float f[E];
#pragma unroll
  for (int i = 0; i < E; ++i) f[i] = from_dtype((uint16_t)(w[i / 2] >> (16 * (i & 1))), dtype);
  float lo = f[0], hi = f[0];
  bool fin = true;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    lo = fminf(lo, f[i]);
    hi = fmaxf(hi, f[i]);
    fin = fin && __builtin_isfinite(f[i]);
  }
  const float kInf = __builtin_inff();
  lo = wave_min(on ? lo : kInf);
  hi = wave_max(on ? hi : -kInf);
  // the type's own rounding of the step: codes are chosen for the step that readers see
  const float tiny = dtype == kF16 ? 5.9604644775390625e-08f : 1.1754943508222875e-38f;
  const float raw = fmaxf((hi - lo) / 15.0f, fmaxf(hi, -lo) * 6.103515625e-05f);
  const float s = fmaxf(from_dtype(to_dtype(raw, dtype), dtype), tiny);
  const bool good = __ballot(on && !fin) == 0 && __builtin_isfinite(s) && __builtin_isfinite(raw);
#pragma unroll
  for (int i = 0; i < E; ++i)
    c[i] = good ? (uint32_t)fminf(fmaxf(__builtin_rintf((f[i] - lo) / s), 0.0f), 15.0f) : 0u;
  const uint32_t nan = dtype == kF16 ? 0x7e007e00u : 0x7fc07fc0u;
  sm = good ? (uint32_t)to_dtype(s, dtype) | ((uint32_t)to_dtype(lo, dtype) << 16) : nan;
}

template <int D>
__global__ void __launch_bounds__(256)
kv4_append_kernel(const uint16_t* __restrict__ k, int64_t ldk, int64_t hk, const uint16_t* __restrict__ v, int64_t ldv,
                  int64_t hv, int dtype, Kv4Cache c, Kv4Batch s) {
  constexpr int E = D == 256 ? 4 : 2, NL = D / E;
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t i = id / c.H;
  const int h = (int)(id - i * c.H);
  if (i >= s.T) return;
  const int b = kv4_sequence(s, i);
  int64_t start;
  int n;
  kv4_rows(s, b, start, n);
  if (i < start || i >= start + n) return;
  const int64_t pos = s.lens[b] - (start + n - i);
  if (pos < 0 || !((pos & 7) == 0 || i == start)) return;
  const int page = kv4_page(c, s, b, pos);
  if (page < 0) return;
  const int j0 = (int)(pos & 7);
  const int cnt = (int)(start + n - i < 8 - j0 ? start + n - i : 8 - j0);
  const bool on = lane < NL;
  const int ch = (on ? lane : 0) * E;

  uint32_t kw[8][E / 2], vw[8][E / 2];
  const uint16_t* kp = k + i * ldk + h * hk + ch;
  const uint16_t* vp = v + i * ldv + h * hv + ch;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < cnt) {
      load_e<E>(kp + j * ldk, kw[j]);
      load_e<E>(vp + j * ldv, vw[j]);
    }
  const int64_t blk = kv4_block(c, page, h, (int)(pos & ~(int64_t)7 & ((1 << c.shift) - 1)));
  uint8_t* kd = c.k + blk * (4 * D);
  uint32_t* vd = reinterpret_cast<uint32_t*>(c.v + blk * (4 * D)) + ch;
  uint32_t words[E];
#pragma unroll
  for (int e = 0; e < E; ++e) words[e] = cnt < 8 && on ? vd[e] : 0u;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < cnt) {
      uint32_t cc[E], sm;
      quantize<E>(kw[j], dtype, on, cc, sm);
      uint8_t* row = kd + (j0 + j) * (D / 2) + ch / 2;
      if (on) {
        if constexpr (E == 2) *row = (uint8_t)(cc[0] | (cc[1] << 4));
        else *reinterpret_cast<uint16_t*>(row) = (uint16_t)(cc[0] | (cc[1] << 4) | (cc[2] << 8) | (cc[3] << 12));
      }
      if (lane == 0) c.ks[blk * 8 + j0 + j] = sm;
      quantize<E>(vw[j], dtype, on, cc, sm);
#pragma unroll
      for (int e = 0; e < E; ++e)
        words[e] = (words[e] & ~(15u << (4 * (j0 + j)))) | (cc[e] << (4 * (j0 + j)));
      if (lane == 0) c.vs[blk * 8 + j0 + j] = sm;
    }
  if (on)
#pragma unroll
    for (int e = 0; e < E; ++e) vd[e] = words[e];
}

// Rows of the cache as values in the model's type: s c + m with one rounding to f32 (the product is
// exact) and one to the type. A row without a place in the cache (before the sequence's first token,
// on a page that does not exist) is NaN.
template <int D>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4Cache c, Kv4Batch s, int dtype, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
  constexpr int E = D == 256 ? 4 : 2, NL = D / E;
  const int lane = threadIdx.x & 63;
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t i = id / c.H;
  const int h = (int)(id - i * c.H);
  if (i >= s.T || lane >= NL) return;
  const int b = kv4_sequence(s, i);
  int64_t start;
  int n;
  kv4_rows(s, b, start, n);
  if (i < start || i >= start + n) return;
  const int64_t pos = s.lens[b] - (start + n - i);
  const int page = kv4_page(c, s, b, pos);
  const int ch = lane * E;
  uint32_t kc[E], vc[E], ks, vs;
  if (page < 0) {
    ks = vs = dtype == kF16 ? 0x7e007e00u : 0x7fc07fc0u;
#pragma unroll
    for (int e = 0; e < E; ++e) kc[e] = vc[e] = 0;
  } else {
    const int j = (int)(pos & 7);
    const int64_t blk = kv4_block(c, page, h, (int)(pos & ~(int64_t)7 & ((1 << c.shift) - 1)));
    const uint8_t* row = c.k + blk * (4 * D) + j * (D / 2) + ch / 2;
    const uint32_t* vd = reinterpret_cast<const uint32_t*>(c.v + blk * (4 * D)) + ch;
    ks = c.ks[blk * 8 + j];
    vs = c.vs[blk * 8 + j];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      kc[e] = (row[e / 2] >> (4 * (e & 1))) & 15u;
      vc[e] = (vd[e] >> (4 * j)) & 15u;
    }
  }
  const int64_t at = (i * c.H + h) * D + ch;
  auto put = [&](uint16_t* o, const uint32_t (&cc)[E], uint32_t sm) {
    const float st = from_dtype((uint16_t)(sm & 0xffffu), dtype), m = from_dtype((uint16_t)(sm >> 16), dtype);
    uint32_t w[E / 2];
#pragma unroll
    for (int e = 0; e < E; e += 2)
      w[e / 2] = (uint32_t)to_dtype(__builtin_fmaf((float)cc[e], st, m), dtype) |
                 ((uint32_t)to_dtype(__builtin_fmaf((float)cc[e + 1], st, m), dtype) << 16);
    if constexpr (E == 2) *reinterpret_cast<uint32_t*>(o + at) = w[0];
    else *reinterpret_cast<uint2*>(o + at) = make_uint2(w[0], w[1]);
  };
  put(k, kc, ks);
  put(v, vc, vs);
}

int launch_kv4_append(const void* k, int64_t ldk, int64_t hk, const void* v, int64_t ldv, int64_t hv, int dtype, int D,
                      const Kv4Cache& c, const Kv4Batch& s, hipStream_t st) {
  const dim3 g((unsigned)((s.T * c.H + 3) / 4));
  auto kp = reinterpret_cast<const uint16_t*>(k), vp = reinterpret_cast<const uint16_t*>(v);
  if (D == 64) hipLaunchKernelGGL(kv4_append_kernel<64>, g, dim3(256), 0, st, kp, ldk, hk, vp, ldv, hv, dtype, c, s);
  else if (D == 128) hipLaunchKernelGGL(kv4_append_kernel<128>, g, dim3(256), 0, st, kp, ldk, hk, vp, ldv, hv, dtype, c, s);
  else hipLaunchKernelGGL(kv4_append_kernel<256>, g, dim3(256), 0, st, kp, ldk, hk, vp, ldv, hv, dtype, c, s);
  return hipGetLastError() == hipSuccess ? kOk : kErrHip;
}

int launch_kv4_read(const Kv4Cache& c, const Kv4Batch& s, int dtype, int D, void* k, void* v, hipStream_t st) {
  const dim3 g((unsigned)((s.T * c.H + 3) / 4));
  auto kp = reinterpret_cast<uint16_t*>(k), vp = reinterpret_cast<uint16_t*>(v);
  if (D == 64) hipLaunchKernelGGL(kv4_read_kernel<64>, g, dim3(256), 0, st, c, s, dtype, kp, vp);
  else if (D == 128) hipLaunchKernelGGL(kv4_read_kernel<128>, g, dim3(256), 0, st, c, s, dtype, kp, vp);
  else hipLaunchKernelGGL(kv4_read_kernel<256>, g, dim3(256), 0, st, c, s, dtype, kp, vp);
  return hipGetLastError() == hipSuccess ? kOk : kErrHip;
}

}  // namespace w4a8
