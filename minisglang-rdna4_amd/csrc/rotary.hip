// Rotary positions: pair i of a head's first R channels, (x[i], x[i + R/2]) or (x[2i], x[2i + 1]), is turned by
// t = position[axis(i)] f_i:   a' = s (a cos t - b sin t),  b' = s (a sin t + b cos t).
//
// Angles. Positions are whole numbers, so t in turns is position * (f_i / 2 pi) modulo 1, and with f_i / 2 pi as a
// fraction of 2^64 that is one 64-bit integer product that overflows as it should and rounds nothing: off by the position times
// the fraction's 2^-65, where an f32 product is off by 4e-3 at position 131072. Its upper 32 bits are cut into quarters of a turn and a rest within an
// eighth, whose sine and cosine are Taylor's polynomials (to x^9 and x^10: the next terms are below 2e-9 and 2e-10).
//
// A thread has one token and one unit of 8 pairs, 16 bytes each of a and b, works its 8 angles out once, and turns that
// unit in `per` heads. Bound by memory for prompts (8191 tokens of 40 heads of 128, 168 MB in and out: 34 to 40 us, 4.2 to 5
// TB/s), by the launch for decode (3.5 us).
#include "rotary.h"

namespace w4a8 {

__device__ __forceinline__ void sincos_turn(uint32_t turn, float& s, float& c) {
  const uint32_t quarter = (turn + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(turn - (quarter << 30)) * 1.4629180792671596e-9f;  // 2 pi / 2^32: within pi / 4
  const float y = x * x;
  float sn = __builtin_fmaf(y, 2.7557319e-6f, -1.9841270e-4f);
  sn = __builtin_fmaf(y, sn, 8.3333333e-3f);
  sn = __builtin_fmaf(y, sn, -1.6666667e-1f);
  sn = __builtin_fmaf(y * x, sn, x);
  float cs = __builtin_fmaf(y, -2.7557319e-7f, 2.4801587e-5f);
  cs = __builtin_fmaf(y, cs, -1.3888889e-3f);
  cs = __builtin_fmaf(y, cs, 4.1666667e-2f);
  cs = __builtin_fmaf(y, cs, -0.5f);
  cs = __builtin_fmaf(y, cs, 1.f);
  const bool swap = quarter & 1;
  s = swap ? cs : sn;
  c = swap ? sn : cs;
  s = quarter & 2 ? -s : s;
  c = (quarter + 1) & 2 ? -c : c;
}

template <int DT>
__device__ __forceinline__ v4u pack8(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)to_dtype(f[2 * i], DT) | ((uint32_t)to_dtype(f[2 * i + 1], DT) << 16);
  return v4u{w[0], w[1], w[2], w[3]};
}

constexpr int kHeads = 4;  // of a thread, at most

template <int DT, bool ADJ, bool NT>
__global__ void __launch_bounds__(256)
rotary_kernel(const Rotary p) {
  const int groups = (p.heads + p.per - 1) / p.per;  // of heads
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t rest = id / p.units;
  const int unit = (int)(id - rest * p.units);
  const int64_t t = rest / groups;
  const int h0 = (int)(rest - t * groups) * p.per;
  if (t >= p.T) return;
  const int h1 = min(h0 + p.per, p.heads);
  auto at = [&](int h, const uint16_t*& in, uint16_t*& out) {
    const bool q = h < p.q.heads;
    const RotaryRows& r = q ? p.q : p.k;
    const int hh = q ? h : h - p.q.heads;
    in = r.in + t * r.ldi + hh * r.hi;
    out = r.out + t * r.ldo + hh * r.ho;
  };
  const int turning = p.R / 16;
  if (unit >= turning) {  // channels behind R: as they are
    const int c = p.R + (unit - turning) * 8;
    for (int h = h0; h < h1; ++h) {
      const uint16_t* in;
      uint16_t* out;
      at(h, in, out);
      *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(in + c);
    }
    return;
  }
  const int ca = ADJ ? unit * 16 : unit * 8, cb = ADJ ? ca + 8 : p.R / 2 + ca;
  v4u a[kHeads], b[kHeads];
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {  // before the angles, which take a chain of reads too
    const uint16_t* in;
    uint16_t* out;
    at(min(h0 + u, h1 - 1), in, out);
    a[u] = stream_read<NT>(in + ca);
    b[u] = stream_read<NT>(in + cb);
  }
  float sn[8], cs[8];
  auto position = [&](int axis) -> uint64_t {
    const int64_t i = axis * p.ldp + t;
    return p.pos64 ? static_cast<const uint64_t*>(p.pos)[i] : (uint64_t)(int64_t) static_cast<const int32_t*>(p.pos)[i];
  };
  const uint64_t first = p.axis ? 0 : position(0);
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int i = unit * 8 + e;
    const uint64_t pos = p.axis ? position(p.axis[i]) : first;
    sincos_turn((uint32_t)((pos * p.turn[i]) >> 32), sn[e], cs[e]);
    sn[e] *= p.scale;
    cs[e] *= p.scale;
  }
#pragma unroll
  for (int u = 0; u < kHeads; ++u) {
    if (h0 + u >= h1) break;
    float x[8], y[8], v[8], w[8];
    unpack8(make_uint4(a[u].x, a[u].y, a[u].z, a[u].w), DT, x);
    unpack8(make_uint4(b[u].x, b[u].y, b[u].z, b[u].w), DT, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if constexpr (ADJ) {
        float* src = e < 4 ? x : y;
        float* dst = e < 4 ? v : w;
        const int j = 2 * (e & 3);
        dst[j] = __builtin_fmaf(src[j], cs[e], -(src[j + 1] * sn[e]));
        dst[j + 1] = __builtin_fmaf(src[j], sn[e], src[j + 1] * cs[e]);
      } else {
        v[e] = __builtin_fmaf(x[e], cs[e], -(y[e] * sn[e]));
        w[e] = __builtin_fmaf(x[e], sn[e], y[e] * cs[e]);
      }
    }
    const uint16_t* in;
    uint16_t* out;
    at(h0 + u, in, out);
    stream_write<NT>(out + ca, pack8<DT>(v));
    stream_write<NT>(out + cb, pack8<DT>(w));
  }
}

template <bool NT>
static void launch(const Rotary& p, int dtype, dim3 g, hipStream_t st) {
  const dim3 b(256);
  if (dtype == kBF16) {
    if (p.adjacent) hipLaunchKernelGGL((rotary_kernel<kBF16, true, NT>), g, b, 0, st, p);
    else hipLaunchKernelGGL((rotary_kernel<kBF16, false, NT>), g, b, 0, st, p);
  } else {
    if (p.adjacent) hipLaunchKernelGGL((rotary_kernel<kF16, true, NT>), g, b, 0, st, p);
    else hipLaunchKernelGGL((rotary_kernel<kF16, false, NT>), g, b, 0, st, p);
  }
}

int launch_rotary(Rotary& p, int D, int dtype, hipStream_t st) {
  p.heads = p.q.heads + p.k.heads;
  const bool rest = p.R < D && (p.q.in != p.q.out || (p.k.heads && p.k.in != p.k.out));  // in place they stay
  p.units = p.R / 16 + (rest ? (D - p.R) / 8 : 0);
  // more heads a thread while the card stays full (8 waves per SIMD: 524288 threads); 8 in flight 45 us
  const int64_t rows = p.T * p.heads * p.units;
  p.per = (int)(rows / 524288 < 1 ? 1 : rows / 524288 > kHeads ? kHeads : rows / 524288);
  const int64_t threads = p.T * ((p.heads + p.per - 1) / p.per) * p.units, wgs = (threads + 255) / 256;
  if (wgs > kMaxGrid) return kErrUnsupported;
  // Past the caches where both halves of a head are whole lines of 128 bytes and the rows more than the caches could keep for who
  // reads them next. us, 40 heads, in and out, other rows each time, past / through the caches (kv4_append behind it in
  // brackets): 128 channels 42 MB 18.0 / 15.7 (26.9 / 24.5), 84 MB 22.7 / 21.8 (36.0 / 35.1), 106 MB 25.7 / 26.3 (43.0 / 43.0),
  // 168 MB 33.5 / 39.8 (55.1 / 60.0). Parts of lines are slower past them at any size: 64 channels 168 MB 42.6 / 40.3,
  // neighbours as pairs 50.3 / 40.8, 96 of 128 channels 50.5 / 49.6.
  if (!p.adjacent && p.R % 128 == 0 && p.T * p.heads * D * 4 > 96 << 20) launch<true>(p, dtype, dim3((unsigned)wgs), st);
  else launch<false>(p, dtype, dim3((unsigned)wgs), st);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

}  // namespace w4a8
