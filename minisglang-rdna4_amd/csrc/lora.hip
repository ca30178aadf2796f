// y = base + scaling[a] (x A_a^T) B_a^T for rows of many adapters: two launches.
//
// A block of 16 rows is the tile of both. Its distinct adapters are found from the ids by ballots and
// taken one after another (or by as many workgroups side by side, `slots`): the tile's product with one
// adapter's matrix, of which only that adapter's rows are kept. Rows come in any order, nothing is
// sorted, and a prompt's blocks have one adapter. Rows of other adapters are dropped by selection,
// never by a zero operand, so that an infinity in one user's weights stays with that user.
//   down: v[m, i] = sum_k x[m, k] A[a, i, k]     f32 partial sums over `kc` parts of K, in a fixed order
//   up:   y[m, n] = base + scaling sum_r v[m, slice * rank + r] B[a, n, r], rounded once
// v keeps f32: it enters the second product as two terms of the model's type (v's first 16 bits for bf16,
// 22 for fp16), scaled by a power of two per row so that neither fp16's range nor its subnormals matter.
#include "lora.h"

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

__device__ __forceinline__ v4w load16(const uint16_t* p, bool on) {
  const uint4 u = on ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
  return v4w{u.x, u.y, u.z, u.w};
}

// The adapters of 16 rows: each lane its row's (lane & 15), and the rows whose adapter is yet to come.
struct Rows {
  int id;
  uint32_t left;
};
__device__ __forceinline__ Rows row_adapters(const LoraArgs& p, int64_t m0, int lane) {
  const int64_t m = m0 + (lane & 15);
  const int id = m < p.M ? p.ids[m] : -1;
  const bool on = id >= 0 && id < p.L;
  return {on ? id : -1, (uint32_t)__ballot(on) & 0xffffu};
}
// the next adapter (wave-uniform); its rows leave `left`
__device__ __forceinline__ int next_adapter(Rows& r) {
  const int a = __builtin_amdgcn_readlane(r.id, __builtin_ctz(r.left));
  r.left &= ~((uint32_t)__ballot(r.id == a) & 0xffffu);
  return a;
}

// grid: (blocks of 16 rows * groups of 16 RB ranks * parts of K, 1, slots). Each of the 4 waves takes every
// fourth 128 inputs of the part: lane (row, g) of an operand holds inputs 32 g .. 32 g + 31 of them, 64
// bytes in a line, as 4 steps; the order of the summed index is free as long as both operands agree.
template <int DT, int RB>
__global__ void __launch_bounds__(256)
lora_down_kernel(const LoraArgs p) {
  __shared__ v4f red[3][RB][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int g = lane >> 4, c = lane & 15;
  const int R = p.slices * p.rank;
  const int groups = (R + 16 * RB - 1) / (16 * RB);
  const uint32_t part = blockIdx.x % (uint32_t)p.kc, tile = blockIdx.x / (uint32_t)p.kc;
  const int64_t m0 = (int64_t)(tile / (uint32_t)groups) * 16;
  const int r0 = (int)(tile % (uint32_t)groups) * 16 * RB;
  const int64_t k0 = (int64_t)part * p.kstep;
  const int64_t k1 = k0 + p.kstep < p.K ? k0 + p.kstep : p.K;
  Rows rows = row_adapters(p, m0, lane);
  for (int i = 0; rows.left; ++i) {
    const int a = next_adapter(rows);
    if (i % (int)gridDim.z != (int)blockIdx.z) continue;
    const bool mine = rows.id == a;
    const uint16_t* xp = p.x + (m0 + (mine ? c : 0)) * p.ldx;
    const uint16_t* ap[RB];
    bool ron[RB];
#pragma unroll
    for (int t = 0; t < RB; ++t) {
      const int r = r0 + 16 * t + c;
      ron[t] = r < R;
      ap[t] = p.a + ((int64_t)a * R + (ron[t] ? r : 0)) * p.K;
    }
    v4f acc[RB];
#pragma unroll
    for (int t = 0; t < RB; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int64_t k = k0 + wave * 128 + g * 32; k < k1 + g * 32; k += 512) {
      v4w xv[4], av[RB][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool in = k + 8 * j < k1;
        xv[j] = load16(xp + k + 8 * j, in && mine);
#pragma unroll
        for (int t = 0; t < RB; ++t) av[t][j] = load16(ap[t] + k + 8 * j, in && ron[t]);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int t = 0; t < RB; ++t) acc[t] = mfma16<DT>(av[t][j], xv[j], acc[t]);
    }
    if (wave)
#pragma unroll
      for (int t = 0; t < RB; ++t) red[wave - 1][t][lane] = acc[t];
    __syncthreads();
    if (wave == 0)
#pragma unroll
      for (int t = 0; t < RB; ++t) {
        const v4f s = (acc[t] + red[0][t][lane]) + (red[1][t][lane] + red[2][t][lane]);
        const int r = r0 + 16 * t + 4 * g;  // rank is a multiple of 8, so are 4 in a row inside R or outside
        if (mine && r < R)
          *reinterpret_cast<v4f*>(p.v + ((int64_t)part * p.M + m0 + c) * R + r) = s;
      }
    __syncthreads();
  }
}

// grid: (4 chunks of 64 columns of one slice * blocks of 16 RB rows, 1, slots). A wave per chunk: row (4 q + i) of
// its j-th product is column 16 q + 4 j + i of the chunk, so a lane ends with 16 neighbouring columns. The
// workgroup first sums the parts of v for its rows and slice, once for its four chunks, into LDS. (The chunks
// of a workgroup are of one slice: launch_lora counts them so.) An adapter's B stays in registers over the RB
// blocks of 16 rows, where its rank is up to 64.
template <int DT, int RB, bool F32>
__global__ void __launch_bounds__(256, RB == 4 ? 2 : 4)
lora_up_kernel(const LoraArgs p) {
  constexpr int kPad = 4;  // floats between rows: the rows of a read start 16 bytes apart, modulo the banks
  extern __shared__ float vs[];  // (16 RB, rank + kPad), then the rows' largest |v|
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const uint32_t quads = (uint32_t)p.chunk[p.slices];
  const uint32_t quad = blockIdx.x % quads;
  int s = 0;
  while (quad >= p.chunk[s + 1]) ++s;
  const int64_t nend = p.col[s + 1];
  const int64_t n0 = p.col[s] + (int64_t)(quad - p.chunk[s]) * 256 + wave * 64;
  const int64_t m0 = (int64_t)(blockIdx.x / quads) * (16 * RB);
  const int R = p.slices * p.rank, ld = p.rank + kPad;
  const bool work = n0 < nend;  // this wave's columns exist (the last workgroup of a slice may have fewer)

  Rows rows[RB];
  uint4 base[RB][F32 ? 4 : 2];
  const int64_t n = n0 + 16 * g;
  const bool cols = work && n < nend;
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    rows[b] = row_adapters(p, m0 + 16 * b, lane);
    const int64_t m = m0 + 16 * b + c;
    if (cols && m < p.M) {
      const uint4* bp = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p.base) + (m * p.ldb + n) * (F32 ? 4 : 2));
#pragma unroll
      for (int j = 0; j < (F32 ? 4 : 2); ++j) base[b][j] = bp[j];
    }
  }
  // v of the rows that this workgroup's slot does: the i-th adapter of the rows is slot i's, modulo the slots
  v4f acc[RB][4];
  bool write[RB], mine_any = false;
#pragma unroll
  for (int b = 0; b < RB; ++b) {
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[b][j] = v4f{0.f, 0.f, 0.f, 0.f};
    write[b] = rows[b].id < 0 && blockIdx.z == 0;  // rows without an adapter are the base itself, the first slot's
  }
  // a row is done by this slot when its adapter's place among the rows' adapters is the slot's
  bool todo[RB];
#pragma unroll
  for (int b = 0; b < RB; ++b) todo[b] = false;
  {
    Rows r[RB];
#pragma unroll
    for (int b = 0; b < RB; ++b) r[b] = rows[b];
    for (int i = 0;; ++i) {
      int a = -1;
#pragma unroll
      for (int b = 0; b < RB; ++b)
        if (a < 0 && r[b].left) a = __builtin_amdgcn_readlane(r[b].id, __builtin_ctz(r[b].left));
      if (a < 0) break;
#pragma unroll
      for (int b = 0; b < RB; ++b) {
        const bool m = r[b].id == a;
        r[b].left &= ~((uint32_t)__ballot(m) & 0xffffu);
        if (i % (int)gridDim.z == (int)blockIdx.z) todo[b] = todo[b] || m;
      }
    }
  }
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    rows[b].left &= (uint32_t)__ballot(todo[b]) & 0xffffu;
    mine_any = mine_any || rows[b].left != 0;
    write[b] = write[b] || todo[b];
  }
  if (mine_any) {
    // four ranks a thread, parts of K in order; rows of other slots are skipped
    const int per = p.rank / 4;
    for (int t = threadIdx.x; t < 16 * RB * per; t += 256) {
      const int row = t / per, r = (t - row * per) * 4;
      uint32_t left = 0;
#pragma unroll
      for (int b = 0; b < RB; ++b) left = row / 16 == b ? rows[b].left : left;
      v4f v = {0.f, 0.f, 0.f, 0.f};
      if ((left >> (row & 15)) & 1) {
        const float* vp = p.v + (m0 + row) * R + s * p.rank + r;
        const int64_t part = p.M * R;
        int q = 0;
        for (; q + 4 <= p.kc; q += 4) {
          const v4f a0 = *reinterpret_cast<const v4f*>(vp + q * part), a1 = *reinterpret_cast<const v4f*>(vp + (q + 1) * part),
                    a2 = *reinterpret_cast<const v4f*>(vp + (q + 2) * part), a3 = *reinterpret_cast<const v4f*>(vp + (q + 3) * part);
          v = (((v + a0) + a1) + a2) + a3;
        }
        for (; q < p.kc; ++q) v += *reinterpret_cast<const v4f*>(vp + q * part);
      }
      *reinterpret_cast<v4f*>(&vs[row * ld + r]) = v;
    }
    __syncthreads();
  }
  if (!work) return;

  bool some = mine_any;
  while (some) {
    int a = -1;
#pragma unroll
    for (int b = 0; b < RB; ++b)
      if (a < 0 && rows[b].left) a = __builtin_amdgcn_readlane(rows[b].id, __builtin_ctz(rows[b].left));
    const float scale = p.scaling[a];
    const uint16_t* bp = p.b + (int64_t)a * p.N * p.rank;
    auto load_b = [&](int rr, v4w (&bw)[4]) {
      const int r = rr + 8 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t nn = n0 + (c >> 2) * 16 + j * 4 + (c & 3);
        const bool in = r < p.rank && nn < nend;
        bw[j] = load16(bp + (in ? nn * p.rank + r : 0), in);
      }
    };
    v4w b0[4], b1[4];
    load_b(0, b0);
    if (p.rank > 32) load_b(32, b1);
#pragma unroll
    for (int b = 0; b < RB; ++b) {
      const bool mine = rows[b].id == a && todo[b];
      const uint32_t which = (uint32_t)__ballot(mine) & 0xffffu;
      if (!which) continue;
      rows[b].left &= ~which;
      const float* vr = vs + (16 * b + c) * ld;
      float top = 0.f;
      for (int r = 8 * g; r < p.rank; r += 32)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(vr[r + e]));
      top = mine ? top : 0.f;
      auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
      auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false, false);
      top = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
      // 2^-e with 2^e the power of two at or below the largest |v|; NaN and infinity pass through as they are
      const uint32_t ex = (__float_as_uint(top) >> 23) & 255u;
      const bool plain = ex > 1 && ex < 253;
      const float down = plain ? __uint_as_float((254u - ex) << 23) : 1.f;
      const float up = (plain ? __uint_as_float(ex << 23) : 1.f) * scale;
      v4f d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = v4f{0.f, 0.f, 0.f, 0.f};
      auto product = [&](int rr, const v4w (&bw)[4]) {
        const int r = rr + 8 * g;
        const bool in = mine && r < p.rank;
        v4w hi, lo;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float v0 = in ? vr[r + 2 * e] * down : 0.f, v1 = in ? vr[r + 2 * e + 1] * down : 0.f;
          const uint16_t h0 = to_dtype(v0, DT), h1 = to_dtype(v1, DT);
          hi[e] = (uint32_t)h0 | ((uint32_t)h1 << 16);
          lo[e] = (uint32_t)to_dtype(v0 - from_dtype(h0, DT), DT) | ((uint32_t)to_dtype(v1 - from_dtype(h1, DT), DT) << 16);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          d[j] = mfma16<DT>(bw[j], hi, d[j]);
          d[j] = mfma16<DT>(bw[j], lo, d[j]);
        }
      };
      product(0, b0);
      if (p.rank > 32) product(32, b1);
      for (int rr = 64; rr < p.rank; rr += 32) {
        v4w bw[4];
        load_b(rr, bw);
        product(rr, bw);
      }
      if (mine)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[b][j] = d[j] * up;
    }
    some = false;
#pragma unroll
    for (int b = 0; b < RB; ++b) some = some || rows[b].left != 0;
  }
#pragma unroll
  for (int b = 0; b < RB; ++b) {
    const int64_t m = m0 + 16 * b + c;
    if (!write[b] || m >= p.M || !cols) continue;
    uint32_t w[8];
    if constexpr (F32) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const v4f y = __builtin_bit_cast(v4f, base[b][j]) + acc[b][j];
        w[2 * j] = (uint32_t)to_dtype(y[0], DT) | ((uint32_t)to_dtype(y[1], DT) << 16);
        w[2 * j + 1] = (uint32_t)to_dtype(y[2], DT) | ((uint32_t)to_dtype(y[3], DT) << 16);
      }
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        float f[8];
        unpack8(base[b][t], DT, f);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          w[4 * t + e] = (uint32_t)to_dtype(f[2 * e] + acc[b][2 * t + e / 2][(2 * e) & 3], DT) |
                         ((uint32_t)to_dtype(f[2 * e + 1] + acc[b][2 * t + e / 2][(2 * e + 1) & 3], DT) << 16);
      }
    }
    uint16_t* op = p.out + m * p.ldo + n;
    *reinterpret_cast<uint4*>(op) = make_uint4(w[0], w[1], w[2], w[3]);
    *reinterpret_cast<uint4*>(op + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  }
}

// parts of K: enough workgroups for a few rows, one part for many
int lora_parts(int64_t M, int64_t K) {
  const int64_t blocks = (M + 15) / 16, most = (K + 511) / 512;
  int64_t kc = 256 / (blocks > 0 ? blocks : 1);
  if (kc > most) kc = most;
  if (kc > 16) kc = 16;
  return kc < 1 ? 1 : (int)kc;
}

int64_t lora_workspace(int64_t M, int64_t K, int64_t R) { return lora_parts(M, K) * M * R * 4; }

int launch_lora(LoraArgs& p, int dtype, hipStream_t st) {
  const int R = p.slices * p.rank;
  p.kc = lora_parts(p.M, p.K);
  p.kstep = (p.K + p.kc * 512 - 1) / (p.kc * 512) * 512;
  const int64_t blocks = (p.M + 15) / 16;
  p.slots = p.M <= 64 ? (int)(p.M < 16 ? p.M : 16) : 1;
  const int rb = R <= 16 ? 1 : R <= 32 ? 2 : 4;
  const int64_t groups = (R + 16 * rb - 1) / (16 * rb);
  const dim3 gd((unsigned)(blocks * groups * p.kc), 1, (unsigned)p.slots), bl(256);
  // blocks of 64 rows where they fill the card (prompts), of 16 else
  const int64_t quads = p.chunk[p.slices];
  const int up_rows = p.slots == 1 && !p.base_f32 && p.rank <= 128 && quads * ((p.M + 63) / 64) >= 1024 ? 64 : 16;
  const dim3 gu((unsigned)(quads * ((p.M + up_rows - 1) / up_rows)), 1, (unsigned)p.slots);
  const unsigned lds = (unsigned)(up_rows * (p.rank + 4) * 4);
#define W4A8_LORA(DT_)                                                                        \
  do {                                                                                        \
    if (rb == 1) hipLaunchKernelGGL((lora_down_kernel<DT_, 1>), gd, bl, 0, st, p);            \
    else if (rb == 2) hipLaunchKernelGGL((lora_down_kernel<DT_, 2>), gd, bl, 0, st, p);       \
    else hipLaunchKernelGGL((lora_down_kernel<DT_, 4>), gd, bl, 0, st, p);                    \
    if (hipGetLastError() != hipSuccess) return kErrHip;                                      \
    if (up_rows == 64) hipLaunchKernelGGL((lora_up_kernel<DT_, 4, false>), gu, bl, lds, st, p);    \
    else if (p.base_f32) hipLaunchKernelGGL((lora_up_kernel<DT_, 1, true>), gu, bl, lds, st, p);   \
    else hipLaunchKernelGGL((lora_up_kernel<DT_, 1, false>), gu, bl, lds, st, p);                  \
  } while (0)
  if (dtype == kBF16) W4A8_LORA(kBF16);
  else W4A8_LORA(kF16);
#undef W4A8_LORA
  return hipGetLastError() == hipSuccess ? kOk : kErrHip;
}

}  // namespace w4a8
