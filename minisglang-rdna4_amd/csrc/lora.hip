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
//
// Measured, first and second kernel: one row, K = N = 4096, rank 16: 2.3 and 4.8 us, latency; 48 rows of 40 adapters,
// K = 14336, N = 4096, rank 64 (A 73 MB, B 21 MB): 16.7 (4.4 TB/s) and 10.4 us; 4096 rows, K = 4096, N = 28672 in two
// slices, rank 16: 18.6 and 126 us (y in and out, 470 MB, 3.7 TB/s). The second kernel with 64 rows a workgroup and
// all their sums in registers took 161 us there: 240 registers a wave, and less of y in flight.
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

__device__ __forceinline__ v4w load16(const uint16_t* p) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
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
    // Rows of other adapters and ranks past R are loaded as some row that is there, and their sums dropped below:
    // a column of the product is one row's, a row of it one rank's.
    const bool mine = rows.id == a;
    const int some = __builtin_ctz((uint32_t)__ballot(mine));
    const uint16_t* xp = p.x + (m0 + (mine ? c : some)) * p.ldx;
    const uint16_t* ap[RB];
#pragma unroll
    for (int t = 0; t < RB; ++t) {
      const int r = r0 + 16 * t + c;
      ap[t] = p.a + ((int64_t)a * R + (r < R ? r : R - 1)) * p.K;
    }
    v4f acc[RB];
#pragma unroll
    for (int t = 0; t < RB; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};
    for (int64_t kb = k0 + wave * 128; kb < k1; kb += 512) {
      const int64_t k = kb + g * 32;
      v4w xv[4], av[RB][4];
      if (kb + 128 <= k1) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          xv[j] = load16(xp + k + 8 * j);
#pragma unroll
          for (int t = 0; t < RB; ++t) av[t][j] = load16(ap[t] + k + 8 * j);
        }
      } else {
        // K's last inputs: past them x and A are zeros
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool in = k + 8 * j < k1;
          const v4w zero = {0, 0, 0, 0};
          xv[j] = in ? load16(xp + k + 8 * j) : zero;
#pragma unroll
          for (int t = 0; t < RB; ++t) av[t][j] = in ? load16(ap[t] + k + 8 * j) : zero;
        }
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

// grid: (spans of p.span columns of one slice * blocks of 16 rows, 1, slots). The workgroup first sums the parts of v
// for its rows and slice into LDS. Then, adapter by adapter, its waves walk the span, 64 columns each at a time: row
// (4 q + i) of the j-th product is column 16 q + 4 j + i of them, so a lane ends with 16 neighbouring columns of its
// row, of which only the adapter's rows are read and written. The next columns' base is loaded while these are
// computed. NS: steps of 32 ranks whose v operands stay in registers over the span; 0: any rank, from LDS each time.
template <int DT, bool F32, int NS>
__global__ void __launch_bounds__(256)
lora_up_kernel(const LoraArgs p) {
  extern __shared__ float vs[];  // (16, rank + 4)
  constexpr int NB = F32 ? 4 : 2;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4, c = lane & 15;
  const uint32_t spans = (uint32_t)p.chunk[p.slices], span = blockIdx.x % spans;
  int s = 0;
  while (span >= p.chunk[s + 1]) ++s;
  const int64_t m0 = (int64_t)(blockIdx.x / spans) * 16, m = m0 + c;
  const int64_t first = p.col[s] + (span - p.chunk[s]) * p.span;
  const int64_t end = first + p.span < p.col[s + 1] ? first + p.span : p.col[s + 1];
  const int R = p.slices * p.rank, ld = p.rank + 4;
  const Rows rows = row_adapters(p, m0, lane);

  const uint8_t* brow = reinterpret_cast<const uint8_t*>(p.base) + (m < p.M ? m : m0) * p.ldb * (F32 ? 4 : 2);
  uint16_t* orow = p.out + (m < p.M ? m : m0) * p.ldo;
  uint4 base[NB];
  auto load_base = [&](int64_t n, bool on) {
    if (on && n < end)
#pragma unroll
      for (int j = 0; j < NB; ++j) base[j] = reinterpret_cast<const uint4*>(brow + n * (F32 ? 4 : 2))[j];
  };
  // base (f32 or the type's) plus d, rounded, at column n of this lane's row
  auto store = [&](const uint4 (&y)[NB], const v4f (&d)[4], float up, int64_t n) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v4f f;
      if constexpr (F32) f = __builtin_bit_cast(v4f, y[j]);
      else {
        const uint32_t a = j & 1 ? y[j / 2].z : y[j / 2].x, b = j & 1 ? y[j / 2].w : y[j / 2].y;
        f = v4f{from_dtype((uint16_t)(a & 0xffffu), DT), from_dtype((uint16_t)(a >> 16), DT),
                from_dtype((uint16_t)(b & 0xffffu), DT), from_dtype((uint16_t)(b >> 16), DT)};
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __builtin_fmaf(d[j][e], up, f[e]);
      w[2 * j] = (uint32_t)to_dtype(f[0], DT) | ((uint32_t)to_dtype(f[1], DT) << 16);
      w[2 * j + 1] = (uint32_t)to_dtype(f[2], DT) | ((uint32_t)to_dtype(f[3], DT) << 16);
    }
    uint4* op = reinterpret_cast<uint4*>(orow + n);
    op[0] = make_uint4(w[0], w[1], w[2], w[3]);
    op[1] = make_uint4(w[4], w[5], w[6], w[7]);
  };

  // the rows of this workgroup's adapters: the i-th of the block is slot i's, modulo the slots
  uint32_t todo = 0;
  {
    Rows r = rows;
    for (int i = 0; r.left; ++i) {
      const uint32_t before = r.left;
      next_adapter(r);
      if (i % (int)gridDim.z == (int)blockIdx.z) todo |= before & ~r.left;
    }
  }
  const bool bare = blockIdx.z == 0 && rows.id < 0 && m < p.M && (F32 || p.base != p.out);
  if (!todo && !__ballot(bare)) return;

  // four ranks a thread, the parts of K in their order
  const int per = p.rank / 4;
  for (int t = threadIdx.x; t < 16 * per; t += 256) {
    const int row = t / per, r = (t - row * per) * 4;
    if (!((todo >> row) & 1)) continue;
    const float* vp = p.v + (m0 + row) * R + s * p.rank + r;
    const int64_t part = p.M * R;
    v4f v = {0.f, 0.f, 0.f, 0.f};
    for (int q = 0; q < p.kc; q += 8) {
      v4f x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) x[u] = *reinterpret_cast<const v4f*>(vp + (q + u < p.kc ? q + u : 0) * part);
#pragma unroll
      for (int u = 0; u < 8; ++u) v += q + u < p.kc ? x[u] : v4f{0.f, 0.f, 0.f, 0.f};
    }
    *reinterpret_cast<v4f*>(&vs[row * ld + r]) = v;
  }
  // rows without an adapter are the base, rounded to the type
  if (__ballot(bare)) {
    const v4f zero[4] = {v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}, v4f{0.f, 0.f, 0.f, 0.f}};
    for (int64_t n = first + wave * 64 + 16 * g; n < end; n += 256) {
      load_base(n, bare);
      if (bare) store(base, zero, 0.f, n);
    }
  }
  __syncthreads();

  Rows r = rows;
  while (r.left) {
    const int a = next_adapter(r);
    const bool mine = rows.id == a && ((todo >> c) & 1);
    if (!__ballot(mine)) continue;
    load_base(first + wave * 64 + 16 * g, mine);
    const float scale = p.scaling[a];
    const float* vr = vs + c * ld + 8 * g;
    float top = 0.f;
    for (int q = 0; q + 8 * g < p.rank; q += 32)
#pragma unroll
      for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(vr[q + e]));
    top = mine ? top : 0.f;
    auto x = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
    auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(top), __float_as_uint(top), false, false);
    top = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
    // 2^-e with 2^e the power of two at or below the largest |v|. A row with an infinity is not scaled, and the infinity
    // becomes NaN: its second term is inf - inf
    const uint32_t ex = (__float_as_uint(top) >> 23) & 255u;
    const bool plain = ex > 1 && ex < 253;
    const float down = plain ? __uint_as_float((254u - ex) << 23) : 1.f;
    const float up = (plain ? __uint_as_float(ex << 23) : 1.f) * scale;
    // v of ranks q .. q + 31 as two terms
    auto operand = [&](int q, v4w& hi, v4w& lo) {
      const bool in = mine && q + 8 * g < p.rank;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float v0 = in ? vr[q + 2 * e] * down : 0.f, v1 = in ? vr[q + 2 * e + 1] * down : 0.f;
        const uint16_t h0 = to_dtype(v0, DT), h1 = to_dtype(v1, DT);
        hi[e] = (uint32_t)h0 | ((uint32_t)h1 << 16);
        lo[e] = (uint32_t)to_dtype(v0 - from_dtype(h0, DT), DT) | ((uint32_t)to_dtype(v1 - from_dtype(h1, DT), DT) << 16);
      }
    };
    v4w hi[NS + 1], lo[NS + 1];
#pragma unroll
    for (int q = 0; q < NS; ++q) operand(32 * q, hi[q], lo[q]);
    const uint16_t* bp = p.b + (int64_t)a * p.N * p.rank;
    for (int64_t n0 = first + wave * 64; n0 < end; n0 += 256) {
      uint4 cur[NB];
#pragma unroll
      for (int j = 0; j < NB; ++j) cur[j] = base[j];
      v4f d[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = v4f{0.f, 0.f, 0.f, 0.f};
      const int64_t nb = n0 + (c >> 2) * 16 + (c & 3);
      // slices are multiples of 16 columns: those past the end are the first 16 again, and not stored
      const uint16_t* bn = bp + (nb - (c & 3) < end ? nb : n0 + (c & 3)) * p.rank;
      auto product = [&](int q, const v4w& h, const v4w& l) {
        const int rk = q + 8 * g;
        v4w bw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) bw[j] = load16(bn + 4 * j * p.rank + (rk < p.rank ? rk : 0));  // v is 0 past the rank
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          d[j] = mfma16<DT>(bw[j], h, d[j]);
          d[j] = mfma16<DT>(bw[j], l, d[j]);
        }
      };
      if constexpr (NS > 0) {
#pragma unroll
        for (int q = 0; q < NS; ++q) product(32 * q, hi[q], lo[q]);
      } else {
        for (int q = 0; q < p.rank; q += 32) {
          operand(q, hi[0], lo[0]);
          product(q, hi[0], lo[0]);
        }
      }
      load_base(n0 + 256 + 16 * g, mine);
      if (mine && n0 + 16 * g < end) store(cur, d, up, n0 + 16 * g);
    }
  }
}

// How a call is cut. Few rows (up to 64): every adapter of a block of 16 rows has a workgroup of its own (slots), and
// 16 ranks; more rows, which are prompts as a rule: 64 ranks and a block's adapters one after another. Parts of K, of
// at least 512 inputs, to about 1024 workgroups; up to 8, since the second kernel sums them in one round of loads.
// us for K = N = 4096 and rank 16, slots / one after another. Each row with an adapter of its own: 17 rows 11 / 43, 64
// 13 / 42, 65 14 / 42, 128 21 / 52, 256 33 / 53, 512 56 / 57, 1024 99 / 65; six prompts: 64 rows 8.3 / 10.5, 256
// 9.8 / 10.6, 512 14.8 / 11.6, 4096 49 / 32. So from 65 to 512 rows batches of many users pay for prompts here (K = 14336,
// rank 64, 128 users: 62 / 192).
struct LoraPlan {
  int slots, rb, kc;
  int64_t kstep;
};
static LoraPlan lora_plan(int64_t M, int64_t K, int64_t R) {
  LoraPlan pl;
  const bool few = M <= 64;
  pl.slots = few ? (int)(M < 16 ? M : 16) : 1;
  pl.rb = few || R <= 16 ? 1 : R <= 32 ? 2 : 4;
  const int64_t tiles = (few ? M : (M + 15) / 16) * ((R + 16 * pl.rb - 1) / (16 * pl.rb));
  int64_t kc = (1024 + tiles - 1) / tiles, most = (K + 511) / 512;
  if (kc > most) kc = most;
  if (kc > 8) kc = 8;
  pl.kc = (int)kc;
  pl.kstep = (K + kc * 512 - 1) / (kc * 512) * 512;
  return pl;
}

int64_t lora_workspace(int64_t M, int64_t K, int64_t R) { return lora_plan(M, K, R).kc * M * R * 4; }

int launch_lora(LoraArgs& p, int dtype, hipStream_t st) {
  const int R = p.slices * p.rank;
  const LoraPlan pl = lora_plan(p.M, p.K, R);
  p.kc = pl.kc;
  p.kstep = pl.kstep;
  const int64_t blocks = (p.M + 15) / 16, groups = (R + 16 * pl.rb - 1) / (16 * pl.rb);
  const dim3 gd((unsigned)(blocks * groups * p.kc), 1, (unsigned)pl.slots), bl(256);
  // the second product's spans: one step of the four waves, or up to 8 where the rows fill the card
  const int64_t quads = (p.N + 255) / 256;
  int64_t steps = quads * blocks / 2048;
  steps = steps < 1 ? 1 : steps > 8 ? 8 : steps;
  p.span = 256 * steps;
  int64_t spans = 0;
  for (int i = 0; i <= kLoraMaxSlices; ++i) {
    p.chunk[i] = spans;
    if (i < p.slices) spans += (p.col[i + 1] - p.col[i] + p.span - 1) / p.span;
  }
  if (blocks * groups * p.kc > kMaxGrid || spans * blocks > kMaxGrid) return kErrUnsupported;
  const dim3 gu((unsigned)(spans * blocks), 1, (unsigned)pl.slots);
  const unsigned lds = (unsigned)(16 * (p.rank + 4) * 4);
#define W4A8_LORA_UP(DT_, F32_)                                                                       \
  do {                                                                                                \
    if (p.rank <= 32) hipLaunchKernelGGL((lora_up_kernel<DT_, F32_, 1>), gu, bl, lds, st, p);         \
    else if (p.rank <= 64) hipLaunchKernelGGL((lora_up_kernel<DT_, F32_, 2>), gu, bl, lds, st, p);    \
    else hipLaunchKernelGGL((lora_up_kernel<DT_, F32_, 0>), gu, bl, lds, st, p);                      \
  } while (0)
#define W4A8_LORA(DT_)                                                                                \
  do {                                                                                                \
    if (pl.rb == 1) hipLaunchKernelGGL((lora_down_kernel<DT_, 1>), gd, bl, 0, st, p);                 \
    else if (pl.rb == 2) hipLaunchKernelGGL((lora_down_kernel<DT_, 2>), gd, bl, 0, st, p);            \
    else hipLaunchKernelGGL((lora_down_kernel<DT_, 4>), gd, bl, 0, st, p);                            \
    if (hipPeekAtLastError() != hipSuccess) return kErrHip;                                           \
    if (p.base_f32) W4A8_LORA_UP(DT_, true);                                                          \
    else W4A8_LORA_UP(DT_, false);                                                                    \
  } while (0)
  if (dtype == kBF16) W4A8_LORA(kBF16);
  else W4A8_LORA(kF16);
#undef W4A8_LORA
#undef W4A8_LORA_UP
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

}  // namespace w4a8
