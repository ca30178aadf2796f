// What moves in the 4-bit cache (layout: kv4.h) beside the appending of tokens: pages are copied, and of a tree of
// drafted tokens the accepted ones are put behind the context. Both take several layers' caches in one launch, since
// each moves little per layer. And the tree itself: from each node's parent, which nodes it sees, and where it stands.
#include "kv4.h"

namespace w4a8 {

// ---- pages: a workgroup copies 1024 vectors of 16 bytes of one pair's page, 4 a lane and all in flight, of its K codes, its
// V codes, or its scales (K's, then V's). Nothing branches before the loads, so that what they wait for is read at once:
// the pair, the cache's pointers. 64 pairs of 17 KB in 4 layers 4.4 us (18.8 with 2048 vectors a workgroup over all four arrays
// in a row, whose places were worked out one after another).
constexpr int kCopyPart = 1024;  // vectors of a workgroup

template <bool NT>
__global__ void __launch_bounds__(256)
kv4_copy_kernel(const Kv4Caches cs, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int pages, int parts,
                uint32_t codes, uint32_t scales) {
  const int pair = blockIdx.x, part = blockIdx.y;
  const Kv4Arrays c = cs.c[blockIdx.z];
  const int s = src[pair], d = dst[pair];
  const bool on = s >= 0 && s < pages && d >= 0 && d < pages && s != d;
  const int64_t from = on ? s : 0, to = on ? d : 0;
  const bool of_k = part < parts, of_v = !of_k && part < 2 * parts;
  const uint32_t i0 = (uint32_t)(of_k ? part : of_v ? part - parts : part - 2 * parts) * kCopyPart + threadIdx.x;
  v4u x[4];
  if (of_k || of_v) {
    v4u* base = reinterpret_cast<v4u*>(of_k ? c.k : c.v);
    const v4u* in = base + from * codes;
    v4u* out = base + to * codes;
#pragma unroll
    for (int u = 0; u < 4; ++u) x[u] = in[min(i0 + 256 * u, codes - 1)];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (on && i0 + 256 * u < codes) stream_write<NT>(out + i0 + 256 * u, x[u]);
  } else {
    v4u *ks = reinterpret_cast<v4u*>(c.ks), *vs = reinterpret_cast<v4u*>(c.vs);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t i = min(i0 + 256 * u, 2 * scales - 1);
      x[u] = i < scales ? ks[from * scales + i] : vs[from * scales + i - scales];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t i = i0 + 256 * u;
      if (on && i < scales) ks[to * scales + i] = x[u];
      if (on && i >= scales && i < 2 * scales) vs[to * scales + i - scales] = x[u];
    }
  }
}

int launch_kv4_copy(const Kv4Caches& cs, int caches, const int32_t* src, const int32_t* dst, int64_t n, int64_t pages,
                    int64_t codes, int64_t scales, hipStream_t st) {
  const int64_t parts = (codes + kCopyPart - 1) / kCopyPart, all = 2 * parts + (2 * scales + kCopyPart - 1) / kCopyPart;
  if (n > kMaxGrid || all > 65535) return kErrUnsupported;
  const dim3 g((unsigned)n, (unsigned)all, (unsigned)caches), b(256);
  // us, bytes in and out, past / through the caches, and with kv4_read behind it: 34 MB 9 / 9, 29 / 24; 68 MB 13 / 16, 52 / 45;
  // 136 MB 29 / 35, 112 / 108; 207 MB 50 / 51, 157 / 146; 238 MB 57 / 58, 179 / 177; 290 MB 68 / 69, 218 / 220; 373 MB 86 / 87, 274 / 293
  if (n * caches * (codes + scales) * 64 > 256 << 20)
    hipLaunchKernelGGL((kv4_copy_kernel<true>), g, b, 0, st, cs, src, dst, (int)pages, (int)parts, (uint32_t)codes, (uint32_t)scales);
  else
    hipLaunchKernelGGL((kv4_copy_kernel<false>), g, b, 0, st, cs, src, dst, (int)pages, (int)parts, (uint32_t)codes, (uint32_t)scales);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

// ---- accepted tokens. Slot j behind the context gets what slot keep[j] >= j holds. A workgroup has one sequence, head
// and layer. It looks 64 slots up at once, a lane each (the list's first entries are read beside the lengths), and takes the 8
// slots of one block at a time, in order: all 8 are read before the first is written, and what is read lies behind what is
// written, so no block reads what an earlier one has written. A thread has one channel of V (words of 8 tokens, a nibble
// of each moves), and words of the tokens' K. Bound by a chain of dependent reads, lengths -> page -> codes.
template <int D>
__global__ void __launch_bounds__(D < 128 ? 128 : D)
kv4_keep_kernel(const Kv4Caches cs, Kv4Cache c, Kv4Batch s, const int32_t* __restrict__ keep, int64_t ldk, int width,
                const int32_t* __restrict__ kept, int32_t* __restrict__ now) {
  constexpr int kThreads = D < 128 ? 128 : D;
  constexpr int KW = D / 8;                       // words of a token's K codes
  constexpr int PASS = (8 * KW + kThreads - 1) / kThreads;
  __shared__ int lst[64], s_where[64];
  __shared__ int64_t s_from[64], s_to[8];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Kv4Arrays a = cs.c[blockIdx.z];
  const int32_t* list = keep + b * ldk;
  int64_t start;
  int n;
  if (tid < 64 && tid < width) lst[tid] = list[tid];
  kv4_rows(s, b, start, n);
  const int64_t base = (int64_t)s.lens[b] - n;  // the first new token
  const int m = min(max(kept[b], 0), min(n, width));
  if (now && h == 0 && blockIdx.z == 0 && tid == 0) now[b] = (int32_t)(base + m);
  // block of a position, or -1
  auto block = [&](int64_t pos) -> int64_t {
    const int page = kv4_page(c, s, b, pos);
    return page < 0 ? -1 : kv4_block(c, page, h, (int)(pos & ~(int64_t)7));
  };
  for (int64_t p64 = base & ~(int64_t)7; p64 < base + m; p64 += 64) {
    __syncthreads();
    if (tid < 64) {
      const int64_t p = p64 + tid;
      const int j = (int)(p - base);
      int i = -1;
      if (j >= 0 && j < m) i = j < 64 ? lst[j] : list[j];
      const bool moves = j >= 0 && i > j && i < n;
      s_from[tid] = moves ? block(base + i) : -1;
      s_where[tid] = (int)((base + i) & 7);
      if ((tid & 7) == 0) s_to[tid >> 3] = j + 8 > 0 && j < m ? block(p) : -1;
    }
    __syncthreads();
    for (int e0 = 0; e0 < 64 && p64 + e0 < base + m; e0 += 8) {
      const int64_t to = s_to[e0 >> 3];
      if (to < 0) continue;
      int64_t from[8];
      int where[8];
      bool some = false;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        from[e] = s_from[e0 + e];
        where[e] = s_where[e0 + e];
        some = some || from[e] >= 0;
      }
      if (!some) continue;
      uint32_t kw[PASS], ksm = 0, vsm = 0, word = 0, vw[8];
      int64_t kf[PASS], sf = -1;
      const bool channel = tid < D;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        vw[e] = channel && from[e] >= 0 ? reinterpret_cast<const uint32_t*>(a.v)[from[e] * D + tid] : 0u;
      if (channel) word = reinterpret_cast<const uint32_t*>(a.v)[to * D + tid];
#pragma unroll
      for (int u = 0; u < PASS; ++u) {
        const int id = tid + u * kThreads, e = (id / KW) & 7;
        kf[u] = id < 8 * KW ? s_from[e0 + e] : -1;
        kw[u] = kf[u] >= 0 ? reinterpret_cast<const uint32_t*>(a.k)[(kf[u] * 8 + s_where[e0 + e]) * KW + id % KW] : 0u;
      }
      if (tid < 8) {
        sf = s_from[e0 + tid];
        if (sf >= 0) {
          ksm = a.ks[sf * 8 + s_where[e0 + tid]];
          vsm = a.vs[sf * 8 + s_where[e0 + tid]];
        }
      }
      __syncthreads();  // all is read, and arrived
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (from[e] >= 0) word = (word & ~(15u << (4 * e))) | (((vw[e] >> (4 * where[e])) & 15u) << (4 * e));
      if (channel) reinterpret_cast<uint32_t*>(a.v)[to * D + tid] = word;
#pragma unroll
      for (int u = 0; u < PASS; ++u) {
        const int id = tid + u * kThreads;
        if (kf[u] >= 0) reinterpret_cast<uint32_t*>(a.k)[(to * 8 + id / KW) * KW + id % KW] = kw[u];
      }
      if (sf >= 0) {
        a.ks[to * 8 + tid] = ksm;
        a.vs[to * 8 + tid] = vsm;
      }
    }
  }
}

int launch_kv4_keep(const Kv4Caches& cs, int caches, int D, const Kv4Cache& c, const Kv4Batch& s, const int32_t* keep, int64_t ldk,
                    int width, const int32_t* kept, int32_t* now, hipStream_t st) {
  const dim3 g((unsigned)c.H, (unsigned)s.B, (unsigned)caches);
  if (D == 64) hipLaunchKernelGGL((kv4_keep_kernel<64>), g, dim3(128), 0, st, cs, c, s, keep, ldk, width, kept, now);
  else if (D == 128) hipLaunchKernelGGL((kv4_keep_kernel<128>), g, dim3(128), 0, st, cs, c, s, keep, ldk, width, kept, now);
  else hipLaunchKernelGGL((kv4_keep_kernel<256>), g, dim3(256), 0, st, cs, c, s, keep, ldk, width, kept, now);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

// ---- a tree. A workgroup per sequence, its parents in LDS; a thread walks from its node to the root and writes the
// node's row of bits word by word, from the highest.
constexpr int kTreeNodes = 4096;

__global__ void __launch_bounds__(256)
kv4_tree_kernel(const int32_t* __restrict__ parents, Kv4Batch s, int words, int window, uint32_t* __restrict__ bits,
                int32_t* __restrict__ pos) {
  __shared__ int up[kTreeNodes];
  const int b = blockIdx.x;
  int64_t start;
  int n;
  kv4_rows(s, b, start, n);
  const int held = min(n, kTreeNodes);
  for (int i = threadIdx.x; i < held; i += 256) up[i] = parents[start + i];
  __syncthreads();
  const int base = (int)((uint32_t)s.lens[b] - (uint32_t)n);
  for (int i = threadIdx.x; i < n; i += 256) {
    uint32_t* row = bits + (start + i) * words;
    int w = words - 1, depth = -1;
    uint32_t acc = 0;
    for (int j = i; j >= 0;) {
      if (window == 0 || depth + 1 < window) {
        const int jw = j >> 5;
        for (; w > jw; --w) {
          row[w] = acc;
          acc = 0;
        }
        if (jw == w) acc |= 1u << (j & 31);
      }
      ++depth;
      const int u = j < kTreeNodes ? up[j] : parents[start + j];
      j = u < j ? u : -1;  // a parent stands before its children
    }
    for (; w >= 0; --w) {
      row[w] = acc;
      acc = 0;
    }
    pos[start + i] = base + depth;
  }
}

int launch_kv4_tree(const int32_t* parents, const Kv4Batch& s, int words, int window, uint32_t* bits, int32_t* pos,
                    hipStream_t st) {
  hipLaunchKernelGGL(kv4_tree_kernel, dim3((unsigned)s.B), dim3(256), 0, st, parents, s, words, window, bits, pos);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

}  // namespace w4a8
