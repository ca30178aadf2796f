// What moves in the 4-bit cache (layout: kv4.h) beside the appending of tokens: pages are copied, and of a tree of
// drafted tokens the accepted ones are put behind the context. Both take several layers' caches in one launch, since
// each moves little per layer. And the tree itself: from each node's parent, which nodes it sees, and where it stands.
#include "kv4.h"

namespace w4a8 {

// ---- pages: a workgroup copies 32 KB of one pair's page, 4 loads of 16 bytes a lane in flight. The page's four arrays
// are taken as one row of vectors: K codes, V codes, K scales, V scales.
constexpr int kCopyPart = 2048;  // vectors of a workgroup

__global__ void __launch_bounds__(256)
kv4_copy_kernel(const Kv4Caches cs, const int32_t* __restrict__ src, const int32_t* __restrict__ dst, int64_t pages, int parts,
                int64_t codes, int64_t scales) {
  const uint32_t pair = blockIdx.x / (uint32_t)parts, part = blockIdx.x - pair * (uint32_t)parts;
  const int64_t s = src[pair], d = dst[pair];
  if (s < 0 || s >= pages || d < 0 || d >= pages || s == d) return;
  const Kv4Arrays& c = cs.c[blockIdx.y];
  const int64_t total = 2 * (codes + scales);
  const int64_t lo = (int64_t)part * kCopyPart, hi = lo + kCopyPart < total ? lo + kCopyPart : total;
  auto at = [&](int64_t i, uint4*& base, int64_t& n) {  // vector i's array, and the page's vectors there; its place in them
    if (i < codes) { base = reinterpret_cast<uint4*>(c.k); n = codes; return i; }
    i -= codes;
    if (i < codes) { base = reinterpret_cast<uint4*>(c.v); n = codes; return i; }
    i -= codes;
    if (i < scales) { base = reinterpret_cast<uint4*>(c.ks); n = scales; return i; }
    base = reinterpret_cast<uint4*>(c.vs);
    n = scales;
    return i - scales;
  };
  for (int64_t i0 = lo + threadIdx.x; i0 < hi; i0 += 1024) {
    uint4 x[4];
    uint4* to[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = i0 + 256 * u;
      uint4* base;
      int64_t n;
      const int64_t j = at(i < hi ? i : i0, base, n);
      x[u] = base[s * n + j];
      to[u] = base + d * n + j;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + 256 * u < hi) *to[u] = x[u];
  }
}

int launch_kv4_copy(const Kv4Caches& cs, int caches, const int32_t* src, const int32_t* dst, int64_t n, int64_t pages,
                    int64_t codes, int64_t scales, hipStream_t st) {
  const int64_t parts = (2 * (codes + scales) + kCopyPart - 1) / kCopyPart;
  if (n * parts > kMaxGrid) return kErrUnsupported;
  hipLaunchKernelGGL(kv4_copy_kernel, dim3((unsigned)(n * parts), (unsigned)caches), dim3(256), 0, st, cs, src, dst, pages,
                     (int)parts, codes, scales);
  return hipPeekAtLastError() == hipSuccess ? kOk : kErrHip;
}

// ---- accepted tokens. Slot j behind the context gets what slot keep[j] >= j holds. A workgroup has one sequence, head
// and layer and takes the 8 slots of one block at a time, in order: all 8 are read before the first is written, and
// what is read lies behind what is written, so no block reads what an earlier one has written. A thread has one
// channel of V (words of 8 tokens, a nibble of each moves), and words of the tokens' K.
template <int D>
__global__ void __launch_bounds__(D < 128 ? 128 : D)
kv4_keep_kernel(const Kv4Caches cs, Kv4Cache c, Kv4Batch s, const int32_t* __restrict__ keep, int64_t ldk, int width,
                const int32_t* __restrict__ kept, int32_t* __restrict__ now) {
  constexpr int kThreads = D < 128 ? 128 : D;
  constexpr int KW = D / 8;                       // words of a token's K codes
  constexpr int PASS = (8 * KW + kThreads - 1) / kThreads;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Kv4Arrays& a = cs.c[blockIdx.z];
  int64_t start;
  int n;
  kv4_rows(s, b, start, n);
  const int64_t base = (int64_t)s.lens[b] - n;  // the first new token
  const int m = min(max(kept[b], 0), min(n, width));
  if (now && h == 0 && blockIdx.z == 0 && tid == 0) now[b] = (int32_t)(base + m);
  const int32_t* list = keep + b * ldk;
  // slot j's source, or -1: it stays as it is
  auto source = [&](int j) -> int64_t {
    if (j < 0 || j >= m) return -1;
    const int i = list[j];
    return i > j && i < n ? base + i : -1;
  };
  // block and place in it of a position, or -1
  auto block = [&](int64_t pos) -> int64_t {
    const int page = kv4_page(c, s, b, pos);
    return page < 0 ? -1 : kv4_block(c, page, h, (int)(pos & ~(int64_t)7));
  };
  for (int64_t p0 = base & ~(int64_t)7; p0 < base + m; p0 += 8) {
    const int64_t to = p0 < 0 ? -1 : block(p0);
    if (to < 0) continue;
    int64_t from[8];
    int where[8];
    bool some = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int64_t src = source((int)(p0 + e - base));
      from[e] = src < 0 ? -1 : block(src);
      where[e] = (int)(src & 7);
      some = some || from[e] >= 0;
    }
    if (!some) continue;
    uint32_t kw[PASS], ksm = 0, vsm = 0, word = 0, vw[8];
    const bool channel = tid < D;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      vw[e] = channel && from[e] >= 0 ? reinterpret_cast<const uint32_t*>(a.v)[from[e] * D + tid] : 0u;
    if (channel) word = reinterpret_cast<const uint32_t*>(a.v)[to * D + tid];
    auto pick = [&](int e, int64_t& f, int& w) {  // from[e] and where[e], e a lane's own
      f = -1;
      w = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i == e) { f = from[i]; w = where[i]; }
    };
    int64_t kf[PASS], sf = -1;
    int kx[PASS], sx = 0;
#pragma unroll
    for (int u = 0; u < PASS; ++u) {
      const int id = tid + u * kThreads;
      pick(id / KW, kf[u], kx[u]);
      kw[u] = kf[u] >= 0 ? reinterpret_cast<const uint32_t*>(a.k)[(kf[u] * 8 + kx[u]) * KW + id % KW] : 0u;
    }
    if (tid < 8) pick(tid, sf, sx);
    if (sf >= 0) {
      ksm = a.ks[sf * 8 + sx];
      vsm = a.vs[sf * 8 + sx];
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
