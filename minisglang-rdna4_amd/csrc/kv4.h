// A paged cache of keys and values in 4 bits.
//
// A vector x of one token and key/value head is D codes c in 0..15 with a step s and a least value m in
// the model's type, and stands for s c + m:
//   m = min x, s = max((max x - min x) / 15, 2^-14 max |x|) rounded to the type and at least its smallest
//   positive value (2^-24 for fp16, 2^-126 for bf16), c = clamp(rint((x - m) / s), 0, 15), in f32.
// m is exact, and c is the nearest code for the step as it is stored. The floor on s keeps m / s, which
// nothing divides by zero, within 2^14. A vector that holds an infinity or a NaN, or whose max x - min x
// passes f32's range, has s = m = NaN, c = 0: whoever attends to it gets NaN, and nobody else.
//
// Memory, for pages of `page` tokens (a power of two from 16): everything is in blocks of 8 tokens of
// one head, block ((p * H + h) * page + t) / 8 of slot t in page p,
//   K codes   8 rows of D / 2 bytes, code d of a row in nibble d % 8 of its 32-bit word d / 8;
//   V codes   D 32-bit words, one per channel: nibble j of it is the code of the block's token j;
//   K, V scale  8 dwords, s in the low half, m in the high one.
// K codes lie along the channels because q k sums over them, V codes along the tokens because p v sums
// over those: a lane's load is in either case what v_mfma_f32_16x16x32's A operand wants in one lane,
// 8 codes of the summed index per 32-bit word, and no code crosses a lane.
#pragma once
#include "w4a8_common.h"

namespace w4a8 {

struct Kv4Cache {
  uint8_t* k;
  uint8_t* v;
  uint32_t* ks;
  uint32_t* vs;
  int64_t pages;
  int shift;  // log2 of the page's tokens
  int H;
};

// Which tokens: sequence b of B has lens[b] tokens, the last cu[b+1] - cu[b] of which are rows cu[b],
// cu[b]+1, ... of the call's T; table[b * ldt + i] is the page of its tokens i * page ...
struct Kv4Batch {
  const int32_t* table;
  int64_t ldt;
  int width;
  const int32_t* cu;
  const int32_t* lens;
  int B;
  int64_t T;
};

struct Kv4Attn {
  const uint16_t* q;
  int64_t ldq, hq;  // elements between tokens and between heads
  uint16_t* out;
  int64_t ldo, ho;
  float* lse;       // (T, Hq) or null
  float lse_more;   // what kv4_join_kernel adds to it
  Kv4Cache c;
  Kv4Batch s;
  int G;            // query heads per key/value head
  uint32_t gmul;    // ceil(2^31 / G): x / G is the high half of 2 x gmul for x below 2^31 / G
  float scale;      // softmax scale times log2(e)
  int causal;
  int window;       // keys before position - window + 1 are not seen; 0: all are
  int splits;       // of the tokens, over the grid
  float* po;        // (splits, T, Hq, D) partial outputs
  float* pml;       // (splits, T, Hq, 2) their maximum and sum
  // a tree of drafted tokens, or null: bit j of row i is whether it sees its sequence's new token j, and pos[i] is its
  // position, which the window counts from
  const uint32_t* bits;
  int64_t ldb;      // words between rows
  int words;        // words of a row
  const int32_t* pos;
};

// Several layers' caches of one shape, for one launch
constexpr int kKv4Caches = 64;
struct Kv4Arrays {
  uint8_t* k;
  uint8_t* v;
  uint32_t* ks;
  uint32_t* vs;
};
struct Kv4Caches {
  Kv4Arrays c[kKv4Caches];
};

// How a call is cut. few: 16 columns and the waves of a workgroup over the tokens; else nq * 16 columns per
// wave, the waves side by side.
// kv4_tree_attn_kernel's parts are 2^-15 of the sums, which then stay in f32 where the values do
constexpr float kWidePart = 0x1p-15f, kWideLse = 15.f * 0.69314718055994531f;

struct Kv4Plan {
  bool few;
  int nq;
  int splits;      // of the tokens, over the grid
  int64_t qgrid;   // tiles of columns per sequence and head
  int wide;        // waves of kv4_tree_attn_kernel, 32 columns each, or 0
};

// rows [start, start + n) of sequence b, kept inside the call's rows whatever cu holds
__device__ __forceinline__ void kv4_rows(const Kv4Batch& s, int b, int64_t& start, int& n) {
  const int64_t lo = s.cu[b], hi = s.cu[b + 1];
  start = lo < 0 ? 0 : lo;
  const int64_t end = hi < s.T ? hi : s.T;
  n = end > start ? (int)(end - start) : 0;
}

// block of slot t of `page`, a multiple of 8
__device__ __forceinline__ int kv4_block(const Kv4Cache& c, int page, int h, int t) {
  return ((page * c.H + h) << (c.shift - 3)) + ((t & ((1 << c.shift) - 1)) >> 3);
}

// page of token t, or -1 where the table has none that exists
__device__ __forceinline__ int kv4_page(const Kv4Cache& c, const Kv4Batch& s, int b, int64_t t) {
  const int64_t i = t >> c.shift;
  if (t < 0 || i >= s.width) return -1;
  const int page = s.table[b * s.ldt + i];
  return page >= 0 && page < c.pages ? page : -1;
}

// A sequence of the call: its rows and its length. Columns are its queries in order, G heads each.
struct Span {
  int64_t start;
  int n, cols, len, first_pos;  // new tokens, columns, length, position of the first new token
  int cut;                      // of a tree: what was taken off the length, and off every position
};
template <bool TREE>
__device__ __forceinline__ Span kv4_span(const Kv4Attn& p, int b) {
  Span s;
  kv4_rows(p.s, b, s.start, s.n);
  s.cols = s.n * p.G;
  const int64_t cap = (int64_t)p.s.width << p.c.shift;
  const int len = max(p.s.lens[b], 0);  // -2^31 has no position n rows before it
  // One token past the table's end stands for all of them: its page is missing. Of a tree each node has its own, behind that
  // one, and positions move with them: a window that saw some of the missing tokens before the nodes sees the one.
  s.len = len > cap ? (int)min((int64_t)len, cap + (TREE ? s.n + 1 : 1)) : len;
  s.cut = TREE ? len - s.len : 0;
  s.first_pos = len - s.cut - s.n;
  return s;
}
// The sequence of the launch's z-th workgroups: the longest first, up to 64 sequences (a lane's each), so that short ones fill the
// launch's end. The whole wave calls. us, in this order / as they come: 48 sequences of up to 26 drafted tokens on up to 8192
// 193 / 269. More come as the caller has them, and want sorting by who builds the batch: 65 361, sorted 285; 128 627 and 480.
__device__ __forceinline__ int kv4_longest(const Kv4Batch& s, int z) {
  if (s.B > 64 || s.B == 1) return z;
  const int lane = threadIdx.x & 63;
  const int mine = lane < s.B ? s.lens[lane] : 0;
  int before = 0;  // sequences that come before the lane's
  for (int j = 0; j < s.B; ++j) {
    const int other = __builtin_amdgcn_readlane(mine, j);
    before += other > mine || (other == mine && j < lane);
  }
  return __builtin_ctzll(__ballot(before == z && lane < s.B));
}
// Of a tree: the first cached key that query i sees, and its 8 bits of the tokens at .. at + 7, counted from the
// first new one
__device__ __forceinline__ int tree_from(const Kv4Attn& p, const Span& s, int i) {
  if (!p.window) return 0;
  const int64_t lo = (int64_t)p.pos[s.start + i] - s.cut - p.window + 1;
  return lo < 0 ? 0 : lo > 0x7fffffff ? 0x7fffffff : (int)lo;
}
__device__ __forceinline__ uint32_t tree_bits(const Kv4Attn& p, const Span& s, int i, int at) {
  if (at <= -8 || at >= s.n) return 0;
  const uint32_t* row = p.bits + (s.start + i) * p.ldb;
  const int w = at >> 5;
  const uint64_t lo = w >= 0 && w < p.words ? row[w] : 0, hi = w + 1 < p.words ? row[w + 1] : 0;
  const uint32_t b = (uint32_t)((lo | (hi << 32)) >> (at & 31)) & 0xffu;
  return s.n - at < 8 ? b & ((1u << (s.n - at)) - 1) : b;
}
}  // namespace w4a8
