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
};

// How a call is cut. few: 16 columns and the waves of a workgroup over the tokens; else nq * 16 columns per
// wave, the waves side by side.
struct Kv4Plan {
  bool few;
  int nq;
  int splits;      // of the tokens, over the grid
  int64_t qgrid;   // tiles of columns per sequence and head
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

}  // namespace w4a8
