// Attention over whole prompts in 16 bits: the arguments that prompt_attn.hip and its entry point share.
#pragma once
#include "w4a8_common.h"

namespace w4a8 {

struct PromptAttn {
  const uint16_t *q, *k, *v;
  int64_t ldq, hq, ldk, hk, ldv, hv;  // elements between tokens and between heads
  uint16_t* out;
  int64_t ldo, ho;
  float* lse;          // (T, H G) or null
  const int32_t* cu;   // (B + 1): rows cu[b] .. cu[b + 1] - 1 are sequence b's
  int B;
  int64_t T;
  int H, G;            // key/value heads, query heads of each
  uint32_t gmul;       // ceil(2^31 / G): x / G is the high half of 2 x gmul for x below 2^31 / G
  float scale;         // softmax scale times log2(e)
  int causal;
  int window;          // keys before position - window + 1 are not seen; 0: all are
};

}  // namespace w4a8
