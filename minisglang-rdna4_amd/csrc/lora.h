// Low-rank adapters of many requests beside a shared projection (lora.hip).
#pragma once
#include "w4a8_common.h"

namespace w4a8 {

constexpr int kLoraMaxSlices = 8;
constexpr int kLoraMaxRank = 256;

struct LoraArgs {
  const uint16_t* x;  // (M, ldx)
  int64_t ldx, M, K;
  const uint16_t* a;  // (L, slices * rank, K)
  const uint16_t* b;  // (L, N, rank)
  const float* scaling;  // (L,)
  const int32_t* ids;    // (M,): adapter of each row; outside 0 .. L-1: none
  int L, rank, slices;
  int64_t N;
  int64_t col[kLoraMaxSlices + 1];    // first column of each slice, then N
  int64_t span;                       // columns per workgroup of the second product, a multiple of 256
  int64_t chunk[kLoraMaxSlices + 1];  // each slice's first span, then all of them
  const void* base;  // (M, ldb): the projection's output, in the model's type or f32
  int64_t ldb;
  int base_f32;
  uint16_t* out;     // (M, ldo); may be base
  int64_t ldo;
  float* v;          // (kc, M, slices * rank) partial x A^T
  int kc;            // parts of K
  int64_t kstep;     // its length, a multiple of 512
};

}  // namespace w4a8
