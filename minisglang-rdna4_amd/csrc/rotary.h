// Rotary positions: the arguments that rotary.hip and its entry point share.
#pragma once
#include "w4a8_common.h"

namespace w4a8 {

constexpr int kRotaryMaxAxes = 8;

// rows of heads to turn: q's, and k's behind them
struct RotaryRows {
  const uint16_t* in;
  uint16_t* out;
  int64_t ldi, hi, ldo, ho;  // elements between tokens and between heads
  int heads;
};
struct Rotary {
  RotaryRows q, k;
  const void* pos;        // (axes, T) of 32 or 64 bits
  int64_t ldp;            // entries from one axis to the next
  int pos64;
  const uint64_t* turn;   // (R / 2): a pair's turns per position, in 2^-64
  const int32_t* axis;    // (R / 2): a pair's axis; null: 0
  int64_t T;
  int R, units;           // channels that turn, and units of 16 of them and of 8 others that a head has
  int adjacent;
  float scale;
  int heads, per;         // of q and k together, and of them per thread
};

}  // namespace w4a8
