// What the C entry points over (T, H, D) rows check in the same way.
#pragma once
#include <stdarg.h>
#include <stdio.h>

#include "w4a8_common.h"

namespace w4a8 {
int set_last_error(int code, const char* msg);

inline int fail(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  return set_last_error(code, msg);
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

inline int launched(int rc, const char* who) {
  if (rc == kOk) return kOk;
  if (rc == kErrUnsupported) return fail(rc, "%s: past its index ranges", who);
  return fail(kErrHip, "%s: HIP launch failed (%s)", who, hipGetErrorString(hipGetLastError()));
}

// whether a (T, H, D) tensor of these strides has each element in a place of its own
inline bool apart(int64_t T, int64_t ld, int64_t H, int64_t hd, int64_t D) {
  if (T <= 1) ld = H * (hd > D ? hd : D);
  if (H <= 1) hd = T * (ld > D ? ld : D);
  const bool rows_in = ld <= hd;  // the rows of a head are neighbours
  return rows_in ? ld >= D && hd >= (T - 1) * ld + D : hd >= D && ld >= (H - 1) * hd + D;
}

// whether (T, H, D) tensors at a and b of 16-bit elements may share some, as far as their strides tell
inline bool collide(const void* a, int64_t lda, int64_t ha, const void* b, int64_t ldb, int64_t hb, int64_t T, int64_t H,
                    int64_t D) {
  // the longer stride outside, a row of the other inside
  auto order = [&](int64_t ld, int64_t h, int64_t& outer, int64_t& n, int64_t& inner) {
    const bool heads_in = H <= 1 || (T > 1 && ld >= h);
    outer = heads_in ? ld : h;
    n = heads_in ? T : H;
    inner = heads_in ? (H > 1 ? (H - 1) * h : 0) + D : (T > 1 ? (T - 1) * ld : 0) + D;
    if (n <= 1) outer = 0;
  };
  int64_t oa, na, ia, ob, nb, ib;
  order(lda, ha, oa, na, ia);
  order(ldb, hb, ob, nb, ib);
  const int64_t pa = (int64_t)(reinterpret_cast<uintptr_t>(a) / 2), pb = (int64_t)(reinterpret_cast<uintptr_t>(b) / 2);
  if (pa + (na - 1) * oa + ia <= pb || pb + (nb - 1) * ob + ib <= pa) return false;
  auto apart_by = [&](int64_t stride, int64_t wa, int64_t wb) {
    const int64_t d = ((pb - pa) % stride + stride) % stride;
    return d >= wa && d + wb <= stride;
  };
  if (oa == ob && na == nb && oa > 0 && apart_by(oa, ia, ib)) return false;  // rows beside each other
  // heads beside each other
  if (ha == hb && ha > 0 && (T <= 1 || (lda == ldb && lda % ha == 0)) && apart_by(ha, D, D)) return false;
  return true;
}

// the same for rows of Ha and of Hb heads: apart where they are columns of one buffer's rows, heads inside
inline bool collide_rows(const void* a, int64_t lda, int64_t ha, int64_t Ha, const void* b, int64_t ldb, int64_t hb, int64_t Hb,
                         int64_t T, int64_t D) {
  auto reach = [&](int64_t ld, int64_t h, int64_t H) { return (T > 1 ? (T - 1) * ld : 0) + (H > 1 ? (H - 1) * h : 0) + D; };
  const int64_t pa = (int64_t)(reinterpret_cast<uintptr_t>(a) / 2), pb = (int64_t)(reinterpret_cast<uintptr_t>(b) / 2);
  if (pa + reach(lda, ha, Ha) <= pb || pb + reach(ldb, hb, Hb) <= pa) return false;
  const int64_t wa = (Ha > 1 ? (Ha - 1) * ha : 0) + D, wb = (Hb > 1 ? (Hb - 1) * hb : 0) + D;
  if (T > 1 && lda == ldb && lda > 0) {
    const int64_t d = ((pb - pa) % lda + lda) % lda;
    return d < wa || d + wb > lda;
  }
  return true;
}

// (T, H, D) rows that 16-byte loads reach; a stride that leads nowhere may be anything
inline bool rows_ok(const void* p, int64_t T, int64_t ld, int64_t H, int64_t hd) {
  return p && aligned16(p) && (T <= 1 || ld % 8 == 0) && (H <= 1 || hd % 8 == 0);
}

}  // namespace w4a8
