// extern "C" entry points of the 4-bit cache and its attention (declared in include/w4a8_mi355x.h).
#include <stdarg.h>
#include <stdio.h>

#include "kv4.h"
#include "../../include/w4a8_mi355x.h"

namespace w4a8 {
int set_last_error(int code, const char* msg);
int launch_kv4_append(const void* k, int64_t ldk, int64_t hk, const void* v, int64_t ldv, int64_t hv, int dtype, int D,
                      const Kv4Cache& c, const Kv4Batch& s, hipStream_t st);
int launch_kv4_read(const Kv4Cache& c, const Kv4Batch& s, int dtype, int D, void* k, void* v, hipStream_t st);
Kv4Plan kv4_plan(int64_t T, int B, int H, int G, int D, int64_t max_q, int64_t max_kv);
int64_t kv4_workspace(int64_t T, int Hq, int D, int splits);
int launch_kv4_attention(Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, void* ws, hipStream_t st);
}  // namespace w4a8

using namespace w4a8;

static int fail(int code, const char* fmt, ...) {
  char msg[400];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(msg, sizeof msg, fmt, ap);
  va_end(ap);
  return set_last_error(code, msg);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

static int launched(int rc, const char* who) {
  if (rc == kOk) return kOk;
  if (rc == kErrUnsupported) return fail(rc, "%s: past its index ranges", who);
  return fail(kErrHip, "%s: HIP launch failed (%s)", who, hipGetErrorString(hipGetLastError()));
}

// the shapes that every call shares
static int shapes(const char* who, int dtype, int64_t T, int64_t H, int64_t D, int64_t pages, int64_t page_size, int64_t B,
                  int64_t width) {
  if (dtype != kBF16 && dtype != kF16) return fail(kErrInvalid, "%s: bf16 or fp16 (dtype %d)", who, dtype);
  if (D != 64 && D != 128 && D != 256)
    return fail(kErrUnsupported, "%s: heads of 64, 128 or 256 channels, got %lld", who, (long long)D);
  if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)))
    return fail(kErrUnsupported, "%s: pages of a power of two tokens from 16 to 65536, got %lld", who, (long long)page_size);
  if (T < 0 || B < 0 || H < 1 || pages < 1 || width < 0)
    return fail(kErrInvalid, "%s: sizes T=%lld B=%lld H=%lld pages=%lld table width=%lld", who, (long long)T, (long long)B,
                (long long)H, (long long)pages, (long long)width);
  // blocks of 8 tokens, rows and a sequence's tokens, to the end of the tile that has the last, are indexed in 32 bits
  if (B > 65535 || H > 65535 || T > 0x7fffffff || T * H > 0x7fffff00 || width > (0x7fffffff - 32) / page_size ||
      pages > ((int64_t)1 << 31) / (H * (page_size / 8)) - 1)
    return fail(kErrUnsupported, "%s: past its index ranges (T=%lld B=%lld H=%lld pages=%lld of %lld, width=%lld)", who,
                (long long)T, (long long)B, (long long)H, (long long)pages, (long long)page_size, (long long)width);
  return kOk;
}

static int operands(const char* who, void* kc, void* vc, void* ks, void* vs, int64_t pages, int64_t page_size, int64_t H,
                    const int32_t* table, int64_t ldt, int64_t width, const int32_t* cu, const int32_t* lens, int64_t B,
                    int64_t T, Kv4Cache& c, Kv4Batch& s) {
  if (!kc || !vc || !ks || !vs || !aligned16(kc) || !aligned16(vc) || !aligned16(ks) || !aligned16(vs))
    return fail(kErrInvalid, "%s: the cache's four arrays must be 16-byte aligned", who);
  if (!cu || !lens || (width > 0 && !table) || ldt < width)
    return fail(kErrInvalid, "%s: needs cu, seq_lens and a page table with stride >= width", who);
  int shift = 0;
  while (((int64_t)1 << shift) < page_size) ++shift;
  c.k = static_cast<uint8_t*>(kc);
  c.v = static_cast<uint8_t*>(vc);
  c.ks = static_cast<uint32_t*>(ks);
  c.vs = static_cast<uint32_t*>(vs);
  c.pages = pages; c.shift = shift; c.H = (int)H;
  s.table = table; s.ldt = ldt; s.width = (int)width;
  s.cu = cu; s.lens = lens; s.B = (int)B; s.T = T;
  return kOk;
}

// whether a (T, H, D) tensor of these strides has each element in a place of its own
static bool apart(int64_t T, int64_t ld, int64_t H, int64_t hd, int64_t D) {
  if (T <= 1) ld = H * (hd > D ? hd : D);
  if (H <= 1) hd = T * (ld > D ? ld : D);
  const bool rows_in = ld <= hd;  // the rows of a head are neighbours
  return rows_in ? ld >= D && hd >= (T - 1) * ld + D : hd >= D && ld >= (H - 1) * hd + D;
}

// whether (T, H, D) tensors at a and b of 16-bit elements may share some, as far as their strides tell
static bool collide(const void* a, int64_t lda, int64_t ha, const void* b, int64_t ldb, int64_t hb, int64_t T, int64_t H,
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

// (T, H, D) rows that 16-byte loads reach; a stride that leads nowhere may be anything
static bool rows_ok(const void* p, int64_t T, int64_t ld, int64_t H, int64_t hd) {
  return p && aligned16(p) && (T <= 1 || ld % 8 == 0) && (H <= 1 || hd % 8 == 0);
}

extern "C" {

int w4a8_kv4_append(const void* k, int64_t ldk, int64_t hk, const void* v, int64_t ldv, int64_t hv, int dtype, int64_t T,
                    int64_t H, int64_t D, void* k_codes, void* v_codes, void* k_scale, void* v_scale, int64_t pages,
                    int64_t page_size, const int32_t* table, int64_t ldt, int64_t width, const int32_t* cu,
                    const int32_t* seq_lens, int64_t B, void* stream) {
  const char* who = "w4a8_kv4_append";
  int rc = shapes(who, dtype, T, H, D, pages, page_size, B, width);
  if (rc || T == 0 || B == 0) return rc;
  Kv4Cache c;
  Kv4Batch s;
  rc = operands(who, k_codes, v_codes, k_scale, v_scale, pages, page_size, H, table, ldt, width, cu, seq_lens, B, T, c, s);
  if (rc) return rc;
  if (!rows_ok(k, T, ldk, H, hk) || !rows_ok(v, T, ldv, H, hv))
    return fail(kErrInvalid, "%s: k and v rows must be 16-byte aligned, with strides that are multiples of 8 elements", who);
  return launched(launch_kv4_append(k, ldk, hk, v, ldv, hv, dtype, (int)D, c, s, (hipStream_t)stream), who);
}

int w4a8_kv4_read(const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, int dtype,
                  int64_t pages, int64_t page_size, int64_t H, int64_t D, const int32_t* table, int64_t ldt, int64_t width,
                  const int32_t* cu, const int32_t* seq_lens, int64_t B, int64_t T, void* k, void* v, void* stream) {
  const char* who = "w4a8_kv4_read";
  int rc = shapes(who, dtype, T, H, D, pages, page_size, B, width);
  if (rc || T == 0 || B == 0) return rc;
  Kv4Cache c;
  Kv4Batch s;
  rc = operands(who, const_cast<void*>(k_codes), const_cast<void*>(v_codes), const_cast<void*>(k_scale),
                const_cast<void*>(v_scale), pages, page_size, H, table, ldt, width, cu, seq_lens, B, T, c, s);
  if (rc) return rc;
  if (!k || !v || !aligned16(k) || !aligned16(v)) return fail(kErrInvalid, "%s: k and v must be 16-byte aligned", who);
  return launched(launch_kv4_read(c, s, dtype, (int)D, k, v, (hipStream_t)stream), who);
}

int64_t w4a8_kv4_attention_workspace_bytes(int64_t T, int64_t Hq, int64_t H, int64_t D, int64_t B, int64_t max_q,
                                           int64_t max_kv) {
  if (T < 0 || B < 0 || H < 1 || Hq < H || Hq % H || max_q < 0 || max_kv < 0 || (D != 64 && D != 128 && D != 256) ||
      T > 0x7fffffff || B > 65535 || Hq > 32768 || max_q > 0x7fffffff || max_kv > 0x7fffffff)
    return -1;
  if (T == 0 || B == 0) return 0;
  return kv4_workspace(T, (int)Hq, (int)D, kv4_plan(T, (int)B, (int)H, (int)(Hq / H), (int)D, max_q, max_kv).splits);
}

int w4a8_kv4_attention(const void* q, int dtype, int64_t ldq, int64_t hq, int64_t T, int64_t Hq, int64_t H, int64_t D,
                       const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, int64_t pages,
                       int64_t page_size, const int32_t* table, int64_t ldt, int64_t width, const int32_t* cu,
                       const int32_t* seq_lens, int64_t B, float scale, int causal, int64_t window, int64_t max_q,
                       int64_t max_kv, void* out, int64_t ldo, int64_t ho, float* lse, void* workspace,
                       int64_t workspace_bytes, void* stream) {
  const char* who = "w4a8_kv4_attention";
  int rc = shapes(who, dtype, T, H, D, pages, page_size, B, width);
  if (rc) return rc;
  if (Hq < H || Hq % H || Hq > 32768)
    return fail(kErrInvalid, "%s: %lld query heads (up to 32768) for %lld key/value heads", who, (long long)Hq, (long long)H);
  if (!(scale > 0.f && scale < 65536.f))  // times a large query's power of two it has to stay in f32
    return fail(kErrInvalid, "%s: the softmax scale must be positive and below 65536", who);
  if (T * Hq > 0x3fffffff)  // queries times heads are columns, indexed in 32 bits
    return fail(kErrUnsupported, "%s: past its index ranges (T=%lld, %lld query heads)", who, (long long)T, (long long)Hq);
  if (window < 0 || window > 0x7fffffff || max_q < 0 || max_kv < 0 || max_q > 0x7fffffff || max_kv > 0x7fffffff)
    return fail(kErrInvalid, "%s: window=%lld max_q=%lld max_kv=%lld", who, (long long)window, (long long)max_q,
                (long long)max_kv);
  if (T == 0 || B == 0) return kOk;
  Kv4Attn p = {};
  rc = operands(who, const_cast<void*>(k_codes), const_cast<void*>(v_codes), const_cast<void*>(k_scale),
                const_cast<void*>(v_scale), pages, page_size, H, table, ldt, width, cu, seq_lens, B, T, p.c, p.s);
  if (rc) return rc;
  if (!rows_ok(q, T, ldq, Hq, hq) || !rows_ok(out, T, ldo, Hq, ho))
    return fail(kErrInvalid, "%s: q and out rows must be 16-byte aligned, with strides that are multiples of 8 elements", who);
  if (!apart(T, ldo, Hq, ho, D))
    return fail(kErrInvalid, "%s: out's rows overlap (strides %lld and %lld)", who, (long long)ldo, (long long)ho);
  const Kv4Plan pl = kv4_plan(T, (int)B, (int)H, (int)(Hq / H), (int)D, max_q, max_kv);
  const int64_t need = kv4_workspace(T, (int)Hq, (int)D, pl.splits);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(kErrInvalid, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)workspace_bytes);
  // a workgroup reads its queries where it writes their outputs, and nowhere else
  if (!(q == out && (T <= 1 || ldq == ldo) && (Hq <= 1 || hq == ho)) && collide(q, ldq, hq, out, ldo, ho, T, Hq, D))
    return fail(kErrInvalid, "%s: out overlaps q without being q itself", who);
  p.q = static_cast<const uint16_t*>(q);
  p.ldq = ldq; p.hq = hq;
  p.out = static_cast<uint16_t*>(out);
  p.ldo = ldo; p.ho = ho;
  p.lse = lse;
  p.G = (int)(Hq / H);
  p.gmul = (uint32_t)((((uint64_t)1 << 31) + p.G - 1) / p.G);
  p.scale = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.window = (int)window;
  return launched(launch_kv4_attention(p, (int)D, dtype, pl, workspace, (hipStream_t)stream), who);
}

}  // extern "C"
