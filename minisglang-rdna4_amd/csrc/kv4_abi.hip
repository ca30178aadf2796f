// extern "C" entry points of the 4-bit cache and its attention (declared in include/w4a8_mi355x.h).
#include "abi_checks.h"
#include "kv4.h"
#include "../../include/w4a8_mi355x.h"

namespace w4a8 {
int launch_kv4_append(const void* k, int64_t ldk, int64_t hk, const void* v, int64_t ldv, int64_t hv, int dtype, int D,
                      const Kv4Cache& c, const Kv4Batch& s, hipStream_t st);
int launch_kv4_read(const Kv4Cache& c, const Kv4Batch& s, int dtype, int D, void* k, void* v, hipStream_t st);
Kv4Plan kv4_plan(int64_t T, int B, int H, int G, int D, int64_t max_q, int64_t max_kv);
Kv4Plan kv4_tree_plan(int64_t T, int B, int H, int G, int D, int64_t window, int64_t max_q, int64_t max_kv);
int64_t kv4_workspace(int64_t T, int Hq, int D, int splits);
int launch_kv4_attention(Kv4Attn& p, int D, int dtype, const Kv4Plan& pl, void* ws, hipStream_t st);
int launch_kv4_copy(const Kv4Caches& cs, int caches, const int32_t* src, const int32_t* dst, int64_t n, int64_t pages,
                    int64_t codes, int64_t scales, hipStream_t st);
int launch_kv4_keep(const Kv4Caches& cs, int caches, int D, const Kv4Cache& c, const Kv4Batch& s, const int32_t* keep, int64_t ldk,
                    int width, const int32_t* kept, int32_t* now, hipStream_t st);
int launch_kv4_tree(const int32_t* parents, const Kv4Batch& s, int words, int window, uint32_t* bits, int32_t* pos,
                    hipStream_t st);
}  // namespace w4a8

using namespace w4a8;

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

// w4a8_kv4_attention, and with bits w4a8_kv4_tree_attention
static int attend(const char* who, const void* q, int dtype, int64_t ldq, int64_t hq, int64_t T, int64_t Hq, int64_t H, int64_t D,
                  const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, int64_t pages,
                  int64_t page_size, const int32_t* table, int64_t ldt, int64_t width, const int32_t* cu,
                  const int32_t* seq_lens, int64_t B, float scale, int causal, int64_t window, int64_t max_q, int64_t max_kv,
                  const uint32_t* bits, int64_t ldb, int words, const int32_t* pos, void* out, int64_t ldo, int64_t ho,
                  float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
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
  const Kv4Plan pl = bits ? kv4_tree_plan(T, (int)B, (int)H, (int)(Hq / H), (int)D, window, max_q, max_kv)
                          : kv4_plan(T, (int)B, (int)H, (int)(Hq / H), (int)D, max_q, max_kv);
  const int64_t need = kv4_workspace(T, (int)Hq, (int)D, pl.splits);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return fail(kErrInvalid, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)workspace_bytes);
  // a workgroup reads its queries where it writes their outputs, and nowhere else
  if (!(q == out && (T <= 1 || ldq == ldo) && (Hq <= 1 || hq == ho)) && collide(q, ldq, hq, out, ldo, ho, T, Hq, D))
    return fail(kErrInvalid, "%s: out overlaps q without being q itself", who);
  p.bits = bits; p.ldb = ldb; p.words = words; p.pos = pos;
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

// a host array of each cache's four pointers
static int gather(const char* who, const void* const* arrays, int64_t caches, int64_t first, Kv4Caches& cs) {
  for (int64_t i = first; i < caches && i < first + kKv4Caches; ++i) {
    const void* const* a = arrays + 4 * i;
    for (int j = 0; j < 4; ++j)
      if (!a[j] || !aligned16(a[j])) return fail(kErrInvalid, "%s: the caches' arrays must be 16-byte aligned", who);
    Kv4Arrays& c = cs.c[i - first];
    c.k = static_cast<uint8_t*>(const_cast<void*>(a[0]));
    c.v = static_cast<uint8_t*>(const_cast<void*>(a[1]));
    c.ks = static_cast<uint32_t*>(const_cast<void*>(a[2]));
    c.vs = static_cast<uint32_t*>(const_cast<void*>(a[3]));
  }
  return kOk;
}
static int distinct(const char* who, const void* const* arrays, int64_t caches) {
  for (int64_t i = 0; i < caches; ++i)
    for (int64_t j = 0; j < i; ++j)
      if (arrays[4 * i] == arrays[4 * j]) return fail(kErrInvalid, "%s: a cache is given twice", who);
  return kOk;
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
  return attend("w4a8_kv4_attention", q, dtype, ldq, hq, T, Hq, H, D, k_codes, v_codes, k_scale, v_scale, pages, page_size, table,
                ldt, width, cu, seq_lens, B, scale, causal, window, max_q, max_kv, nullptr, 0, 0, nullptr, out, ldo, ho, lse,
                workspace, workspace_bytes, stream);
}

int w4a8_kv4_tree(const int32_t* parents, int64_t T, const int32_t* cu, const int32_t* seq_lens, int64_t B, int64_t words,
                  int64_t window, uint32_t* bits, int32_t* positions, void* stream) {
  const char* who = "w4a8_kv4_tree";
  if (T < 0 || B < 0 || words < 1 || words > 128 || window < 0 || window > 0x7fffffff)
    return fail(kErrInvalid, "%s: T=%lld B=%lld words=%lld (1 to 128) window=%lld", who, (long long)T, (long long)B,
                (long long)words, (long long)window);
  if (B > 0x7fffff || T > 0x7fffffff)
    return fail(kErrUnsupported, "%s: past its index ranges (T=%lld B=%lld)", who, (long long)T, (long long)B);
  if (T == 0 || B == 0) return kOk;
  if (!parents || !cu || !seq_lens || !bits || !positions)
    return fail(kErrInvalid, "%s: needs parents, cu, seq_lens, bits and positions", who);
  Kv4Batch s = {};
  s.cu = cu; s.lens = seq_lens; s.B = (int)B; s.T = T;
  return launched(launch_kv4_tree(parents, s, (int)words, (int)window, bits, positions, (hipStream_t)stream), who);
}

int64_t w4a8_kv4_tree_attention_workspace_bytes(int64_t T, int64_t Hq, int64_t H, int64_t D, int64_t B, int64_t window,
                                                int64_t max_q, int64_t max_kv) {
  if (w4a8_kv4_attention_workspace_bytes(T, Hq, H, D, B, max_q, max_kv) < 0 || window < 0) return -1;
  if (T == 0 || B == 0) return 0;
  return kv4_workspace(T, (int)Hq, (int)D, kv4_tree_plan(T, (int)B, (int)H, (int)(Hq / H), (int)D, window, max_q, max_kv).splits);
}

int w4a8_kv4_tree_attention(const void* q, int dtype, int64_t ldq, int64_t hq, int64_t T, int64_t Hq, int64_t H, int64_t D,
                            const void* k_codes, const void* v_codes, const void* k_scale, const void* v_scale, int64_t pages,
                            int64_t page_size, const int32_t* table, int64_t ldt, int64_t width, const int32_t* cu,
                            const int32_t* seq_lens, int64_t B, float scale, int64_t window, int64_t max_q, int64_t max_kv,
                            const uint32_t* bits, int64_t ldb, int64_t words, const int32_t* positions, void* out,
                            int64_t ldo, int64_t ho, float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "w4a8_kv4_tree_attention";
  if (T > 0 && B > 0 && (!bits || words < 1 || words > 128 || ldb < words || (window > 0 && !positions)))
    return fail(kErrInvalid, "%s: needs rows of 1 to 128 words of bits, and with a window positions", who);
  // a node past the table's end has a place of its own behind it
  if (page_size > 0 && page_size <= 65536 && width > (0x7fffffff - 64 - (T > 0 ? T : 0)) / page_size)
    return fail(kErrUnsupported, "%s: past its index ranges (T=%lld, width=%lld)", who, (long long)T, (long long)width);
  return attend(who, q, dtype, ldq, hq, T, Hq, H, D, k_codes, v_codes, k_scale, v_scale, pages, page_size, table, ldt, width, cu,
                seq_lens, B, scale, 1, window, max_q, max_kv, bits, ldb, (int)words, positions, out, ldo, ho, lse, workspace,
                workspace_bytes, stream);
}

int w4a8_kv4_copy_pages(const void* const* arrays, int64_t caches, int64_t pages, int64_t page_size, int64_t H, int64_t D,
                        const int32_t* src, const int32_t* dst, int64_t n, void* stream) {
  const char* who = "w4a8_kv4_copy_pages";
  int rc = shapes(who, kBF16, 0, H, D, pages, page_size, 1, 0);
  if (rc) return rc;
  if (caches < 0 || caches > 65535 || n < 0 || n > 0x7fffffff)
    return fail(kErrInvalid, "%s: %lld caches, %lld pairs", who, (long long)caches, (long long)n);
  if (caches == 0 || n == 0) return kOk;
  if (!arrays || !src || !dst) return fail(kErrInvalid, "%s: needs the caches' arrays, src and dst", who);
  if ((rc = distinct(who, arrays, caches))) return rc;
  const int64_t rows = H * page_size;  // in vectors of 16 bytes
  for (int64_t i = 0; i < caches; i += kKv4Caches) {
    Kv4Caches cs = {};
    if ((rc = gather(who, arrays, caches, i, cs))) return rc;
    const int64_t some = caches - i < kKv4Caches ? caches - i : kKv4Caches;
    rc = launched(launch_kv4_copy(cs, (int)some, src, dst, n, pages, rows * D / 32, rows / 4, (hipStream_t)stream), who);
    if (rc) return rc;
  }
  return kOk;
}

int w4a8_kv4_keep(const void* const* arrays, int64_t caches, int64_t pages, int64_t page_size, int64_t H, int64_t D,
                  const int32_t* table, int64_t ldt, int64_t width, const int32_t* cu, const int32_t* seq_lens, int64_t B,
                  const int32_t* keep, int64_t ldk, int64_t most, const int32_t* kept, int32_t* new_lens, void* stream) {
  const char* who = "w4a8_kv4_keep";
  int rc = shapes(who, kBF16, 0, H, D, pages, page_size, B, width);
  if (rc) return rc;
  if (caches < 1 || caches > 65535 || most < 0 || most > 0x7fffffff)
    return fail(kErrInvalid, "%s: %lld caches, up to %lld kept tokens", who, (long long)caches, (long long)most);
  if (B == 0) return kOk;
  if (!arrays || !kept || (most > 0 && !keep) || ldk < most)
    return fail(kErrInvalid, "%s: needs the caches' arrays, kept, and keep with a stride of at least its width", who);
  const struct { const int32_t* p; int64_t n; const char* name; } read[] = {
      {seq_lens, B, "seq_lens"}, {cu, B + 1, "cu"}, {kept, B, "kept"}, {keep, most > 0 ? (B - 1) * ldk + most : 0, "keep"},
      {table, width > 0 ? (B - 1) * ldt + width : 0, "the page table"}};
  for (const auto& r : read)
    if (new_lens && r.p && r.n > 0 && new_lens < r.p + r.n && r.p < new_lens + B)
      return fail(kErrInvalid, "%s: new_lens overlaps %s, which every workgroup reads", who, r.name);
  if ((rc = distinct(who, arrays, caches))) return rc;
  for (int64_t i = 0; i < caches; i += kKv4Caches) {
    Kv4Caches cs = {};
    if ((rc = gather(who, arrays, caches, i, cs))) return rc;
    Kv4Cache c;
    Kv4Batch s;
    rc = operands(who, cs.c[0].k, cs.c[0].v, cs.c[0].ks, cs.c[0].vs, pages, page_size, H, table, ldt, width, cu, seq_lens, B,
                  0x7fffffff, c, s);
    if (rc) return rc;
    const int64_t some = caches - i < kKv4Caches ? caches - i : kKv4Caches;
    rc = launched(launch_kv4_keep(cs, (int)some, (int)D, c, s, keep, ldk, (int)most, kept, i == 0 ? new_lens : nullptr,
                                  (hipStream_t)stream), who);
    if (rc) return rc;
  }
  return kOk;
}

}  // extern "C"
