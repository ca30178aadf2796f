// extern "C" entry points of rotary positions and of attention over whole prompts (declared in include/w4a8_mi355x.h).
#include "abi_checks.h"
#include "prompt_attn.h"
#include "rotary.h"
#include "../../include/w4a8_mi355x.h"

namespace w4a8 {
int launch_prompt_attention(const PromptAttn& p, int D, int dtype, int64_t max_q, hipStream_t st);
int launch_rotary(Rotary& p, int D, int dtype, hipStream_t st);
}

using namespace w4a8;

extern "C" {

int w4a8_prompt_attention(const void* q, int64_t ldq, int64_t hq, const void* k, int64_t ldk, int64_t hk, const void* v,
                          int64_t ldv, int64_t hv, int dtype, int64_t T, int64_t Hq, int64_t H, int64_t D,
                          const int32_t* cu, int64_t B, float scale, int causal, int64_t window, int64_t max_q, void* out,
                          int64_t ldo, int64_t ho, float* lse, void* stream) {
  const char* who = "w4a8_prompt_attention";
  if (dtype != kBF16 && dtype != kF16) return fail(kErrInvalid, "%s: bf16 or fp16 (dtype %d)", who, dtype);
  if (D != 64 && D != 128 && D != 256)
    return fail(kErrUnsupported, "%s: heads of 64, 128 or 256 channels, got %lld", who, (long long)D);
  if (T < 0 || B < 0 || H < 1 || Hq < H || Hq % H || Hq > 32768)
    return fail(kErrInvalid, "%s: T=%lld B=%lld, %lld query heads (up to 32768) for %lld key/value heads", who, (long long)T,
                (long long)B, (long long)Hq, (long long)H);
  if (!(scale > 0.f && scale < 65536.f))
    return fail(kErrInvalid, "%s: the softmax scale must be positive and below 65536", who);
  if (window < 0 || window > 0x7fffffff || max_q < 0 || max_q > 0x7fffffff)
    return fail(kErrInvalid, "%s: window=%lld max_q=%lld", who, (long long)window, (long long)max_q);
  if (B > 65535 || T > 0x3fffffff / Hq)  // queries times heads are columns, indexed in 32 bits
    return fail(kErrUnsupported, "%s: past its index ranges (T=%lld, %lld query heads, B=%lld)", who, (long long)T,
                (long long)Hq, (long long)B);
  if (T == 0 || B == 0) return kOk;
  if (!cu) return fail(kErrInvalid, "%s: needs cu", who);
  if (!rows_ok(q, T, ldq, Hq, hq) || !rows_ok(k, T, ldk, H, hk) || !rows_ok(v, T, ldv, H, hv) || !rows_ok(out, T, ldo, Hq, ho))
    return fail(kErrInvalid, "%s: rows must be 16-byte aligned, with strides that are multiples of 8 elements", who);
  if (T <= 1) ldk = ldv = D;
  // a tile's rows are bounded, and reached, by 32-bit offsets
  if (ldk < D || ldv < D || ldk >= (1 << 23) || ldv >= (1 << 23))
    return fail(kErrUnsupported, "%s: k and v rows must be D to 2^23 elements apart, got %lld and %lld", who, (long long)ldk,
                (long long)ldv);
  if (!apart(T, ldo, Hq, ho, D))
    return fail(kErrInvalid, "%s: out's rows overlap (strides %lld and %lld)", who, (long long)ldo, (long long)ho);
  // a workgroup reads its queries where it writes their outputs, and nowhere else
  if (!(q == out && (T <= 1 || ldq == ldo) && (Hq <= 1 || hq == ho)) && collide(q, ldq, hq, out, ldo, ho, T, Hq, D))
    return fail(kErrInvalid, "%s: out overlaps q without being q itself", who);
  if (collide_rows(out, ldo, ho, Hq, k, ldk, hk, H, T, D) || collide_rows(out, ldo, ho, Hq, v, ldv, hv, H, T, D))
    return fail(kErrInvalid, "%s: out overlaps k or v", who);
  PromptAttn p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.ldq = ldq; p.hq = hq; p.ldk = ldk; p.hk = hk; p.ldv = ldv; p.hv = hv;
  p.out = static_cast<uint16_t*>(out);
  p.ldo = ldo; p.ho = ho;
  p.lse = lse;
  p.cu = cu;
  p.B = (int)B; p.T = T;
  p.H = (int)H; p.G = (int)(Hq / H);
  p.gmul = (uint32_t)((((uint64_t)1 << 31) + p.G - 1) / p.G);
  p.scale = scale * 1.4426950408889634f;
  p.causal = causal != 0;
  p.window = (int)window;
  return launched(launch_prompt_attention(p, (int)D, dtype, max_q, (hipStream_t)stream), who);
}

int w4a8_rotary(const void* q, int64_t ldq, int64_t hq, int64_t Hq, const void* k, int64_t ldk, int64_t hk, int64_t Hk,
                int dtype, int64_t T, int64_t D, int64_t R, int adjacent, const void* positions, int positions_64,
                int64_t axes, int64_t ldp, const uint64_t* turns, const int32_t* axis, float scale, void* q_out,
                int64_t ldqo, int64_t hqo, void* k_out, int64_t ldko, int64_t hko, void* stream) {
  const char* who = "w4a8_rotary";
  if (dtype != kBF16 && dtype != kF16) return fail(kErrInvalid, "%s: bf16 or fp16 (dtype %d)", who, dtype);
  if (D < 16 || D > 1024 || D % 8 || R < 16 || R > D || R % 16)
    return fail(kErrUnsupported, "%s: heads of 16 to 1024 channels (a multiple of 8), a multiple of 16 of which turn, got %lld "
                "of %lld", who, (long long)R, (long long)D);
  if (T < 0 || Hq < 1 || Hk < 0 || axes < 1 || axes > kRotaryMaxAxes || (axes > 1 && !axis))
    return fail(kErrInvalid, "%s: T=%lld, %lld and %lld heads, %lld axes (up to %d, with each pair's)", who, (long long)T,
                (long long)Hq, (long long)Hk, (long long)axes, kRotaryMaxAxes);
  if (T > 0x7fffffff || Hq > 32768 || Hk > 32768)
    return fail(kErrUnsupported, "%s: past its index ranges (T=%lld, %lld and %lld heads)", who, (long long)T, (long long)Hq,
                (long long)Hk);
  if (T == 0) return kOk;
  if (!positions || !turns) return fail(kErrInvalid, "%s: needs positions and turns", who);
  const struct { const void* in; int64_t ldi, hi; void* out; int64_t ldo, ho, H; const char* name; } rows[2] = {
      {q, ldq, hq, q_out, ldqo, hqo, Hq, "q"}, {k, ldk, hk, k_out, ldko, hko, Hk, "k"}};
  for (const auto& r : rows) {
    if (r.H == 0) continue;
    if (!rows_ok(r.in, T, r.ldi, r.H, r.hi) || !rows_ok(r.out, T, r.ldo, r.H, r.ho))
      return fail(kErrInvalid, "%s: rows must be 16-byte aligned, with strides that are multiples of 8 elements", who);
    if (!apart(T, r.ldo, r.H, r.ho, D))
      return fail(kErrInvalid, "%s: %s's output rows overlap (strides %lld and %lld)", who, r.name, (long long)r.ldo,
                  (long long)r.ho);
    // a thread reads what it writes, and nothing else
    if (!(r.in == r.out && (T <= 1 || r.ldi == r.ldo) && (r.H <= 1 || r.hi == r.ho)) &&
        collide(r.in, r.ldi, r.hi, r.out, r.ldo, r.ho, T, r.H, D))
      return fail(kErrInvalid, "%s: %s's output overlaps it without being it", who, r.name);
  }
  if (Hk && (collide_rows(q_out, ldqo, hqo, Hq, k, ldk, hk, Hk, T, D) || collide_rows(k_out, ldko, hko, Hk, q, ldq, hq, Hq, T, D) ||
             collide_rows(q_out, ldqo, hqo, Hq, k_out, ldko, hko, Hk, T, D)))
    return fail(kErrInvalid, "%s: q and k overlap", who);
  Rotary p = {};
  p.q = {static_cast<const uint16_t*>(q), static_cast<uint16_t*>(q_out), ldq, hq, ldqo, hqo, (int)Hq};
  p.k = {static_cast<const uint16_t*>(k), static_cast<uint16_t*>(k_out), ldk, hk, ldko, hko, (int)Hk};
  p.pos = positions;
  p.pos64 = positions_64 != 0;
  p.ldp = ldp;
  p.turn = turns;
  p.axis = axes > 1 ? axis : nullptr;
  p.T = T;
  p.R = (int)R;
  p.adjacent = adjacent != 0;
  p.scale = scale;
  return launched(launch_rotary(p, (int)D, dtype, (hipStream_t)stream), who);
}

}  // extern "C"
