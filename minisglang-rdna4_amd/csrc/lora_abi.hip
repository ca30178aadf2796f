// extern "C" entry points of the low-rank adapters (declared in include/w4a8_mi355x.h).
#include <stdarg.h>
#include <stdio.h>

#include "lora.h"
#include "../../include/w4a8_mi355x.h"

namespace w4a8 {
int set_last_error(int code, const char* msg);
int64_t lora_workspace(int64_t M, int64_t K, int64_t R);
int launch_lora(LoraArgs& p, int dtype, hipStream_t st);
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

// whether M rows of wa bytes, lda apart, may share bytes with M rows of wb bytes, ldb apart
static bool collide(const void* a, int64_t lda, int64_t wa, const void* b, int64_t ldb, int64_t wb, int64_t M) {
  const int64_t pa = (int64_t)reinterpret_cast<uintptr_t>(a), pb = (int64_t)reinterpret_cast<uintptr_t>(b);
  if (pa + (M - 1) * lda + wa <= pb || pb + (M - 1) * ldb + wb <= pa) return false;
  if (M > 1 && lda == ldb) {  // columns of one buffer
    const int64_t d = ((pb - pa) % lda + lda) % lda;
    return d < wa || d + wb > lda;
  }
  return true;
}

extern "C" {

int64_t w4a8_lora_workspace_bytes(int64_t M, int64_t K, int64_t rank, int slices) {
  if (M < 0 || K <= 0 || rank <= 0 || rank > kLoraMaxRank || rank % 8 || slices < 1 || slices > kLoraMaxSlices) return -1;
  return M == 0 ? 0 : lora_workspace(M, K, rank * slices);
}

int w4a8_lora_add(const void* x, int dtype, int64_t M, int64_t K, int64_t ldx, const void* a, const void* b,
                  const float* scaling, int64_t L, int64_t rank, const int64_t* slice_cols, int slices,
                  const int32_t* adapters, const void* base, int base_dtype, int64_t ldb, void* out, int64_t ldo,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "w4a8_lora_add";
  if (dtype != kBF16 && dtype != kF16) return fail(kErrInvalid, "%s: bf16 or fp16 (dtype %d)", who, dtype);
  if (base_dtype != dtype && base_dtype != kF32)
    return fail(kErrInvalid, "%s: base must be f32 or of x's type (dtype %d)", who, base_dtype);
  if (M < 0 || K <= 0 || K % 8 || L < 1 || L > 0x7fffffff)
    return fail(kErrInvalid, "%s: M=%lld K=%lld (a multiple of 8) adapters=%lld", who, (long long)M, (long long)K, (long long)L);
  if (rank <= 0 || rank > kLoraMaxRank || rank % 8)
    return fail(kErrUnsupported, "%s: ranks that are multiples of 8 up to %d, got %lld (pad A and B with zeros)", who,
                kLoraMaxRank, (long long)rank);
  if (slices < 1 || slices > kLoraMaxSlices || !slice_cols)
    return fail(kErrUnsupported, "%s: 1 to %d slices, got %d", who, kLoraMaxSlices, slices);
  LoraArgs p = {};
  int64_t n = 0;
  for (int i = 0; i < slices; ++i) {
    if (slice_cols[i] <= 0 || slice_cols[i] % 16 || slice_cols[i] > 0x7fffffff)
      return fail(kErrInvalid, "%s: slice %d has %lld columns (multiples of 16)", who, i, (long long)slice_cols[i]);
    p.col[i] = n;
    n += slice_cols[i];
  }
  for (int i = slices; i <= kLoraMaxSlices; ++i) p.col[i] = n;
  if (M == 0) return kOk;
  if (M > (1 << 26))
    return fail(kErrUnsupported, "%s: past its index ranges (M=%lld, N=%lld)", who, (long long)M, (long long)n);
  if (!x || !a || !b || !scaling || !adapters || !base || !out || !aligned16(x) || !aligned16(a) || !aligned16(b) ||
      !aligned16(base) || !aligned16(out))
    return fail(kErrInvalid, "%s: x, a, b, base and out must be 16-byte aligned, scaling and adapters given", who);
  if (ldx < K || ldx % 8 || ldo < n || ldo % 8 || ldb < n || ldb % 8)
    return fail(kErrInvalid, "%s: row strides must be multiples of 8 that hold a row (ldx=%lld ldb=%lld ldo=%lld)", who,
                (long long)ldx, (long long)ldb, (long long)ldo);
  // a row's workgroups read base where they write out, and nowhere else
  const int64_t bs = base_dtype == kF32 ? 4 : 2;
  if (!(base == out && bs == 2 && (M == 1 || ldb == ldo)) && collide(base, ldb * bs, n * bs, out, ldo * 2, n * 2, M))
    return fail(kErrInvalid, "%s: out overlaps base without being base itself", who);
  const int64_t need = lora_workspace(M, K, rank * slices);
  if (!workspace || workspace_bytes < need || !aligned16(workspace))
    return fail(kErrInvalid, "%s: needs a 16-byte aligned workspace of %lld bytes, got %lld", who, (long long)need,
                (long long)workspace_bytes);
  p.x = static_cast<const uint16_t*>(x);
  p.ldx = ldx; p.M = M; p.K = K;
  p.a = static_cast<const uint16_t*>(a);
  p.b = static_cast<const uint16_t*>(b);
  p.scaling = scaling; p.ids = adapters;
  p.L = (int)L; p.rank = (int)rank; p.slices = slices; p.N = n;
  p.base = base; p.ldb = ldb; p.base_f32 = base_dtype == kF32;
  p.out = static_cast<uint16_t*>(out);
  p.ldo = ldo;
  p.v = static_cast<float*>(workspace);
  const int rc = launch_lora(p, dtype, (hipStream_t)stream);
  if (rc == kErrUnsupported)
    return fail(rc, "%s: past its index ranges (M=%lld, N=%lld)", who, (long long)M, (long long)n);
  if (rc != kOk)
    return fail(kErrHip, "%s: HIP launch failed (%s)", who, hipGetErrorString(hipGetLastError()));
  return kOk;
}

}  // extern "C"
