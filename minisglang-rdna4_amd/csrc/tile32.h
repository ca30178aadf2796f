// 32x32x16 products of 16-bit operands, and tiles of rows in LDS that both of attention's products read without bank
// conflicts (prompt_attn.hip, kv4_tree_attn.hip).
#pragma once
#include "w4a8_common.h"

namespace w4a8 {

typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4w __attribute__((ext_vector_type(4)));
typedef uint32_t v2w __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef short v4s __attribute__((__vector_size__(8)));


template <int DT>
__device__ __forceinline__ v16f mfma32(const v4w& a, const v4w& b, const v16f& c) {
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ uint32_t pack16(float a, float b) {
  if constexpr (DT == kBF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2b));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2h));
}

// both halves of a packed pair onto an f32 sum
template <int DT>
__device__ __forceinline__ float add_pair(uint32_t w, float c) {
#if defined(__HIP_DEVICE_COMPILE__)
  if constexpr (DT == kBF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, w), __builtin_bit_cast(v2b, 0x3f803f80u), c, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), __builtin_bit_cast(v2h, 0x3c003c00u), c, false);
#else
  return c;
#endif
}

// over the two lanes that hold a column (xor 32)
__device__ __forceinline__ float pair_max(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float pair_sum(float v) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// the maximum m itself where m times its factor is past what one f32 number holds to within 1, else 0
__device__ __forceinline__ float far_off(float m, float sc) {
  return fabsf(m) * sc >= 16777216.f && m != -__builtin_inff() ? m : 0.f;
}

// Where the 16 bytes `chunk` (8 channels) of row `r` lie in a tile of D channels, for the DMA and both kinds of read
template <int D>
struct Place {
  // keys. 256 channels: 8 waves share a tile (copies into LDS weigh most there: 4 waves 517 TFLOP/s, 8 waves 768)
  static constexpr int kTile = D == 256 ? 32 : 64;
  // rows of 64 channels come 8 to a DMA; the second 4 of them swap neighbouring chunks
  static constexpr int kGroup = D == 64 ? 1024 + 32 : 8 * D + 16;  // bytes from one group of rows to the next
  static constexpr int kRows = D == 64 ? 8 : 4;                    // rows of a group
  static constexpr int kBytes = kTile / kRows * kGroup;
  static constexpr int kDmas = kTile * D / 8 / 64;                 // wave-wide DMAs of a tile
  static __device__ __forceinline__ constexpr int at(int r, int chunk) {
    if (D == 64)
      return (r >> 3) * kGroup + ((r >> 2) & 1) * 512 + (chunk >> 2) * 256 + (r & 3) * 64 + ((chunk & 3) ^ ((r >> 2) & 1)) * 16;
    return (r >> 2) * kGroup + (chunk >> 2) * 256 + (r & 3) * 64 + (chunk & 3) * 16;
  }
  // DMA x's place in LDS, and the row and chunk that its lane brings there
  static __device__ __forceinline__ constexpr int dma_at(int x) {
    return D == 256 ? (x >> 1) * kGroup + (x & 1) * 1024 : x * kGroup;
  }
  static __device__ __forceinline__ int dma_row(int x, int lane) {
    return D == 64 ? x * 8 + ((lane >> 5) << 2) + ((lane >> 2) & 3) : (D == 256 ? x >> 1 : x) * 4 + ((lane >> 2) & 3);
  }
  static __device__ __forceinline__ int dma_chunk(int x, int lane) {
    if (D == 64) return ((lane >> 4) & 1) * 4 + ((lane & 3) ^ (lane >> 5));
    return (D == 256 ? (x & 1) * 16 : 0) + (lane >> 4) * 4 + (lane & 3);
  }
};

__device__ __forceinline__ v4w lds_read(const unsigned char* p) { return *reinterpret_cast<const v4w*>(p); }
// 4 keys of this lane's channel: the 16 lanes of a group give the addresses of 4 rows times 16 channels
__device__ __forceinline__ v2w lds_read_tr(const unsigned char* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(v2w, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p));
#else
  return v2w{0, 0};
#endif
}

}  // namespace w4a8
