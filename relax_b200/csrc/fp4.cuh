// Microscaled 4-bit floats: the formats, the layout of their scales, and conversions.
//
// A value is an e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign) times the scale of its block of consecutive k:
//   kMx  blocks of 32, scale 2^(byte - 127), byte 255 is NaN (e8m0)
//   kNv  blocks of 16, scale e4m3 without a sign, 0x7f is NaN, and one fp32 factor for the whole tensor
// Codes are rows of k / 2 bytes, the even k in the lower nibble.
//
// Scales lie in tiles of 128 rows x 4 blocks, 512 bytes each, tile (row / 128, block / 4) at
// (row / 128) * ceil(blocks / 4) + block / 4; inside a tile, row r and block b are at (r % 32) * 16 + (r / 32) * 4 + b.
// That is the order in which the tensor cores take scales from tensor memory: a row's four blocks are one 32-bit word, and
// a tile is one copy of 32 lanes x 16 bytes.  Rows and blocks past the matrix are zero (scale zero times code zero: what
// is beyond k adds nothing).
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"

namespace rb200 {
namespace f4 {

enum { kMx = 0, kNv = 1 };
enum { kF16 = 0, kBf16 = 1, kF32 = 2 };  // RB200_DTYPE_*

__host__ __device__ constexpr int block_of(int fmt) { return fmt == kMx ? 32 : 16; }
__host__ __device__ inline int64_t scale_row_tiles(int64_t rows) { return (rows + 127) / 128; }
__host__ __device__ inline int64_t scale_k_tiles(int64_t k, int fmt) { return (k / block_of(fmt) + 3) / 4; }
__host__ __device__ inline int64_t scale_bytes(int64_t rows, int64_t k, int fmt) {
  return scale_row_tiles(rows) * scale_k_tiles(k, fmt) * 512;
}
// byte offset of the word that holds blocks 4q .. 4q + 3 of a row
__host__ __device__ inline int64_t scale_word(int64_t row, int64_t q, int64_t k_tiles) {
  return ((row >> 7) * k_tiles + q) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// k must be whole blocks and rows whole 16-byte vectors of codes
#define RB200_FP4_CHECK_SHAPE(FMT, ROWS, K)                                                                       \
  RB200_CHECK((FMT) == f4::kMx || (FMT) == f4::kNv, "unknown 4-bit format %d", (int)(FMT));                       \
  RB200_CHECK((ROWS) >= 0 && (ROWS) < (1ll << 31) && (K) > 0 && (K) % 32 == 0 && (K) < (1ll << 30),               \
              "4-bit floats need k %% 32 == 0 and fewer than 2^31 rows (rows=%lld, k=%lld)", (long long)(ROWS), (long long)(K))

#ifdef __CUDACC__

// eight values -> eight codes (round to nearest, ties to the even code, saturating); element 0 in the lowest nibble
__device__ __forceinline__ uint32_t to_codes8(const float (&v)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
// eight codes -> four f16x2, in order
__device__ __forceinline__ void from_codes8(uint32_t w, uint32_t (&h)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "mov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
}
// e4m3 of a non-negative number: round to nearest even, saturating at 448
__device__ __forceinline__ uint32_t to_e4m3(float v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(0.0f), "f"(v));
  return r & 0x7fu;
}
// two e4m3 bytes -> f16x2
__device__ __forceinline__ uint32_t from_e4m3x2(uint32_t two) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  return r;
}
__device__ __forceinline__ float e4m3_value(uint32_t byte) {
  const uint32_t h = from_e4m3x2(byte & 0x7fu);
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}
__device__ __forceinline__ float e8m0_value(uint32_t byte) {  // 2^-127 is a subnormal
  return byte == 255u ? __uint_as_float(0x7fc00000u) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
template <int FMT>
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return FMT == kMx ? e8m0_value(byte) : e4m3_value(byte);
}

template <class T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(float v) { return v; }

#endif  // __CUDACC__

}  // namespace f4
}  // namespace rb200
