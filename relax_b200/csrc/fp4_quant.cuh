// Sixteen consecutive elements of a row into 4-bit floats: what the quantiser and the linears of few rows do alike.
//
// kMx is exact in fp32 as it stands (division by a power of two).  kNv divides by s * ts, which fp32 cannot hold: x is
// multiplied by 1 / (s ts) taken once 2^-21 too small and once too large, and where the two codes differ - x lies next to the
// border between them - x and the border are compared in 64 bits, where border * s * ts is exact (3 + 4 + 24 bits).  The scale
// itself is settled the same way, by a 64-bit quotient where fp32 leaves it open: see e4m3_of.
#pragma once

#include "fp4.cuh"

namespace rb200 {
namespace f4 {

#ifdef __CUDACC__

// 16 consecutive elements as they lie in memory, their values, and the bits of their largest magnitude as fp32 (a NaN's are
// above infinity's)
template <class T>
struct Sixteen {
  static constexpr int kVectors = sizeof(T);  // of 16 bytes
  uint4 raw[kVectors];
  __device__ __forceinline__ void load(const T* p, bool wide) {
    if (wide) {  // 32-byte loads: the lanes' halves of a sector in one request
#pragma unroll
      for (int i = 0; i < kVectors; i += 2)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(raw[i].x), "=r"(raw[i].y), "=r"(raw[i].z), "=r"(raw[i].w), "=r"(raw[i + 1].x), "=r"(raw[i + 1].y),
                       "=r"(raw[i + 1].z), "=r"(raw[i + 1].w)
                     : "l"(reinterpret_cast<const uint4*>(p) + i));
    } else {
#pragma unroll
      for (int i = 0; i < kVectors; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kVectors; ++i) raw[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ uint32_t word(int i) const {
    const uint4& q = raw[i >> 2];
    return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
  }
  __device__ __forceinline__ float2 two(int i) const;  // elements 2i, 2i + 1
  __device__ __forceinline__ uint32_t top() const;
};
template <>
__device__ __forceinline__ float2 Sixteen<__half>::two(int i) const {
  const uint32_t w = word(i);
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 Sixteen<__nv_bfloat16>::two(int i) const {
  return make_float2(__uint_as_float(word(i) << 16), __uint_as_float(word(i) & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 Sixteen<float>::two(int i) const {
  return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
}
// (magnitudes of either 16-bit type order as integers, two at a time)
template <class T>
__device__ __forceinline__ uint32_t top_pair(const Sixteen<T>& v) {
  uint32_t m = v.word(0) & 0x7fff7fffu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, v.word(i) & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}
template <>
__device__ __forceinline__ uint32_t Sixteen<__half>::top() const {
  return __float_as_uint(__half2float(__ushort_as_half((unsigned short)top_pair(*this))));
}
template <>
__device__ __forceinline__ uint32_t Sixteen<__nv_bfloat16>::top() const {
  return top_pair(*this) << 16;
}
template <>
__device__ __forceinline__ uint32_t Sixteen<float>::top() const {
  uint32_t m = 0u;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, word(i) & 0x7fffffffu);
  return m;
}

// RNE_e4m3 of amax / (6 ts), r = that quotient in 64 bits (off by a few 2^-53).  The borders between e4m3 values have five
// bits, so the true quotient is on one or at least 2^-35 from it.  The detour through fp32 must not move it onto one:
// it is cut to fp32 and, where something larger than the error was cut off, made odd.
__device__ __forceinline__ uint32_t e4m3_of(double r) {
  const double up = r * (1.0 + 0x1p-46);
  float f = __double2float_rz(up);
  if (up - (double)f > r * 0x1p-45) f = __uint_as_float(__float_as_uint(f) | 1u);
  return to_e4m3(f);
}

// The same from fp32 where that settles it: the quotient once too small, once too large.
__device__ __forceinline__ uint32_t e4m3_of(float top, float per_six, double per_six_exact) {
  const float r = top * per_six;
  if (r >= 0x1p-12f && r <= 0x1p12f) {
    uint16_t two;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(two) : "f"(r * (1.0f + 0x1p-21f)), "f"(r * (1.0f - 0x1p-21f)));
    if ((two & 0xffu) == (two >> 8)) return two & 0x7fu;
  }
  return e4m3_of((double)top * per_six_exact);
}

// The border between codes c and c + 1 (magnitudes).
__device__ __forceinline__ double border_above(uint32_t c) {
  return c < 4 ? 0.25 + 0.5 * c : c == 4 ? 2.5 : c == 5 ? 3.5 : 5.0;
}
// The code's magnitude of |x| / unit, by comparisons in 64 bits.
static __device__ __noinline__ uint32_t code_by_borders(double ax, double unit) {
  uint32_t c = 0;
  for (; c < 7; ++c) {
    const double b = border_above(c) * unit;
    if (!(ax > b || (ax == b && (c & 1u)))) break;  // on a border: the even one of the two
  }
  return c;
}

// eight values times f -> codes
template <class T>
__device__ __forceinline__ uint32_t scaled_codes(const Sixteen<T>& v, int half, float f) {
  float y[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 q = v.two(4 * half + i);
    // both products in one instruction
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%0, %1};\n\tmov.b64 b, {%2, %2};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "+f"(q.x), "+f"(q.y)
        : "f"(f));
    y[2 * i] = q.x;
    y[2 * i + 1] = q.y;
  }
  return to_codes8(y);
}

// codes of 16 elements
template <int FMT, class T>
__device__ __forceinline__ void codes16(const Sixteen<T>& v, uint32_t byte, float ts, uint32_t (&out)[2]) {
  if (FMT == kMx) {
    const float inv = __uint_as_float((254u - byte) << 23);
    out[0] = scaled_codes(v, 0, inv);
    out[1] = scaled_codes(v, 1, inv);
    return;
  }
  const float s = e4m3_value(byte), unit = s * ts;
  if (byte == 0u) {
    out[0] = out[1] = 0u;
    return;
  }
  const bool plain = unit >= 0x1p-100f && unit <= 0x1p100f;
  const float inv = __frcp_rn(unit), below = inv * (1.0f - 0x1p-21f), above = inv * (1.0f + 0x1p-21f);
  uint32_t hi[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    out[h] = scaled_codes(v, h, below);
    hi[h] = scaled_codes(v, h, above);
  }
  if (out[0] == hi[0] && out[1] == hi[1] && plain) return;
  const double exact_unit = (double)s * (double)ts;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int sh = 4 * (i & 7);
    const uint32_t lo = (out[i >> 3] >> sh) & 15u, up = (hi[i >> 3] >> sh) & 15u;
    if (lo != up || !plain) {
      const float2 q = v.two(i >> 1);
      const float x = (i & 1) ? q.y : q.x;
      const double ax = fabs((double)x);
      uint32_t c;
      if (plain) {
        const double b = border_above(lo & 7u) * exact_unit;
        c = ax > b || (ax == b && (lo & 1u)) ? up : lo;
      } else {
        c = code_by_borders(ax, exact_unit) | (__float_as_uint(x) >> 28 & 8u);
      }
      out[i >> 3] = (out[i >> 3] & ~(15u << sh)) | (c << sh);
    }
  }
}


// A tensor's scale as the elements need it.
template <int FMT>
struct TensorScale {
  float ts, per_six;
  double per_six_exact;
  bool bad;  // every block gets the NaN scale
  __device__ __forceinline__ explicit TensorScale(float value) : ts(FMT == kNv ? value : 1.0f) {
    bad = FMT == kNv && !(ts > 0.0f && ts <= 3.402823466e38f);
    per_six_exact = FMT == kNv ? 1.0 / (6.0 * (double)ts) : 0.0;
    per_six = (float)per_six_exact;
  }
};
// The scale byte and the codes of 16 elements; kMx: neighbouring lanes (xor 1) hold a block together.
template <int FMT, class T>
__device__ __forceinline__ uint32_t quantise(const Sixteen<T>& v, const TensorScale<FMT>& ts, uint32_t (&c)[2]) {
  uint32_t top = v.top(), byte;
  if (FMT == kMx) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  const bool nan = top >= 0x7f800000u || ts.bad;
  c[0] = c[1] = 0u;
  if (nan) return FMT == kMx ? 255u : 0x7fu;
  if (FMT == kMx) {
    byte = top >> 23;
    byte = byte > 2u ? byte - 2u : 0u;
  } else {
    byte = e4m3_of(__uint_as_float(top), ts.per_six, ts.per_six_exact);
  }
  codes16<FMT>(v, byte, ts.ts, c);
  return byte;
}

#endif  // __CUDACC__

}  // namespace f4
}  // namespace rb200
