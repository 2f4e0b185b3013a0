// Quantising to microscaled 4-bit floats, reading them back, and the layout of their scales.
//
// Definition, in real numbers with the named roundings only (RNE: to nearest, ties to the even code):
//   kMx  e = max(floor(log2(max |x|)) - 2, -127),  scale 2^e,             q = RNE_e2m1(x / 2^e),      |q| <= 6
//   kNv  s = RNE_e4m3(max |x| / (6 ts)) <= 448,    ts the tensor's scale, q = RNE_e2m1(x / (s ts)),   |q| <= 6
// over the blocks of a row; a block whose s is 0 has codes 0, one with an infinity or a NaN the NaN scale and codes 0, and
// where ts is not a positive finite number every block has the NaN scale.
//
// One pass over x: a lane takes 16 consecutive k, a warp 512, two rows on their way.  kMx is exact in fp32 as it stands (division by a power of
// two).  kNv divides by s * ts, which fp32 cannot hold: x is multiplied by 1 / (s ts) taken once 2^-21 too small and once too
// large, and where the two codes differ - x lies next to the border between them - x and the border are compared in 64
// bits, where border * s * ts is exact (3 + 4 + 24 bits).  The scale itself is rounded from a 64-bit quotient: see
// e4m3_of.  Memory bounds it: 2 bytes read and 0.53 or 0.56 written per fp16 element.
#include "../../include/relax_b200.h"
#include "fp4_encode.h"

namespace rb200 {
namespace {
using namespace f4;

constexpr int kWarps = 8;
constexpr int kRowsPerCta = 32;  // a CTA's rows, of 512 k

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
__device__ __noinline__ uint32_t code_by_borders(double ax, double unit) {
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

struct EncodeParams {
  const void* x;
  int64_t ldx, batch_stride;
  int64_t rows, row_groups;  // groups of kRowsPerCta, scale tiles' padding rows among them
  int64_t batch;
  int k, k_tiles, wide;
  const float* ts;
  uint8_t* codes;
  uint8_t* scales;
};

template <int FMT, class T>
__global__ void __launch_bounds__(kWarps * 32, FMT == kMx ? 4 : 6) encode_fp4_kernel(const EncodeParams p, bool activations) {
  constexpr int kLanesPerBlock = FMT == kMx ? 2 : 1, kAhead = FMT == kMx ? 2 : 1;  // rows on their way (kNv: its instructions bound it)
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seg = (int)blockIdx.x * 32 + lane, k0 = seg * 16, q = seg / (4 * kLanesPerBlock);
  griddep_wait();
  // (weights, scales and zero points are never written by a kernel that lets its dependents start: matmuls may read them
  // ahead of their wait)
  if (activations) griddep_launch_dependents();
  for (int64_t e = blockIdx.z; e < p.batch; e += gridDim.z) {
    const float ts = FMT == kNv && p.ts ? p.ts[e] : 1.0f;
    const bool bad = FMT == kNv && !(ts > 0.0f && ts <= 3.402823466e38f);
    const double per_six_exact = FMT == kNv ? 1.0 / (6.0 * (double)ts) : 0.0;
    const float per_six = (float)per_six_exact;
    uint8_t* scales = p.scales + e * (p.row_groups * kRowsPerCta / 128) * p.k_tiles * 512;
    for (int64_t group = blockIdx.y; group < p.row_groups; group += gridDim.y) {
#pragma unroll 1
      for (int i = 0; i < kRowsPerCta / kWarps; i += kAhead) {
        const int64_t row = group * kRowsPerCta + i * kWarps + warp;
        Sixteen<T> v[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          if (row + j * kWarps < p.rows && k0 < p.k)
            v[j].load(static_cast<const T*>(p.x) + e * p.batch_stride + (row + j * kWarps) * p.ldx + k0, p.wide != 0);
          else
            v[j].clear();
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
          const int64_t r = row + j * kWarps;
          const bool real = r < p.rows && k0 < p.k;
          uint32_t top = v[j].top(), byte;
          if (FMT == kMx) top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          const bool nan = top >= 0x7f800000u || bad;
          if (FMT == kMx) {
            byte = top >> 23;
            byte = byte > 2u ? byte - 2u : 0u;
          } else {
            byte = nan ? 0u : e4m3_of(__uint_as_float(top), per_six, per_six_exact);
          }
          uint32_t c[2] = {0u, 0u};
          if (nan) byte = FMT == kMx ? 255u : 0x7fu;
          else codes16<FMT>(v[j], byte, ts, c);
          if (real)
            *reinterpret_cast<uint2*>(p.codes + (e * p.rows + r) * (int64_t)(p.k / 2) + k0 / 2) = make_uint2(c[0], c[1]);
          else
            byte = 0u;
          // four blocks of a row are one word
          uint32_t w = byte << (8 * ((lane / kLanesPerBlock) & 3));
          w |= __shfl_xor_sync(0xffffffffu, w, kLanesPerBlock);
          w |= __shfl_xor_sync(0xffffffffu, w, 2 * kLanesPerBlock);
          if (lane % (4 * kLanesPerBlock) == 0 && q < p.k_tiles) *reinterpret_cast<uint32_t*>(scales + scale_word(r, q, p.k_tiles)) = w;
        }
      }
    }
  }
}

struct DecodeParams {
  const uint8_t* codes;
  const uint8_t* scales;
  int64_t rows, row_groups, row_tiles, batch;
  int k, k_tiles;
  const float* ts;
  void* out;
};

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  constexpr int kPer = 16 / sizeof(T);
#pragma unroll
  for (int i = 0; i < 8 / kPer; ++i) {
    __align__(16) T t[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) t[j] = narrow<T>(v[i * kPer + j]);
    reinterpret_cast<uint4*>(p)[i] = *reinterpret_cast<const uint4*>(t);
  }
}

// A warp takes 512 k of a row, a lane eight and eight further on by 256: what it stores is next to its neighbours'.
template <int FMT, class T>
__global__ void __launch_bounds__(kWarps * 32) decode_fp4_kernel(const DecodeParams p) {
  constexpr int kAhead = 4;
  griddep_wait();
  const int warp = threadIdx.x >> 5, k0 = (int)blockIdx.x * 512 + (threadIdx.x & 31) * 8;
  for (int64_t e = blockIdx.z; e < p.batch; e += gridDim.z) {
    const float ts = FMT == kNv && p.ts ? p.ts[e] : 1.0f;
    const uint8_t* scales = p.scales + e * p.row_tiles * p.k_tiles * 512;
    for (int64_t group = blockIdx.y; group < p.row_groups; group += gridDim.y) {
      uint32_t c[kAhead][2], byte[kAhead][2];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t r = group * kRowsPerCta + j * kWarps + warp;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = k0 + h * 256, blk = k / block_of(FMT);
          if (r < p.rows && k < p.k) {
            c[j][h] = *reinterpret_cast<const uint32_t*>(p.codes + (e * p.rows + r) * (int64_t)(p.k / 2) + k / 2);
            byte[j][h] = scales[scale_word(r, blk >> 2, p.k_tiles) + (blk & 3)];
          }
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const int64_t r = group * kRowsPerCta + j * kWarps + warp;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = k0 + h * 256;
          if (r < p.rows && k < p.k) {
            const float s = scale_value<FMT>(byte[j][h]);
            uint32_t w[4];
            from_codes8(c[j][h], w);
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
              v[2 * i] = FMT == kMx ? f.x * s : f.x * s * ts;  // code * scale is exact in fp32
              v[2 * i + 1] = FMT == kMx ? f.y * s : f.y * s * ts;
            }
            store8(static_cast<T*>(p.out) + (e * p.rows + r) * (int64_t)p.k + k, v);
          }
        }
      }
    }
  }
}
static_assert(kRowsPerCta == 4 * kWarps, "a warp's rows");

// a thread per word of the result
__global__ void __launch_bounds__(256) tile_scales_kernel(const uint8_t* src, uint32_t* dst, int64_t words, int64_t rows, int row_tiles,
                                                          int k_tiles, int blocks) {
  griddep_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= words) return;
  const int in_tile = (int)(i & 127);
  const int64_t tile = i >> 7, q = tile % k_tiles, rt = (tile / k_tiles) % row_tiles, e = tile / ((int64_t)k_tiles * row_tiles);
  const int64_t row = rt * 128 + (in_tile & 3) * 32 + (in_tile >> 2);
  uint32_t w = 0u;
  if (row < rows) {
    const uint8_t* s = src + (e * rows + row) * blocks + q * 4;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (q * 4 + b < blocks) w |= (uint32_t)s[b] << (8 * b);
  }
  dst[i] = w;
}

// a CTA per 512 k, rows and matrices beyond the grid's limits by loops
dim3 grid_of(int spans, int64_t row_groups, int64_t batch) {
  return dim3((unsigned)spans, (unsigned)(row_groups < 65535 ? row_groups : 65535), (unsigned)(batch < 65535 ? batch : 65535));
}

template <int FMT>
int encode_typed(const EncodeParams& p, int dtype, bool activations, cudaStream_t stream) {
  const dim3 grid = grid_of((p.k_tiles * 4 * block_of(FMT) + 511) / 512, p.row_groups, p.batch);
  if (dtype == kF16)
    RB200_CUDA(launch_dependent(encode_fp4_kernel<FMT, __half>, grid, kWarps * 32, 0, stream, p, activations));
  else if (dtype == kBf16)
    RB200_CUDA(launch_dependent(encode_fp4_kernel<FMT, __nv_bfloat16>, grid, kWarps * 32, 0, stream, p, activations));
  else
    RB200_CUDA(launch_dependent(encode_fp4_kernel<FMT, float>, grid, kWarps * 32, 0, stream, p, activations));
  return 0;
}
template <int FMT>
int decode_typed(const DecodeParams& p, int dtype, cudaStream_t stream) {
  const dim3 grid = grid_of((p.k + 511) / 512, p.row_groups, p.batch);
  if (dtype == kF16) RB200_CUDA(launch_dependent(decode_fp4_kernel<FMT, __half>, grid, kWarps * 32, 0, stream, p));
  else if (dtype == kBf16) RB200_CUDA(launch_dependent(decode_fp4_kernel<FMT, __nv_bfloat16>, grid, kWarps * 32, 0, stream, p));
  else RB200_CUDA(launch_dependent(decode_fp4_kernel<FMT, float>, grid, kWarps * 32, 0, stream, p));
  return 0;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace

int fp4_encode_launch(const void* x, int dtype, int64_t batch, int64_t rows, int64_t k, int64_t ldx, int64_t batch_stride, int fmt,
                      const float* tensor_scale, void* codes, void* scales, bool activations, cudaStream_t stream) {
  EncodeParams p;
  p.x = x;
  p.ldx = ldx;
  p.batch_stride = batch_stride;
  p.rows = rows;
  p.row_groups = scale_row_tiles(rows) * (128 / kRowsPerCta);
  p.batch = batch;
  p.k = (int)k;
  p.k_tiles = (int)scale_k_tiles(k, fmt);
  const int64_t width = dtype == kF32 ? 4 : 2;
  p.wide = reinterpret_cast<uintptr_t>(x) % 32 == 0 && ldx * width % 32 == 0 && batch_stride * width % 32 == 0;
  p.ts = tensor_scale;
  p.codes = static_cast<uint8_t*>(codes);
  p.scales = static_cast<uint8_t*>(scales);
  if (batch == 0 || rows == 0) return 0;
  return fmt == kMx ? encode_typed<kMx>(p, dtype, activations, stream) : encode_typed<kNv>(p, dtype, activations, stream);
}

}  // namespace rb200

using namespace rb200;

extern "C" {

size_t rb200_fp4_scale_bytes(int64_t rows, int64_t k, int format) {
  if ((format != f4::kMx && format != f4::kNv) || rows < 0 || k <= 0) return 0;
  return (size_t)f4::scale_bytes(rows, k, format);
}

int rb200_encode_fp4(const void* x, int dtype, int64_t batch, int64_t rows, int64_t k, int64_t ldx, int format,
                     const float* tensor_scale, void* codes, void* scales, void* stream) {
  RB200_FP4_CHECK_SHAPE(format, rows, k);
  RB200_CHECK(dtype >= f4::kF16 && dtype <= f4::kF32, "unknown element type %d", dtype);
  RB200_CHECK(batch >= 0, "batch must not be negative");
  if (batch == 0 || rows == 0) return 0;
  RB200_CHECK(x && codes && scales, "x, codes and scales must be non-NULL");
  RB200_CHECK(format == f4::kNv || !tensor_scale, "the mx format has no tensor scale");
  const int64_t width = dtype == f4::kF32 ? 4 : 2;
  RB200_CHECK(ldx >= k && ldx * width % 16 == 0 && aligned16(x) && aligned16(codes) && aligned16(scales),
              "x rows, codes and scales must be 16-byte aligned (ldx=%lld)", (long long)ldx);
  return fp4_encode_launch(x, dtype, batch, rows, k, ldx, rows * ldx, format, tensor_scale, codes, scales, false,
                           static_cast<cudaStream_t>(stream));
}

int rb200_decode_fp4(const void* codes, const void* scales, int64_t batch, int64_t rows, int64_t k, int format,
                     const float* tensor_scale, void* out, int dtype, void* stream) {
  RB200_FP4_CHECK_SHAPE(format, rows, k);
  RB200_CHECK(dtype >= f4::kF16 && dtype <= f4::kF32, "unknown element type %d", dtype);
  RB200_CHECK(batch >= 0, "batch must not be negative");
  if (batch == 0 || rows == 0) return 0;
  RB200_CHECK(codes && scales && out, "codes, scales and out must be non-NULL");
  RB200_CHECK(format == f4::kNv || !tensor_scale, "the mx format has no tensor scale");
  RB200_CHECK(aligned16(codes) && aligned16(scales) && aligned16(out), "codes, scales and out must be 16-byte aligned");
  DecodeParams p;
  p.codes = static_cast<const uint8_t*>(codes);
  p.scales = static_cast<const uint8_t*>(scales);
  p.rows = rows;
  p.row_groups = (rows + kRowsPerCta - 1) / kRowsPerCta;
  p.row_tiles = f4::scale_row_tiles(rows);
  p.batch = batch;
  p.k = (int)k;
  p.k_tiles = (int)f4::scale_k_tiles(k, format);
  p.ts = tensor_scale;
  p.out = out;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return format == f4::kMx ? decode_typed<f4::kMx>(p, dtype, s) : decode_typed<f4::kNv>(p, dtype, s);
}

int rb200_preprocess_fp4_scales(const void* src, void* dst, int64_t batch, int64_t rows, int64_t k, int format, void* stream) {
  RB200_FP4_CHECK_SHAPE(format, rows, k);
  RB200_CHECK(batch >= 0, "batch must not be negative");
  if (batch == 0 || rows == 0) return 0;
  RB200_CHECK(src && dst && src != dst, "src and dst must be non-NULL and different");
  RB200_CHECK(aligned16(dst), "dst must be 16-byte aligned");
  const int64_t row_tiles = f4::scale_row_tiles(rows), k_tiles = f4::scale_k_tiles(k, format), words = batch * row_tiles * k_tiles * 128;
  RB200_CHECK((words + 255) / 256 < (1ll << 31), "too many scales for one call");
  RB200_CUDA(launch_dependent(tile_scales_kernel, dim3((unsigned)((words + 255) / 256)), 256, 0, static_cast<cudaStream_t>(stream),
                              static_cast<const uint8_t*>(src), static_cast<uint32_t*>(dst), words, rows, (int)row_tiles, (int)k_tiles,
                              (int)(k / f4::block_of(format))));
  return 0;
}

}  // extern "C"
