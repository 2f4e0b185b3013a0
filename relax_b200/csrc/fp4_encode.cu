// Quantising to microscaled 4-bit floats, reading them back, and the layout of their scales.
//
// Definition, in real numbers with the named roundings only (RNE: to nearest, ties to the even code):
//   kMx  e = max(floor(log2(max |x|)) - 2, -127),  scale 2^e,             q = RNE_e2m1(x / 2^e),      |q| <= 6
//   kNv  s = RNE_e4m3(max |x| / (6 ts)) <= 448,    ts the tensor's scale, q = RNE_e2m1(x / (s ts)),   |q| <= 6
// over the blocks of a row; a block whose s is 0 has codes 0, one with an infinity or a NaN the NaN scale and codes 0, and
// where ts is not a positive finite number every block has the NaN scale.
//
// One pass over x: a lane takes 16 consecutive k, a warp 512 of a row (fp4_quant.cuh).  Memory bounds kMx (2 bytes read and 0.53
// written per fp16 element; 150 instructions a warp's 512 elements) and reading back, instruction issue kNv: 360
// instructions, most of them for the two products of every element, issued in 74 % of the clocks.
// Measured (fp16 and bf16, inputs out of memory): 1733 x 11008 in kMx 11.0 us (48 MB, 4.4 TB/s), back 9.2 us; 28672 x 8192 in
// kNv 150 us (602 MB, 4.0 TB/s), back 90 us (6.7 TB/s); one row of 4096 in kNv 3.1 us, back 2.1 us.
// A checkpoint's scales into tiles: 14.7 MB (28672 x 8192 in kNv) 56 us, 0.5 TB/s: a warp reads four bytes each of 32 rows, an
// eighth of each sector.  Done once per weight, so left as simple as it is.
#include "../../include/relax_b200.h"
#include "fp4_encode.h"
#include "fp4_quant.cuh"

namespace rb200 {
namespace {
using namespace f4;

constexpr int kWarps = 8;
constexpr int kRowsPerCta = 32;  // a CTA's rows, of 512 k (the quantiser's, of a small input: fewer)

struct EncodeParams {
  const void* x;
  int64_t ldx, batch_stride;
  int64_t rows, row_groups;  // groups of turns * kWarps, scale tiles' padding rows among them
  int64_t scale_stride;      // bytes from matrix to matrix
  int turns;                 // rows of a warp
  int64_t batch;
  int k, k_tiles, wide;
  const float* ts;
  uint8_t* codes;
  uint8_t* scales;
};

template <int FMT>
constexpr int kCtas = FMT == kMx ? 4 : 6;  // of an SM
template <int FMT>
constexpr int kRowsAhead = FMT == kMx ? 2 : 1;  // rows on their way to a warp (kNv: its instructions bound it)

template <int FMT, class T>
__global__ void __launch_bounds__(kWarps * 32, kCtas<FMT>) encode_fp4_kernel(const EncodeParams p, bool activations) {
  constexpr int kLanesPerBlock = FMT == kMx ? 2 : 1, kAhead = kRowsAhead<FMT>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int seg = (int)blockIdx.x * 32 + lane, k0 = seg * 16, q = seg / (4 * kLanesPerBlock);
  griddep_wait();
  // (weights, scales and zero points are never written by a kernel that lets its dependents start: matmuls may read them
  // ahead of their wait)
  if (activations) griddep_launch_dependents();
  for (int64_t e = blockIdx.z; e < p.batch; e += gridDim.z) {
    const TensorScale<FMT> ts(p.ts ? p.ts[e] : 1.0f);
    uint8_t* scales = p.scales + e * p.scale_stride;
    for (int64_t group = blockIdx.y; group < p.row_groups; group += gridDim.y) {
#pragma unroll 1
      for (int i = 0; i < p.turns; i += kAhead) {
        const int64_t row = (group * p.turns + i) * kWarps + warp;
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
          uint32_t c[2], byte = quantise<FMT>(v[j], ts, c);
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
int encode_typed(EncodeParams& p, int dtype, bool activations, cudaStream_t stream) {
  // A warp's rows come one after another (kMx: two by two), each a trip to memory: as few as fill the SMs once
  // (kNv, 48 rows of 28672: 8.9 us with four, 4.8 with one; 256 of 4096: 7.5 and 4.2).
  const int spans = (p.k_tiles * 4 * block_of(FMT) + 511) / 512;
  const int64_t room = (int64_t)kCtas<FMT> * sm_count_current();
  p.turns = kRowsPerCta / kWarps;
  while (p.turns > kRowsAhead<FMT> && p.rows * spans * p.batch <= room * kWarps * (p.turns / 2)) p.turns /= 2;
  p.row_groups = scale_row_tiles(p.rows) * 128 / (p.turns * kWarps);
  const dim3 grid = grid_of(spans, p.row_groups, p.batch);
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
  p.batch = batch;
  p.k = (int)k;
  p.k_tiles = (int)scale_k_tiles(k, fmt);
  p.scale_stride = scale_row_tiles(rows) * p.k_tiles * 512;
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
