// out = unary(binary(act(ta tw sum_k a[m, k] w[n, k] + bias[n]), residual[m, n])) of two microscaled 4-bit operands.
//
// The tensor cores take codes and block scales as they are (tcgen05.mma, block_scale): nothing is decoded.  Here are batches
// of at most 64 rows, fp4_pair.cu has the larger ones.  The tile is out^T, 128 rows of w by the batch (nb, rounded up to 16,
// is the MMA's N); a stage is 256 k: two tensor-map loads of codes and the scale tiles, which the MMA's thread copies into
// tensor memory ahead of the MMAs that read them.
// With few tiles k is cut over the CTAs of a cluster: each keeps its partial tile in shared memory (the stages' memory, done
// with by then), and each adds up its share of the batch rows in the order of the ranks, so that a result does not depend
// on timing.
//
// What bounds it is reading w once: k 28672 x n 8192 in the mx format, 125 MB, takes 24.1 us for one row out of memory (the
// kernel alone, 5.2 TB/s), 22.1 a call in a row of calls; two CTAs an SM keep some 200 KB on their way there.  Small ones are
// launch and one trip to memory and back through the cluster: k 4096 x n 4096 in the nv format, 9.4 MB, 6.5 us a call in a row,
// 8.2 to 8.8 the kernel alone out of memory, of which the reading is 1.5.
#include <atomic>

#include <cstring>

#include "fp4_encode.h"
#include "fp4_gemm.h"
#include "fp4_mma.cuh"
#include "fp4_out.cuh"
#include "fp4_quant.cuh"
#include "tensormap.h"

namespace rb200 {
namespace f4 {
namespace {

using ug::elect_one;
using ug::make_b_desc;
using ug::tc_commit;
using ug::tc_fence_after;
using ug::tc_fence_before;
using ug::tc_ld16;
using ug::tmem_alloc;
using ug::tmem_dealloc;
using ug::tmem_relinquish;

constexpr int kThreads = 192;
constexpr int kTileN = 128;
constexpr int kMaxStages = 8;
constexpr int kWBytes = kTileN * 128;

__device__ int g_status;

struct Params {
  Output o;
  const uint8_t* a_scales;
  const uint8_t* w_scales;
  int k, k_tiles;
  int nb, stages, tmem_cols, cluster, early;
  const void* x;  // QX: the batch as it is, of out's type
  int64_t ldx;
};

size_t stage_bytes(int fmt, int nb) {
  return (size_t)kWBytes + (size_t)nb * 128 + (size_t)stage_tiles(fmt) * 512 * 2;
}
size_t smem_bytes(int fmt, int nb, int stages) { return 1024 + stages * stage_bytes(fmt, nb) + (2 * kMaxStages + 2) * 8 + 32; }

// QX: `a` is quantised here, by the warps that have nothing to do before the epilogue, one chunk a warp.
template <int FMT, class T, bool QX>
__global__ void __launch_bounds__(kThreads)
    fp4_gemm_kernel(const Params p, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a) {
  constexpr int NT = stage_tiles(FMT);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int nb = p.nb, stages = p.stages;
  const int code_bytes = kWBytes + nb * 128;
  constexpr int scale_bytes = NT * 512 * 2;
  uint8_t* codes = smem;                                   // [stage][w | a]
  uint8_t* scales = smem + (size_t)stages * code_bytes;    // [stage][w tiles | a tiles]
  uint64_t* full = reinterpret_cast<uint64_t*>(scales + (size_t)stages * scale_bytes);
  uint64_t* empty = full + kMaxStages;
  uint64_t* d_full = empty + kMaxStages;
  uint32_t* holder = reinterpret_cast<uint32_t*>(d_full + 2);  // [0] tensor memory, [1] a CTA of the cluster failed

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), n0 = (int)blockIdx.x / p.cluster * kTileN;
  const int chunks = (p.k + kStageK - 1) / kStageK;
  const int c0 = (int)((int64_t)chunks * rank / p.cluster), c1 = (int)((int64_t)chunks * (rank + 1) / p.cluster);

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], QX ? 2 : 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(d_full, 1);
    holder[1] = 0u;
    mbar_fence_init();
  }
  if (warp == 1) {
    tmem_alloc(holder, (uint32_t)p.tmem_cols);
    tmem_relinquish();
  }
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = holder[0];
  const int w_col = (nb + 31) / 32 * 32, a_col = w_col + 4 * NT;  // tensor memory columns of the scales
  bool ok = true;

  if (warp == 0) {
    // ============================================================ loads
    const bool leader = elect_one();
    // bytes of the scale tiles of chunk c for 128 rows
    auto tiles_of = [&](int c) { return (uint32_t)min(NT, p.k_tiles - c * NT) * 512u; };
    auto load_w = [&](int s, int c) {
      uint8_t* at = scales + (size_t)s * scale_bytes;
      mbar_arrive_expect_tx(&full[s], (uint32_t)(QX ? kWBytes : code_bytes) + tiles_of(c) * (QX ? 1 : 2));
      tma_load(codes + (size_t)s * code_bytes, &tmap_w, c * 128, n0, &full[s]);
      bulk_g2s(at, p.w_scales + ((int64_t)(n0 >> 7) * p.k_tiles + c * NT) * 512, tiles_of(c), &full[s]);
    };
    auto load_a = [&](int s, int c) {
      if (QX) return;
      uint8_t* at = scales + (size_t)s * scale_bytes + NT * 512;
      tma_load(codes + (size_t)s * code_bytes + kWBytes, &tmap_a, c * 128, 0, &full[s]);
      bulk_g2s(at, p.a_scales + (int64_t)c * NT * 512, tiles_of(c), &full[s]);
    };
    const int first = min(stages, c1 - c0);  // stages filled before any is free again
    if (leader) {
      if (p.early) {
        for (int s = 0; s < first; ++s) load_w(s, c0 + s);
      } else {
        for (int s = 0; s < first; ++s) tma_prefetch(&tmap_w, (c0 + s) * 128, n0);
      }
    }
    griddep_wait();
    if (leader)
      for (int s = 0; s < first; ++s) {
        if (!p.early) load_w(s, c0 + s);
        load_a(s, c0 + s);
      }
    int s = 0, issued = first;
    uint32_t ph = 0;
    for (int c = c0 + first; c < c1; ++c) {
      if (!mbar_wait_parked(&empty[s], ph, &g_status)) {
        ok = false;
        break;
      }
      if (leader) {
        load_w(s, c);
        load_a(s, c);
      }
      ++issued;
      __syncwarp();
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    // nothing may be on its way into this CTA's memory when it leaves: the last fill of every stage
    for (int i = max(0, issued - stages); i < issued; ++i)
      ok = mbar_wait_parked(&full[i % stages], (uint32_t)(i / stages) & 1u, &g_status) && ok;
  } else if (warp == 1) {
    // ============================================================ scales into tensor memory, MMAs
    const bool leader = elect_one();
    const uint32_t idesc = mma_desc<FMT>(kTileN, nb);
    const uint64_t w_desc0 = make_b_desc(smem_u32(codes)), sc0 = scale_desc(smem_u32(scales));
    int s = 0;
    uint32_t ph = 0;
    for (int c = c0; c < c1; ++c) {
      ok = mbar_wait_parked(&full[s], ph, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      if (leader) {
        const uint64_t w_desc = w_desc0 + (uint64_t)(s * (code_bytes >> 4)), a_desc = w_desc + (uint64_t)(kWBytes >> 4);
        const uint64_t sc = sc0 + (uint64_t)(s * (scale_bytes >> 4));
        const int mmas = min(kStageK, p.k - c * kStageK + kMmaK - 1) / kMmaK;
        // (scale tiles past the last k are copied as they lie there; no MMA reads them)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          copy_scales(tmem + w_col + 4 * t, sc + (uint64_t)(t * (512 >> 4)));
          copy_scales(tmem + a_col + 4 * t, sc + (uint64_t)((NT + t) * (512 >> 4)));
        }
#pragma unroll
        for (int j = 0; j < kStageK / kMmaK; ++j) {
          const int t = FMT == kMx ? j >> 1 : j;
          if (j < mmas)
            mma_scaled<FMT>(tmem, w_desc + j * 2, a_desc + j * 2, FMT == kMx && (j & 1) ? upper_half(idesc) : idesc, tmem + w_col + 4 * t,
                            tmem + a_col + 4 * t, (c > c0 || j > 0) ? 1u : 0u);
        }
        tc_commit(&empty[s]);
      }
      __syncwarp();
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
    if (ok && leader) tc_commit(d_full);
    __syncwarp();
  } else if (QX) {
    // ============================================================ the batch's rows, quantised into the stages
    griddep_wait();
    const TensorScale<FMT> ts(p.o.a_ts ? *p.o.a_ts : 1.0f);
    for (int i = warp - 2; i < c1 - c0; i += kThreads / 32 - 2) {
      const int s = i % stages, c = c0 + i;
      ok = mbar_wait_parked(&empty[s], ((uint32_t)(i / stages) & 1u) ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      uint8_t* a = codes + (size_t)s * code_bytes + kWBytes;
      uint8_t* sc = scales + (size_t)s * scale_bytes + NT * 512;
      for (int j = lane; j < (p.o.m * 16 + 31) / 32 * 32; j += 32) {  // (whole warps: lanes exchange maxima)
        const int row = j >> 4, seg = j & 15, k = c * kStageK + seg * 16;
        Sixteen<T> v;
        const bool real = row < p.o.m && k < p.k;
        if (real) v.load(static_cast<const T*>(p.x) + row * p.ldx + k, false);
        else v.clear();
        uint32_t q[2];
        const uint32_t byte = quantise<FMT>(v, ts, q);
        if (row < p.o.m) {
          // 128-byte rows, their 16-byte columns swizzled as the tensor maps do it
          *reinterpret_cast<uint2*>(a + row * 128 + (((seg >> 1) ^ (row & 7)) << 4) + (seg & 1) * 8) = make_uint2(q[0], q[1]);
          const int blk = FMT == kMx ? seg >> 1 : seg;
          if (FMT == kNv || (seg & 1) == 0) sc[(blk >> 2) * 512 + (row & 31) * 16 + (blk & 3)] = (uint8_t)(real ? byte : 0u);
        }
      }
      fence_proxy_async();  // the tensor cores read it
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[s]);
    }
  }

  // ============================================================ the tile, by batch rows: [nb][128] fp32 where the stages were
  float* part = reinterpret_cast<float*>(smem);
  griddep_wait();
  const float alpha = out_scale(p.o);
  const int lo = p.o.m * rank / p.cluster, hi = p.o.m * (rank + 1) / p.cluster;  // this CTA's rows of the result
  const int n = n0 + lane * 4;
  float bias[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) bias[i] = bias_at<T>(p.o, n + i);
  if (p.o.residual && n < p.o.n)
    for (int m = lo + warp; m < hi; m += kThreads / 32) prefetch_line(static_cast<const T*>(p.o.residual) + m * p.o.ld_res + n);
  ok = mbar_wait_parked(d_full, 0, &g_status) && ok;  // every stage has been read
  ok = __all_sync(0xffffffffu, ok);
  if (!ok) {
    for (int r = 0; r < p.cluster; ++r) st_cluster(at_rank(smem_u32(holder + 1), r), 1u);
  }
  __syncthreads();
  tc_fence_after();
  if (warp >= 2 && ok) {
    const int quad = warp & 3;
    const uint32_t lane_taddr = (uint32_t)(32 * quad) << 16;
    for (int c = 0; c < nb; c += 16) {
      float v[16];
      tc_ld16(lane_taddr | (tmem + c), v);
#pragma unroll
      for (int i = 0; i < 16; ++i) part[(c + i) * kTileN + quad * 32 + lane] = v[i];
    }
  }
  tc_fence_before();
  if (p.cluster > 1) cluster_sync();
  else __syncthreads();
  if (holder[1] == 0u) {
    T* out = static_cast<T*>(p.o.out);
    const bool wide = n + 4 <= p.o.n && (reinterpret_cast<uintptr_t>(out) & (4 * sizeof(T) - 1)) == 0 && p.o.ldo % 4 == 0;
    for (int m = lo + warp; m < hi; m += kThreads / 32) {
      const uint32_t at = smem_u32(part + m * kTileN + lane * 4);
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int q = 0; q < p.cluster; ++q) {
        const float4 o = ld_cluster4(p.cluster > 1 ? at_rank(at, q) : at);
        v.x += o.x;
        v.y += o.y;
        v.z += o.z;
        v.w += o.w;
      }
      float f[4] = {v.x, v.y, v.z, v.w};
      float x[4];
      if (p.o.residual) load_residual<T, false>(p.o, x, m, n);
      finish<false>(p.o, f, alpha, bias, x);
      __align__(16) T t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = narrow<T>(f[i]);
      T* dst = out + m * p.o.ldo + n;
      if (wide) {
        if (sizeof(T) == 2) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(t);
        else *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(t);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (n + i < p.o.n) dst[i] = t[i];
      }
    }
  }
  if (p.cluster > 1) cluster_sync();  // others may still be reading this CTA's part
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, (uint32_t)p.tmem_cols);
  }
}

constexpr int kMaxDevices = 64;
std::atomic<bool> g_launched[kMaxDevices];  // devices whose status word a wait may have set

// CTAs that share a tile's k: as many as leave two CTAs an SM and two chunks each.  The kernel alone out of memory, us, with
// 1 / 2 / 4 / 8 of them: mx, one row, k 28672 x n 8192 33.9 / 26.0 / 24.2 / 28.3 (4 taken); mx, 7 rows, k 4096 x n 32016
// 16.2 / 20.0 / 27.6 / 46.8 (1); nv, 48 rows, k 28672 x n 8192 40.3 / 29.6 / 26.5 / 32.4 (4); mx, 16 rows, k 8192 x n 2048
// 13.1 / 10.2 / 8.2 / 8.3 (8); mx, 4 rows, k 4096 x n 1024 9.0 / 7.9 / 6.9 / 6.5 (8); nv, one row, k = n = 4096
// 8.9 / 8.1 / 7.6 / 8.2 (8: four would be 7 % less); nv, 16 rows, k 4096 x n 14336 10.9 / 11.7 / 15.6 / 25.2 (2: one would be
// 7 % less).
int cluster_of(int tiles, int64_t k) {
  const int chunks = (int)((k + kStageK - 1) / kStageK);
  int c = 1;
  while (c < 8 && tiles * c * 2 <= 2 * sm_count_current() && chunks >= 4 * c) c *= 2;
  return c;
}

template <int FMT, class T, bool QX>
int launch_typed(Params& p, const CUtensorMap& tw, const CUtensorMap& ta, cudaStream_t stream) {
  auto kern = fp4_gemm_kernel<FMT, T, QX>;
  static thread_local int configured_device = -1;
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (configured_device != dev) {
    RB200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_device = dev;
  }
  const int tiles = (p.o.n + kTileN - 1) / kTileN;
  p.cluster = cluster_of(tiles, p.k);
  p.stages = kMaxStages;
  while (smem_bytes(FMT, p.nb, p.stages) > 113 * 1024) --p.stages;  // two CTAs an SM; three stages or more
  const size_t smem = smem_bytes(FMT, p.nb, p.stages);  // (three stages hold 48 KB of w, a tile of sums 32)
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.cluster), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  RB200_CUDA(cudaLaunchKernelEx(&cfg, kern, p, tw, ta));
  return 0;
}

template <int FMT, bool QX>
int launch_fmt(Params& p, int dtype, const CUtensorMap& tw, const CUtensorMap& ta, cudaStream_t stream) {
  switch (dtype) {
    case kF16: return launch_typed<FMT, __half, QX>(p, tw, ta, stream);
    case kBf16: return launch_typed<FMT, __nv_bfloat16, QX>(p, tw, ta, stream);
    default: return launch_typed<FMT, float, QX>(p, tw, ta, stream);
  }
}

// Few rows are quantised by the product's CTAs, each its share of k for itself, where that takes less than a kernel before it:
// one or two rows (k 4096 x n 4096: 13.3 -> 12.3 us with the launches and cold, k 28672 x n 8192: 33.8 -> 30.7), and three or four
// where a CTA's four warps have at most two turns of 256 k x two rows each (k 4096 x n 4096: four rows, two turns, 13.3 -> 12.4;
// eight rows, four turns, 13.3 -> 14.3; k 4096 x n 11008, four rows, four turns, 15.4 -> 16.4).
bool quantises_itself(int64_t m, int64_t n, int64_t k) {
  if (m <= 2) return true;
  const int tiles = (int)((n + kTileN - 1) / kTileN), per = (int)((k + kStageK - 1) / kStageK + cluster_of(tiles, k) - 1) / cluster_of(tiles, k);
  return m <= 4 && (per + 3) / 4 * ((m + 1) / 2) <= 2;
}

}  // namespace
}  // namespace f4

int fp4_gemm_read_status(int* status_out) {
  *status_out = 0;
  int dev = -1;
  RB200_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= f4::kMaxDevices || !f4::g_launched[dev].load(std::memory_order_relaxed)) return 0;
  int v = 0, pairs = 0;
  RB200_CUDA(cudaMemcpyFromSymbol(&v, f4::g_status, sizeof(int)));
  if (v != 0) {
    const int zero = 0;
    RB200_CUDA(cudaMemcpyToSymbol(f4::g_status, &zero, sizeof(int)));
  }
  if (fp4_pair_read_status(&pairs) != 0) return -1;
  *status_out = v != 0 ? v : pairs;
  return 0;
}

static int fp4_few_launch(const rb200_gemm_fp4_desc& d, const void* x, int64_t ldx, cudaStream_t stream) {
  using namespace f4;
  Params p;
  memset(&p, 0, sizeof(p));
  p.o = output_of(d);
  p.a_scales = static_cast<const uint8_t*>(d.a_scales);
  p.w_scales = static_cast<const uint8_t*>(d.w_scales);
  p.k = (int)d.k;
  p.k_tiles = (int)scale_k_tiles(d.k, d.format);
  p.early = launch_overlap_enabled() ? 1 : 0;
  p.nb = (int)((d.m + 15) / 16 * 16);
  const int cols = (p.nb + 31) / 32 * 32 + 4 * stage_tiles(d.format) * 2;
  p.tmem_cols = cols <= 64 ? 64 : 128;
  CUtensorMap tw, ta;
  if (make_tensor_map_2d(&tw, d.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)d.k / 2, (unsigned long long)d.n,
                         (unsigned long long)d.k / 2, 128, kTileN, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) != 0 ||
      (!x &&
       make_tensor_map_2d(&ta, d.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)d.k / 2, (unsigned long long)d.m,
                          (unsigned long long)d.k / 2, 128, (unsigned)p.nb, CU_TENSOR_MAP_SWIZZLE_128B) != 0))
    return -1;
  if (x) {
    ta = tw;
    p.x = x;
    p.ldx = ldx;
    return d.format == kMx ? launch_fmt<kMx, true>(p, d.out_dtype, tw, ta, stream) : launch_fmt<kNv, true>(p, d.out_dtype, tw, ta, stream);
  }
  return d.format == kMx ? launch_fmt<kMx, false>(p, d.out_dtype, tw, ta, stream) : launch_fmt<kNv, false>(p, d.out_dtype, tw, ta, stream);
}

// Up to 64 rows here, more by pairs of CTAs (us out of memory, this kernel / pairs; it can be built for 128 rows): 64 rows
// k 4096 x n 11008 12.2 / 11.5, k = n = 4096 10.8 / 10.6, k 28672 x n 8192 27.9 / 30.6, k 14336 x n 4096 13.8 / 16.2, k 4096 x
// n 22016 16.3 / 18.3, x n 1024 8.0 / 10.3; 96 rows 13.4 / 12.4, 11.8 / 10.6, 29.0 / 30.5, 14.9 / 16.5, 18.3 / 19.8, 8.2 / 10.3; 128 rows
// 14.9 / 12.7, 13.1 / 10.7, 30.4 / 31.3, 16.2 / 16.6, 20.0 / 20.0, 9.1 / 10.4.  A limit by shape would save up to a fifth between.
int fp4_gemm_launch(const rb200_gemm_fp4_desc& d, const void* x, int64_t ldx, cudaStream_t stream) {
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < f4::kMaxDevices) f4::g_launched[dev].store(true, std::memory_order_relaxed);
  return d.m > 64 ? fp4_pair_launch(d, stream) : fp4_few_launch(d, x, ldx, stream);
}

}  // namespace rb200

using namespace rb200;

namespace {
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// what rb200_gemm_fp4 and rb200_linear_fp4 check alike
int check_gemm(const rb200_gemm_fp4_desc* d) {
  RB200_CHECK(d != nullptr && d->struct_size == sizeof(rb200_gemm_fp4_desc), "rb200_gemm_fp4_desc has a wrong struct_size");
  RB200_FP4_CHECK_SHAPE(d->format, d->m, d->k);
  RB200_CHECK(d->n > 0 && d->n < (1ll << 30), "n=%lld out of range", (long long)d->n);
  RB200_CHECK(d->out_dtype >= f4::kF16 && d->out_dtype <= f4::kF32, "unknown element type %d", d->out_dtype);
  RB200_CHECK(d->activation >= RB200_ACT_IDENTITY && d->activation <= RB200_ACT_GELU, "unknown activation %d", d->activation);
  RB200_CHECK(d->binary_op >= RB200_BIN_NONE && d->binary_op <= RB200_BIN_MULTIPLY, "unknown binary op %d", d->binary_op);
  RB200_CHECK(d->unary_op >= RB200_UN_IDENTITY && d->unary_op <= RB200_UN_RELU, "unknown unary op %d", d->unary_op);
  RB200_CHECK(d->ldo >= d->n, "ldo=%lld is less than n", (long long)d->ldo);
  RB200_CHECK(d->format == f4::kNv || (!d->a_tensor_scale && !d->w_tensor_scale), "the mx format has no tensor scale");
  if (d->m == 0) return 0;  // (an empty residual has no address)
  RB200_CHECK((d->binary_op != RB200_BIN_NONE) == (d->residual != nullptr), "a residual needs a binary op, and the other way round");
  RB200_CHECK(d->w && d->w_scales && d->out, "w, w_scales and out must be non-NULL");
  RB200_CHECK(aligned16(d->w) && aligned16(d->w_scales), "codes and scales must be 16-byte aligned");
  const uintptr_t width = d->out_dtype == f4::kF32 ? 4 : 2;
  RB200_CHECK(reinterpret_cast<uintptr_t>(d->out) % width == 0 && reinterpret_cast<uintptr_t>(d->bias) % width == 0 &&
                  reinterpret_cast<uintptr_t>(d->residual) % width == 0,
              "out, bias and residual must be aligned to their elements");
  return 0;
}
}  // namespace

extern "C" {

int rb200_gemm_fp4(const rb200_gemm_fp4_desc* d, void* stream) {
  if (check_gemm(d) != 0) return -1;
  if (d->m == 0) return 0;
  RB200_CHECK(d->a && d->a_scales && aligned16(d->a) && aligned16(d->a_scales), "a and a_scales must be non-NULL and 16-byte aligned");
  return fp4_gemm_launch(*d, nullptr, 0, static_cast<cudaStream_t>(stream));
}

size_t rb200_linear_fp4_workspace_bytes(int64_t m, int64_t k, int format) {
  if ((format != f4::kMx && format != f4::kNv) || m <= 0 || k <= 0) return 0;
  return (size_t)((m * (k / 2) + 255) / 256 * 256 + f4::scale_bytes(m, k, format));
}

int rb200_linear_fp4(const void* x, int x_dtype, int64_t ldx, const rb200_gemm_fp4_desc* desc, void* workspace,
                     size_t workspace_bytes, void* stream) {
  if (check_gemm(desc) != 0) return -1;
  RB200_CHECK(x_dtype >= f4::kF16 && x_dtype <= f4::kF32, "unknown element type %d", x_dtype);
  if (desc->m == 0) return 0;
  rb200_gemm_fp4_desc d = *desc;
  const int64_t width = x_dtype == f4::kF32 ? 4 : 2;
  RB200_CHECK(x && ldx >= d.k && ldx * width % 16 == 0 && aligned16(x), "x must be non-NULL, its rows 16-byte aligned (ldx=%lld)",
              (long long)ldx);
  RB200_CHECK(workspace && (reinterpret_cast<uintptr_t>(workspace) & 255u) == 0 &&
                  workspace_bytes >= rb200_linear_fp4_workspace_bytes(d.m, d.k, d.format),
              "the workspace must be 256-byte aligned and hold rb200_linear_fp4_workspace_bytes");
  // (a product that quantises x reads it in the CTAs of every tile, while others already store: not where out lies over x)
  const uintptr_t x0 = reinterpret_cast<uintptr_t>(x), out0 = reinterpret_cast<uintptr_t>(d.out);
  const uintptr_t x1 = x0 + ((d.m - 1) * ldx + d.k) * width, out1 = out0 + ((d.m - 1) * d.ldo + d.n) * (d.out_dtype == f4::kF32 ? 4 : 2);
  const bool apart = x1 <= out0 || out1 <= x0;
  if (apart && x_dtype == d.out_dtype && f4::quantises_itself(d.m, d.n, d.k)) return fp4_gemm_launch(d, x, ldx, static_cast<cudaStream_t>(stream));
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + (d.m * (d.k / 2) + 255) / 256 * 256;
  if (fp4_encode_launch(x, x_dtype, 1, d.m, d.k, ldx, 0, d.format, d.a_tensor_scale, codes, scales, true,
                        static_cast<cudaStream_t>(stream)) != 0)
    return -1;
  d.a = codes;
  d.a_scales = scales;
  return fp4_gemm_launch(d, nullptr, 0, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
