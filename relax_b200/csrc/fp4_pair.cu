// Large batches of the 4-bit float product: pairs of CTAs on one 256 x 256 tile.
//
// The tile is out^T again: 256 rows of w, 128 in each CTA of the pair, by up to 256 rows of a, of which each CTA holds half
// (tcgen05.mma, cta_group::2).  A stage is 256 k; everything it needs - codes, and scale tiles as rows of 128 words - comes
// by tensor-map loads that count on rank 0's barrier, and rank 0's MMA thread copies the scales of both CTAs into tensor
// memory.  What bounds a stage is the tensor cores (540 clocks at their nominal rate) and, close behind, what an SM takes
// from L2: 38 KB at 64 bytes a clock are 600 clocks; tiles of 128 x 256 per SM without pairing would need 54 KB.
// Accumulator and scales leave no room for a second accumulator, so the drain takes all 256 columns into registers (eight
// warps, up to 128 columns each) and hands the tensor memory back before it applies the epilogue and stores: the MMAs of the next
// tile wait for the reading only.  The drain itself is a loop over 16 columns: out of a cold instruction cache the same code for
// all 128 columns took 8 to 26 us in its first tile, the loop takes 3.5 (warm, it costs 3 % at 2048 rows, k 4096).
// The 128 sums and the loop want more than the 168 registers a thread that 384 threads share evenly: the form without shared k
// spills 120 to 128 bytes a thread (192 to 204 bytes of stores), written and read back once a tile.
//
// Measured: 4096 rows, k 8192 x n 28672 in the mx format 300 us, 6.4 PFLOP/s, 387 with the quantiser and at the power cap; 2048
// rows, k 4096 x n 22016 in the nv format 77 us (4.8), 108; 333 rows, k 4096 x n 11008 with bias and silu 19 us (1.6), 20.6.
#include <cstring>

#include "fp4_gemm.h"
#include "fp4_index.h"
#include "fp4_mma.cuh"
#include "fp4_out.cuh"
#include "tensormap.h"

namespace rb200 {
namespace f4 {
namespace {

using ug::elect_one;
using ug::make_b_desc;
using ug::tc_fence_after;
using ug::tc_fence_before;

constexpr int kThreads = 384;
constexpr int kDrainWarps = 8;
constexpr int kTileN = 128;  // rows of w in a CTA
constexpr int kNb = 256;     // rows of a
constexpr int kMaxStages = 6;
constexpr int kRows = 16;    // of a, that a drain warp finishes and stores at once, by 32 columns
constexpr int kBuffers = 4;  // for that many of them, each warp

__device__ int g_status;

struct Params {
  Output o;
  int n_tiles, m_tiles, n_first, stages, early, tma_store, staged, k;
};

template <int FMT>
__host__ __device__ constexpr int stage_bytes() {
  return kTileN * 128 + kNb / 2 * 128 + stage_tiles(FMT) * 512 * 3;
}

__device__ __forceinline__ void tmem_alloc2(uint32_t* holder, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(holder)), "r"(cols) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc2(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
// loads of either CTA, counted on rank 0's barrier
__device__ __forceinline__ void tma_load2(void* dst, const CUtensorMap* map, int c0, int c1, uint32_t bar0) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(bar0)
      : "memory");
}
__device__ __forceinline__ void tma_load3(void* dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar0) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar0)
      : "memory");
}
__device__ __forceinline__ void tma_store(const CUtensorMap* map, int c0, int c1, const void* src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1),
               "r"(smem_u32(src))
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int LEFT>
__device__ __forceinline__ void stores_read() {  // all but the last LEFT stores have read shared memory
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void commit2(uint64_t* bar, int first) {  // arrives at both CTAs' barrier
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)(3 << first))
      : "memory");
}
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void copy_scales2(uint32_t taddr, uint64_t desc) {  // in both CTAs, each from its own shared memory
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int FMT>
__device__ __forceinline__ void mma_scaled2(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales,
                                            uint32_t b_scales, uint32_t accumulate) {
  if (FMT == kMx)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {  // 32 columns of this warp's lanes; tcgen05.wait::ld follows
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
      "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// SPLIT: the k of a tile is cut over the two pairs of a cluster.
template <int FMT, class T, bool SPLIT>
__global__ void __launch_bounds__(kThreads, 1)
    fp4_pair_kernel(const Params p, const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                    const __grid_constant__ CUtensorMap tmap_ws, const __grid_constant__ CUtensorMap tmap_as,
                    const __grid_constant__ CUtensorMap tmap_out) {
  constexpr int NT = stage_tiles(FMT), kA = kTileN * 128, kWs = kA + kNb / 2 * 128, kAs = kWs + NT * 512;
  constexpr int kWCol = kNb, kACol = kNb + 4 * NT;  // tensor memory columns of the scales
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  const int stages = p.stages;
  T* store = reinterpret_cast<T*>(smem + (size_t)stages * stage_bytes<FMT>());  // [drain warp][kBuffers][kRows][32]
  uint64_t* full = reinterpret_cast<uint64_t*>(store + kDrainWarps * kBuffers * kRows * 32);  // the first CTA's are used
  uint64_t* empty = full + kMaxStages;
  uint64_t* d_full = empty + kMaxStages;
  uint64_t* d_empty = d_full + 1;  // the first CTA's is used
  uint32_t* holder = reinterpret_cast<uint32_t*>(d_empty + 1);  // [0] tensor memory, [1] a CTA of the cluster failed

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int split = SPLIT ? 2 : 1;
  // rank in the pair, the pair's place in the cluster, its first CTA
  const int rank = (int)cluster_rank() & 1, part = (int)cluster_rank() >> 1, first = part * 2;
  const int pair = (int)blockIdx.x / (2 * split), pairs = (int)gridDim.x / (2 * split);
  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(d_full, 1);
    mbar_init(d_empty, 2 * kDrainWarps);
    holder[1] = 0u;
    mbar_fence_init();
  }
  if (warp == 1) tmem_alloc2(holder, 512u);
  fence_proxy_async();
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // every CTA's barriers exist before any remote arrival
  tc_fence_after();
  griddep_launch_dependents();
  const uint32_t tmem = holder[0];
  const int chunks = (p.k + kStageK - 1) / kStageK, items = p.n_tiles * p.m_tiles;
  const int c0 = chunks * part / split, c1 = chunks * (part + 1) / split;
  // The rounds of items go forth and back over the pairs: with two rounds the last ones, the smaller, follow the smallest of the
  // first (333 rows, k 4096 x n 11008: 24.2 -> 20.4 us).
  auto index_at = [&](int round) { return round * pairs + (round % 2 ? pairs - 1 - pair : pair); };
  struct Item {
    int n0, m0, width;  // this CTA's first row of w, the tile's first row of a, columns of the MMA
    int share;          // of them, for the drain warps' first half (100 rows, k 4096 x n 11008, silu: 18.3 -> 16.1 us by halves)
  };
  auto item_at = [&](int i) {
    const int nt = p.n_first ? i % p.n_tiles : i / p.m_tiles, mt = p.n_first ? i / p.n_tiles : i % p.m_tiles;
    Item it;
    it.n0 = (2 * nt + rank) * kTileN;
    it.m0 = mt * kNb;
    it.width = tile_width(p.o.m, it.m0, kNb);
    it.share = (it.width + 63) / 64 * 32;
    return it;
  };

  bool ok = true;
  if (warp == 0) {
    // ============================================================ loads
    const bool leader = elect_one();
    int s = 0;
    uint32_t ph = 1;
    bool waited = false;
    auto load_w = [&](const Item& it, int c, int s) {
      uint8_t* at = smem + (size_t)s * stage_bytes<FMT>();
      const uint32_t bar0 = at_rank(smem_u32(&full[s]), first);
      if (rank == 0) mbar_arrive_expect_tx(&full[s], 2u * (uint32_t)stage_bytes<FMT>());
      tma_load2(at, &tmap_w, c * 128, it.n0, bar0);
      tma_load3(at + kWs, &tmap_ws, 0, c * NT, it.n0 >> 7, bar0);
    };
    auto load_a = [&](const Item& it, int c, int s) {
      uint8_t* at = smem + (size_t)s * stage_bytes<FMT>();
      const uint32_t bar0 = at_rank(smem_u32(&full[s]), first);
      tma_load2(at + kA, &tmap_a, c * 128, it.m0 + rank * (it.width / 2), bar0);
      tma_load3(at + kAs, &tmap_as, 0, c * NT, it.m0 >> 7, bar0);
    };
    if (!p.early) {
      if (leader && pair < items) {
        const Item it = item_at(pair);
        for (int c = c0; c < min(c0 + stages, c1); ++c) tma_prefetch(&tmap_w, c * 128, it.n0);
      }
      griddep_wait();
      waited = true;
    }
    // before the wait only weights are read: as many stages as there are, in the first tile
    int ahead = 0;
    if (!waited) {
      ahead = pair < items ? min(stages, c1 - c0) : 0;
      if (leader) {
        const Item it = item_at(pair);
        for (int c = 0; c < ahead; ++c) load_w(it, c0 + c, c);
      }
      __syncwarp();
      griddep_wait();
    }
    for (int round = 0, i; ok && (i = index_at(round)) < items; ++round) {
      const Item it = item_at(i);
      for (int c = c0; c < c1; ++c) {
        ok = mbar_wait_parked(&empty[s], ph, &g_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (leader) {
          if (ahead == 0) load_w(it, c, s);
          load_a(it, c, s);
        }
        __syncwarp();
        if (ahead > 0) --ahead;
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
    }
    // every commit to this CTA's barriers has arrived, so every load has landed, before it may leave
    for (int j = 0; ok && j < stages; ++j) {
      ok = mbar_wait_parked(&empty[s], ph, &g_status);
      if (++s == stages) {
        s = 0;
        ph ^= 1u;
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ============================================================ scales into tensor memory, MMAs
    const bool leader = elect_one();
    const uint64_t w_desc0 = make_b_desc(smem_u32(smem)), ws_desc0 = scale_desc(smem_u32(smem + kWs));
    int s = 0;
    uint32_t ph = 0, dph = 1;
    for (int round = 0, i; ok && (i = index_at(round)) < items; ++round, dph ^= 1u) {
      const uint32_t idesc = mma_desc<FMT>(256, item_at(i).width);
      const int a_tiles = item_at(i).width > 128 ? 2 : 1;
      ok = mbar_wait_parked(d_empty, dph, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      for (int c = c0; c < c1; ++c) {
        ok = mbar_wait_parked(&full[s], ph, &g_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tc_fence_after();
        if (leader) {
          const uint64_t off = (uint64_t)(s * (stage_bytes<FMT>() >> 4));
          const uint64_t w_desc = w_desc0 + off, a_desc = w_desc + (uint64_t)(kA >> 4), sc = ws_desc0 + off;
          const int mmas = min(kStageK, p.k - c * kStageK + kMmaK - 1) / kMmaK;
#pragma unroll
          for (int t = 0; t < NT; ++t) copy_scales2(tmem + kWCol + 4 * t, sc + (uint64_t)(t * 32));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            copy_scales2(tmem + kACol + 8 * t, sc + (uint64_t)((NT + t) * 32));
            if (a_tiles == 2) copy_scales2(tmem + kACol + 8 * t + 4, sc + (uint64_t)((2 * NT + t) * 32));
          }
#pragma unroll
          for (int j = 0; j < kStageK / kMmaK; ++j) {
            const int t = FMT == kMx ? j >> 1 : j;
            if (j < mmas)
              mma_scaled2<FMT>(tmem, w_desc + j * 2, a_desc + j * 2, FMT == kMx && (j & 1) ? upper_half(idesc) : idesc,
                               tmem + kWCol + 4 * t, tmem + kACol + 8 * t, (c > c0 || j > 0) ? 1u : 0u);
          }
          commit2(&empty[s], first);
        }
        __syncwarp();
        if (++s == stages) {
          s = 0;
          ph ^= 1u;
        }
      }
      if (ok && leader) commit2(d_full, first);
      __syncwarp();
    }
  }

  // ============================================================ drain
  const int dw = warp - 4, quad = warp & 3, half = dw >> 2;
  T* mine = store + dw * kBuffers * kRows * 32;
  const uint32_t taddr = tmem + ((uint32_t)(32 * quad) << 16);
  // A warp's columns of the accumulator (rows of a) by kRows of them.  SPLIT: of its four groups of 32 columns the first pair
  // has the even ones, the second the odd ones.
  constexpr int kTurns = SPLIT ? 4 : 8;
  auto column = [&](int turn) { return SPLIT ? (turn >> 1) * 64 + part * 32 + (turn & 1) * kRows : turn * kRows; };
  auto first_of = [&](const Item& it) { return half * it.share; };  // this warp's first column, and how many rows of a it has
  auto rows_of = [&](const Item& it) { return min(it.share, p.o.m - it.m0 - first_of(it)); };
  // the residual goes to where the result of that turn will be stored from, two turns ahead
  auto fetch = [&](const Item& it, int turn) {
    constexpr int kPer = 16 / (int)sizeof(T), kPieces = 32 / kPer;
    const int n = it.n0 + quad * 32, m = it.m0 + first_of(it) + column(turn), rows = min(kRows, rows_of(it) - column(turn));
    if (turn < kTurns)
      for (int i = lane; i < rows * kPieces; i += 32) {
        const int r = i / kPieces, c = i % kPieces * kPer;
        if (n + c < p.o.n)
          copy16(mine + ((turn % kBuffers) * kRows + r) * 32 + c, static_cast<const T*>(p.o.residual) + (m + r) * p.o.ld_res + n + c);
      }
    copies_commit();
  };
  // before an item's sums are there; returns what a lane adds to its column of the result
  auto prepare = [&](const Item& it) {
    stores_read<0>();
    __syncwarp();
    if (p.staged) {
      fetch(it, 0);
      fetch(it, 1);
    }
    return bias_at<T>(p.o, it.n0 + quad * 32 + lane);
  };
  auto put = [&](const Item& it, int turn, float (&v)[kRows], float alpha, float bias) {
    const int n = it.n0 + quad * 32, m = it.m0 + first_of(it) + column(turn);
    T* st = mine + (turn % kBuffers) * kRows * 32 + lane;
    float x[kRows];
    if (p.staged) {
      stores_read<1>();
      __syncwarp();
      fetch(it, turn + 2);
      copies_wait<2>();
      __syncwarp();
#pragma unroll
      for (int r = 0; r < kRows; ++r) x[r] = widen(st[r * 32]);
    } else {
      stores_read<kBuffers - 1>();
      __syncwarp();
      if (p.o.residual) load_residual<T, true>(p.o, x, m, n + lane);
    }
    finish<true>(p.o, v, alpha, &bias, x);
    if (p.tma_store) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) st[r * 32] = narrow<T>(v[r]);
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) tma_store(&tmap_out, n, m, st);
    } else if (n + lane < p.o.n) {
      T* dst = static_cast<T*>(p.o.out) + (int64_t)m * p.o.ldo + n + lane;
#pragma unroll
      for (int r = 0; r < kRows; ++r)
        if (m + r < p.o.m) dst[r * p.o.ldo] = narrow<T>(v[r]);
    }
  };
  if (!SPLIT && warp >= 4) {
    griddep_wait();
    const float alpha = out_scale(p.o);
    uint32_t ph = 0;
    for (int round = 0, i; (i = index_at(round)) < items; ++round, ph ^= 1u) {
      const Item it = item_at(i);
      const float bias = prepare(it);
      ok = mbar_wait_parked(d_full, ph, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int rows = rows_of(it);
      float v[128];
      if (rows > 0) {
#pragma unroll
        for (int c = 0; c < 128; c += 32) tmem_ld32(taddr + first_of(it) + c, v + c);
        ug::tc_wait_ld();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) arrive_cluster(at_rank(smem_u32(d_empty), first));
      if (it.n0 + quad * 32 >= p.o.n) continue;
#pragma unroll 1
      for (int turn = 0; column(turn) < rows; ++turn) {
        float t[kRows];
        switch (turn) {
#define RB200_TAKE(j)                                              \
  case j:                                                          \
    _Pragma("unroll") for (int r = 0; r < kRows; ++r) t[r] = v[j * kRows + r]; \
    break;
          RB200_TAKE(0)
          RB200_TAKE(1)
          RB200_TAKE(2)
          RB200_TAKE(3)
          RB200_TAKE(4)
          RB200_TAKE(5)
          RB200_TAKE(6)
          default:
            RB200_TAKE(7)
#undef RB200_TAKE
        }
        put(it, turn, t, alpha, bias);
      }
    }
    copies_wait<0>();
    stores_read<0>();
  }
  if (SPLIT) {
    // each pair sends the other what it does not keep, by columns of 128 rows of w, into the memory of its stages
    griddep_wait();
    const Item it = item_at(pair);
    const float alpha = out_scale(p.o), bias = warp >= 4 ? prepare(it) : 0.0f;
    ok = mbar_wait_parked(d_full, 0, &g_status) && ok;
    ok = __all_sync(0xffffffffu, ok);
    if (!ok)
      for (int r = 0; r < 4; ++r) st_cluster(at_rank(smem_u32(holder + 1), r), 1u);
    __syncthreads();
    cluster_sync();  // both pairs' stages have been read
    tc_fence_after();
    const int rows = rows_of(it);
    const bool work = warp >= 4 && holder[1] == 0u;
    // [half][group / 2][32][128] fp32
    float* slots = reinterpret_cast<float*>(smem) + half * 2 * 32 * 128 + quad * 32 + lane;
    if (work) {
#pragma unroll 1
      for (int c = 32 * (1 - part); c < rows; c += 64) {
        float v[32];
        tmem_ld32(taddr + first_of(it) + c, v);
        ug::tc_wait_ld();
        const uint32_t at = at_rank(smem_u32(slots + (c >> 6) * 32 * 128), (1 - part) * 2 + rank);
#pragma unroll
        for (int i = 0; i < 32; ++i) st_cluster_f32(at + i * 512, v[i]);
      }
    }
    __syncwarp();
    cluster_sync();
    if (work && it.n0 + quad * 32 < p.o.n) {
#pragma unroll 1
      for (int turn = 0; turn < kTurns && column(turn) < rows; ++turn) {
        const int c = column(turn);
        float v[kRows];
        ug::tc_ld16(taddr + first_of(it) + c, v);
        const float* from = slots + ((c >> 6) * 32 + (c & 31)) * 128;
#pragma unroll
        for (int i = 0; i < kRows; ++i) v[i] += from[i * 128];
        put(it, turn, v, alpha, bias);
      }
    }
    copies_wait<0>();
    stores_read<0>();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // the other CTA may still have been reading this one's tiles, or arriving here
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc2(tmem, 512u);
  }
}

// Two pairs share a tile's k where that fills empty SMs and leaves each pair eight stages: handing over half of the sums and
// meeting twice costs about 3 us, a stage 0.27 (256 rows, k 4096 x n 4096: 18.5 -> 17.3 us, k 28672 x n 8192: 50 -> 36; at k 3328
// it is even).  A tenth of the SMs is left out, since clusters of four do not find room everywhere: with 34 tiles one waits for
// another to end (128 rows, k 8192: n 8448 20.4 us, n 8704 30.9, without sharing 24).
bool splits(int tiles, int64_t k) { return tiles * 40 <= 9 * sm_count_current() && k >= 16 * kStageK; }

template <int FMT, class T, bool SPLIT>
int launch_split(Params& p, const CUtensorMap (&maps)[5], cudaStream_t stream) {
  auto kern = fp4_pair_kernel<FMT, T, SPLIT>;
  const size_t tail = (size_t)kDrainWarps * kBuffers * kRows * 32 * sizeof(T) + (2 * kMaxStages + 2) * 8 + 16 + 1024;
  p.stages = kMaxStages;
  while (p.stages > 2 && p.stages * (size_t)stage_bytes<FMT>() + tail > 227 * 1024) --p.stages;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = p.stages * (size_t)stage_bytes<FMT>() + tail;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = SPLIT ? 4 : 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  static thread_local int configured_device = -1;
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (configured_device != dev) {
    RB200_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_device = dev;
  }
  const int items = p.n_tiles * p.m_tiles, pairs = sm_count_current() / 2;
  cfg.gridDim = dim3((unsigned)(SPLIT ? 4 * items : 2 * (items < pairs ? items : pairs)), 1, 1);
  RB200_CUDA(cudaLaunchKernelEx(&cfg, kern, p, maps[0], maps[1], maps[2], maps[3], maps[4]));
  return 0;
}
template <int FMT, class T>
int launch_typed(Params& p, const CUtensorMap (&maps)[5], cudaStream_t stream) {
  return splits(p.n_tiles * p.m_tiles, p.k) ? launch_split<FMT, T, true>(p, maps, stream) : launch_split<FMT, T, false>(p, maps, stream);
}
template <int FMT>
int launch_fmt(Params& p, int dtype, const CUtensorMap (&maps)[5], cudaStream_t stream) {
  switch (dtype) {
    case kF16: return launch_typed<FMT, __half>(p, maps, stream);
    case kBf16: return launch_typed<FMT, __nv_bfloat16>(p, maps, stream);
    default: return launch_typed<FMT, float>(p, maps, stream);
  }
}

// scales as rows of 128 words: [row tiles][k tiles][128], a stage's tiles of `row_tiles` x 128 rows a load
int scale_map(CUtensorMap* map, const void* scales, int64_t rows, int64_t k, int fmt, unsigned row_tiles) {
  const unsigned long long dims[3] = {128, (unsigned long long)scale_k_tiles(k, fmt), (unsigned long long)scale_row_tiles(rows)};
  const unsigned long long strides[2] = {512, 512 * dims[1]};
  const unsigned box[3] = {128, (unsigned)stage_tiles(fmt), row_tiles};
  return make_tensor_map(map, scales, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}

}  // namespace
}  // namespace f4

int fp4_pair_launch(const rb200_gemm_fp4_desc& d, cudaStream_t stream) {
  using namespace f4;
  Params p;
  memset(&p, 0, sizeof(p));
  p.o = output_of(d);
  p.k = (int)d.k;
  p.early = launch_overlap_enabled() ? 1 : 0;
  RB200_CHECK((d.n + 2 * kTileN - 1) / (2 * kTileN) * ((d.m + kNb - 1) / kNb) < (1ll << 30), "the product is too large (m=%lld, n=%lld)", (long long)d.m,
              (long long)d.n);
  p.n_tiles = (int)((d.n + 2 * kTileN - 1) / (2 * kTileN));
  p.m_tiles = (int)((d.m + kNb - 1) / kNb);
  // Two tiles of a, the second one usually smaller: all the large ones first.  More: neighbours share a tile of w.
  p.n_first = p.m_tiles <= 2;
  const int width = d.out_dtype == kF32 ? 4 : 2;
  p.tma_store = reinterpret_cast<uintptr_t>(d.out) % 16 == 0 && d.ldo * width % 16 == 0;
  p.staged = p.tma_store && d.residual && reinterpret_cast<uintptr_t>(d.residual) % 16 == 0 && p.o.ld_res * width % 16 == 0;
  CUtensorMap maps[5];
  if (make_tensor_map_2d(&maps[0], d.w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)d.k / 2, (unsigned long long)d.n,
                         (unsigned long long)d.k / 2, 128, kTileN, CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
      make_tensor_map_2d(&maps[1], d.a, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)d.k / 2, (unsigned long long)d.m,
                         (unsigned long long)d.k / 2, 128, kNb / 2, CU_TENSOR_MAP_SWIZZLE_128B) != 0 ||
      scale_map(&maps[2], d.w_scales, d.n, d.k, d.format, 1) != 0 || scale_map(&maps[3], d.a_scales, d.m, d.k, d.format, 2) != 0)
    return -1;
  maps[4] = maps[0];
  if (p.tma_store &&
      make_tensor_map_2d(&maps[4], d.out,
                         d.out_dtype == kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                         : d.out_dtype == kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                         (unsigned long long)d.n, (unsigned long long)d.m, (unsigned long long)d.ldo * width, 32,
                         (unsigned)kRows, CU_TENSOR_MAP_SWIZZLE_NONE) != 0)
    return -1;
  return d.format == kMx ? launch_fmt<kMx>(p, d.out_dtype, maps, stream) : launch_fmt<kNv>(p, d.out_dtype, maps, stream);
}

int fp4_pair_read_status(int* v) {
  RB200_CUDA(cudaMemcpyFromSymbol(v, f4::g_status, sizeof(int)));
  if (*v != 0) {
    const int zero = 0;
    RB200_CUDA(cudaMemcpyToSymbol(f4::g_status, &zero, sizeof(int)));
  }
  return 0;
}

}  // namespace rb200
