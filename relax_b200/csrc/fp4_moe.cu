// A whole expert layer for a few tokens over weights in microscaled 4-bit floats, in two kernels:
//   up    routing; h[r] = silu(x Wg^T) * (x Wu^T) for the (token, expert) pairs r, ordered by expert
//   down  out[t] = sum over the token's experts of gate * (h[r] Wd^T)
//
// What bounds it is reading the weights of the chosen experts once, so activations keep their 16 bits: codes become fp16
// pairs in registers (one conversion per pair, exact) and go through mma.sync with up to eight rows as its columns, which
// at these batch sizes costs less than the reading.  kMx scales multiply the fp32 sums of a block; kNv scales have too few
// k for that and multiply the fp16 pairs, exactly (two and four significant bits, at least 2^-10, at most 2688).
//
// Routing is a few hundred clocks for a few tokens, so every CTA does it for itself from the logits: no kernel before these
// two, no hand-over through memory.  `down` does it, and asks for its first weights, while `up` still runs.
//
// Weights come by tensor-map loads in 128-byte rows, swizzled; a lane's code words are then free of bank conflicts.  A
// warp's lane (g, t) holds, of the 32 k of a chunk, k 8t .. 8t + 7 of rows g and g + 8: the MMAs' k slots are a permutation
// of k, the same one for x, whose eight values are one 16-byte word.
// `down` cuts the (expert, k) sequence of 64 output columns over the CTAs of a cluster; each adds gate times its sums in
// shared memory, every word by one thread in the order of the sequence, and the cluster's parts are added in rank order:
// nothing depends on timing.
#include <atomic>
#include <cstring>

#include "../../include/relax_b200.h"
#include "fp4_mma.cuh"
#include "tensormap.h"

namespace rb200 {
namespace f4 {
namespace {

using ug::elect_one;

constexpr int kMaxTokens = 32, kMaxExperts = 256, kMaxTopK = 8;
constexpr int kConsumers = 8;  // warps: four blocks of 16 rows, gate and up or two halves of k
constexpr int kThreads = (kConsumers + 2) * 32;  // and a warp for the weights' loads, one for x's
constexpr int kTile = 64;      // rows of a weight box
constexpr int kBox = kTile * 128;
constexpr int kMaxStages = 6;

__device__ int g_status;

// Rows are the (token, expert) pairs by expert; an entry is at most 8 NT rows of one expert.  NT = 1 has at most eight tokens.
template <int NT>
struct alignas(16) Routing {
  static constexpr int kRows = (NT == 1 ? 8 : kMaxTokens) * kMaxTopK;
  uint32_t mask[kMaxExperts];  // tokens of an expert
  float gate_of_row[kRows];
  float gate_of[kRows];        // by token and choice
  int warp_sum[kConsumers];
  int entries;
  int failed;
  uint16_t entry_row[kRows + 2];
  uint8_t entry_expert[kRows];
  uint8_t token_of_row[kRows];
  uint8_t expert_of[kRows];
};

struct Params {
  const __half* x;
  const float* logits;
  const uint8_t* s1;
  const uint8_t* s2;
  const float* ts1;
  const float* ts2;
  __half* h;
  __half* out;
  int64_t s1_expert, s2_expert;  // bytes of an expert's scales
  int tokens, experts, top_k, renormalize;
  int hidden, ffn, k_tiles1, k_tiles2;
  int stages, cluster;
};

// order of floats as unsigned numbers, NaN lowest
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return v == v ? ((b & 0x80000000u) ? ~b : b | 0x80000000u) : 0u;
}

// U tokens (t, t + 8, ..) by a warp, side by side: what takes the time is the latency of each step.  PER experts a lane.
template <int U, int PER, int NT>
__device__ __forceinline__ void choose(const Params& p, Routing<NT>& r, int t) {
  const int lane = threadIdx.x & 31;
  float v[U][PER], top[U], sum[U], chosen[U], mine[U];
  uint32_t key[U][PER];
  int my_expert[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool token = t + u * kConsumers < p.tokens;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = i * 32 + lane;
      v[u][i] = token && e < p.experts ? __ldcg(p.logits + (t + u * kConsumers) * p.experts + e) : -INFINITY;
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    top[u] = v[u][0];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      top[u] = fmaxf(top[u], v[u][i]);
      key[u][i] = i * 32 + lane < p.experts ? max(order_key(v[u][i]), 1u) : 0u;  // 0: not there, or taken
    }
    chosen[u] = mine[u] = 0.0f;
    my_expert[u] = 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], o));
#pragma unroll
  for (int u = 0; u < U; ++u) {
    sum[u] = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 32 + lane < p.experts) sum[u] += expf(v[u][i] - top[u]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] += __shfl_xor_sync(0xffffffffu, sum[u], o);
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best[U], all[U];
    int at[U], e[U];
    float val[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      best[u] = key[u][0];
      at[u] = lane;
      val[u] = v[u][0];
#pragma unroll
      for (int i = 1; i < PER; ++i)
        if (key[u][i] > best[u]) {
          best[u] = key[u][i];
          at[u] = i * 32 + lane;
          val[u] = v[u][i];
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) all[u] = __reduce_max_sync(0xffffffffu, best[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) e[u] = (int)__reduce_min_sync(0xffffffffu, best[u] == all[u] ? (uint32_t)at[u] : 0xffffu);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float w = expf(__shfl_sync(0xffffffffu, val[u], e[u] & 31) - top[u]);
      chosen[u] += w;
      if (lane == j) {
        mine[u] = w;
        my_expert[u] = e[u];
      }
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (i * 32 + lane == e[u]) key[u][i] = 0u;
    }
  }
  // (a NaN among the logits, or nothing but -inf: sum is NaN, and so is every gate)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int token = t + u * kConsumers;
    if (token < p.tokens && lane < p.top_k) {
      r.expert_of[token * p.top_k + lane] = (uint8_t)my_expert[u];
      r.gate_of[token * p.top_k + lane] = p.renormalize && sum[u] == sum[u] ? mine[u] / chosen[u] : mine[u] / sum[u];
      atomicOr(&r.mask[my_expert[u]], 1u << token);
    }
  }
}

// The routing, by every thread of the CTA: the top_k largest logits of a token (equal ones: lower expert first), gates
// softmax over all experts or over the chosen ones; rows and entries in expert order.
template <int NT>
__device__ void route(const Params& p, Routing<NT>& r) {
  constexpr int U = NT == 1 ? 1 : kMaxTokens / kConsumers, most = NT * 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < kMaxExperts) r.mask[tid] = 0u;
  __syncthreads();
  if (warp < kConsumers && warp < p.tokens) {
    if (p.experts <= 32) choose<U, 1>(p, r, warp);
    else if (p.experts <= 64) choose<U, 2>(p, r, warp);
    else choose<U, kMaxExperts / 32>(p, r, warp);
  }
  __syncthreads();
  const uint32_t m = tid < kMaxExperts ? r.mask[tid] : 0u;
  const int n = __popc(m), parts = (n + most - 1) / most;
  int upto = n | parts << 16;  // rows and entries counted together
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (warp < kConsumers && lane == 31) r.warp_sum[warp] = upto;
  __syncthreads();
  if (warp < kConsumers) {
    int before = upto - (n | parts << 16);
    for (int w = 0; w < warp; ++w) before += r.warp_sum[w];
    const int row = before & 0xffff, a = before >> 16;
    for (int i = 0; i < parts; ++i) {
      r.entry_expert[a + i] = (uint8_t)tid;
      r.entry_row[a + i] = (uint16_t)(row + i * most);
    }
    uint32_t left = m;
    for (int i = 0; i < n; ++i, left &= left - 1u) {
      const int t = __ffs((int)left) - 1;
      float gate = 0.0f;
      for (int j = 0; j < p.top_k; ++j)
        if (r.expert_of[t * p.top_k + j] == tid) gate = r.gate_of[t * p.top_k + j];
      r.token_of_row[row + i] = (uint8_t)t;
      r.gate_of_row[row + i] = gate;
    }
    if (tid == kMaxExperts - 1) {
      r.entries = a + parts;
      r.entry_row[a + parts] = (uint16_t)(row + n);
    }
  }
  __syncthreads();
}

// 16 bytes of global memory, or zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// arrives at the barrier when this thread's copies so far have landed (the barrier counts these arrivals)
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory"); }

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The scales of rows g and g + 8 over 128 k, as the products take them.
template <int FMT>
struct Scales {
  // kMx: fp32 scales of the four blocks of either row.  kNv: f16x2, this lane's scale of row g and of row g + 8, by chunk
  float f0[4], f8[4];
  uint32_t both[4];
  __device__ __forceinline__ void take(const uint8_t* at, int t) {  // `at`: row g's word in the (first) tile
    if (FMT == kMx) {
      expand(*reinterpret_cast<const uint32_t*>(at), f0);
      expand(*reinterpret_cast<const uint32_t*>(at + 8 * 16), f8);
    } else {
      // blocks 2i and 2i + 1 of chunk i; lanes t < 2 hold k of the first, the others of the second
      const uint32_t sel = t < 2 ? 0x40u : 0x51u;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t a = *reinterpret_cast<const uint32_t*>(at + q * 512) & 0x7f7f7f7fu;
        const uint32_t b = *reinterpret_cast<const uint32_t*>(at + q * 512 + 8 * 16) & 0x7f7f7f7fu;
        both[2 * q] = from_e4m3x2(__byte_perm(a, b, sel));
        both[2 * q + 1] = from_e4m3x2(__byte_perm(a, b, sel + 0x22u));
      }
    }
  }
  static __device__ __forceinline__ void expand(uint32_t w, float (&f)[4]) {
    uint32_t lo, hi;  // bf16 has the exponents of e8m0
    asm("{\n\t.reg .b16 a, b;\n\t"
        "mov.b32 {a, b}, %2;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %0, a;\n\t"
        "cvt.rn.bf16x2.ue8m0x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
    f[0] = __uint_as_float(lo << 16);
    f[1] = __uint_as_float(lo & 0xffff0000u);
    f[2] = __uint_as_float(hi << 16);
    f[3] = __uint_as_float(hi & 0xffff0000u);
  }
};

// Rows g and g + 8 of a 16-row block over the 32 k of chunk i: sums of the products with the x words of the column tiles.
template <int FMT, int NT>
__device__ __forceinline__ void chunk(float (&acc)[NT][4], uint32_t w0, uint32_t w8, const Scales<FMT>& s, int i, const uint4 (&x)[NT],
                                      int tiles) {
  uint32_t a0[4], a8[4];
  from_codes8(w0, a0);
  from_codes8(w8, a8);
  if (FMT == kNv) {
    const uint32_t p0 = __byte_perm(s.both[i], 0u, 0x1010), p8 = __byte_perm(s.both[i], 0u, 0x3232);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      a0[q] = mul2(a0[q], p0);
      a8[q] = mul2(a8[q], p8);
    }
  }
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    if (j > 0 && j >= tiles) break;
    if (FMT == kNv) {
      mma(acc[j], a0[0], a8[0], a0[1], a8[1], x[j].x, x[j].y);
      mma(acc[j], a0[2], a8[2], a0[3], a8[3], x[j].z, x[j].w);
    } else {
      float part[4];
      mma_first(part, a0[0], a8[0], a0[1], a8[1], x[j].x, x[j].y);
      mma(part, a0[2], a8[2], a0[3], a8[3], x[j].z, x[j].w);
      acc[j][0] = fmaf(part[0], s.f0[i], acc[j][0]);
      acc[j][1] = fmaf(part[1], s.f0[i], acc[j][1]);
      acc[j][2] = fmaf(part[2], s.f8[i], acc[j][2]);
      acc[j][3] = fmaf(part[3], s.f8[i], acc[j][3]);
    }
  }
}

// A warp's share of a stage: 16 rows over 256 k, eight chunks of 32.  `w` row g of the block in a box of 128-byte rows, swizzled,
// at this lane's word; `x` row g of the stage's x at this lane's 16 bytes; `sc` row g's word in the first scale tile.
template <int FMT, int NT>
struct Walk {
  int off[8], xoff[2];
  __device__ __forceinline__ explicit Walk(int g) {
#pragma unroll
    for (int i = 0; i < 8; ++i) off[i] = (i ^ g) << 4;
#pragma unroll
    for (int i = 0; i < 2; ++i) xoff[i] = (i ^ (g & 1)) * 64;
  }
  __device__ __forceinline__ void stage(float (&acc)[NT][4], const uint8_t* w, const uint8_t* x0, const uint8_t* sc, int t, int tiles) const {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      Scales<FMT> s;
      s.take(sc + q * (stage_tiles(FMT) / 2) * 512, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4 x[NT];
#pragma unroll
        for (int j = 0; j < NT; ++j)
          x[j] = *reinterpret_cast<const uint4*>(x0 + xoff[i & 1] + q * 256 + (i >> 1) * 128 + j * 8 * (kStageK * 2));
        chunk<FMT, NT>(acc, *reinterpret_cast<const uint32_t*>(w + off[q * 4 + i]),
                       *reinterpret_cast<const uint32_t*>(w + off[q * 4 + i] + 8 * 128), s, i, x, tiles);
      }
    }
  }
};

// Shared memory: [codes of all stages][scales][x][barriers][routing][sums], offsets from the aligned base.
struct Layout {
  int code_bytes, scale_bytes, x_bytes;  // of a stage
};
template <int FMT, int NT>
__host__ __device__ constexpr Layout layout_up() {
  return {2 * kBox, 2 * stage_tiles(FMT) * 512, NT * 8 * kStageK * 2};
}
template <int FMT, int NT>
__host__ __device__ constexpr Layout layout_down() {
  return {2 * kBox, 2 * stage_tiles(FMT) * 512, NT * 8 * 2 * kStageK * 2};
}
__host__ __device__ constexpr int stage_total(const Layout& l) { return l.code_bytes + l.scale_bytes + l.x_bytes; }

// Position in the ring of stages.
struct Ring {
  int stages, s;
  uint32_t ph;
  __device__ __forceinline__ void next() {
    if (++s == stages) {
      s = 0;
      ph ^= 1u;
    }
  }
};
__device__ __forceinline__ void init_ring(uint64_t* full, uint64_t* empty, int stages) {
  for (int i = 0; i < stages; ++i) {
    mbar_init(&full[i], 1 + 32);       // the loads' bytes, a lane's copies of x each
    mbar_init(&empty[i], kConsumers);
  }
  mbar_fence_init();
}
// No load may be on its way when the CTA leaves: the last fill of every stage.
__device__ __forceinline__ void drain_ring(uint64_t* full, int stages, int issued) {
  for (int i = max(0, issued - stages); i < issued; ++i) mbar_wait_parked(&full[i % stages], (uint32_t)(i / stages) & 1u, &g_status);
}
// `tiles` consecutive scale tiles from `from` on, those past `last` replaced by the last one: it has the same rows' scales, and
// what is past k is zero codes and zeros of x.
__device__ __forceinline__ void load_scale_tiles(uint8_t* dst, const uint8_t* base, int from, int tiles, int last, uint64_t* bar) {
  const int there = min(tiles, last + 1 - from);
  bulk_g2s(dst, base + (int64_t)from * 512, (uint32_t)there * 512u, bar);
  for (int i = there; i < tiles; ++i) bulk_g2s(dst + i * 512, base + (int64_t)last * 512, 512u, bar);
}
// 16-byte column of x in its row's 512 bytes, so that a quarter-warp's reads (two rows, four columns) meet no bank twice
__device__ __forceinline__ int x_column(int row, int column) { return column ^ ((row & 1) << 2); }

constexpr int kRoutingOffset = 2 * kMaxStages * 8;
__host__ __device__ constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NT)) moe_fp4_up_kernel(const Params p, const __grid_constant__ CUtensorMap tmap_w) {
  constexpr Layout L = layout_up<FMT, NT>();
  constexpr int TILES = stage_tiles(FMT);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const scales = smem + p.stages * L.code_bytes;
  uint8_t* const xs = scales + p.stages * L.scale_bytes;
  uint64_t* const full = reinterpret_cast<uint64_t*>(xs + p.stages * L.x_bytes);
  uint64_t* const empty = full + kMaxStages;
  Routing<NT>& r = *reinterpret_cast<Routing<NT>*>(reinterpret_cast<uint8_t*>(full) + kRoutingOffset);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    init_ring(full, empty, p.stages);
    r.failed = 0;
  }
  fence_proxy_async();
  griddep_wait();
  griddep_launch_dependents();
  route<NT>(p, r);

  const int f_tiles = p.ffn / kTile, items = r.entries * f_tiles, chunks = (p.hidden + kStageK - 1) / kStageK;
  Ring ring = {p.stages, 0, 0u};
  if (warp == kConsumers) {
    // ============================================================ weights
    const bool leader = elect_one();
    int issued = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int a = item / f_tiles, f0 = (item - a * f_tiles) * kTile, e = r.entry_expert[a];
      const uint8_t* s_gate = p.s1 + e * p.s1_expert + (int64_t)(f0 >> 7) * p.k_tiles1 * 512;
      const uint8_t* s_up = p.s1 + e * p.s1_expert + (int64_t)((p.ffn + f0) >> 7) * p.k_tiles1 * 512;
      for (int c = 0; c < chunks; ++c) {
        ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (leader) {
          uint64_t* bar = &full[ring.s];
          uint8_t* w = smem + ring.s * L.code_bytes;
          uint8_t* sc = scales + ring.s * L.scale_bytes;
          mbar_arrive_expect_tx(bar, L.code_bytes + L.scale_bytes);
          tma_load(w, &tmap_w, c * 128, e * 2 * p.ffn + f0, bar);
          tma_load(w + kBox, &tmap_w, c * 128, e * 2 * p.ffn + p.ffn + f0, bar);
          load_scale_tiles(sc, s_gate, c * TILES, TILES, p.k_tiles1 - 1, bar);
          load_scale_tiles(sc + TILES * 512, s_up, c * TILES, TILES, p.k_tiles1 - 1, bar);
        }
        __syncwarp();
        ++issued;
        ring.next();
      }
    }
    drain_ring(full, p.stages, issued);
  } else if (warp == kConsumers + 1) {
    // ============================================================ x
    int issued = 0;
    bool ok = true;
    for (int item = blockIdx.x; ok && item < items; item += gridDim.x) {
      const int a = item / f_tiles, row0 = r.entry_row[a], rows = r.entry_row[a + 1] - row0;
      const __half* src[NT * 8];
#pragma unroll
      for (int i = 0; i < NT * 8; ++i) src[i] = p.x + (int64_t)r.token_of_row[row0 + min(i, rows - 1)] * p.hidden + lane * 8;
      for (int c = 0; c < chunks; ++c) {
        ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const int k = c * kStageK;
        const bool there = k + lane * 8 < p.hidden;
        const uint32_t dst = smem_u32(xs + ring.s * L.x_bytes);
#pragma unroll
        for (int i = 0; i < NT * 8; ++i)
          if (i < rows) cp_async16(dst + i * (kStageK * 2) + x_column(i, lane) * 16, there ? src[i] + k : p.x, there);
        cp_async_arrive(&full[ring.s]);
        ++issued;
        ring.next();
      }
    }
    drain_ring(full, p.stages, issued);
  } else {
    // ============================================================ products: warps 0 to 3 gate rows, 4 to 7 up rows
    const int fb = warp & 3, is_up = warp >> 2, g = lane >> 2, t = lane & 3;
    float* red = reinterpret_cast<float*>(&r + 1);  // [fb][value][lane]
    const Walk<FMT, NT> walk(g);
    const uint8_t* const w_at = smem + is_up * kBox + (fb * 16 + g) * 128 + t * 4;
    const uint8_t* const x_at = xs + g * (kStageK * 2) + t * 16;
    bool ok = true;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
      const int a = item / f_tiles, f0 = (item - a * f_tiles) * kTile, e = r.entry_expert[a];
      const int row0 = r.entry_row[a], rows = r.entry_row[a + 1] - row0, tiles = (rows + 7) / 8;
      float acc[NT][4];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
      // this lane's words in the scale tiles of its rows
      const uint8_t* const s_at = scales + is_up * TILES * 512 + (int)scale_word(((is_up ? p.ffn + f0 : f0) & 127) + fb * 16 + g, 0, 1);
      for (int c = 0; c < chunks; ++c) {
        if (ok) ok = mbar_wait_parked(&full[ring.s], ring.ph, &g_status);
        walk.stage(acc, w_at + ring.s * L.code_bytes, x_at + ring.s * L.x_bytes, s_at + ring.s * L.scale_bytes, t, tiles);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[ring.s]);
        ring.next();
      }
      // gate and up meet; rows g, g + 8 of columns 2t, 2t + 1
      if (!ok) r.failed = 1;
      if (is_up) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) red[((fb * NT + j) * 4 + i) * 32 + lane] = acc[j][i];
      }
      consumers_sync();
      if (!is_up && r.failed == 0) {
        const float ts = p.ts1 ? p.ts1[e] : 1.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float gv = acc[j][i] * ts, uv = red[((fb * NT + j) * 4 + i) * 32 + lane] * ts;
            const int row = j * 8 + 2 * t + (i & 1), f = f0 + fb * 16 + g + (i >> 1) * 8;
            // (h is rounded to fp16: it is the next product's operand, 2^-11 of itself at most, the error of its sum is
            // below that of the output's own rounding)
            if (row < rows) p.h[(int64_t)(row0 + row) * p.ffn + f] = __float2half_rn(gv / (1.0f + __expf(-gv)) * uv);
          }
      }
      consumers_sync();
    }
  }
}

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NT)) moe_fp4_down_kernel(const Params p, const __grid_constant__ CUtensorMap tmap_w) {
  constexpr Layout L = layout_down<FMT, NT>();
  constexpr int TILES = stage_tiles(FMT), kUnitK = 2 * kStageK;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const scales = smem + p.stages * L.code_bytes;
  uint8_t* const xs = scales + p.stages * L.scale_bytes;
  uint64_t* const full = reinterpret_cast<uint64_t*>(xs + p.stages * L.x_bytes);
  uint64_t* const empty = full + kMaxStages;
  Routing<NT>& r = *reinterpret_cast<Routing<NT>*>(reinterpret_cast<uint8_t*>(full) + kRoutingOffset);
  float* sums = reinterpret_cast<float*>(&r + 1);  // [half of k][token][64 columns]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = (int)cluster_rank(), n0 = (int)(blockIdx.x / p.cluster) * kTile;
  if (tid == 0) {
    init_ring(full, empty, p.stages);
    r.failed = 0;
  }
  for (int i = tid; i < 2 * p.tokens * kTile; i += kThreads) sums[i] = 0.0f;
  fence_proxy_async();
  // The logits and the weights are older than the kernel before this one, which let this one start only after its own wait
  // (the logits are read past L1, which may hold what was there before them).
  route<NT>(p, r);

  const int per = (p.ffn + kUnitK - 1) / kUnitK, units = r.entries * per;
  const int u0 = (int)((int64_t)units * rank / p.cluster), u1 = (int)((int64_t)units * (rank + 1) / p.cluster);
  Ring ring = {p.stages, 0, 0u};
  if (warp == kConsumers) {
    // ============================================================ weights (older than the kernel before, too)
    const bool leader = elect_one();
    int issued = 0;
    for (int u = u0; u < u1; ++u) {
      bool ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (leader) {
        const int a = u / per, c = u - a * per, e = r.entry_expert[a];
        uint64_t* bar = &full[ring.s];
        uint8_t* w = smem + ring.s * L.code_bytes;
        const bool two = c * kUnitK + kStageK < p.ffn;  // (else the second box keeps what it had: its x is zeros)
        mbar_arrive_expect_tx(bar, (two ? 2 * kBox : kBox) + L.scale_bytes);
        tma_load(w, &tmap_w, c * 256, e * p.hidden + n0, bar);
        if (two) tma_load(w + kBox, &tmap_w, c * 256 + 128, e * p.hidden + n0, bar);
        load_scale_tiles(scales + ring.s * L.scale_bytes, p.s2 + e * p.s2_expert + (int64_t)(n0 >> 7) * p.k_tiles2 * 512, c * 2 * TILES,
                         2 * TILES, p.k_tiles2 - 1, bar);
      }
      __syncwarp();
      ++issued;
      ring.next();
    }
    drain_ring(full, p.stages, issued);
  } else if (warp == kConsumers + 1) {
    // ============================================================ h
    griddep_wait();  // the kernel before's
    int issued = 0;
    for (int u = u0; u < u1; ++u) {
      bool ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int a = u / per, c = u - a * per, row0 = r.entry_row[a], rows = r.entry_row[a + 1] - row0;
      const uint32_t dst = smem_u32(xs + ring.s * L.x_bytes);
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int k = c * kUnitK + half * kStageK + lane * 8;
        const bool there = k < p.ffn;
        const __half* src = p.h + (int64_t)row0 * p.ffn + (there ? k : 0);
#pragma unroll
        for (int i = 0; i < NT * 8; ++i)
          if (i < rows) cp_async16(dst + (half * NT * 8 + i) * (kStageK * 2) + x_column(i, lane) * 16, src + (int64_t)i * p.ffn, there);
      }
      cp_async_arrive(&full[ring.s]);
      ++issued;
      ring.next();
    }
    drain_ring(full, p.stages, issued);
  } else {
    // ============================================================ products
    const int fb = warp & 3, kh = warp >> 2, g = lane >> 2, t = lane & 3;
    const uint8_t* const w_at = smem + kh * kBox + (fb * 16 + g) * 128 + t * 4;
    const uint8_t* const x_at = xs + (kh * NT * 8 + g) * (kStageK * 2) + t * 16;
    const uint8_t* const s_at = scales + kh * TILES * 512 + (int)scale_word((n0 & 127) + fb * 16 + g, 0, 1);
    const Walk<FMT, NT> walk(g);
    bool ok = true;
    float acc[NT][4];
    for (int u = u0; u < u1; ++u) {
      const int a = u / per, c = u - a * per;
      const int row0 = r.entry_row[a], rows = r.entry_row[a + 1] - row0, tiles = (rows + 7) / 8;
      if (u == u0 || c == 0) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[j][i] = 0.0f;
      }
      if (ok) ok = mbar_wait_parked(&full[ring.s], ring.ph, &g_status);
      walk.stage(acc, w_at + ring.s * L.code_bytes, x_at + ring.s * L.x_bytes, s_at + ring.s * L.scale_bytes, t, tiles);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[ring.s]);
      ring.next();
      if (u + 1 == u1 || c + 1 == per) {
        // this entry's part is complete here: gate times it, into the tokens' sums (a word belongs to one lane)
        const float ts = p.ts2 ? p.ts2[r.entry_expert[a]] : 1.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = j * 8 + 2 * t + (i & 1);
            if (row < rows) {
              float* at = sums + ((kh * p.tokens + r.token_of_row[row0 + row]) * kTile + fb * 16 + g + (i >> 1) * 8);
              *at = fmaf(r.gate_of_row[row0 + row] * ts, acc[j][i], *at);
            }
          }
        __syncwarp();
      }
    }
    if (!ok)
      for (int q = 0; q < p.cluster; ++q) st_cluster(at_rank(smem_u32(&r.failed), q), 1u);
  }
  griddep_wait();
  griddep_launch_dependents();
  __syncthreads();
  cluster_sync();
  if (r.failed == 0) {
    // four columns of a token a thread
    const int quads = p.tokens * (kTile / 4);
    for (int i = rank * kThreads + tid; i < quads; i += p.cluster * kThreads) {
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int q = 0; q < p.cluster; ++q)
        for (int half = 0; half < 2; ++half) {
          const float4 o = ld_cluster4(at_rank(smem_u32(sums + half * p.tokens * kTile + i * 4), q));
          v.x += o.x;
          v.y += o.y;
          v.z += o.z;
          v.w += o.w;
        }
      const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
      const int token = i / (kTile / 4), n = n0 + (i % (kTile / 4)) * 4;
      *reinterpret_cast<uint2*>(p.out + (int64_t)token * p.hidden + n) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  }
  cluster_sync();  // others may still be reading this CTA's sums
}

constexpr int kMaxDevices = 64;
std::atomic<bool> g_launched[kMaxDevices];  // devices whose status word a wait may have set

template <int NT>
size_t smem_bytes(const Layout& l, int stages, size_t extra) {
  return 1024 + (size_t)stages * stage_total(l) + kRoutingOffset + sizeof(Routing<NT>) + extra;
}

template <int FMT, int NT>
int launch(Params p, const CUtensorMap& t1, const CUtensorMap& t2, cudaStream_t stream) {
  auto up = moe_fp4_up_kernel<FMT, NT>;
  auto down = moe_fp4_down_kernel<FMT, NT>;
  static thread_local int configured_device = -1;
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (configured_device != dev) {
    RB200_CUDA(cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    RB200_CUDA(cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_device = dev;
  }
  const int ctas = ctas_per_sm(NT) * sm_count_current();
  const size_t room = (size_t)(NT == 1 ? 75 : 113) * 1024;  // so that they fit an SM's 228 KB, 1 KB more each
  const int rows = p.tokens * p.top_k;

  const size_t red = (size_t)4 * NT * 4 * 32 * 4;
  p.stages = kMaxStages;
  while (p.stages > 2 && smem_bytes<NT>(layout_up<FMT, NT>(), p.stages, red) > room) --p.stages;
  const int64_t items = (int64_t)rows * (p.ffn / kTile);  // at most
  RB200_CUDA(launch_dependent(up, dim3((unsigned)(items < ctas ? items : ctas)), kThreads,
                              smem_bytes<NT>(layout_up<FMT, NT>(), p.stages, red), stream, p, t1));

  const size_t sums = (size_t)2 * p.tokens * kTile * 4;
  p.stages = kMaxStages;
  while (p.stages > 2 && smem_bytes<NT>(layout_down<FMT, NT>(), p.stages, sums) > room) --p.stages;
  const int n_tiles = p.hidden / kTile, per = (p.ffn + 2 * kStageK - 1) / (2 * kStageK);
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem_bytes<NT>(layout_down<FMT, NT>(), p.stages, sums);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  // Clusters do not fill the SMs evenly, so how many of each size run at a time is asked for (once: the sums' share of
  // shared memory at its largest, which changes no stage count).  Time goes with waves / size.
  static thread_local int places_device = -1, places[9];
  if (places_device != dev) {
    cfg.numAttrs = 1;
    cudaLaunchConfig_t ask = cfg;
    ask.dynamicSmemBytes = room;
    for (int c = 1; c <= 8; ++c) {
      attr[0].val.clusterDim.x = (unsigned)c;
      ask.gridDim = dim3((unsigned)(ctas / c * c), 1, 1);
      RB200_CUDA(cudaOccupancyMaxActiveClusters(&places[c], down, &ask));
    }
    places_device = dev;
  }
  p.cluster = 1;
  for (int c = 2; c <= 8 && c <= p.top_k * per; ++c) {  // (a token's experts are top_k different ones)
    auto waves = [&](int size) { return places[size] < 1 ? 1 << 20 : (n_tiles + places[size] - 1) / places[size]; };
    if (waves(c) * p.cluster < waves(p.cluster) * c) p.cluster = c;
  }
  cfg.gridDim = dim3((unsigned)(n_tiles * p.cluster), 1, 1);
  attr[0].val.clusterDim.x = (unsigned)p.cluster;
  cfg.numAttrs = 2;
  RB200_CUDA(cudaLaunchKernelEx(&cfg, down, p, t2));
  return 0;
}

template <int FMT>
int launch_fmt(const Params& p, const CUtensorMap& t1, const CUtensorMap& t2, cudaStream_t stream) {
  return p.tokens <= 8 ? launch<FMT, 1>(p, t1, t2, stream) : launch<FMT, 2>(p, t1, t2, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace
}  // namespace f4

int fp4_moe_read_status(int* status_out) {
  *status_out = 0;
  int dev = -1;
  RB200_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= f4::kMaxDevices || !f4::g_launched[dev].load(std::memory_order_relaxed)) return 0;
  int v = 0;
  RB200_CUDA(cudaMemcpyFromSymbol(&v, f4::g_status, sizeof(int)));
  if (v != 0) {
    const int zero = 0;
    RB200_CUDA(cudaMemcpyToSymbol(f4::g_status, &zero, sizeof(int)));
  }
  *status_out = v;
  return 0;
}

}  // namespace rb200

using namespace rb200;

extern "C" {

size_t rb200_moe_layer_fp4_workspace_bytes(int64_t tokens, int64_t top_k, int64_t ffn) {
  return tokens > 0 && top_k > 0 && ffn > 0 ? (size_t)(tokens * top_k * ffn) * 2 : 0;
}

int rb200_moe_layer_fp4(const rb200_moe_layer_fp4_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  RB200_CHECK(d != nullptr && d->struct_size == sizeof(rb200_moe_layer_fp4_desc), "rb200_moe_layer_fp4_desc has a wrong struct_size");
  RB200_CHECK(d->format == f4::kMx || d->format == f4::kNv, "unknown 4-bit format %d", d->format);
  RB200_CHECK(d->tokens >= 0 && d->tokens <= f4::kMaxTokens, "tokens=%lld outside [0, %d]", (long long)d->tokens, f4::kMaxTokens);
  RB200_CHECK(d->num_experts >= 1 && d->num_experts <= f4::kMaxExperts, "num_experts=%lld outside [1, %d]", (long long)d->num_experts,
              f4::kMaxExperts);
  RB200_CHECK(d->top_k >= 1 && d->top_k <= f4::kMaxTopK && d->top_k <= d->num_experts, "top_k=%lld outside [1, min(%d, experts)]",
              (long long)d->top_k, f4::kMaxTopK);
  RB200_CHECK(d->hidden > 0 && d->hidden % 64 == 0 && d->ffn > 0 && d->ffn % 64 == 0 && d->hidden < (1 << 24) && d->ffn < (1 << 24) &&
                  d->num_experts * 2 * d->ffn < (1ll << 31) && d->num_experts * d->hidden < (1ll << 31),
              "hidden and ffn must be multiples of 64 (hidden=%lld, ffn=%lld)", (long long)d->hidden, (long long)d->ffn);
  RB200_CHECK(d->format == f4::kNv || (!d->gate_up_tensor_scale && !d->down_tensor_scale), "the mx format has no tensor scale");
  if (d->tokens == 0) return 0;
  RB200_CHECK(d->x && d->logits && d->w_gate_up && d->gate_up_scales && d->w_down && d->down_scales && d->out && workspace,
              "NULL argument");
  RB200_CHECK(f4::aligned16(d->x) && f4::aligned16(d->w_gate_up) && f4::aligned16(d->gate_up_scales) && f4::aligned16(d->w_down) &&
                  f4::aligned16(d->down_scales) && f4::aligned16(d->out) && f4::aligned16(workspace) &&
                  (reinterpret_cast<uintptr_t>(d->logits) & 3u) == 0,
              "tensors must be 16-byte aligned");
  RB200_CHECK(workspace_bytes >= rb200_moe_layer_fp4_workspace_bytes(d->tokens, d->top_k, d->ffn),
              "the workspace must hold rb200_moe_layer_fp4_workspace_bytes");
  f4::Params p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const __half*>(d->x);
  p.logits = d->logits;
  p.s1 = static_cast<const uint8_t*>(d->gate_up_scales);
  p.s2 = static_cast<const uint8_t*>(d->down_scales);
  p.ts1 = d->gate_up_tensor_scale;
  p.ts2 = d->down_tensor_scale;
  p.h = static_cast<__half*>(workspace);
  p.out = static_cast<__half*>(d->out);
  p.s1_expert = f4::scale_bytes(2 * d->ffn, d->hidden, d->format);
  p.s2_expert = f4::scale_bytes(d->hidden, d->ffn, d->format);
  p.tokens = (int)d->tokens;
  p.experts = (int)d->num_experts;
  p.top_k = (int)d->top_k;
  p.renormalize = d->renormalize;
  p.hidden = (int)d->hidden;
  p.ffn = (int)d->ffn;
  p.k_tiles1 = (int)f4::scale_k_tiles(d->hidden, d->format);
  p.k_tiles2 = (int)f4::scale_k_tiles(d->ffn, d->format);
  CUtensorMap t1, t2;
  if (make_tensor_map_2d(&t1, d->w_gate_up, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)d->hidden / 2,
                         (unsigned long long)(d->num_experts * 2 * d->ffn), (unsigned long long)d->hidden / 2, 128, f4::kTile,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) != 0 ||
      make_tensor_map_2d(&t2, d->w_down, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)d->ffn / 2,
                         (unsigned long long)(d->num_experts * d->hidden), (unsigned long long)d->ffn / 2, 128, f4::kTile,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B) != 0)
    return -1;
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < f4::kMaxDevices) f4::g_launched[dev].store(true, std::memory_order_relaxed);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return d->format == f4::kMx ? f4::launch_fmt<f4::kMx>(p, t1, t2, s) : f4::launch_fmt<f4::kNv>(p, t1, t2, s);
}

}  // extern "C"
