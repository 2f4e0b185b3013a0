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
// two, no hand-over through memory.  `down` does it, and asks for its first weights, as soon as CTAs of `up` leave it room on
// their SM: two of either fill one.
//
// Weights come by tensor-map loads in 128-byte rows, swizzled; a lane's code words are then free of bank conflicts.  A
// warp's lane (g, t) holds, of the 32 k of a chunk, k 8t .. 8t + 7 of rows g and g + 8: the MMAs' k slots are a permutation
// of k, the same one for x, whose eight values are one 16-byte word.
// `down` cuts the sequence of (64 output columns, entry, 512 k) evenly over the CTAs.  Each adds gate times its sums in shared
// memory, every word by one thread at a time in the order of the sequence; what it has of a column tile that is not its own
// alone goes to the workspace, and the last CTA to come adds the parts up in the order of the CTAs: nothing depends on timing.
//
// Measured, hidden 4096, ffn 14336, eight experts, two a token: one token in the mx format 50 us, 187 MB (3.7 TB/s), in nv 52; eight
// in the nv format 143 to 175 us by where their weights lie, 712 MB (5.0 to 4.1 TB/s); 29 tokens, hidden 2048, ffn 1408, 64 experts,
// six a token 80 us, 277 MB (3.5 TB/s).
// Boxes out of memory come at 6 TB/s at the most.  Below that, kNv is held by issue (63 instructions per 512 bytes of codes,
// issued in 63 % of the clocks), few or small experts by the starts and last tiles of two kernels.
#include <atomic>
#include <cstring>
#include <type_traits>

#include "../../include/relax_b200.h"
#include "fp4_mma.cuh"
#include "fp4_out.cuh"
#include "handover.h"
#include "tensormap.h"

namespace rb200 {
namespace f4 {
namespace {

using ug::elect_one;

constexpr int kMaxTokens = 32, kMaxExperts = 256, kMaxTopK = 8;
constexpr int kConsumers = 8;  // warps: four blocks of 16 rows, gate and up or two halves of k
constexpr int kThreads = (kConsumers + 2) * 32;  // and a warp for the weights' loads, one for x's
constexpr int kTile = 64;      // rows of a weight box: four 16-row blocks, inside one tile of scales
constexpr int kBox = kTile * 128;
constexpr int kMaxStages = 6;
constexpr int kMaxCtas = 512;  // that the workspace has room for

__device__ int g_status;

// Rows are the (token, expert) pairs by expert; an entry is at most 8 NT rows of one expert.
template <int NT>
struct alignas(16) Routing {
  static constexpr int kRows = kMaxTokens * kMaxTopK;
  uint32_t mask[kMaxExperts];  // tokens of an expert
  float gate_of_row[kRows];
  float gate_of[kRows];        // by token and choice
  int warp_sum[kConsumers];
  int entries;
  int failed, scaled;
  uint32_t ticket;
  uint16_t first_row[kMaxExperts];  // of an expert
  uint16_t entry_row[kRows + 2];
  uint8_t entry_expert[kRows];
  uint8_t token_of_row[kRows];
  uint8_t expert_of[kRows];
  int8_t exponent_of_row[kRows];  // down: its h is 2^exponent times what the products take
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
  int stages;
  float* parts;       // down: two tiles [tokens][64] a CTA
  uint32_t* tickets;  // down: a tile's parts that are there
  uint32_t* words;    // up: hand-over words, or nullptr
  int8_t* exponents;  // of h: a row's sixteens of f
  uint32_t* states;   // of up's CTAs, written by every call
  int absent;         // up: the CTA that hands over nothing (self-test), or -1
  uint64_t wait_ns;   // bound of the wait for them
};

// h between the kernels is fp16 times 2^exponent, an exponent for 16 f of a row: fp16 alone ends at 65504, and below 2^-14 it
// loses bits.  Where the largest of the sixteen lies in [2^-16, 2^11) the exponent is kPlain, and if it is everywhere, `down`
// takes the numbers as they lie.  Else it is in steps of 16, such that the largest becomes 2^-1 to 2^15, and `down` brings a row
// to its largest exponent (few sixteens have another), which multiplies the row's sums.  Either way an element is off by 2^-12 of
// itself, or by 2^-28, or, of a row whose largest is outside [2^-16, 2^11), by 2^-23 of that largest.  (The
// measured cases: exponents cost 48.1 -> 48.7 us for one token, 141.9 -> 142.7 for eight; with h some 2^10 times larger the same
// layers take 52.3 and 194 to 202.)
constexpr int kPlain = -4, kLowest = -100;
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // -126 .. 127
// of the bits of sixteen numbers' largest finite magnitude
__device__ __forceinline__ int h_exponent(uint32_t top) {
  const int x = (int)(top >> 23) - 127;
  return top == 0u ? kLowest : x >= -16 && x < 11 ? kPlain : max(kPlain + ((x + 5) >> 4) * 16, kLowest);
}
__device__ __forceinline__ uint32_t finite_bits(float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u ? b : 0u;
}

// order of floats as unsigned numbers, NaN lowest
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return v == v ? ((b & 0x80000000u) ? ~b : b | 0x80000000u) : 0u;
}

// order_key's inverse (NaN for 0)
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 0u ? __uint_as_float(0x7fffffffu) : __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

// A token by a warp, PER experts a lane.  Loops stay loops: the kernel's instructions are not in the caches when it starts, so
// what is executed once costs its fetch (29 tokens, 64 experts: 6.6 us unrolled over four tokens, the rounds alone 3).
template <int PER, int NT>
__device__ __forceinline__ void choose(const Params& p, Routing<NT>& r, const float* logits, int t) {
  const int lane = threadIdx.x & 31;
  uint32_t key[PER];  // 0: not there, or taken
  bool nan = false;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    const bool there = e < p.experts;
    const float v = (there ? logits[t * p.experts + e] : 0.0f) + 0.0f;  // (-0 is +0 then)
    nan = nan || v != v;
    key[i] = there ? max(order_key(v), 1u) : 0u;
  }
  uint32_t first[PER], my_key = 0u;
  int my_expert = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) first[i] = key[i];
#pragma unroll 1
  for (int j = 0; j < p.top_k; ++j) {
    uint32_t best = key[0];
    int at = lane;
#pragma unroll
    for (int i = 1; i < PER; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i * 32 + lane;
      }
    const uint32_t all = __reduce_max_sync(0xffffffffu, best);
    int e;
    if (PER == 1) e = __ffs((int)__ballot_sync(0xffffffffu, best == all)) - 1;
    else e = (int)__reduce_min_sync(0xffffffffu, best == all ? (uint32_t)at : 0xffffu);
    if (lane == j) {
      my_key = all;
      my_expert = e;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i * 32 + lane == e) key[i] = 0u;
  }
  const float top = key_value(__shfl_sync(0xffffffffu, my_key, 0));
  const float mine = lane < p.top_k ? expf(key_value(my_key) - top) : 0.0f;
  float sum = 0.0f;
  if (p.renormalize) {  // over the chosen ones, else over all experts
    sum = mine;
  } else {
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (first[i] != 0u) sum += expf(key_value(first[i]) - top);
  }
#pragma unroll 1
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  // (an infinite maximum: its difference to itself is NaN)
  nan = __any_sync(0xffffffffu, nan);
  if (lane < p.top_k) {
    r.expert_of[t * p.top_k + lane] = (uint8_t)my_expert;
    r.gate_of[t * p.top_k + lane] = nan ? __uint_as_float(0x7fffffffu) : mine / sum;
    atomicOr(&r.mask[my_expert], 1u << t);
  }
}

// The routing, by every thread of the CTA: the top_k largest logits of a token (equal ones: lower expert first), gates
// softmax over all experts or over the chosen ones; rows and entries in expert order.  The entries are there when it
// returns, the rows' tokens and gates after rows_sync, in which the weights' warp takes no part.
// `scratch`: tokens x experts floats, where loads go later.
template <int NT>
__device__ __forceinline__ void route(const Params& p, Routing<NT>& r, float* scratch) {
  constexpr int most = NT * 8;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid < kMaxExperts) r.mask[tid] = 0u;
#pragma unroll 1
  for (int i = tid; i < p.tokens * p.experts; i += 8 * kThreads) {  // (eight loads on their way: one after the other is a microsecond each)
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j * kThreads < p.tokens * p.experts) v[j] = __ldcg(p.logits + i + j * kThreads);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i + j * kThreads < p.tokens * p.experts) scratch[i + j * kThreads] = v[j];
  }
  __syncthreads();
#pragma unroll 1
  for (int t = warp; t < p.tokens; t += kThreads / 32) {
    if (p.experts <= 32) choose<1>(p, r, scratch, t);
    else if (p.experts <= 64) choose<2>(p, r, scratch, t);
    else choose<kMaxExperts / 32>(p, r, scratch, t);
  }
  fence_proxy_async();  // bulk copies write the scratch next
  __syncthreads();
  const int n = tid < kMaxExperts ? __popc(r.mask[tid]) : 0, parts = (n + most - 1) / most;
  int upto = n | parts << 16;  // rows and entries counted together
#pragma unroll 1
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += u;
  }
  if (warp < kConsumers && lane == 31) r.warp_sum[warp] = upto;
  __syncthreads();
  if (warp < kConsumers) {
    int before = upto - (n | parts << 16);
#pragma unroll 1
    for (int w = 0; w < warp; ++w) before += r.warp_sum[w];
    const int row = before & 0xffff, a = before >> 16;
    r.first_row[tid] = (uint16_t)row;
#pragma unroll 1
    for (int i = 0; i < parts; ++i) {
      r.entry_expert[a + i] = (uint8_t)tid;
      r.entry_row[a + i] = (uint16_t)(row + i * most);
    }
    if (tid == kMaxExperts - 1) {
      r.entries = a + parts;
      r.entry_row[a + parts] = (uint16_t)(row + n);
    }
  }
  __syncthreads();
  if (tid < p.tokens * p.top_k) {
    const int e = r.expert_of[tid], t = tid / p.top_k, row = r.first_row[e] + __popc(r.mask[e] & ((1u << t) - 1u));
    r.token_of_row[row] = (uint8_t)t;
    r.gate_of_row[row] = r.gate_of[tid];
    r.exponent_of_row[row] = kPlain;
  }
}
__device__ __forceinline__ void rows_sync() {
  if ((threadIdx.x >> 5) == kConsumers) asm volatile("bar.arrive 2, %0;" ::"n"(kThreads) : "memory");
  else asm volatile("bar.sync 2, %0;" ::"n"(kThreads) : "memory");
}

// 16 bytes of global memory, or zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void cp_async_wait() {  // all but the last LEFT groups have landed
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
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
// Four 8 x 16-byte matrices: lane i names row i % 8 of matrix i / 8, and lane (g, t) gets word t of row g of each.
__device__ __forceinline__ void load_matrices(uint32_t (&v)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(at)
               : "memory");
}

// The scales of rows g and g + 8 over 128 k, as the products take them.
template <int FMT>
struct Scales {
  // kMx: fp32 scales of the four blocks of either row.  kNv: this lane's scales of row g (low half) and of row g + 8, by chunk
  float f0[4], f8[4];
  uint32_t both[4];
  __device__ __forceinline__ void take(const uint8_t* at0, const uint8_t* at8, int t) {  // their words in the (first) tile
    if (FMT == kMx) {
      expand(*reinterpret_cast<const uint32_t*>(at0), f0);
      expand(*reinterpret_cast<const uint32_t*>(at8), f8);
    } else {
      // blocks 2i and 2i + 1 of chunk i; lanes t < 2 hold k of the first, the others of the second
      const uint32_t sel = t < 2 ? 0x40u : 0x51u;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint32_t a = *reinterpret_cast<const uint32_t*>(at0 + q * 512) & 0x7f7f7f7fu;
        const uint32_t b = *reinterpret_cast<const uint32_t*>(at8 + q * 512) & 0x7f7f7f7fu;
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
    const __half2 both = *reinterpret_cast<const __half2*>(&s.both[i]);
    const __half2 p0 = __low2half2(both), p8 = __high2half2(both);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      __half2 v0 = __hmul2(*reinterpret_cast<const __half2*>(&a0[q]), p0), v8 = __hmul2(*reinterpret_cast<const __half2*>(&a8[q]), p8);
      a0[q] = *reinterpret_cast<const uint32_t*>(&v0);
      a8[q] = *reinterpret_cast<const uint32_t*>(&v8);
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

// A warp's share of a stage: 16 rows over 256 k, eight chunks of 32.  `w` the block's first row in a box of 128-byte rows,
// swizzled; `x` row g of the stage's x at this lane's 16 bytes; `s0`, `s8` rows g's and g + 8's words in the first scale tile.
// kNv adds the chunks to two accumulators in turn: one MMA after the other into one is a chain of 20 clocks a link.
template <int FMT, int NT>
struct Walk {
  static constexpr int kSums = FMT == kNv ? 2 : 1;
  uint32_t off[4];
  int xoff[2];
  __device__ __forceinline__ explicit Walk(int lane) {
    const int r = lane & 7, m = lane >> 3;  // rows r, r + 8 of chunk 2j, then of chunk 2j + 1
#pragma unroll
    for (int j = 0; j < 4; ++j) off[j] = (uint32_t)(((m & 1) * 8 + r) * 128 + (((2 * j + (m >> 1)) ^ r) << 4));
#pragma unroll
    for (int i = 0; i < 2; ++i) xoff[i] = (i ^ ((lane >> 2) & 1)) * 64;
  }
  __device__ __forceinline__ void stage(float (&acc)[kSums][NT][4], uint32_t w, const uint8_t* x0, const uint8_t* s0, const uint8_t* s8, int t,
                                        int tiles) const {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      Scales<FMT> s;
      s.take(s0 + q * (stage_tiles(FMT) / 2) * 512, s8 + q * (stage_tiles(FMT) / 2) * 512, t);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t v[4];
        load_matrices(v, w + off[q * 2 + h]);
        uint4 x[2][NT];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < NT; ++j)
            x[i][j] = *reinterpret_cast<const uint4*>(x0 + xoff[i] + q * 256 + h * 128 + j * 8 * (kStageK * 2));
        chunk<FMT, NT>(acc[0], v[0], v[1], s, 2 * h, x[0], tiles);
        chunk<FMT, NT>(acc[kSums - 1], v[2], v[3], s, 2 * h + 1, x[1], tiles);
      }
    }
  }
};

// Shared memory: [codes of all stages][scales][x][barriers][routing][sums], offsets from the aligned base.
struct Layout {
  int code_bytes, scale_bytes, x_bytes;  // of a stage
};
// up: boxes of gate and of up, with their scale tiles; down: two boxes of consecutive k, theirs
template <int FMT, int NT, bool UP>
__host__ __device__ constexpr Layout layout() {
  return {2 * kBox, 2 * stage_tiles(FMT) * 512, NT * 8 * (UP ? 1 : 2) * kStageK * 2};
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

// Rows src + i * pitch elements (or, with tokens, src + token * pitch) of 256 k into a stage's x, 16 bytes a lane.
__device__ __forceinline__ void copy_rows(uint32_t dst, const __half* src, int64_t pitch, const uint8_t* tokens, int rows, bool there) {
  const int lane = threadIdx.x & 31;
#pragma unroll 2
  for (int i = 0; i < rows; ++i)
    cp_async16(dst + i * (kStageK * 2) + x_column(i, lane) * 16, src + (tokens ? tokens[i] : i) * pitch, there);
}

// Exponents of rows: the largest of their sixteens.  By a warp, two rows at once.
template <int NT>
__device__ __forceinline__ void take_exponents(const Params& p, Routing<NT>& r, int row0, int rows) {
  const int lane = threadIdx.x & 31, words = p.ffn / 64;
#pragma unroll 1
  for (int i = 0; i < rows; i += 2) {
    const int more = i + 1 < rows ? words : 0;
    const uint32_t* from = reinterpret_cast<const uint32_t*>(p.exponents) + (int64_t)(row0 + i) * words;
    uint32_t top[2] = {0x80808080u, 0x80808080u};
#pragma unroll 1
    for (int w = lane; w < words; w += 8 * 32) {
      uint32_t v[2][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[0][j] = w + j * 32 < words ? __ldcg(from + w + j * 32) : 0x80808080u;
        v[1][j] = w + j * 32 < more ? __ldcg(from + words + w + j * 32) : 0x80808080u;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        top[0] = __vmaxs4(top[0], v[0][j]);
        top[1] = __vmaxs4(top[1], v[1][j]);
      }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      top[q] = __vmaxs4(top[q], top[q] >> 16 | top[q] << 16);
      top[q] = __vmaxs4(top[q], top[q] >> 8 | top[q] << 24);
      const int e = __reduce_max_sync(0xffffffffu, (int)(int8_t)top[q]);
      if (lane == 0 && i + q < rows) r.exponent_of_row[row0 + i + q] = (int8_t)e;
    }
  }
  __syncwarp();
}
// What this lane's copies brought of rows' h, eight numbers of either half at `k` and `k` + 256, from the exponents of their
// sixteens to those of the rows.  All copies but those of the last LEFT groups are waited for.
template <int LEFT, int NT>
__device__ __forceinline__ void rescale_rows(const Params& p, const Routing<NT>& r, uint8_t* x, int k, int row0, int rows) {
  const int lane = threadIdx.x & 31;
  const signed char* const from = reinterpret_cast<const signed char*>(p.exponents) + (int64_t)row0 * (p.ffn / 16) + k / 16;
#pragma unroll 1
  for (int base = 0; base < rows; base += 4) {
    int own[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int half = 0; half < 2; ++half)
        own[half][i] = base + i < rows && k + half * kStageK < p.ffn ? __ldcg(from + (int64_t)(base + i) * (p.ffn / 16) + half * (kStageK / 16)) : 127;
    cp_async_wait<LEFT>();
#pragma unroll 1
    for (int i = 0; i < 4 && base + i < rows; ++i) {
      const int row = base + i;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int e = i == 0 ? own[half][0] : i == 1 ? own[half][1] : i == 2 ? own[half][2] : own[half][3];
        const int by = e - r.exponent_of_row[row0 + row];
        if (e == 127 || by == 0) continue;
        // (fp16's powers of two end at -24; a number times 2^-48 is zero, an infinity stays one)
        const __half2 one = __float2half2_rn(power_of_two(max(by, -24))), two = __float2half2_rn(power_of_two(max(min(by + 24, 0), -24)));
        __half2* v = reinterpret_cast<__half2*>(x + half * (NT * 8 * kStageK * 2) + row * (kStageK * 2) + x_column(row, lane) * 16);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = __hmul2(__hmul2(v[q], one), two);
      }
    }
  }
}

template <int S, int NT>
__device__ __forceinline__ void zero(float (&sum)[S][NT][4]) {
#pragma unroll
  for (int q = 0; q < S; ++q)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[q][j][i] = 0.0f;
}
template <int S, int NT>
__device__ __forceinline__ void join(float (&sum)[S][NT][4]) {  // all into the first
#pragma unroll
  for (int q = 1; q < S; ++q)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[0][j][i] += sum[q][j][i];
}

constexpr int kRoutingOffset = 2 * kMaxStages * 8;
constexpr int kCtasPerSm = 2;

// A sequence of units cut evenly over the CTAs.
struct Share {
  int total, ctas;  // units, CTAs with some
  __device__ __forceinline__ int begin(int cta) const { return (int)((int64_t)total * cta / ctas); }
  __device__ __forceinline__ int owner(int unit) const { return (int)(((int64_t)(unit + 1) * ctas - 1) / total); }
};
// A unit's place, (tile, a, c) for `down`, (a, tile, c) for `up`, kept by counting: the divisions took as long as a unit's
// products.
template <bool UP>
struct Place {
  int tile, a, c, per, inner;  // chunks of an inner item, items of an outer one
  __device__ __forceinline__ Place(int unit, int per_, int inner_) : per(per_), inner(inner_) {
    const int outer = unit / (per * inner), v = unit - outer * (per * inner), in = v / per;
    tile = UP ? in : outer;
    a = UP ? outer : in;
    c = v - in * per;
  }
  __device__ __forceinline__ bool last_of_entry() const { return c + 1 == per; }
  __device__ __forceinline__ bool last_of_tile() const { return last_of_entry() && a + 1 == inner; }
  __device__ __forceinline__ void next() {
    if (++c == per) {
      c = 0;
      int& in = UP ? tile : a;
      if (++in == inner) {
        in = 0;
        ++(UP ? a : tile);
      }
    }
  }
};

// What `down` has to know of up's CTAs, a word of each (one for all of them would have to be cleared first).
constexpr uint32_t kFailed = 1u;  // a wait ran out: parts of h are not there
constexpr uint32_t kScaled = 2u;  // some exponent of h is not kPlain

// Hand-over words (handover.h): a warp's sums of a part of a 64-row tile.  A word is its own flag, vacant (all bits set) at rest.
constexpr uint32_t kVacant = 0xffffffffu;
template <int NT>
__host__ __device__ constexpr int part_words() {
  return kConsumers * NT * 4 * 32;
}
template <int NT>
__device__ __forceinline__ uint4* part_of(uint32_t* words, int cta, int j) {
  return reinterpret_cast<uint4*>(words + (int64_t)cta * part_words<NT>()) + ((threadIdx.x >> 5) * NT + j) * 32 + (threadIdx.x & 31);
}
template <int NT>
__device__ __forceinline__ void publish(uint32_t* words, int cta, const float (&acc)[NT][4]) {
#pragma unroll
  for (int j = 0; j < NT; ++j) {
    uint32_t v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = __float_as_uint(acc[j][i]);
      if (v[i] == kVacant) v[i] = 0x7fffffffu;
    }
    asm volatile("st.volatile.global.v4.u32 [%0], {%1, %2, %3, %4};" ::"l"(part_of<NT>(words, cta, j)), "r"(v[0]), "r"(v[1]), "r"(v[2]),
                 "r"(v[3])
                 : "memory");
  }
}
// acc += the part of `cta`, whose words are left vacant; false when the wait for them ran out
template <int NT>
__device__ __forceinline__ bool absorb(uint32_t* words, int cta, float (&acc)[NT][4], uint64_t limit_ns) {
#pragma unroll 1
  for (int j = 0; j < NT; ++j) {
    uint4* at = part_of<NT>(words, cta, j);
    uint32_t v[4];
    uint64_t began = 0;
    for (;;) {
      asm volatile("ld.volatile.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "l"(at) : "memory");
      if (v[0] != kVacant && v[1] != kVacant && v[2] != kVacant && v[3] != kVacant) break;
      uint64_t now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (began == 0) began = now;
      if (now - began > limit_ns) {
        atomicExch(&g_status, kStatusWaitTimeout);
        return false;
      }
    }
    asm volatile("st.volatile.global.v4.u32 [%0], {%1, %1, %1, %1};" ::"l"(at), "r"(kVacant) : "memory");
#pragma unroll
    for (int q = 0; q < NT; ++q)  // (registers have no index)
      if (q == j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[q][i] += __uint_as_float(v[i]);
      }
  }
  return true;
}

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) moe_fp4_up_kernel(const Params p, const __grid_constant__ CUtensorMap tmap_w) {
  constexpr int TILES = stage_tiles(FMT);
  constexpr Layout L = layout<FMT, NT, true>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const scales = smem + p.stages * L.code_bytes;
  uint8_t* const xs = scales + p.stages * L.scale_bytes;
  uint64_t* const full = reinterpret_cast<uint64_t*>(xs + p.stages * L.x_bytes);
  uint64_t* const empty = full + kMaxStages;
  Routing<NT>& r = *reinterpret_cast<Routing<NT>*>(reinterpret_cast<uint8_t*>(full) + kRoutingOffset);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    tma_prefetch_map(&tmap_w);
    init_ring(full, empty, p.stages);
    r.failed = r.scaled = 0;
  }
  fence_proxy_async();
  griddep_wait();
  griddep_launch_dependents();
  if (blockIdx.x == 0)
    for (int i = tid; i < p.hidden / kTile; i += kThreads) p.tickets[i] = 0u;
  route<NT>(p, r, reinterpret_cast<float*>(smem));
  rows_sync();

  // (entry, 64 f, 256 k) units.  With words to hand over parts in, the CTAs get equal shares: whoever has an item's first k adds
  // what the CTAs behind it did of it, which they do first; else whole items.
  const int f_tiles = p.ffn / kTile, items = r.entries * f_tiles, chunks = (p.hidden + kStageK - 1) / kStageK;
  Share share;
  share.total = p.words ? items * chunks : items;
  share.ctas = min((int)gridDim.x, p.words ? max(share.total / 2, 1) : items);
  const bool any = (int)blockIdx.x < share.ctas;
  const int unit = p.words ? 1 : chunks;
  const int u0 = any ? share.begin(blockIdx.x) * unit : 0, u1 = any ? share.begin(blockIdx.x + 1) * unit : 0;
  Ring ring = {p.stages, 0, 0u};
  if (warp == kConsumers) {
    // ============================================================ weights
    const bool leader = elect_one();
    int issued = 0;
    Place<true> at(u0, chunks, f_tiles);
    for (int u = u0; u < u1; ++u, at.next()) {
      bool ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (leader) {
        const int c = at.c, f0 = at.tile * kTile, e = r.entry_expert[at.a];
        const uint8_t* s_e = p.s1 + e * p.s1_expert;
        uint64_t* bar = &full[ring.s];
        uint8_t* w = smem + ring.s * L.code_bytes;
        uint8_t* sc = scales + ring.s * L.scale_bytes;
        mbar_arrive_expect_tx(bar, L.code_bytes + L.scale_bytes);
        tma_load(w, &tmap_w, c * 128, e * 2 * p.ffn + f0, bar);
        tma_load(w + kBox, &tmap_w, c * 128, e * 2 * p.ffn + p.ffn + f0, bar);
        load_scale_tiles(sc, s_e + (int64_t)(f0 >> 7) * p.k_tiles1 * 512, c * TILES, TILES, p.k_tiles1 - 1, bar);
        load_scale_tiles(sc + TILES * 512, s_e + (int64_t)((p.ffn + f0) >> 7) * p.k_tiles1 * 512, c * TILES, TILES, p.k_tiles1 - 1, bar);
      }
      __syncwarp();
      ++issued;
      ring.next();
    }
    drain_ring(full, p.stages, issued);
  } else if (warp == kConsumers + 1) {
    // ============================================================ x
    int issued = 0;
    Place<true> at(u0, chunks, f_tiles);
    for (int u = u0; u < u1; ++u, at.next()) {
      bool ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int row0 = r.entry_row[at.a], rows = r.entry_row[at.a + 1] - row0, k = at.c * kStageK + lane * 8;
      const bool there = k < p.hidden;
      copy_rows(smem_u32(xs + ring.s * L.x_bytes), p.x + (there ? k : 0), p.hidden, r.token_of_row + row0, rows, there);
      cp_async_arrive(&full[ring.s]);
      ++issued;
      ring.next();
    }
    drain_ring(full, p.stages, issued);
  } else {
    // ============================================================ products: warps 0 to 3 gate rows, 4 to 7 up rows
    const int fb = warp & 3, is_up = warp >> 2, g = lane >> 2, t = lane & 3;
    float* red = reinterpret_cast<float*>(&r + 1);  // [fb][value][lane]
    const Walk<FMT, NT> walk(lane);
    constexpr int kSums = Walk<FMT, NT>::kSums;
    const uint32_t w_at = smem_u32(smem) + is_up * kBox + fb * 16 * 128;
    const uint8_t* const x_at = xs + g * (kStageK * 2) + t * 16;
    bool ok = true;
    Place<true> at(u0, chunks, f_tiles);
    for (int u = u0; u < u1;) {
      const int f0 = at.tile * kTile, e = r.entry_expert[at.a], first = at.c, n = min(chunks - first, u1 - u);
      const int row0 = r.entry_row[at.a], rows = r.entry_row[at.a + 1] - row0, tiles = (rows + 7) / 8;
      float sum[kSums][NT][4];
      zero(sum);
      // this lane's words in the scale tiles of its rows
      const uint8_t* const s0 = scales + is_up * TILES * 512 + (int)scale_word(((is_up ? p.ffn + f0 : f0) & 127) + fb * 16 + g, 0, 1);
      const uint8_t* const s8 = scales + is_up * TILES * 512 + (int)scale_word(((is_up ? p.ffn + f0 : f0) & 127) + fb * 16 + g + 8, 0, 1);
      for (int i = 0; i < n; ++i, at.next()) {
        if (ok) ok = mbar_wait_parked(&full[ring.s], ring.ph, &g_status);
        walk.stage(sum, w_at + ring.s * L.code_bytes, x_at + ring.s * L.x_bytes, s0 + ring.s * L.scale_bytes, s8 + ring.s * L.scale_bytes, t,
                   tiles);
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[ring.s]);
        ring.next();
      }
      u += n;
      float(&acc)[NT][4] = sum[0];
      join(sum);
      if (first > 0) {
        if (ok && (int)blockIdx.x != p.absent) publish<NT>(p.words, blockIdx.x, acc);
        continue;
      }
      if (n < chunks) {
        const int last = share.owner(u - n + chunks - 1);
        for (int q = blockIdx.x + 1; ok && q <= last; ++q) ok = absorb<NT>(p.words, q, acc, p.wait_ns);
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
        const int f = f0 + fb * 16;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          float h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = silu(acc[j][i] * ts) * (red[((fb * NT + j) * 4 + i) * 32 + lane] * ts);
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t top = max(finite_bits(h[q]), finite_bits(h[2 + q]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            const int row = j * 8 + 2 * t + q, exponent = h_exponent(top);
            if (row < rows) {
              const float by = power_of_two(-exponent);
              __half* to = p.h + (int64_t)(row0 + row) * p.ffn + f + g;
              to[0] = __float2half_rn(h[q] * by);
              to[8] = __float2half_rn(h[2 + q] * by);
              if (g == 0) p.exponents[(int64_t)(row0 + row) * (p.ffn / 16) + f / 16] = (int8_t)exponent;
              if (exponent != kPlain && top != 0u) r.scaled = 1;
            }
          }
        }
      }
      consumers_sync();
    }
    if (!ok) r.failed = 1;
  }
  __syncthreads();
  if (tid == 0) p.states[blockIdx.x] = (r.failed ? kFailed : 0u) | (r.scaled ? kScaled : 0u);
}

template <int FMT, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) moe_fp4_down_kernel(const Params p, const __grid_constant__ CUtensorMap tmap_w) {
  constexpr int TILES = stage_tiles(FMT), kUnitK = 2 * kStageK;
  constexpr Layout L = layout<FMT, NT, false>();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* const scales = smem + p.stages * L.code_bytes;
  uint8_t* const xs = scales + p.stages * L.scale_bytes;
  uint64_t* const full = reinterpret_cast<uint64_t*>(xs + p.stages * L.x_bytes);
  uint64_t* const empty = full + kMaxStages;
  Routing<NT>& r = *reinterpret_cast<Routing<NT>*>(reinterpret_cast<uint8_t*>(full) + kRoutingOffset);
  float* sums = reinterpret_cast<float*>(&r + 1);  // [half of k][token][64 columns]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    tma_prefetch_map(&tmap_w);
    init_ring(full, empty, p.stages);
    r.failed = r.scaled = 0;
  }
  for (int i = tid; i < 2 * p.tokens * kTile; i += kThreads) sums[i] = 0.0f;
  fence_proxy_async();
  // The logits and the weights are older than the kernel before this one, which let this one start only after its own wait
  // (the logits are read past L1, which may hold what was there before them).
  route<NT>(p, r, reinterpret_cast<float*>(smem));
  rows_sync();

  const int per = (p.ffn + kUnitK - 1) / kUnitK;
  const int per_tile = r.entries * per;
  Share share;
  share.total = p.hidden / kTile * per_tile;
  share.ctas = (int)gridDim.x;
  // as many CTAs a column tile where that is nearly all of them: every CTA then has a part of one tile only
  const int each = share.ctas / (p.hidden / kTile);
  if (each * (p.hidden / kTile) * 16 >= share.ctas * 15) share.ctas = each * (p.hidden / kTile);
  share.ctas = min(share.ctas, share.total);
  const bool any = (int)blockIdx.x < share.ctas;
  const int u0 = any ? share.begin(blockIdx.x) : 0, u1 = any ? share.begin(blockIdx.x + 1) : 0;
  Ring ring = {p.stages, 0, 0u};
  if (warp == kConsumers) {
    // ============================================================ weights (older than the kernel before, too)
    const bool leader = elect_one();
    int issued = 0;
    Place<false> at(u0, per, r.entries);
    for (int u = u0; u < u1; ++u, at.next()) {
      bool ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (leader) {
        const int tile = at.tile, c = at.c, e = r.entry_expert[at.a];
        uint64_t* bar = &full[ring.s];
        uint8_t* w = smem + ring.s * L.code_bytes;
        const bool two = c * kUnitK + kStageK < p.ffn;  // (else the second box keeps what it had: its x is zeros)
        mbar_arrive_expect_tx(bar, (two ? 2 * kBox : kBox) + L.scale_bytes);
        tma_load(w, &tmap_w, c * 256, e * p.hidden + tile * kTile, bar);
        if (two) tma_load(w + kBox, &tmap_w, c * 256 + 128, e * p.hidden + tile * kTile, bar);
        load_scale_tiles(scales + ring.s * L.scale_bytes, p.s2 + e * p.s2_expert + (int64_t)(tile >> 1) * p.k_tiles2 * 512, c * 2 * TILES,
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
    griddep_launch_dependents();
    // The words of state are asked for first and looked at when the copies of the first unit are on their way, too (one token
    // 47.7 -> 48.1 us; looked at after the copies of every stage 48.8).
    uint32_t state = 0u;
    {
      uint32_t word[kMaxCtas / 32];
#pragma unroll
      for (int i = 0; i < kMaxCtas / 32; ++i) word[i] = i * 32 + lane < (int)gridDim.x ? __ldcg(p.states + i * 32 + lane) : 0u;
#pragma unroll
      for (int i = 0; i < kMaxCtas / 32; ++i) state |= word[i];
    }
    int issued = 0;
    Place<false> at(u0, per, r.entries), behind = at;
    int behind_s = 0;
    bool first = true;
    auto finish_behind = [&](auto left) {
      const int row0 = r.entry_row[behind.a], rows = r.entry_row[behind.a + 1] - row0;
      if (first || behind.c == 0) take_exponents(p, r, row0, rows);
      first = false;
      rescale_rows<decltype(left)::value>(p, r, xs + behind_s * L.x_bytes, behind.c * kUnitK + lane * 8, row0, rows);
      mbar_arrive(&full[behind_s]);
      behind.next();
      if (++behind_s == p.stages) behind_s = 0;
    };
    for (int u = u0; u < u1; ++u, at.next()) {
      bool ok = mbar_wait_parked(&empty[ring.s], ring.ph ^ 1u, &g_status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      const int c = at.c, row0 = r.entry_row[at.a], rows = r.entry_row[at.a + 1] - row0;
#pragma unroll 1
      for (int half = 0; half < 2; ++half) {
        const int k = c * kUnitK + half * kStageK + lane * 8;
        const bool there = k < p.ffn;
        copy_rows(smem_u32(xs + ring.s * L.x_bytes) + half * (NT * 8 * kStageK * 2), p.h + (int64_t)row0 * p.ffn + (there ? k : 0), p.ffn,
                  nullptr, rows, there);
      }
      ++issued;
      if (u == u0) {
        state = __reduce_or_sync(0xffffffffu, state);
        if (state & kFailed) r.failed = 1;  // (who waits for a unit sees it)
      }
      if (state & kScaled) {  // one unit's copies are on their way while the unit before is seen to
        cp_async_commit();
        if (u > u0) finish_behind(std::integral_constant<int, 1>());
        if (u + 1 == u1) finish_behind(std::integral_constant<int, 0>());
      } else {
        cp_async_arrive(&full[ring.s]);
      }
      ring.next();
    }
    drain_ring(full, p.stages, issued);
  } else {
    // ============================================================ products
    griddep_wait();  // for what is written below
    const int fb = warp & 3, kh = warp >> 2, g = lane >> 2, t = lane & 3;
    const uint32_t w_at = smem_u32(smem) + kh * kBox + fb * 16 * 128;
    const uint8_t* const x_at = xs + (kh * NT * 8 + g) * (kStageK * 2) + t * 16;
    const int s_row = (int)scale_word(fb * 16 + g, 0, 1), s_row8 = (int)scale_word(fb * 16 + g + 8, 0, 1);
    const Walk<FMT, NT> walk(lane);
    constexpr int kSums = Walk<FMT, NT>::kSums;
    bool ok = true;
    float sum[kSums][NT][4];
    float(&acc)[NT][4] = sum[0];
    int tile_first = u0;  // this CTA's first unit of the tile at hand
    Place<false> at(u0, per, r.entries);
    int rows = 0, tiles = 0, token[NT][2];
    float gate[NT][2];
    for (int u = u0; u < u1; ++u, at.next()) {
      const int tile = at.tile;
      if (u == u0 || at.c == 0) {
        zero(sum);
        const int row0 = r.entry_row[at.a];
        rows = r.entry_row[at.a + 1] - row0;
        tiles = (rows + 7) / 8;
        const float ts = p.ts2 ? p.ts2[r.entry_expert[at.a]] : 1.0f;
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) {  // of this lane's columns of the sums
            const int row = row0 + min(j * 8 + 2 * t + q, rows - 1);
            token[j][q] = r.token_of_row[row];
            gate[j][q] = r.gate_of_row[row] * ts;
          }
      }
      if (ok) ok = mbar_wait_parked(&full[ring.s], ring.ph, &g_status);
      const uint8_t* sc = scales + ring.s * L.scale_bytes + kh * TILES * 512 + (tile & 1) * 8;  // rows 64 .. 127 of a scale tile: words 2, 3
      walk.stage(sum, w_at + ring.s * L.code_bytes, x_at + ring.s * L.x_bytes, sc + s_row, sc + s_row8, t, tiles);
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[ring.s]);
      ring.next();
      const bool tile_ends = u + 1 == u1 || at.last_of_tile();
      if (tile_ends || at.last_of_entry()) {
        join(sum);
        // this entry's part is complete here: gate times it and the row's power of two, into the tokens' sums (a word belongs to one lane at a time)
        float* word[NT][2];
        float had[NT][4], gate_here[NT][2];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            word[j][q] = sums + (kh * p.tokens + token[j][q]) * kTile + fb * 16 + g;
            had[j][q] = word[j][q][0];
            had[j][2 + q] = word[j][q][8];
            gate_here[j][q] = gate[j][q] * power_of_two(r.exponent_of_row[r.entry_row[at.a] + min(j * 8 + 2 * t + q, rows - 1)]);
          }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            if (j * 8 + 2 * t + q < rows) {
              word[j][q][0] = fmaf(gate_here[j][q], acc[j][q], had[j][q]);
              word[j][q][8] = fmaf(gate_here[j][q], acc[j][2 + q], had[j][2 + q]);
            }
        __syncwarp();
      }
      if (tile_ends) {
        if (!ok) r.failed = 1;
        consumers_sync();
        // The tile as far as this CTA has it: written as it is if that is all of it, else put with the parts of other CTAs; who
        // comes last adds them up, in the order of the CTAs.
        constexpr int quads = kTile / 4;
        const int first = share.owner(tile * per_tile), last = share.owner((tile + 1) * per_tile - 1);
        const bool whole = first == last;
        const int size = p.tokens * kTile;
        float* mine = p.parts + (int64_t)(blockIdx.x * 2 + (tile_first == u0 ? 0 : 1)) * size;
        bool write = whole && r.failed == 0;
        if (!whole) {
          for (int i = tid; i < size / 4; i += kConsumers * 32) {
            const float4 x = reinterpret_cast<const float4*>(sums)[i], y = reinterpret_cast<const float4*>(sums + size)[i];
            __stcg(reinterpret_cast<float4*>(mine) + i, make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w));
          }
          __threadfence();
          consumers_sync();
          if (tid == 0) r.ticket = atomicAdd(p.tickets + tile, 1u | (r.failed ? 0x10000u : 0u));
          consumers_sync();
          // (every part is there, and none of a CTA whose wait ran out)
          write = r.ticket == (uint32_t)(last - first) && r.failed == 0;
          __threadfence();
        }
        if (write) {
          for (int i = tid; i < size / 4; i += kConsumers * 32) {
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            auto add = [&](const float4& q) {
              o.x += q.x;
              o.y += q.y;
              o.z += q.z;
              o.w += q.w;
            };
            if (whole) {
              add(reinterpret_cast<const float4*>(sums)[i]);
              add(reinterpret_cast<const float4*>(sums + size)[i]);
            } else {
#pragma unroll 4
              for (int q = first; q <= last; ++q) {
                const int slot = share.begin(q) / per_tile == tile ? 0 : 1;
                add(__ldcg(reinterpret_cast<const float4*>(p.parts + (int64_t)(q * 2 + slot) * size) + i));
              }
            }
            const __half2 lo = __floats2half2_rn(o.x, o.y), hi = __floats2half2_rn(o.z, o.w);
            *reinterpret_cast<uint2*>(p.out + (int64_t)(i / quads) * p.hidden + tile * kTile + (i % quads) * 4) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          }
        }
        tile_first = u + 1;
        if (u + 1 < u1) {
          consumers_sync();
          for (int i = tid; i < 2 * size; i += kConsumers * 32) sums[i] = 0.0f;
          consumers_sync();
        }
      }
    }
  }
}

constexpr int kMaxDevices = 64;
std::atomic<bool> g_launched[kMaxDevices];  // devices whose status word a wait may have set

template <int NT>
size_t smem_bytes(const Layout& l, int stages, size_t extra) {
  return 1024 + (size_t)stages * stage_total(l) + kRoutingOffset + sizeof(Routing<NT>) + extra;
}

struct Weights {
  const void* up;
  const void* down;
};

int weight_map(CUtensorMap* map, const void* w, int64_t rows, int64_t k) {
  return make_tensor_map_2d(map, w, CU_TENSOR_MAP_DATA_TYPE_UINT8, (unsigned long long)k / 2, (unsigned long long)rows,
                            (unsigned long long)k / 2, 128, kTile, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
}

template <int FMT, int NT>
int launch(Params p, const Weights& w, int absent, cudaStream_t stream) {
  auto up = moe_fp4_up_kernel<FMT, NT>;
  auto down = moe_fp4_down_kernel<FMT, NT>;
  const int most_ctas = kCtasPerSm * sm_count_current(), ctas = most_ctas < kMaxCtas ? most_ctas : kMaxCtas;
  const size_t room = (size_t)113 * 1024;  // so that two fit an SM's 228 KB, 1 KB more each
  const size_t red = (size_t)4 * NT * 4 * 32 * 4, sums = (size_t)2 * p.tokens * kTile * 4;
  static thread_local int configured_device = -1;
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (configured_device != dev) {
    RB200_CUDA(cudaFuncSetAttribute(up, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    RB200_CUDA(cudaFuncSetAttribute(down, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
    configured_device = dev;
  }

  Layout l = layout<FMT, NT, true>();
  p.stages = kMaxStages;
  while (p.stages > 2 && smem_bytes<NT>(l, p.stages, red) > room) --p.stages;
  CUtensorMap map;
  if (weight_map(&map, w.up, (int64_t)p.experts * 2 * p.ffn, p.hidden) != 0) return -1;
  p.absent = absent;
  p.words = handover_words(stream, sm_count_current(), (size_t)ctas * part_words<NT>() * sizeof(uint32_t));
  p.wait_ns = (wait_limit_ms() ? (uint64_t)wait_limit_ms() : 2000ull) * 1000000ull;
  RB200_CUDA(launch_dependent(up, dim3((unsigned)ctas), kThreads, smem_bytes<NT>(l, p.stages, red), stream, p, map));

  l = layout<FMT, NT, false>();
  p.stages = kMaxStages;
  while (p.stages > 2 && smem_bytes<NT>(l, p.stages, sums) > room) --p.stages;
  if (weight_map(&map, w.down, (int64_t)p.experts * p.hidden, p.ffn) != 0) return -1;
  RB200_CUDA(launch_dependent(down, dim3((unsigned)ctas), kThreads, smem_bytes<NT>(l, p.stages, sums), stream, p, map));
  return 0;
}

template <int FMT>
int launch_fmt(const Params& p, const Weights& w, int absent, cudaStream_t stream) {
  // Entries of eight rows, or of sixteen where experts have more than eight on average: weights of an expert with more rows than
  // an entry are read again (by then from L2), rows that are not there take shared memory from the stages and clocks from the
  // products.  us with eight / sixteen: hidden 4096, ffn 14336, eight experts of top 2, mx, 9 tokens 130 / 180, 24 (6 rows on average)
  // 168 / 227, 32 (8) 206 / 245; ffn 1536, 16 experts of top 4, nv, 24 (6) 57 / 69, 32 (8) 74.3 / 76.0; hidden = ffn = 4096, four
  // experts of top 2, mx, 32 (16) 74.3 / 72.5.
  return p.tokens * p.top_k <= 8 * p.experts ? launch<FMT, 1>(p, w, absent, stream) : launch<FMT, 2>(p, w, absent, stream);
}

// [h | its exponents | parts | states | tickets]
struct Workspace {
  size_t exponents, parts, states, tickets, bytes;
};
Workspace workspace_of(int64_t tokens, int64_t top_k, int64_t hidden, int64_t ffn) {
  Workspace w;
  w.exponents = (size_t)((tokens * top_k * ffn * 2 + 255) / 256 * 256);
  w.parts = w.exponents + (size_t)((tokens * top_k * ((ffn + 15) / 16) + 255) / 256 * 256);
  w.states = w.parts + (size_t)kMaxCtas * 2 * tokens * kTile * 4;
  w.tickets = w.states + (size_t)kMaxCtas * 4;
  w.bytes = w.tickets + (size_t)((hidden + kTile - 1) / kTile) * 4;
  return w;
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

size_t rb200_moe_layer_fp4_workspace_bytes(int64_t tokens, int64_t top_k, int64_t hidden, int64_t ffn) {
  if (tokens <= 0 || top_k <= 0 || hidden <= 0 || ffn <= 0) return 0;
  return f4::workspace_of(tokens, top_k, hidden, ffn).bytes;
}

int rb200_moe_layer_fp4(const rb200_moe_layer_fp4_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  return rb200_moe_layer_fp4_selftest(d, workspace, workspace_bytes, -1, stream);
}

int rb200_moe_layer_fp4_selftest(const rb200_moe_layer_fp4_desc* d, void* workspace, size_t workspace_bytes, int absent, void* stream) {
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
  RB200_CHECK(d->hidden / 64 * d->tokens * d->top_k * ((d->ffn + 511) / 512) < (1ll << 30) && d->ffn / 64 * d->tokens * d->top_k * ((d->hidden + 255) / 256) < (1ll << 30),
              "the layer is too large (hidden=%lld, ffn=%lld)", (long long)d->hidden, (long long)d->ffn);
  RB200_CHECK(d->format == f4::kNv || (!d->gate_up_tensor_scale && !d->down_tensor_scale), "the mx format has no tensor scale");
  if (d->tokens == 0) return 0;
  RB200_CHECK(d->x && d->logits && d->w_gate_up && d->gate_up_scales && d->w_down && d->down_scales && d->out && workspace,
              "NULL argument");
  RB200_CHECK(f4::aligned16(d->x) && f4::aligned16(d->w_gate_up) && f4::aligned16(d->gate_up_scales) && f4::aligned16(d->w_down) &&
                  f4::aligned16(d->down_scales) && f4::aligned16(d->out) && f4::aligned16(workspace) &&
                  (reinterpret_cast<uintptr_t>(d->logits) & 3u) == 0,
              "tensors must be 16-byte aligned");
  RB200_CHECK(workspace_bytes >= rb200_moe_layer_fp4_workspace_bytes(d->tokens, d->top_k, d->hidden, d->ffn),
              "the workspace must hold rb200_moe_layer_fp4_workspace_bytes");
  f4::Params p;
  memset(&p, 0, sizeof(p));
  p.x = static_cast<const __half*>(d->x);
  p.logits = d->logits;
  p.s1 = static_cast<const uint8_t*>(d->gate_up_scales);
  p.s2 = static_cast<const uint8_t*>(d->down_scales);
  p.ts1 = d->gate_up_tensor_scale;
  p.ts2 = d->down_tensor_scale;
  const f4::Workspace ws = f4::workspace_of(d->tokens, d->top_k, d->hidden, d->ffn);
  p.h = static_cast<__half*>(workspace);
  p.exponents = reinterpret_cast<int8_t*>(static_cast<uint8_t*>(workspace) + ws.exponents);
  p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ws.parts);
  p.states = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + ws.states);
  p.tickets = reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(workspace) + ws.tickets);
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
  const f4::Weights w = {d->w_gate_up, d->w_down};
  int dev = 0;
  RB200_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < f4::kMaxDevices) f4::g_launched[dev].store(true, std::memory_order_relaxed);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return d->format == f4::kMx ? f4::launch_fmt<f4::kMx>(p, w, absent, s) : f4::launch_fmt<f4::kNv>(p, w, absent, s);
}

}  // extern "C"
