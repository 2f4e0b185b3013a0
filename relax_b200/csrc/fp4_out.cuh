// What the products of 4-bit floats do with their sums: scale, bias, activation, residual.
#pragma once

#include "../../include/relax_b200.h"
#include "fp4.cuh"

namespace rb200 {
namespace f4 {

struct Output {
  const float* a_ts;
  const float* w_ts;
  const void* bias;
  const void* residual;
  void* out;
  int64_t ldo, ld_res;
  int m, n;
  int act, binop, unop;
};
inline Output output_of(const rb200_gemm_fp4_desc& d) {
  Output o;
  o.a_ts = d.a_tensor_scale;
  o.w_ts = d.w_tensor_scale;
  o.bias = d.bias;
  o.residual = d.residual;
  o.out = d.out;
  o.ldo = d.ldo;
  o.ld_res = d.n;
  o.m = (int)d.m;
  o.n = (int)d.n;
  o.act = d.activation;
  o.binop = d.residual ? d.binary_op : RB200_BIN_NONE;
  o.unop = d.unary_op;
  return o;
}

#ifdef __CUDACC__
__device__ __forceinline__ float out_scale(const Output& o) { return (o.a_ts ? *o.a_ts : 1.0f) * (o.w_ts ? *o.w_ts : 1.0f); }

// v / (1 + exp(-v)) to 2^-20 of v; a quotient 1 / (1 + exp(-v)) below 2^-126 is taken as 0 (v < -87)
__device__ __forceinline__ float silu(float v) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(v * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return v * r;
}
// (a NaN stays one: it says that a block of an operand was not finite)
__device__ __forceinline__ float relu(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(0.0f));
  return r;
}
__device__ __forceinline__ float gelu(float v) { return 0.5f * v * (1.0f + erff(v * 0.70710678118654752f)); }

// unary(binary(act(alpha v + bias), x)) for R elements of a column (one bias) or of a row (R of them), x the residual's.
// The tests of what there is sit outside the loops over elements, and R is small: out of a cold instruction cache
// the instructions of 128 unrolled elements took five times as long to come as to run.
template <bool COLUMN, int R>
__device__ __forceinline__ void finish(const Output& o, float (&v)[R], float alpha, const float* bias, const float (&x)[R]) {
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = v[i] * alpha + bias[COLUMN ? 0 : i];
  if (o.act == RB200_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = relu(v[i]);
  } else if (o.act == RB200_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = silu(v[i]);
  } else if (o.act == RB200_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = gelu(v[i]);
  }
  if (o.residual) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = o.binop == RB200_BIN_MULTIPLY ? v[i] * x[i] : v[i] + x[i];
  }
  if (o.unop == RB200_UN_RELU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = relu(v[i]);
  }
}
__device__ __forceinline__ void prefetch_line(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory"); }
// R elements of the residual, of a column or of a row; past the matrix the last one's.  Nothing to branch on, so that all are
// on their way together.
template <class T, bool COLUMN, int R>
__device__ __forceinline__ void load_residual(const Output& o, float (&x)[R], int m, int n) {
  const T* r = static_cast<const T*>(o.residual);
#pragma unroll
  for (int i = 0; i < R; ++i) x[i] = widen(r[min(COLUMN ? m + i : m, o.m - 1) * o.ld_res + min(COLUMN ? n : n + i, o.n - 1)]);
}
// bias of column n
template <class T>
__device__ __forceinline__ float bias_at(const Output& o, int n) {
  return o.bias && n < o.n ? widen(static_cast<const T*>(o.bias)[n]) : 0.0f;
}
#endif  // __CUDACC__

}  // namespace f4
}  // namespace rb200
