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

// unary(binary(act(alpha v + bias[n]), residual)) for rows m .. m + R - 1 of column n; rows and columns past the matrix are
// left without it.  The tests of what there is sit outside the loops over elements.
template <class T, int R>
__device__ __forceinline__ void finish_column(const Output& o, float* v, float alpha, int m, int n) {
  const bool there = n < o.n;
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] *= alpha;
  if (o.bias) {
    const float b = there ? widen(static_cast<const T*>(o.bias)[n]) : 0.0f;
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] += b;
  }
  if (o.act == RB200_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = fmaxf(v[i], 0.0f);
  } else if (o.act == RB200_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = v[i] / (1.0f + __expf(-v[i]));
  } else if (o.act == RB200_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = 0.5f * v[i] * (1.0f + erff(v[i] * 0.70710678118654752f));
  }
  if (o.residual) {
    const T* r = static_cast<const T*>(o.residual) + m * o.ld_res + n;
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (there && m + i < o.m) {
        const float x = widen(r[i * o.ld_res]);
        v[i] = o.binop == RB200_BIN_MULTIPLY ? v[i] * x : v[i] + x;
      }
  }
  if (o.unop == RB200_UN_RELU) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] = fmaxf(v[i], 0.0f);
  }
}
// the same for one element
template <class T>
__device__ __forceinline__ float finish(const Output& o, float v, float alpha, int m, int n) {
  finish_column<T, 1>(o, &v, alpha, m, n);
  return v;
}
#endif  // __CUDACC__

}  // namespace f4
}  // namespace rb200
