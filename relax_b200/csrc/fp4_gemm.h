// Host-visible launch of the product of two microscaled 4-bit operands.
#pragma once
#include "../../include/relax_b200.h"
#include "fp4.cuh"

namespace rb200 {
// x not NULL (at most four rows, of out's type): `a` is x, quantised in the kernel.
int fp4_gemm_launch(const rb200_gemm_fp4_desc& d, const void* x, int64_t ldx, cudaStream_t stream);
// The same by pairs of CTAs, for large batches; its status word, read and cleared.
int fp4_pair_launch(const rb200_gemm_fp4_desc& d, cudaStream_t stream);
int fp4_pair_read_status(int* v);
}  // namespace rb200
