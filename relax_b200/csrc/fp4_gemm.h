// Host-visible launch of the product of two microscaled 4-bit operands.
#pragma once
#include "../../include/relax_b200.h"
#include "fp4.cuh"

namespace rb200 {
int fp4_gemm_launch(const rb200_gemm_fp4_desc& d, cudaStream_t stream);
// The same by pairs of CTAs, for large batches; its status word, read and cleared.
int fp4_pair_launch(const rb200_gemm_fp4_desc& d, cudaStream_t stream);
int fp4_pair_read_status(int* v);
}  // namespace rb200
