// Host-visible launch of the product of two microscaled 4-bit operands.
#pragma once
#include "../../include/relax_b200.h"
#include "fp4.cuh"

namespace rb200 {
int fp4_gemm_launch(const rb200_gemm_fp4_desc& d, cudaStream_t stream);
}  // namespace rb200
