// Host-visible launches of the 4-bit float quantiser.
#pragma once
#include "fp4.cuh"

namespace rb200 {
// x [batch][rows][k] (rows ldx elements apart, batches batch_stride) -> codes and tiled scales.  `activations`: the result
// is read by the next kernel as activations are, after its wait for this one, so that kernel may start early.
int fp4_encode_launch(const void* x, int dtype, int64_t batch, int64_t rows, int64_t k, int64_t ldx, int64_t batch_stride, int fmt,
                      const float* tensor_scale, void* codes, void* scales, bool activations, cudaStream_t stream);
}  // namespace rb200
