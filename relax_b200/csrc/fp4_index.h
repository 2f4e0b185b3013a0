// Index arithmetic of the 4-bit float products that host code can run as well.
#pragma once

#ifdef __CUDACC__
#define RB200_F4_HD __host__ __device__ __forceinline__
#else
#define RB200_F4_HD inline
#endif

namespace rb200 {
namespace f4 {

// Columns of the MMA of a tile that starts at row m0 of m: the rows that are left, at most `most`, in steps of 32.  (Bounded
// first: rounding up what is left of 2^31 - 1 rows would overflow.)
RB200_F4_HD int tile_width(int m, int m0, int most) {
  const int left = m - m0 < most ? m - m0 : most;
  return (left + 31) / 32 * 32;
}

}  // namespace f4
}  // namespace rb200
