// Shared helpers of the kernels that work on a rank's attention heads: heads of 16-bit or fp32 elements in registers
// as fp32, and reductions over the lanes that share a row.
#pragma once

#include "common.hpp"

namespace iris_amd {

// N consecutive elements of type DT at `p`, which is aligned to all of them (N 1 to 4), as fp32.
template <int DT, int N>
__device__ inline void load_elems(const IRIS_GLOBAL char* p, float (&v)[N]) {
  static_assert(N == 1 || N == 4, "one element, or four");
  if constexpr (DT == IRIS_DTYPE_F32) {
    if constexpr (N == 4) {
      const f32x4 x = *(const IRIS_GLOBAL f32x4*)p;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = x[e];
    } else {
      v[0] = *(const IRIS_GLOBAL float*)p;
    }
  } else if constexpr (N == 4) {
    const u32x2 x = *(const IRIS_GLOBAL u32x2*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = from16<DT>((unsigned short)(x[e / 2] >> (16 * (e & 1))));
  } else {
    v[0] = from16<DT>(*(const IRIS_GLOBAL unsigned short*)p);
  }
}

template <int DT, int N>
__device__ inline void store_elems(IRIS_GLOBAL char* p, const float (&v)[N]) {
  static_assert(N == 1 || N == 4, "one element, or four");
  if constexpr (DT == IRIS_DTYPE_F32) {
    if constexpr (N == 4)
      *(IRIS_GLOBAL f32x4*)p = f32x4{v[0], v[1], v[2], v[3]};
    else
      *(IRIS_GLOBAL float*)p = v[0];
  } else if constexpr (N == 4) {
    *(IRIS_GLOBAL u32x2*)p = u32x2{pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3])};
  } else {
    *(IRIS_GLOBAL unsigned short*)p = to16<DT>(v[0]);
  }
}

// Sum over groups of `lanes` neighbouring lanes (a power of two up to 64), in every one of them; the same order for
// every lane, so that all hold the same bits.
template <int LANES, class T>
__device__ inline T sum_lanes(T x) {
#pragma unroll
  for (int m = 1; m < LANES; m *= 2) x += __shfl_xor(x, m, 64);
  return x;
}

// A position, slot or page of the caller's lies outside what it indexes (iris_amd.h, IRIS_STATUS_BAD_INDEX).
__device__ inline void report(uint32_t* status, uint32_t bits) {
  if (status) __hip_atomic_fetch_or(status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace iris_amd
