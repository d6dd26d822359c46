// Shared helpers of the kernels that work on a rank's attention heads: heads of 16-bit or fp32 elements in registers
// as fp32, and reductions over the lanes that share a row.
#pragma once

#include "common.hpp"

namespace iris_amd {

// Launches a kernel; its own status, whatever error an earlier call of the thread has left.
template <class Args>
inline hipError_t launch(void (*kernel)(Args), dim3 grid, int threads, size_t lds, void* stream, Args args) {
  void* const list[] = {&args};
  return hipLaunchKernel((const void*)kernel, grid, dim3(threads), const_cast<void**>(list), lds, (hipStream_t)stream);
}

// Division by the launch's page size for dividends below 2^31: with s = ceil(log2 d), m = ceil(2^(31 + s) / d) < 2^32 + 1 and
// m d - 2^(31 + s) < 2^s, so that floor(n m / 2^(31 + s)) = floor(n / d) for n < 2^31.
struct PageDiv {
  uint32_t d, shift;
  uint64_t m;
};
__host__ __device__ inline PageDiv make_page_div(uint32_t d) {
  PageDiv p{d, 31, 0};
  while ((1ull << (p.shift - 31)) < d) ++p.shift;
  p.m = ((1ull << p.shift) + d - 1) / d;
  return p;
}
__host__ __device__ inline uint32_t page_div(uint32_t n, const PageDiv& p) { return (uint32_t)(((uint64_t)n * p.m) >> p.shift); }

// N elements of type DT as they lie in memory (N 1 or 4), and as fp32.
template <int DT, int N>
struct Raw {
  static constexpr bool F32 = DT == IRIS_DTYPE_F32;
  static constexpr int WORDS = F32 ? N : (N + 1) / 2;
  uint32_t w[WORDS];
  __device__ inline void load(const IRIS_GLOBAL char* p) {
    if constexpr (WORDS == 4) {
      const u32x4 x = *(const IRIS_GLOBAL u32x4*)p;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = x[i];
    } else if constexpr (WORDS == 2) {
      const u32x2 x = *(const IRIS_GLOBAL u32x2*)p;
      w[0] = x[0], w[1] = x[1];
    } else if constexpr (F32) {
      w[0] = *(const IRIS_GLOBAL uint32_t*)p;
    } else {
      w[0] = *(const IRIS_GLOBAL unsigned short*)p;
    }
  }
  __device__ inline void store(IRIS_GLOBAL char* p) const {
    if constexpr (WORDS == 4)
      *(IRIS_GLOBAL u32x4*)p = u32x4{w[0], w[1], w[2], w[3]};
    else if constexpr (WORDS == 2)
      *(IRIS_GLOBAL u32x2*)p = u32x2{w[0], w[1]};
    else if constexpr (F32)
      *(IRIS_GLOBAL uint32_t*)p = w[0];
    else
      *(IRIS_GLOBAL unsigned short*)p = (unsigned short)w[0];
  }
  __device__ inline void get(float (&v)[N]) const {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if constexpr (F32)
        v[e] = __builtin_bit_cast(float, w[e]);
      else
        v[e] = from16<DT>((unsigned short)(w[e / 2] >> (16 * (e & 1))));
    }
  }
  __device__ inline void set(const float (&v)[N]) {
    if constexpr (F32) {
#pragma unroll
      for (int e = 0; e < N; ++e) w[e] = __builtin_bit_cast(uint32_t, v[e]);
    } else if constexpr (N == 4) {
      w[0] = pack2<DT>(v[0], v[1]), w[1] = pack2<DT>(v[2], v[3]);
    } else {
      w[0] = to16<DT>(v[0]);
    }
  }
};

// A lane's value from the lane that CTRL (a DPP permutation within 16 lanes) names: a VALU operand, where a shuffle would go through LDS.
template <int CTRL>
__device__ inline float permuted(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
// op over the lanes 16 (32) apart, in each of them.
template <class Op>
__device__ inline float over_16(float x, Op op) {
  const auto r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return op(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
template <class Op>
__device__ inline float over_32(float x, Op op) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
  return op(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// op over groups of LANES neighbouring lanes (8, 16, 32 or 64), the same bits in all of them: neighbours, pairs, from four equal
// lanes on mirror images, and rows and halves of the wave that change places between two copies.
template <int LANES, class Op>
__device__ inline float over_lanes(float x, Op op) {
  constexpr int NEIGHBOURS = 0xB1, PAIRS = 0x4E, MIRROR_8 = 0x141, MIRROR_16 = 0x140;  // quad_perm [1,0,3,2], [2,3,0,1]; row_half_mirror, row_mirror
  x = op(x, permuted<NEIGHBOURS>(x));
  x = op(x, permuted<PAIRS>(x));
  x = op(x, permuted<MIRROR_8>(x));
  if constexpr (LANES >= 16) x = op(x, permuted<MIRROR_16>(x));
  if constexpr (LANES >= 32) x = over_16(x, op);
  if constexpr (LANES >= 64) x = over_32(x, op);
  return x;
}
struct Larger {
  __device__ inline float operator()(float x, float y) const { return fmaxf(x, y); }
};
struct Sum {
  template <class T>
  __device__ inline T operator()(T x, T y) const {
    return x + y;
  }
};
template <int LANES>
__device__ inline float sum_lanes(float x) {
  return over_lanes<LANES>(x, Sum{});
}
template <int LANES>
__device__ inline double sum_lanes(double x) {
  static_assert(LANES == 64, "as single pairs are laid out");
#pragma unroll
  for (int m = 1; m < 64; m *= 2) x += __shfl_xor(x, m, 64);
  return x;
}

// A position, slot or page of the caller's lies outside what it indexes (iris_amd.h, IRIS_STATUS_BAD_INDEX).
__device__ inline void report(uint32_t* status, uint32_t bits) {
  if (status) __hip_atomic_fetch_or(status, bits, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace iris_amd
