// What the attention kernels share: the paged cache's addresses, the keys that rows see, the parts of a split axis.
#pragma once

#include <type_traits>

#include "cache_codes.hpp"

namespace iris_amd {

struct AttentionKArgs {
  iris_attention_args a;
  PageDiv page;
  float scale_log2;   // scale * log2(e): scores are exponents of two
  int group;          // query heads to a key head
  int splits;         // parts of a unit's keys (prompts)
  int by_length;      // rows that see the most keys start first (prompts in tiles): row tiles that take one place a CU; 0: no order
  int grid_units;     // workgroups that share the work (decode)
  float* slots;       // partial results, `slot_elems` floats each
  int32_t* counters;  // arrivals at split units; zero between launches
};

// A cache in 8 bits has scales beside its codes.  CT: the codes' type, or 0 for a cache of the heads' own type.
struct QuantizedKArgs : AttentionKArgs {
  iris_cache_scales s;
  PageDiv block;
};
template <int CT>
using KArgs = std::conditional_t<CT == 0, AttentionKArgs, QuantizedKArgs>;

// The keys that the queries at positions first .. last see, as tiles of BT keys: `front` tiles that hold the first tokens (sinks),
// then tiles from `start` on; `count` in all.
struct KeyTiles {
  int front, start, count;
  int lo;  // the first key inside the window of the first query
  __device__ inline int tile(int j) const { return j < front ? j : start + j - front; }
};
template <int BT>
__device__ inline KeyTiles key_tiles(const iris_attention_args& a, int first, int last) {
  KeyTiles k{0, 0, 0, 0};
  if (last < 0) return k;
  const int end = last / BT + 1;
  if (a.window > 0) {
    k.lo = max(0, max(first, 0) - a.window + 1);
    const int sinks = min(a.sinks, k.lo);
    k.start = k.lo / BT;
    k.front = min((sinks + BT - 1) / BT, k.start);
  }
  k.count = k.front + end - k.start;
  return k;
}
// Does the query at position `at` see key `key`?  (window 0: all up to its own)
__device__ inline bool sees(const iris_attention_args& a, int at, int key) {
  return key <= at && (a.window <= 0 || at - key < a.window || key < a.sinks);
}

// sum + the two 16-bit weights of `w`: sums of the weights as they are multiplied, so that a row whose weight is one key's has that
// key's value and nothing of the weight's rounding.  (Subnormal fp16 weights count.)
template <int DT>
__device__ inline float add_weights(uint32_t w, float sum) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
  if constexpr (DT == IRIS_DTYPE_BF16)
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), bf16x2{(__bf16)1.f, (__bf16)1.f}, sum, false);
  else
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), f16x2{(_Float16)1.f, (_Float16)1.f}, sum, false);
}

// Word i of an array that no kernel writes while this one runs, by a scalar load (i is the wave's).
__device__ inline int scalar_at(const int32_t* p, int64_t i) { return ((const __attribute__((address_space(4))) int32_t*)p)[i]; }

}  // namespace iris_amd
