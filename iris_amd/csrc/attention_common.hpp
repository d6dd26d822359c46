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
  // Strides as 32 bits hold them (the launcher has seen to it), so that a product with a page's number is two scalar instructions.
  uint32_t k_page16, v_page16;  // of pages of codes, in 16 bytes
  uint32_t ks_page, vs_page, ks_block, vs_block;
  uint32_t block16;             // (block_of)
  int dealt;                    // row tiles in the order of dealt() (prompts in tiles)
};
// Where sixteen keys of a cache in 8 bits lie, `at` places into a page.
struct CodesAt {
  uint64_t k, v, k_scale, v_scale;  // bytes from a head's first codes and first scales
};
// at / block for places that are multiples of 16: with d = block / 16 and m = ceil(2^32 / d) - 1, floor((n + 1) m / 2^32) = floor(n / d)
// for (n + 1) d <= 2^32, which pages of up to 2^20 tokens leave.
__host__ inline uint32_t make_block16(uint32_t block) { return (uint32_t)(((1ull << 32) + block / 16 - 1) / (block / 16) - 1); }
__device__ inline uint32_t block_of(const QuantizedKArgs& g, int at) { return __umulhi((uint32_t)at / 16 + 1, g.block16); }
__device__ inline CodesAt codes_at(const QuantizedKArgs& g, int page, int at) {
  const uint32_t block = block_of(g, at);
  return {((uint64_t)(uint32_t)page * g.k_page16) * 16, ((uint64_t)(uint32_t)page * g.v_page16) * 16,
          (uint64_t)(uint32_t)page * g.ks_page + (uint64_t)block * g.ks_block, (uint64_t)(uint32_t)page * g.vs_page + (uint64_t)block * g.vs_block};
}
template <int CT>
using KArgs = std::conditional_t<CT == 0, AttentionKArgs, QuantizedKArgs>;

// A permutation of n items: 256 of them (and what is left, by powers of two) with their numbers' bits reversed.  Row tiles have room for each
// request's without a sum over the requests, which leaves every so many-th of them empty, every other one where requests have one each;
// and XCDs, and engines within them, get workgroups in turn, so that in the items' own order some of them would get all the empty ones.
// (512 requests with 128 rows each behind 8192 keys, heads of 128: 558 us, dealt 363; behind 2048 158 and 93.)
__host__ __device__ inline int dealt(int b, int n) {
  int first = b & ~255, left = n - first < 256 ? n - first : 256, bits = 31 - __builtin_clz(left);
  while (b - first >= 1 << bits) {
    first += 1 << bits;
    left -= 1 << bits;
    bits = 31 - __builtin_clz(left);
  }
  return bits ? first + (int)(__builtin_bitreverse32((uint32_t)(b - first)) >> (32 - bits)) : b;
}

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
