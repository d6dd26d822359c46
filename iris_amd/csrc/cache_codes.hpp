// The numbers of a cache in 8 bits: codes (8-bit floats, CT: IRIS_DTYPE_E4M3 or _E5M2) and the powers of two that scale a block of
// tokens of a head.  A code times a power of two has no more places than the code, so that fp32, bf16 and (in its range) fp16
// hold it as it is, and the conversion's own scale operand multiplies for nothing.
#pragma once

#include "heads_common.hpp"

namespace iris_amd {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// The largest code is 0.875 * 2^TOP.  A code with these bits (or, E5M2, more) beside its sign is no finite number.
template <int CT>
struct Codes {
  static constexpr bool E4M3 = CT == IRIS_DTYPE_E4M3;
  static constexpr int TOP = E4M3 ? 9 : 16;
  static constexpr uint32_t NOT_FINITE = E4M3 ? 0x7F : 0x7C;
};
constexpr int MAX_CODES_PAGE = 1 << 20;  // tokens of a page
constexpr int SCALE_ONE = 127, SCALE_NAN = 255;  // a scale's byte x is 2^(x - 127)
constexpr int SCALE_LEAST = SCALE_ONE - 100;     // of a block that is written: codes times it are ordinary fp32 numbers
constexpr uint32_t NAN_CODES = 0x7F7F7F7Fu;      // (of both kinds)

__device__ inline float scale_of(int byte) { return __builtin_bit_cast(float, byte << 23); }

// The scale byte at p; the same for the whole wave where p is.
__device__ inline uint32_t scale_byte(const uint8_t* p) { return *(const IRIS_GLOBAL uint8_t*)p; }

// Two codes of w (HI: its upper half) times a power of two, as numbers of type DT in a word.
template <int CT, int DT, bool HI>
__device__ inline uint32_t decode2(uint32_t w, float scale) {
  if constexpr (DT == IRIS_DTYPE_BF16) {
    if constexpr (Codes<CT>::E4M3)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, scale, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(w, scale, HI));
  } else {
    static_assert(DT == IRIS_DTYPE_F16);
    if constexpr (Codes<CT>::E4M3)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_bf8(w, scale, HI));
  }
}
// ... as fp32 numbers.
template <int CT, bool HI>
__device__ inline f32x2 decode2_f32(uint32_t w, float scale) {
  if constexpr (Codes<CT>::E4M3)
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(w, scale, HI);
  else
    return __builtin_amdgcn_cvt_scalef32_pk_f32_bf8(w, scale, HI);
}
template <int CT>
__device__ inline f32x4 decode4_f32(uint32_t w, float scale) {
  const f32x2 lo = decode2_f32<CT, false>(w, scale), hi = decode2_f32<CT, true>(w, scale);
  return f32x4{lo[0], lo[1], hi[0], hi[1]};
}

// Numbers over a power of two, rounded to codes: two of type DT in a word (fp32: two words), into the lower or upper half of `into`.
typedef short s16x2 __attribute__((ext_vector_type(2)));
template <int CT, bool HI>
__device__ inline uint32_t encode2_f32(uint32_t into, float a, float b, float scale) {
  const s16x2 old = __builtin_bit_cast(s16x2, into);
  if constexpr (Codes<CT>::E4M3)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(old, a, b, scale, HI));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(old, a, b, scale, HI));
}
template <int CT, int DT, bool HI>
__device__ inline uint32_t encode2(uint32_t into, uint32_t x, float scale) {
  const s16x2 old = __builtin_bit_cast(s16x2, into);
  if constexpr (DT == IRIS_DTYPE_BF16) {
    if constexpr (Codes<CT>::E4M3)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(old, __builtin_bit_cast(bf16x2, x), scale, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf8_bf16(old, __builtin_bit_cast(bf16x2, x), scale, HI));
  } else {
    static_assert(DT == IRIS_DTYPE_F16);
    if constexpr (Codes<CT>::E4M3)
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(old, __builtin_bit_cast(f16x2, x), scale, HI));
    else
      return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf8_f16(old, __builtin_bit_cast(f16x2, x), scale, HI));
  }
}

}  // namespace iris_amd
