// Device side of MX quantisation: one group's scale and E2M1 codes.
#pragma once

#include "mb_elem.h"

namespace mb {

typedef __bf16 elem_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 elem_f16x2 __attribute__((ext_vector_type(2)));
typedef uint16_t elem_u16x2 __attribute__((ext_vector_type(2)));

// Scale byte S of a group whose largest magnitude has these fp32 bits: the
// exponent field less 2, at least 0; 255 for infinities and NaN.
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  const int field = static_cast<int>(largest >> 23);
  return field == 255 ? 255u : static_cast<uint32_t>(field > 2 ? field - 2 : 0);
}

// Largest magnitude so far, in a form that joins by `join` and that
// `magnitude_bits` turns into fp32 bits. 16-bit elements stay packed: without
// the sign their bits order like their magnitudes, NaN and infinities on top.
__device__ __forceinline__ uint32_t join_magnitudes(float, uint32_t a, uint32_t b) { return max(a, b); }
template <class T>
__device__ __forceinline__ uint32_t join_magnitudes(T, uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(elem_u16x2, a),
                                                                __builtin_bit_cast(elem_u16x2, b)));
}

template <class T>
__device__ __forceinline__ uint32_t raw_magnitude(const Raw8<T>& raw) {
  constexpr uint32_t kMask = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < static_cast<int>(2 * sizeof(T)); ++i)
    largest = join_magnitudes(T(), largest, raw.part[i / 4][i % 4] & kMask);
  return largest;
}

template <class T>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t largest) {
  if constexpr (sizeof(T) == 4) {
    return largest;
  } else {
    const uint16_t half = static_cast<uint16_t>(max(largest & 0xffffu, largest >> 16));
    const float value = widen(__builtin_bit_cast(T, half));
    return __builtin_bit_cast(uint32_t, value);
  }
}

// Eight elements as E2M1 codes under the scale S (0 for S = 255). The
// conversion divides by the power of two of its scale operand's exponent field
// (0 stands for 2^-127), rounds to nearest even and saturates at 6.
template <class T>
__device__ __forceinline__ uint32_t encode8(const Raw8<T>& raw, uint32_t scale) {
  const float by = __builtin_bit_cast(float, scale << 23);
  uint32_t word = 0;
  if constexpr (sizeof(T) == 4) {
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, raw[0], raw[1], by, 0);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, raw[2], raw[3], by, 1);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, raw[4], raw[5], by, 2);
    word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(word, raw[6], raw[7], by, 3);
  } else {
    const uint32_t w0 = raw.part[0][0], w1 = raw.part[0][1], w2 = raw.part[0][2], w3 = raw.part[0][3];
    if constexpr (__is_same(T, __bf16)) {
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(elem_bf16x2, w0), by, 0);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(elem_bf16x2, w1), by, 1);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(elem_bf16x2, w2), by, 2);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(word, __builtin_bit_cast(elem_bf16x2, w3), by, 3);
    } else {
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(elem_f16x2, w0), by, 0);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(elem_f16x2, w1), by, 1);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(elem_f16x2, w2), by, 2);
      word = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(word, __builtin_bit_cast(elem_f16x2, w3), by, 3);
    }
  }
  return scale == 255 ? 0 : word;
}

}  // namespace mb
