// Device side of FP8 quantisation with block scales: a block's scale, E4M3 codes,
// and the gate of a feed-forward block.
#pragma once

#include "mb_elem.h"
#include "mb_mx_device.h"

namespace mb {

typedef int16_t elem_s16x2 __attribute__((ext_vector_type(2)));

// Scale byte S = e + 127 of a block whose largest magnitude has these fp32 bits: the
// smallest e with max <= 448 * 2^e, at least -127; 255 for infinities and NaN. 448 is
// 1.75 * 2^8, so a mantissa past 0x600000 carries into the exponent field.
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t largest) {
  const int field = static_cast<int>((largest + 0x1fffffu) >> 23);
  return largest >= 0x7f800000u ? 255u : static_cast<uint32_t>(field > 8 ? field - 8 : 0);
}

// Two elements as E4M3 codes under the scale operand `by` = S << 23: the conversion
// divides by the power of two of its exponent field (0 stands for 2^-127) and rounds
// to nearest even. No quotient passes 448, and a power of two makes it exact, so that
// this is the only rounding.
template <bool HIGH>
__device__ __forceinline__ elem_s16x2 fp8_pair(elem_s16x2 word, float a, float b, float by) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(word, a, b, by, HIGH);
}
template <bool HIGH>
__device__ __forceinline__ elem_s16x2 fp8_pair(elem_s16x2 word, __bf16, uint32_t both, float by) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(word, __builtin_bit_cast(elem_bf16x2, both), by, HIGH);
}
template <bool HIGH>
__device__ __forceinline__ elem_s16x2 fp8_pair(elem_s16x2 word, _Float16, uint32_t both, float by) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(word, __builtin_bit_cast(elem_f16x2, both), by, HIGH);
}

// Four elements as the bytes of a dword; 0 under the scale 255.
__device__ __forceinline__ uint32_t fp8_encode4(float a, float b, float c, float d, uint32_t scale) {
  const float by = __builtin_bit_cast(float, scale << 23);
  elem_s16x2 word = {0, 0};
  word = fp8_pair<false>(word, a, b, by);
  word = fp8_pair<true>(word, c, d, by);
  return scale == 255 ? 0 : __builtin_bit_cast(uint32_t, word);
}

// Eight elements, as they are stored, as two dwords of codes.
template <class T>
__device__ __forceinline__ elem_u32x2 fp8_encode8(const Raw8<T>& raw, uint32_t scale) {
  if constexpr (sizeof(T) == 4) {
    return elem_u32x2{fp8_encode4(raw[0], raw[1], raw[2], raw[3], scale),
                      fp8_encode4(raw[4], raw[5], raw[6], raw[7], scale)};
  } else {
    const float by = __builtin_bit_cast(float, scale << 23);
    elem_u32x2 out;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t low = raw.part[0][2 * h], high = raw.part[0][2 * h + 1];
      elem_s16x2 word = {0, 0};
      word = fp8_pair<false>(word, T(), low, by);
      word = fp8_pair<true>(word, T(), high, by);
      out[h] = scale == 255 ? 0 : __builtin_bit_cast(uint32_t, word);
    }
    return out;
  }
}

// Largest magnitude over the 16 lanes of a row of the wave, in the form of
// join_magnitudes, in all of them.
template <class T>
__device__ __forceinline__ uint32_t row16_magnitude(uint32_t v) {
  v = join_magnitudes(T(), v, quad_swap<kQuadXor1>(v));
  v = join_magnitudes(T(), v, quad_swap<kQuadXor2>(v));
  v = join_magnitudes(T(), v, quad_swap<0x141>(v));  // mirrored in 8 lanes
  return join_magnitudes(T(), v, quad_swap<0x140>(v));  // and in 16
}

__device__ __forceinline__ uint32_t float_bits(float v) { return __builtin_bit_cast(uint32_t, v); }

// Largest magnitude of eight fp32 values, as bits (which order like magnitudes, NaN
// and infinities on top).
__device__ __forceinline__ uint32_t float8_magnitude(const float (&v)[8]) {
  uint32_t largest = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) largest = max(largest, float_bits(v[i]) & 0x7fffffffu);
  return largest;
}

// 1 / (1 + e^-g) and its complement, each to a few units of fp32's last place: the
// power is taken of -|g|, so that neither is a difference, and g log2(e) in two parts,
// so that a large |g| costs the power no bits. Both are of positive terms; below
// 2^-126 (|g| over 87.3) the smaller one is 0.
struct Sigmoid {
  float value, complement;
};
__device__ __forceinline__ Sigmoid sigmoid(float g) {
  constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147182f;
  const float size = fmaxf(-fabsf(g), -128.0f);  // no infinity meets another
  const float high = size * kLog2e;
  const float low = fmaf(size, kLog2e, -high) + size * kLog2eRest;
  const float power = __builtin_amdgcn_exp2f(high);
  const float e = fmaf(power, low * kLn2, power);
  const float r = __builtin_amdgcn_rcpf(1.0f + e);
  return g >= 0 ? Sigmoid{r, e * r} : Sigmoid{e * r, r};
}

// silu(gate) * up.
__device__ __forceinline__ float gated(float gate, float up) { return gate * sigmoid(gate).value * up; }

}  // namespace mb
