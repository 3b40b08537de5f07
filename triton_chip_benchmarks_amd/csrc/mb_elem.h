// Element types of the layer operators (MX quantisation, linear, routing,
// combine): loads to and stores from fp32 registers, eight elements a lane, at
// any element alignment.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mb_internal.h"

namespace mb {

typedef uint32_t elem_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t elem_u32x2 __attribute__((ext_vector_type(2)));
// 16 bytes at any element's address: gfx950 takes a global_load_dwordx4 there.
typedef elem_u32x4 elem_u32x4_any __attribute__((aligned(2)));

// fp32 value of one stored element, and back (round to nearest even).
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return static_cast<float>(v); }
__device__ __forceinline__ float widen(__bf16 v) { return static_cast<float>(v); }

// Eight consecutive elements as they are stored.
template <class T>
struct Raw8 {
  elem_u32x4 part[sizeof(T) / 2];  // one 16-byte vector of 16-bit elements, two of fp32

  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
      part[i] = *reinterpret_cast<const elem_u32x4_any*>(reinterpret_cast<const uint8_t*>(p) + 16 * i);
  }
  // The first `count` of them; the rest zero.
  __device__ __forceinline__ void load(const T* p, int count) {
    if (count >= 8) {
      load(p);
      return;
    }
    T v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < count ? p[i] : T(0);
    __builtin_memcpy(part, v, sizeof(part));
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) part[i] = elem_u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ float operator[](int i) const {
    if constexpr (sizeof(T) == 4) {
      const uint32_t word = part[i / 4][i % 4];  // __builtin_bit_cast of the element itself takes element 0
      return __builtin_bit_cast(float, word);
    } else {
      const uint32_t word = part[0][i / 2];
      const uint16_t half = static_cast<uint16_t>(i % 2 ? word >> 16 : word);
      return widen(__builtin_bit_cast(T, half));
    }
  }
};

template <class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int count) {
  T out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = static_cast<T>(v[i]);
  if (count >= 8) {
    elem_u32x4 part[sizeof(T) / 2];
    __builtin_memcpy(part, out, sizeof(part));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i)
      *reinterpret_cast<elem_u32x4_any*>(reinterpret_cast<uint8_t*>(p) + 16 * i) = part[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < count) p[i] = out[i];
  }
}

// Value of another lane of the same quad: lanes 1,0,3,2 or 2,3,0,1.
template <int PERM>
__device__ __forceinline__ uint32_t quad_swap(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), PERM, 0xf, 0xf, true));
}
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E;

__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, 64);
  return v;
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v = fmaxf(v, __shfl_xor(v, offset, 64));
  return v;
}

// Host: bytes of one element of MB_DTYPE_*, 0 for another code.
inline uint32_t elem_bytes(int dtype) {
  return dtype == MB_DTYPE_F32 ? 4 : dtype == MB_DTYPE_F16 || dtype == MB_DTYPE_BF16 ? 2 : 0;
}

// Host: bytes that `rows` rows of `k` elements span at a row stride (elements).
inline uint64_t strided_bytes(uint64_t rows, uint64_t k, uint64_t row_stride, uint32_t item) {
  return rows && k ? ((rows - 1) * row_stride + k) * item : 0;
}

}  // namespace mb

// call(T{}) for the element type of `dtype`.
#define MB_FOR_DTYPE(dtype, call)          \
  do {                                     \
    if ((dtype) == MB_DTYPE_F32) {         \
      using T = float;                     \
      call;                                \
    } else if ((dtype) == MB_DTYPE_F16) {  \
      using T = _Float16;                  \
      call;                                \
    } else {                               \
      using T = __bf16;                    \
      call;                                \
    }                                      \
  } while (0)
