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

// STREAM: non-temporal, for outputs that the L2s cannot hold (see streams()).
template <bool STREAM, class T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int count) {
  T out[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = static_cast<T>(v[i]);
  if (count >= 8) {
    elem_u32x4 part[sizeof(T) / 2];
    __builtin_memcpy(part, out, sizeof(part));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) {
      elem_u32x4_any* to = reinterpret_cast<elem_u32x4_any*>(reinterpret_cast<uint8_t*>(p) + 16 * i);
      if constexpr (STREAM)
        __builtin_nontemporal_store(part[i], to);
      else
        *to = part[i];
    }
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

// One step of a reduction over the wave: v joined with another lane's, by data
// parallel primitives, which take no LDS trip as a shuffle does (about 8 cycles
// against 60). Lanes that CTRL leaves out get `none`.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_lane(float none, float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none),
                                                               __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}

// f over the wave's lanes, in every lane: rows of 16 by shifts of 1, 2, 4 and 8,
// then row after row; lane 63 has all.
template <class F>
__device__ __forceinline__ float wave_reduce(float v, float none, F&& f) {
  v = f(v, dpp_lane<0x111, 0xf>(none, v));
  v = f(v, dpp_lane<0x112, 0xf>(none, v));
  v = f(v, dpp_lane<0x114, 0xf>(none, v));
  v = f(v, dpp_lane<0x118, 0xf>(none, v));
  v = f(v, dpp_lane<0x142, 0xa>(none, v));  // lane 15 of rows 0 and 2 to rows 1 and 3
  v = f(v, dpp_lane<0x143, 0xc>(none, v));  // lane 31 to rows 2 and 3
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

__device__ __forceinline__ float wave_add(float v) {
  return wave_reduce(v, 0.0f, [](float a, float b) { return a + b; });
}

// f over the lane's team of TEAM lanes (a wave's 64, or its row of 16), the same
// bits in every lane of the team: in a row, partners swap values (lanes 1 and 2
// apart, then mirrored ones of 8 and of 16), so that both join the same two.
template <int TEAM, class F>
__device__ __forceinline__ float team_reduce(float v, float none, F&& f) {
  static_assert(TEAM == 64 || TEAM == 16, "a wave or a row of it");
  if constexpr (TEAM == 64) return wave_reduce(v, none, f);
  v = f(v, dpp_lane<kQuadXor1, 0xf>(none, v));
  v = f(v, dpp_lane<kQuadXor2, 0xf>(none, v));
  v = f(v, dpp_lane<0x141, 0xf>(none, v));
  return f(v, dpp_lane<0x140, 0xf>(none, v));
}

template <int TEAM>
__device__ __forceinline__ float team_add(float v) {
  return team_reduce<TEAM>(v, 0.0f, [](float a, float b) { return a + b; });
}

template <int TEAM>
__device__ __forceinline__ float team_max(float v) {
  return team_reduce<TEAM>(v, -__builtin_inff(), [](float a, float b) { return fmaxf(a, b); });
}

// Host: bytes of one element of MB_DTYPE_*, 0 for another code.
inline uint32_t elem_bytes(int dtype) {
  return dtype == MB_DTYPE_F32 ? 4 : dtype == MB_DTYPE_F16 || dtype == MB_DTYPE_BF16 ? 2 : 0;
}

// Host: whether an output of so many bytes is stored non-temporally: past the 32
// MiB that the eight L2s hold together (combine of 8192x4 rows of 4096 bf16 58 us,
// so 49; smaller outputs stay where the next kernel finds them).
inline bool streams(uint64_t bytes) { return bytes > (32u << 20); }

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
