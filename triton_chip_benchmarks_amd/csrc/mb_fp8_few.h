// Products of FP8 operands for few rows: the weight goes from memory into the
// registers of the matrix instructions, and nothing of it through LDS.
#pragma once

#include <type_traits>

#include "mb_fp8_device.h"
#include "mb_mx_stream.h"

namespace mb {

// Expert and rows of a workgroup's blockIdx.y; false where it has none. With
// fewer rows than experts there is one grid row a row of X, and the first row of
// an expert stands for all of them; its expert is the number of those that end
// at or before it.
__device__ __forceinline__ bool fp8_few_expert(const int32_t* __restrict__ offsets, int experts, int rows, int lane,
                                               int& e, int& first, int& last) {
  e = 0;
  if (offsets) {
    e = blockIdx.y;
    if (rows < experts) {
      int ended = 0;
      for (int base = 0; base < experts; base += 64)
        ended += __builtin_popcountll(__ballot(base + lane < experts && offsets[min(base + lane, experts - 1) + 1] <=
                                                                            static_cast<int>(blockIdx.y)));
      e = ended;
      if (e >= experts || offsets[e] != static_cast<int>(blockIdx.y)) return false;
    }
  }
  expert_rows(offsets, e, rows, first, last);
  return first < last;
}

// What becomes of the sums: the product in Y's type, silu(gate) * up in Y's type (with
// the gate and up themselves, if wanted), or silu(gate) * up as an FP8 operand.
enum Fp8Epilogue { kFp8Plain, kFp8Gated, kFp8GatedFp8 };

// A product's arguments: X [rows] (or [tokens], gathered by `order`) of K = k elements,
// W of experts * (n or, gated, 2n: the gates', then the ups') rows. A scale stands for
// 1 << shift rows.
struct Fp8Product {
  const void* x;
  uint64_t row_stride;  // elements; of an operand, its pitch
  const uint8_t* sx;    // NULL: X is of the output's type, or fp32, fp16 or bf16 anyway
  int x_shift;
  const uint8_t *w, *sw;
  int w_shift;
  void* y;
  uint8_t* sy;
  void* gate_up;
  int rows, n, k;
  const int32_t *offsets, *order;
  int copies, tokens, experts;
};

constexpr int kFp8FewRows = 16;
// Waves of a workgroup, and the workgroups of which a CU's registers hold the waves.
constexpr int fp8_few_waves(int split) { return split == 4 ? 4 : 8; }
constexpr int fp8_few_resident(int fb, int split) { return (fb == 1 ? 16 : 12) / fp8_few_waves(split); }

// LDS of the quantised rows: a row's codes, then a row's scales, each row a bank
// group past the one before. Pairs of blocks: a turn of the kernel takes two.
constexpr uint32_t fp8_staged_blocks(uint32_t k) { return (k + 255) / 256 * 2; }
constexpr uint32_t fp8_code_stride(uint32_t k) { return fp8_staged_blocks(k) * 128 + 16; }
constexpr uint32_t fp8_scale_stride(uint32_t k) { return fp8_staged_blocks(k) + 2; }
constexpr uint64_t fp8_few_lds(uint32_t k, uint32_t rows) {
  return uint64_t{rows} * (fp8_code_stride(k) + fp8_scale_stride(k));
}
constexpr uint64_t fp8_few_parts(int waves, int width) { return uint64_t{1} * waves * kFp8FewRows * (width + 1) * 4; }

// A lane's 32 codes of a block of K and the dword with its scale.
//
// Outputs of 16 bits take v_mfma_scale_f32_16x16x128_f8f6f4, which adds products eight
// at a time, each cut toward zero 13 bits below the power of two of the largest one's
// exponents, and goes on in fp32: 7 * 2^-13 of the products' magnitudes at worst, 2^-16
// to 2^-14 of the result, by its 2-norm, for normal values to values over ten binades:
// under a hundredth of the output's own rounding, at twice the rate. Outputs of fp32
// take the codes to bf16, with the scale, which is exact (from 2^-126 on), and
// v_mfma_f32_16x16x32_bf16, whose sums are of fp32, at half the rate.
struct Fp8Codes {
  i32x4 at[2];
};
struct Fp8Wide {
  bf16x8 at[4];
};

__device__ __forceinline__ Fp8Wide fp8_widen(const Fp8Codes& codes, uint32_t scale) {
  const float by = __builtin_bit_cast(float, (scale & 0xff) << 23);
  Fp8Wide wide;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    elem_bf16x2 pair[4];
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint32_t word = static_cast<uint32_t>(codes.at[g / 2][g % 2 * 2 + w]);
      pair[2 * w] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, by, false);
      pair[2 * w + 1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, by, true);
    }
    __builtin_memcpy(&wide.at[g], pair, sizeof(pair));
  }
  return wide;
}

// Operands of the matrix instructions for sums of type Y; SEL is the scale's byte.
template <bool WIDE, int SEL>
struct Fp8Fragment {
  Fp8Codes codes;
  uint32_t scale;
  __device__ __forceinline__ Fp8Fragment(const Fp8Codes& c, uint32_t s) : codes(c), scale(s) {}
};
template <int SEL>
struct Fp8Fragment<true, SEL> {
  Fp8Wide wide;
  __device__ __forceinline__ Fp8Fragment(const Fp8Codes& c, uint32_t s) : wide(fp8_widen(c, s >> (8 * SEL))) {}
};

template <int SEL>
__device__ __forceinline__ f32x4 fp8_mma16(const Fp8Fragment<false, SEL>& a, const Fp8Fragment<false, SEL>& b,
                                           f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
      __builtin_shufflevector(a.codes.at[0], a.codes.at[1], 0, 1, 2, 3, 4, 5, 6, 7),
      __builtin_shufflevector(b.codes.at[0], b.codes.at[1], 0, 1, 2, 3, 4, 5, 6, 7), c, 0, 0, SEL,
      static_cast<int>(a.scale), SEL, static_cast<int>(b.scale));
}
template <int SEL>
__device__ __forceinline__ f32x4 fp8_mma16(const Fp8Fragment<true, SEL>& a, const Fp8Fragment<true, SEL>& b,
                                           f32x4 c) {
#pragma unroll
  for (int g = 0; g < 4; ++g)
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.wide.at[g], b.wide.at[g], c, 0, 0, 0);
  return c;
}

// A workgroup takes up to 16 rows at a time (of one expert) and TILES tiles of
// FB * 16 rows of W (gated: 16 of the gates' and the same 16 of the ups' each two),
// SPLIT waves sharing a tile's K in turns of 256 elements; they add their parts in LDS
// in a fixed order. X is of fp32, fp16 or bf16, quantised into LDS on the way, or
// (uint8_t) an operand, read where it is. W's rows are the instruction's rows, X's its
// columns: a lane holds 32 bytes of K of a row of each, and four neighbouring features
// of one row of the output.
//
// Reading the weights bounds it, so the next turn's are in flight while one's are
// multiplied (132 to 152 registers with two fragments of W, 12 waves a CU). Workgroups of
// four waves fill those where one of eight leaves four out: the gated pair of 14336 x 4096
// takes 16 rows in 27.5 us and not 31, 64 tokens of eight of 128 experts of 2048 x 2048
// 170 and not 194 (6.3 TB/s). A SPLIT of eight is for as few columns as leave CUs without
// a workgroup, where a wave's turns one after the other are the time: one row of 8192 by
// 2048 columns takes 7.7 us, by four 10.4. With X's codes or a third turn in flight as
// well, a CU holds half the waves, at 1.1 to 1.3 times the time.
template <class X, class Y, int EPILOGUE, int FB, int SPLIT>
__global__ void __launch_bounds__(64 * fp8_few_waves(SPLIT)) fp8_few_kernel(Fp8Product p, int lds_rows) {
#if defined(__HIP_DEVICE_COMPILE__)
  constexpr bool GATED = EPILOGUE != kFp8Plain, STAGED = sizeof(X) > 1, WIDE = sizeof(Y) == 4;
  constexpr int WAVES = fp8_few_waves(SPLIT), ROWS = kFp8FewRows, TILES = WAVES / SPLIT, WIDTH = FB * 16;
  constexpr int COLUMNS = GATED ? WIDTH / 2 : WIDTH;
  static_assert(!GATED || FB % 2 == 0, "pairs");
  static_assert(EPILOGUE != kFp8GatedFp8 || TILES * COLUMNS == 128, "a workgroup holds whole blocks of the output");
  // The staged rows, and then, in their place, the waves' sums: two workgroups of 16
  // rows of K = 4096 fit a CU.
  extern __shared__ __attribute__((aligned(16))) uint8_t staged[];
  float(*const parts)[ROWS][WIDTH + 1] = reinterpret_cast<float(*)[ROWS][WIDTH + 1]>(staged);
  const int lane = threadIdx.x & 63, part = lane >> 4, l16 = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int e, first, last;
  if (!fp8_few_expert(p.offsets, p.experts, p.rows, lane, e, first, last)) return;
  const int n = p.n, k = p.k, width = GATED ? 2 * n : n;
  const int n0 = (blockIdx.x * TILES + wave / SPLIT) * COLUMNS, turn0 = wave % SPLIT;
  const int blocks = (k + 127) / 128, pitch = (k + 15) / 16 * 16, steps = (k + 511) / 512;
  const int turns = ((blocks + 1) / 2 - turn0 + SPLIT - 1) / SPLIT;
  const int w_scales = (width + (1 << p.w_shift) - 1) >> p.w_shift;
  const int x_scales = (p.rows + (1 << p.x_shift) - 1) >> p.x_shift;
  const int code_stride = fp8_code_stride(k), scale_stride = fp8_scale_stride(k);
  uint8_t* const staged_scales = staged + lds_rows * code_stride;
  const uint8_t* wr[FB];
  const uint8_t* swr[FB];
#pragma unroll
  for (int f = 0; f < FB; ++f) {
    const int feature = min(n0 + (GATED ? f / 2 : f) * 16 + l16, n - 1) + (GATED && f % 2 ? n : 0);
    wr[f] = p.w + (int64_t{e} * width + feature) * pitch;
    swr[f] = p.sw + (int64_t{e} * steps * w_scales + (feature >> p.w_shift)) * 4;
  }
  struct Unit {
    Fp8Codes w[FB][2];
    uint32_t s[FB];
  };
  auto load = [&](Unit& unit, int turn) __attribute__((always_inline)) {
    const int b = (turn0 + turn * SPLIT) * 2;
#pragma unroll
    for (int f = 0; f < FB; ++f) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int q = 0; q < 2; ++q)
          unit.w[f][h].at[q] =
              *reinterpret_cast<const i32x4*>(wr[f] + min((b + h) * 128 + part * 32 + q * 16, pitch - 16));
      unit.s[f] = *reinterpret_cast<const uint16_t*>(swr[f] + (int64_t{b >> 2} * w_scales * 4 + (b & 3)));
    }
  };
  for (int m0 = first + static_cast<int>(blockIdx.z) * ROWS; m0 < last; m0 += static_cast<int>(gridDim.z) * ROWS) {
    Unit unit;
    if (turns > 0) load(unit, 0);  // in flight while the rows are quantised
    const int live = min(ROWS, last - m0);
    if constexpr (STAGED) {
      // A wave takes 512 elements of a row at a time, BATCH of them in flight, so that
      // rows and places are the wave's and cost its lanes nothing: quantisation is bound
      // by instructions here, since every workgroup of the launch does it anew.
      constexpr int BATCH = 2;
      const int chunks = (k + 511) / 512, all = fp8_staged_blocks(k);
      int row = 0, chunk = wave;
      auto settle = [&]() __attribute__((always_inline)) {
        while (chunk >= chunks) {
          chunk -= chunks;
          ++row;
        }
      };
      settle();
      while (row < live) {
        Raw8<X> raw[BATCH];
        int rows_at[BATCH], chunk_at[BATCH];
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          rows_at[u] = row;
          chunk_at[u] = chunk;
          if (row < live) {
            int token = m0 + row;
            if (p.order) token = max(0, min(p.order[token] / p.copies, p.tokens - 1));
            const X* from = static_cast<const X*>(p.x) + static_cast<uint64_t>(token) * p.row_stride + chunk * 512;
            if ((chunk + 1) * 512 <= k)
              raw[u].load(from + lane * 8);
            else
              raw[u].load(from + lane * 8, k - chunk * 512 - lane * 8);
          }
          chunk += WAVES;
          settle();
        }
#pragma unroll
        for (int u = 0; u < BATCH; ++u) {
          if (rows_at[u] >= live) break;
          const uint32_t scale = fp8_scale_byte(magnitude_bits<X>(row16_magnitude<X>(raw_magnitude(raw[u]))));
          const int block = chunk_at[u] * 4 + lane / 16;
          if (block < all) {
            *reinterpret_cast<elem_u32x2*>(staged + rows_at[u] * code_stride + chunk_at[u] * 512 + lane * 8) =
                fp8_encode8(raw[u], scale);
            if (lane % 16 == 0) staged_scales[rows_at[u] * scale_stride + block] = static_cast<uint8_t>(scale);
          }
        }
      }
      __syncthreads();
    }
    const int mine = min(l16, live - 1);
    const uint8_t *xc, *xs;
    if constexpr (STAGED) {
      xc = staged + mine * code_stride + part * 32;
      xs = staged_scales + mine * scale_stride;
    } else {
      xc = static_cast<const uint8_t*>(p.x) + static_cast<int64_t>(m0 + mine) * pitch + part * 32;
      xs = p.sx + static_cast<int64_t>((m0 + mine) >> p.x_shift) * 4;
    }
    f32x4 acc[FB] = {};
    auto multiply = [&](const Unit& unit, int turn) __attribute__((always_inline)) {
      const int b = (turn0 + turn * SPLIT) * 2;
      const bool tail = !STAGED && (b + 2) * 128 > pitch;
      const bool past = b + 1 >= blocks;  // of the turn's second block: nothing of it counts, its scales neither
      Fp8Codes codes[2];
      uint32_t scales;
      if constexpr (STAGED) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            codes[h].at[q] = *reinterpret_cast<const i32x4*>(xc + (b + h) * 128 + q * 16);
        scales = *reinterpret_cast<const uint16_t*>(xs + b);
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q)
            codes[h].at[q] =
                *reinterpret_cast<const i32x4*>(xc + min((b + h) * 128 + q * 16, pitch - 16 - part * 32));
        scales = *reinterpret_cast<const uint16_t*>(xs + (int64_t{b >> 2} * x_scales * 4 + (b & 3)));
        if (tail) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int q = 0; q < 2; ++q)
              if ((b + h) * 128 + part * 32 + q * 16 >= pitch) codes[h].at[q] = i32x4{0, 0, 0, 0};
        }
      }
      if (past) scales &= 0xff;
      const Fp8Fragment<WIDE, 0> x0(codes[0], scales);
      const Fp8Fragment<WIDE, 1> x1(codes[1], scales);
#pragma unroll
      for (int f = 0; f < FB; ++f) {
        acc[f] = fp8_mma16(Fp8Fragment<WIDE, 0>(unit.w[f][0], unit.s[f]), x0, acc[f]);
        acc[f] = fp8_mma16(Fp8Fragment<WIDE, 1>(unit.w[f][1], past ? unit.s[f] & 0xff : unit.s[f]), x1, acc[f]);
      }
    };
    for (int turn = 0; turn < turns; ++turn) {
      multiply(unit, turn);
      if (turn + 1 < turns) load(unit, turn + 1);
    }
    if constexpr (STAGED) __syncthreads();  // every wave has read the rows
#pragma unroll
    for (int f = 0; f < FB; ++f)
#pragma unroll
      for (int i = 0; i < 4; ++i) parts[wave][l16][f * 16 + 4 * part + i] = acc[f][i];
    __syncthreads();
    // Column `column` of the workgroup's and row r, of W's rows of parity `odd`.
    auto sum = [&](int r, int column, int odd) __attribute__((always_inline)) {
      const int tile = column / COLUMNS, c = column % COLUMNS;
      const int at = GATED ? (c / 16 * 2 + odd) * 16 + c % 16 : c;
      float v = 0.0f;
#pragma unroll
      for (int s = 0; s < SPLIT; ++s) v += parts[tile * SPLIT + s][r][at];
      return v;
    };
    const int n_wg = blockIdx.x * TILES * COLUMNS;
    if constexpr (EPILOGUE == kFp8GatedFp8) {
      const int y_pitch = (n + 15) / 16 * 16, piece = threadIdx.x % 16, column = n_wg + piece * 8;
      for (int r = threadIdx.x / 16; r < live; r += 4 * WAVES) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
          v[i] = column + i < n ? gated(sum(r, piece * 8 + i, 0), sum(r, piece * 8 + i, 1)) : 0.0f;
        const uint32_t scale = fp8_scale_byte(row16_magnitude<float>(float8_magnitude(v)));
        const int64_t row = m0 + r;
        if (column < y_pitch)
          *reinterpret_cast<elem_u32x2*>(static_cast<uint8_t*>(p.y) + row * y_pitch + column) =
              elem_u32x2{fp8_encode4(v[0], v[1], v[2], v[3], scale), fp8_encode4(v[4], v[5], v[6], v[7], scale)};
        if (piece == 0) {
          const int block = n_wg / 128;
          uint8_t* to = p.sy + (int64_t{block / 4} * p.rows + row) * 4;
          to[block % 4] = static_cast<uint8_t>(scale);
          if (block + 1 == (n + 127) / 128)
            for (int b = block % 4 + 1; b < 4; ++b) to[b] = 127;
        }
      }
    } else {
      for (int i = threadIdx.x; i < live * TILES * COLUMNS; i += 64 * WAVES) {
        const int r = i / (TILES * COLUMNS), column = i % (TILES * COLUMNS);
        if (n_wg + column >= n) continue;
        const int64_t row = m0 + r;
        float v = sum(r, column, 0);
        if constexpr (GATED) {
          const float up = sum(r, column, 1);
          if (p.gate_up) {
            Y* pair = static_cast<Y*>(p.gate_up) + row * 2 * n + n_wg + column;
            pair[0] = static_cast<Y>(v);
            pair[n] = static_cast<Y>(up);
          }
          v = gated(v, up);
        }
        static_cast<Y*>(p.y)[row * n + n_wg + column] = static_cast<Y>(v);
      }
    }
    if (m0 + static_cast<int>(gridDim.z) * ROWS < last) __syncthreads();  // the parts are written again
  }
#endif
}

}  // namespace mb
