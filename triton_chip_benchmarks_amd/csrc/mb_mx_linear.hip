// Products of MXFP4 operands for linear layers: Y = X . W^T, each row of X with
// the weight of its expert where there are several.
#include <cstring>
#include <type_traits>

#include "mb_elem.h"
#include "mb_gemm_ring.h"
#include "mb_mx.h"
#include "mb_mx_device.h"
#include "mb_mx_stream.h"

namespace mb {
namespace {

// One wave computes 16 columns of 16 rows at a time with
// v_mfma_scale_f32_16x16x128_f8f6f4: W's rows as the instruction's rows, X's as
// its columns, so that a lane holds four neighbouring columns of one row.
template <class T>
__global__ void __launch_bounds__(256)
    mx_product_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ sx, const uint8_t* __restrict__ w,
                      const uint8_t* __restrict__ sw, T* __restrict__ y, int rows, int n, int k,
                      const int32_t* __restrict__ offsets) {
  using Op = MfmaMxfp4x16;
  const int lane = threadIdx.x & 63, part = lane >> 4;
  const int n0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * 16;
  if (n0 >= n) return;
  const uint32_t e = blockIdx.y;
  int first, last;
  expert_rows(offsets, e, rows, first, last);
  const int groups = (k + 31) / 32, blocks = (k + 255) / 256;
  const int64_t row_bytes = int64_t{groups} * 16;
  const int wn = min(n0 + (lane & 15), n - 1);
  const uint8_t* wr = w + (int64_t{e} * n + wn) * row_bytes;
  const uint8_t* swr = sw + (int64_t{e} * blocks * n + wn) * 8;
  for (int m0 = first + static_cast<int>(blockIdx.z) * 16; m0 < last; m0 += static_cast<int>(gridDim.z) * 16) {
    const int xm = min(m0 + (lane & 15), last - 1);
    const uint8_t* xr = x + xm * row_bytes;
    const uint8_t* sxr = sx + int64_t{xm} * 8;
    Op::Acc acc = {};
    for (int g0 = 0; g0 < groups; g0 += 4) {
      const int g = g0 + part;
      i32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
      int sa = 127, sb = 127;
      if (g < groups) {
        a = *reinterpret_cast<const i32x4*>(wr + g * 16);
        b = *reinterpret_cast<const i32x4*>(xr + g * 16);
        sa = swr[int64_t{g >> 3} * n * 8 + (g & 7)];
        sb = sxr[int64_t{g >> 3} * rows * 8 + (g & 7)];
      }
      acc = Op::mma(a, b, acc, sa, sb);
    }
    const int m = m0 + (lane & 15);
    if (m < last) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int col = n0 + 4 * part + r;
        if (col < n) y[int64_t{m} * n + col] = static_cast<T>(acc[r]);
      }
    }
  }
}

// ---- few rows ------------------------------------------------------------------

// Rows of X with one expert's weight, for few rows: quantisation and product in
// one launch. A workgroup quantises up to 16 rows into LDS (or copies codes that
// are quantised already), then multiplies them by its features' weight, which
// goes from memory into the registers of v_mfma_scale_f32_16x16x128_f8f6f4 and is
// read once for the 16 rows. SPLIT waves share the K of FB * 16 features, in
// turns of 256 elements, and add their parts in LDS in a fixed order; the
// workgroup's other waves take other features.
//
// Bound by the weight's bytes from memory, and at one row by the latency of a
// launch and one pass over K. A wave keeps one turn's loads in flight (2.2 KiB of
// 32 features): many waves cover the latency better than deep ones, whose
// registers cost them (two turns deep 5 to 20% slower with many experts, four
// 60%), and non-temporal loads lose 5 to 10%. With the weight from HBM (another
// copy of it in each pass): 1x8192x8192 10.4 us (3.4 TB/s; the same weight again,
// from the memory-side cache, 7.5), two rows for each of 128 experts of 2048x4096
// 92 (6.2 TB/s). Quantising in the kernel spares a launch of 2.3 and costs 0.1 at
// 1x8192x8192, nothing beside 128 experts and, since every workgroup does it for
// every row, 2.9 of 16.0 at 16x8192x8192 and 5.2 of 18.5 at 16x4096x14336.
constexpr int kFewWaves = 8, kFewRows = 16;

// Expert and rows of a workgroup's blockIdx.y; false where it has none. With
// fewer rows than experts there is one grid row a row of X, and the first row of
// an expert stands for all of them; its expert is the number of those that end
// at or before it.
__device__ __forceinline__ bool few_expert(const int32_t* __restrict__ offsets, int experts, int rows, int lane, int& e,
                                           int& first, int& last) {
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

// LDS of the quantised rows: a row's codes, then a row's scales, each row a bank
// group past the one before.
constexpr uint32_t few_code_stride(uint32_t blocks) { return blocks * 128 + 16; }
constexpr uint32_t few_scale_stride(uint32_t blocks) { return blocks * 8 + 8; }
constexpr uint64_t few_lds_bytes(uint32_t blocks, uint32_t rows) {
  return uint64_t{rows} * (few_code_stride(blocks) + few_scale_stride(blocks));
}

// X: fp32, fp16 or bf16 rows at `row_stride`, or uint8_t, codes with `sx`.
template <class X, class T, int FB, int SPLIT>
__global__ void __launch_bounds__(64 * kFewWaves)
    mx_few_kernel(const X* __restrict__ x, uint64_t row_stride, const uint8_t* __restrict__ sx,
                  const uint8_t* __restrict__ w, const uint8_t* __restrict__ sw, T* __restrict__ y, int rows, int n,
                  int k, const int32_t* __restrict__ offsets, const int32_t* __restrict__ order, int copies,
                  int tokens, int experts, int lds_rows) {
  using Op = MfmaMxfp4x16;
  constexpr int TILES = kFewWaves / SPLIT, COLUMNS = FB * 16;
  __shared__ float parts[kFewWaves][kFewRows][COLUMNS + 1];
  extern __shared__ __attribute__((aligned(16))) uint8_t staged[];
  const int lane = threadIdx.x & 63, part = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int e, first, last;
  if (!few_expert(offsets, experts, rows, lane, e, first, last)) return;
  const int n0 = (blockIdx.x * TILES + wave / SPLIT) * COLUMNS, turn0 = wave % SPLIT;
  const int groups = (k + 31) / 32, blocks = (k + 255) / 256;
  const int row_bytes = groups * 16;
  const int turns = (blocks - turn0 + SPLIT - 1) / SPLIT;
  const int code_stride = few_code_stride(blocks), scale_stride = few_scale_stride(blocks);
  uint8_t* const staged_scales = staged + lds_rows * code_stride;
  const uint8_t* wr[FB];
  const uint8_t* swr[FB];
#pragma unroll
  for (int f = 0; f < FB; ++f) {
    const int feature = min(n0 + f * 16 + (lane & 15), n - 1);
    wr[f] = w + (int64_t{e} * n + feature) * row_bytes;
    swr[f] = sw + (int64_t{e} * blocks * n + feature) * 8;
  }
  struct Unit {
    i32x4 w[FB][2];
    elem_u32x2 s[FB];
  };
  auto load = [&](Unit& unit, int turn) __attribute__((always_inline)) {
    const int b = turn0 + turn * SPLIT;
#pragma unroll
    for (int f = 0; f < FB; ++f) {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        unit.w[f][h] =
            *reinterpret_cast<const i32x4*>(wr[f] + min(b * 128 + h * 64 + part * 16, row_bytes - 16));
      unit.s[f] = *reinterpret_cast<const elem_u32x2*>(swr[f] + int64_t{b} * n * 8);
    }
  };
  for (int m0 = first; m0 < last; m0 += kFewRows) {
    Unit unit;
    if (turns > 0) load(unit, 0);  // in flight while the rows are quantised
    const int live = min(kFewRows, last - m0);
    for (int task = threadIdx.x; task < live * blocks * 8; task += 64 * kFewWaves) {
      const int row = task / (blocks * 8), group = task % (blocks * 8);
      i32x4 codes = {0, 0, 0, 0};
      uint32_t scale = 0;  // groups past K: zeros of the scale 2^-127
      if constexpr (sizeof(X) == 1) {
        if (group < groups) {
          codes = *reinterpret_cast<const i32x4*>(x + int64_t{m0 + row} * row_bytes + group * 16);
          scale = sx[(int64_t{group >> 3} * rows + m0 + row) * 8 + (group & 7)];
        }
      } else if (group < groups) {
        int token = m0 + row;
        if (order) token = max(0, min(order[token] / copies, tokens - 1));
        const X* from = x + static_cast<uint64_t>(token) * row_stride + group * 32;
        Raw8<X> raw[4];
        if (group * 32 + 32 <= k) {
#pragma unroll
          for (int q = 0; q < 4; ++q) raw[q].load(from + q * 8);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q) raw[q].load(from + q * 8, k - group * 32 - q * 8);
        }
        uint32_t largest = raw_magnitude(raw[0]);
#pragma unroll
        for (int q = 1; q < 4; ++q) largest = join_magnitudes(X(), largest, raw_magnitude(raw[q]));
        scale = scale_byte(magnitude_bits<X>(largest));
#pragma unroll
        for (int q = 0; q < 4; ++q) codes[q] = static_cast<int>(encode8(raw[q], scale));
      }
      *reinterpret_cast<i32x4*>(staged + row * code_stride + group * 16) = codes;
      staged_scales[row * scale_stride + group] = static_cast<uint8_t>(scale);
    }
    __syncthreads();
    const int mine = min(lane & 15, live - 1);
    const uint8_t* xc = staged + mine * code_stride + part * 16;
    const uint8_t* xs = staged_scales + mine * scale_stride;
    Op::Acc acc[FB] = {};
    auto multiply = [&](const Unit& unit, int turn) __attribute__((always_inline)) {
      const int b = turn0 + turn * SPLIT;
      const elem_u32x2 sb = *reinterpret_cast<const elem_u32x2*>(xs + b * 8);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const i32x4 codes = *reinterpret_cast<const i32x4*>(xc + b * 128 + h * 64);
        // Past K the codes are zeros; whatever the weight's scales hold there must not be NaN.
        const bool past = b * 8 + h * 4 + part >= groups;
#pragma unroll
        for (int f = 0; f < FB; ++f)
          acc[f] = Op::mma(unit.w[f][h], codes, acc[f], past ? 0 : static_cast<int>(unit.s[f][h] >> (8 * part)),
                           static_cast<int>(sb[h] >> (8 * part)));
      }
    };
    for (int turn = 0; turn < turns; ++turn) {
      multiply(unit, turn);
      if (turn + 1 < turns) load(unit, turn + 1);
    }
#pragma unroll
    for (int f = 0; f < FB; ++f)
#pragma unroll
      for (int r = 0; r < 4; ++r) parts[wave][lane & 15][f * 16 + 4 * part + r] = acc[f][r];
    __syncthreads();
    const int n_wg = blockIdx.x * TILES * COLUMNS;
    for (int i = threadIdx.x; i < live * TILES * COLUMNS; i += 64 * kFewWaves) {
      const int r = i / (TILES * COLUMNS), column = i % (TILES * COLUMNS), tile = column / COLUMNS;
      float sum = 0.0f;
#pragma unroll
      for (int v = 0; v < SPLIT; ++v) sum += parts[tile * SPLIT + v][r][column % COLUMNS];
      if (n_wg + column < n) y[static_cast<int64_t>(m0 + r) * n + n_wg + column] = static_cast<T>(sum);
    }
  }
}

// ---- tiles through the ring GEMM -----------------------------------------------

// Expert and first row of row tile `tile` (BN rows each, an expert's rows
// starting a tile of their own), for the whole wave.
struct ExpertTile {
  int expert, first, last;
};

template <int BN>
__device__ __forceinline__ int expert_tile_count(const int32_t* __restrict__ offsets, int e, int experts, int rows) {
  if (e >= experts) return 0;
  int first, last;
  expert_rows(offsets, e, rows, first, last);
  return (last - first + BN - 1) / BN;
}

template <int BN>
__device__ __forceinline__ int count_row_tiles(const int32_t* __restrict__ offsets, int experts, int rows, int lane) {
  if (offsets == nullptr) return (rows + BN - 1) / BN;
  int total = 0;
  for (int e = lane; e < experts; e += 64) total += expert_tile_count<BN>(offsets, e, experts, rows);
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) total += __shfl_xor(total, offset, 64);
  return __builtin_amdgcn_readfirstlane(total);
}

template <int BN>
__device__ __forceinline__ ExpertTile find_row_tile(const int32_t* __restrict__ offsets, int experts, int rows,
                                                    int tile, int lane) {
  if (offsets == nullptr) return {0, tile * BN, rows};
  int before = 0;  // tiles of the experts below `base`
  for (int base = 0; base < experts; base += 64) {
    const int mine = expert_tile_count<BN>(offsets, base + lane, experts, rows);
    int scan = mine;
#pragma unroll
    for (int offset = 1; offset < 64; offset <<= 1) {
      const int v = __shfl_up(scan, offset, 64);
      if (lane >= offset) scan += v;
    }
    const uint64_t past = __ballot(before + scan > tile);
    if (past) {
      const int at = __builtin_ctzll(past);
      const int start = before + __builtin_amdgcn_readlane(scan - mine, at);
      const int e = base + at;
      int first, last;
      expert_rows(offsets, e, rows, first, last);
      return {e, first + (tile - start) * BN, last};
    }
    before += __builtin_amdgcn_readlane(scan, 63);
  }
  return {0, rows, rows};  // no such tile
}

// BM columns (features) of BN rows of one expert by gemm_ring_kernel's loop, W as
// its A and X as its B: a lane then holds four neighbouring features of a row.
// The tile leaves through LDS, so that rows are stored in whole 16-byte pieces.
template <class T, int BM, int BN, int STAGES>
__global__ void __launch_bounds__(256)
    mx_product_ring_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ sx,
                           const uint8_t* __restrict__ w, const uint8_t* __restrict__ sw, T* __restrict__ y, int rows,
                           int n, int k, const int32_t* __restrict__ offsets, int experts, int band) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Op = MfmaMxfp4;
  using Tile = RingTile<Op, BM, BN, STAGES>;
  constexpr int FM = Tile::FM, FN = Tile::FN;
  constexpr int LDS_ROW = BM * sizeof(T) + 16;  // padded: neighbouring rows start in other banks
  static_assert(BN * LDS_ROW <= STAGES * Tile::STAGE, "the output tile fits the ring's LDS");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * Tile::STAGE];
  if (k < 0) lds[threadIdx.x] = 0;  // keeps DMA-written reads live; never executed
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  // The grid bounds the number of tiles, which the experts' row counts decide.
  // XCD x (ids x, x + 8, ..) takes a contiguous share of the real ones.
  const int row_tiles = count_row_tiles<BN>(offsets, experts, rows, lane);
  const int columns = (n + BM - 1) / BM;
  if (static_cast<int64_t>(row_tiles) * columns > gridDim.x) return;  // offsets that do not rise: nothing to rely on
  const int count = row_tiles * columns, xcd = blockIdx.x % kXcds, index = blockIdx.x / kXcds;
  if (index >= count / kXcds + (xcd < count % kXcds)) return;
  const int pid = xcd * (count / kXcds) + min(xcd, count % kXcds) + index;
  const int per_band = band * columns, first_tile = pid / per_band * band;
  const int in_band = min(row_tiles - first_tile, band);
  const int row_tile = first_tile + pid % per_band % in_band;
  const int m0 = pid % per_band / in_band * BM;
  const ExpertTile at = find_row_tile<BN>(offsets, experts, rows, row_tile, lane);
  const int n0 = at.first, live = min(BN, at.last - at.first);
  const int64_t e = at.expert;
  const int steps = (k + 255) / 256;

  typename Op::Acc acc[FM][FN];
  ring_accumulate<Op, BM, BN, STAGES>(lds, w + e * n * (k / 2), x, sw + e * steps * n * 8, sx, n, rows, k, m0, n0,
                                      min(BM, n - m0), live, lane, wave, acc);
  lds_barrier();  // every wave's reads of the ring have ended
  const int wm = wave & 1, wn = wave >> 1;
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        T out[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) out[r] = static_cast<T>(acc[i][j][4 * q + r]);
        const int row = wn * Tile::WN + j * 32 + (lane & 31);
        const int column = wm * Tile::WM + i * 32 + Op::out_row(lane, 4 * q);
        __builtin_memcpy(__builtin_assume_aligned(lds + row * LDS_ROW + column * sizeof(T), 4 * sizeof(T)), out,
                         sizeof(out));
      }
  lds_barrier();
  constexpr int PIECE = 16 / sizeof(T), PIECES = BM / PIECE;  // a row's 16-byte pieces
  T* tile_y = y + static_cast<int64_t>(n0) * n + m0;
#pragma unroll 4
  for (int piece = threadIdx.x; piece < BN * PIECES; piece += 256) {
    const int row = piece / PIECES, column = piece % PIECES * PIECE;
    if (row >= live || m0 + column >= n) continue;
    const elem_u32x4 value = *reinterpret_cast<const elem_u32x4*>(lds + row * LDS_ROW + column * sizeof(T));
    T* to = tile_y + static_cast<int64_t>(row) * n + column;
    if (m0 + column + PIECE <= n) {
      *reinterpret_cast<elem_u32x4_any*>(to) = value;
    } else {
      T part[PIECE];
      __builtin_memcpy(part, &value, 16);
#pragma unroll
      for (int i = 0; i < PIECE; ++i)
        if (m0 + column + i < n) to[i] = part[i];
    }
  }
#endif
}

using ProductLauncher = void (*)(const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, void*, int, int, int,
                                 const int32_t*, int, uint32_t, int, hipStream_t);

template <class T, int BM, int BN, int STAGES>
void launch_ring(const uint8_t* x, const uint8_t* sx, const uint8_t* w, const uint8_t* sw, void* y, int rows, int n,
                 int k, const int32_t* offsets, int experts, uint32_t grid, int band, hipStream_t stream) {
  mx_product_ring_kernel<T, BM, BN, STAGES><<<dim3(grid), dim3(256), 0, stream>>>(
      x, sx, w, sw, static_cast<T*>(y), rows, n, k, offsets, experts, band);
}

template <class T, int BM, int BN, int STAGES>
void launch_stream(const uint8_t* x, const uint8_t* sx, const uint8_t* w, const uint8_t* sw, void* y, int rows, int n,
                   int k, const int32_t* offsets, int experts, uint32_t grid, int band, hipStream_t stream) {
  constexpr uint32_t kPlaces = 256 * RingTile<MfmaMxfp4, BM, BN, STAGES>::RESIDENT;
  mx_product_stream_kernel<T, BM, BN, STAGES><<<dim3(grid < kPlaces ? grid : kPlaces), dim3(256), 0, stream>>>(
      x, sx, w, sw, static_cast<T*>(y), rows, n, k, offsets, experts, band);
}

// What a launch takes, in microseconds: `launch` once; for every round of its
// workgroups `tile`, `ragged` more where the rows of Y are not on 16 bytes, and
// for every 256 elements of K from `step_empty` to `step_full` with the filled
// share of the round (the L2s and the power limit slow a step down as more CUs
// run).
struct ProductCost {
  float launch, tile, ragged, step_empty, step_full;
};

// A kernel of BM features by BN rows a tile.
struct ProductKernel {
  int features, rows;
  bool persistent;
  int band;      // row tiles that share their weight's panels in an XCD's L2
  int resident;  // workgroups a CU holds
  ProductCost cost;
  ProductLauncher launch[3];  // by MB_DTYPE_*
  const char* name[3];
};
constexpr bool kPersistent_ring = false, kPersistent_stream = true;
#define MB_SUFFIX_ring
#define MB_SUFFIX_stream "_stream"
#define MB_PRODUCT_NAME(T, KIND, BM, BN) "mx_product_" T "_" #BM "x" #BN MB_SUFFIX_##KIND
#define MB_PRODUCT(KIND, BM, BN, STAGES, BAND, ...)                                                        \
  ProductKernel {                                                                                          \
    BM, BN, kPersistent_##KIND, BAND, RingTile<MfmaMxfp4, BM, BN, STAGES>::RESIDENT, {__VA_ARGS__},        \
        {launch_##KIND<float, BM, BN, STAGES>, launch_##KIND<_Float16, BM, BN, STAGES>,                    \
         launch_##KIND<__bf16, BM, BN, STAGES>},                                                           \
        {MB_PRODUCT_NAME("f32", KIND, BM, BN), MB_PRODUCT_NAME("f16", KIND, BM, BN),                       \
         MB_PRODUCT_NAME("bf16", KIND, BM, BN)}                                                            \
  }
// Fitted to 414 launches on an MI355X (17 to 32768 rows, n and K from 64 to 8192,
// one weight or 8 to 256 experts of uneven popularity, half of the n odd): the
// cheapest estimate costs 2.1% over the fastest of the five on average, over 10%
// in one launch of 17, at most 38% (2 us). Ten kernels were measured; these five's
// best is 0.8% over the ten's, the two that are not persistent alone 12%.
const ProductKernel kProductKernels[] = {
    MB_PRODUCT(ring, 128, 128, 2, 8, 2.10f, 3.59f, 0.25f, 0.303f, 1.426f),
    MB_PRODUCT(ring, 64, 64, 3, 8, 2.90f, 2.86f, 0.12f, 0.056f, 0.495f),
    MB_PRODUCT(stream, 256, 128, 3, 4, 5.45f, 2.34f, 1.66f, 0.510f, 1.204f),
    MB_PRODUCT(stream, 128, 64, 3, 8, 5.31f, 0.90f, 0.48f, 0.179f, 0.918f),
    MB_PRODUCT(stream, 64, 64, 3, 8, 4.84f, 0.83f, 0.28f, 0.102f, 0.768f),
};

#define MB_PRODUCT_REGISTER(T, NAME)                                                                        \
  MB_REGISTER_KERNEL("mx_product_" NAME, mx_product_kernel<T>);                                             \
  MB_REGISTER_KERNEL("mx_product_" NAME "_128x128", (mx_product_ring_kernel<T, 128, 128, 2>));              \
  MB_REGISTER_KERNEL("mx_product_" NAME "_64x64", (mx_product_ring_kernel<T, 64, 64, 3>));                  \
  MB_REGISTER_KERNEL("mx_product_" NAME "_256x128_stream", (mx_product_stream_kernel<T, 256, 128, 3>));     \
  MB_REGISTER_KERNEL("mx_product_" NAME "_128x64_stream", (mx_product_stream_kernel<T, 128, 64, 3>));       \
  MB_REGISTER_KERNEL("mx_product_" NAME "_64x64_stream", (mx_product_stream_kernel<T, 64, 64, 3>))
#define MB_FEW_REGISTER_SPLIT(T, NAME, FB, SPLIT, SIZE)                                             \
  MB_REGISTER_KERNEL("mx_linear_few_" NAME "_" SIZE, (mx_few_kernel<T, T, FB, SPLIT>));            \
  MB_REGISTER_KERNEL("mx_product_few_" NAME "_" SIZE, (mx_few_kernel<uint8_t, T, FB, SPLIT>))
#define MB_FEW_REGISTER(T, NAME)                   \
  MB_FEW_REGISTER_SPLIT(T, NAME, 1, 8, "16x8");    \
  MB_FEW_REGISTER_SPLIT(T, NAME, 2, 8, "32x8");    \
  MB_FEW_REGISTER_SPLIT(T, NAME, 2, 4, "32x4")
MB_FEW_REGISTER(float, "f32");
MB_FEW_REGISTER(_Float16, "f16");
MB_FEW_REGISTER(__bf16, "bf16");
MB_PRODUCT_REGISTER(float, "f32");
MB_PRODUCT_REGISTER(_Float16, "f16");
MB_PRODUCT_REGISTER(__bf16, "bf16");

constexpr uint32_t kMostExperts = 4096;

int check_shape(const char* entry, int dtype, uint64_t rows, uint64_t n, uint64_t k, uint32_t experts) {
  if (!elem_bytes(dtype)) return fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (experts == 0 || experts > kMostExperts)
    return fail(MB_ERR_INVALID, "%s: %u experts outside 1..%u", entry, experts, kMostExperts);
  if (rows > kMxMostRows || n > kMxMostK || k > kMxMostK)
    return fail(MB_ERR_UNSUPPORTED, "%s: %llu x %llu x %llu: at most %u rows, %u columns and %u elements of K", entry,
                (unsigned long long)rows, (unsigned long long)n, (unsigned long long)k, kMxMostRows, kMxMostK,
                kMxMostK);
  return MB_OK;
}

int check_output(const char* entry, int dtype, const void* y, uint64_t y_bytes, uint64_t rows, uint64_t n) {
  const uint32_t item = elem_bytes(dtype);
  if (y == nullptr || y_bytes < rows * n * item)
    return fail(MB_ERR_INVALID, "%s: the output is NULL or too small for %llu x %llu", entry, (unsigned long long)rows,
                (unsigned long long)n);
  if (!aligned(y, item)) return fail(MB_ERR_ALIGNMENT, "%s: the output must lie on its elements' %u bytes", entry, item);
  return MB_OK;
}

int check_offsets(const char* entry, const int32_t* offsets, uint64_t offsets_bytes, uint32_t experts) {
  if (offsets == nullptr)
    return experts == 1 ? MB_OK : fail(MB_ERR_INVALID, "%s: several experts need offsets", entry);
  if (offsets_bytes < (uint64_t{experts} + 1) * 4)
    return fail(MB_ERR_INVALID, "%s: offsets must hold %u entries", entry, experts + 1);
  if (!aligned(offsets, 4)) return fail(MB_ERR_ALIGNMENT, "%s: offsets must lie on 4 bytes", entry);
  return MB_OK;
}

// Row tiles of `tile` rows: at most, and as many as experts of even numbers of
// rows have (a last one half empty on average).
uint64_t most_row_tiles(uint32_t rows, uint32_t experts, int tile) {
  return experts > 1 ? rows / tile + (rows < experts ? rows : experts) : (rows + uint64_t{1} * tile - 1) / tile;
}

double mean_row_tiles(uint32_t rows, uint32_t experts, int tile) {
  if (experts == 1) return static_cast<double>(most_row_tiles(rows, 1, tile));
  const double each = static_cast<double>(rows) / experts;
  return experts * (each >= tile ? each / tile + 0.5 : each >= 1 ? 1.0 : each);
}

// Estimated microseconds of a launch (see ProductCost).
double product_cost(const ProductKernel& kernel, uint32_t rows, uint32_t n, uint32_t steps, uint32_t experts,
                    bool ragged) {
  const double tiles = mean_row_tiles(rows, experts, kernel.rows) * ((n + kernel.features - 1) / kernel.features);
  const double round = 256.0 * kernel.resident, whole = static_cast<double>(static_cast<uint64_t>(tiles / round));
  const double rest = tiles / round - whole;
  const ProductCost& cost = kernel.cost;
  auto one = [&](double filled) {
    return cost.tile + (ragged ? cost.ragged : 0.0f) +
           steps * (cost.step_empty + (cost.step_full - cost.step_empty) * filled);
  };
  return cost.launch + whole * one(1.0) + (rest > 0 ? one(rest) : 0.0);
}

// Whether mx_few_kernel can: its rows' codes fit the LDS.
bool few_fits(uint64_t rows, uint32_t k) {
  return few_lds_bytes((k + 255) / 256, rows < kFewRows ? static_cast<uint32_t>(rows) : kFewRows) <= 128 * 1024;
}

// Whether mx_few_kernel takes a call: up to 16 rows of one weight, up to two an
// expert on average (it reads a weight once for 16 rows, but its rows are
// quantised, or copied, once a workgroup), whose codes fit the LDS. us, weights
// from HBM, it and the tiles with their quantisation: 16x8192x8192 16.0 and 19.0,
// 16x4096x14336 18.5 and 27.7; 128 experts of 2048x4096, two rows each 92 and 103
// (128x64 tiles), four 107 on those, and 92 here for rows that are operands.
bool few_rows(uint64_t rows, uint32_t k, uint32_t experts) {
  const uint64_t most = experts > 1 ? 2 * uint64_t{experts} : kFewRows;
  return rows <= most && few_fits(rows, k);
}

// Forms of mx_few_kernel, by the number of features a workgroup takes: 32 where
// that gives every CU a workgroup, else 16 (operands of 1x4096x14336 9.2 us, with
// 32 11.2; at 8192x8192, with one workgroup of 32 a CU, 10.2 and with 16 9.6); with
// many workgroups, 64 and half the waves on each K (two rows of 128 experts 92.7,
// with all eight 95.1; four 92.2 and 98.9).
enum FewForm { kFew16x8, kFew32x8, kFew32x4, kFewForms };
constexpr uint32_t kFewColumns[kFewForms] = {16, 32, 64};
#define MB_FEW_NAMES(KIND, SIZE) \
  {"mx_" KIND "_few_f32_" SIZE, "mx_" KIND "_few_f16_" SIZE, "mx_" KIND "_few_bf16_" SIZE}
// By form and MB_DTYPE_*: of rows quantised on the way, of operands.
const char* const kLinearFewNames[kFewForms][3] = {MB_FEW_NAMES("linear", "16x8"), MB_FEW_NAMES("linear", "32x8"),
                                                   MB_FEW_NAMES("linear", "32x4")};
const char* const kProductFewNames[kFewForms][3] = {MB_FEW_NAMES("product", "16x8"), MB_FEW_NAMES("product", "32x8"),
                                                    MB_FEW_NAMES("product", "32x4")};
const char* const kPlainNames[3] = {"mx_product_f32", "mx_product_f16", "mx_product_bf16"};

FewForm few_form(uint32_t rows, uint32_t n, uint32_t experts) {
  const uint64_t wide = (n + uint64_t{31}) / 32 * (rows < experts ? rows : experts);
  return wide < 256 ? kFew16x8 : wide < 2048 ? kFew32x8 : kFew32x4;
}

template <class X, class T>
void launch_few(FewForm form, const void* x, uint64_t row_stride, const void* sx, const void* w, const void* sw,
                void* y, uint32_t rows, uint32_t n, uint32_t k, const int32_t* offsets, const int32_t* order,
                uint32_t copies, uint32_t tokens, uint32_t experts, hipStream_t stream) {
  const uint32_t grid_rows = rows < experts ? rows : experts, lds_rows = rows < kFewRows ? rows : kFewRows;
  const uint32_t columns = kFewColumns[form];
  auto launch = [&](auto kernel) {
    kernel<<<dim3((n + columns - 1) / columns, grid_rows), dim3(64 * kFewWaves),
             static_cast<uint32_t>(few_lds_bytes((k + 255) / 256, lds_rows)), stream>>>(
        static_cast<const X*>(x), row_stride, static_cast<const uint8_t*>(sx), static_cast<const uint8_t*>(w),
        static_cast<const uint8_t*>(sw), static_cast<T*>(y), static_cast<int>(rows), static_cast<int>(n),
        static_cast<int>(k), offsets, order, static_cast<int>(copies), static_cast<int>(tokens),
        static_cast<int>(experts), static_cast<int>(lds_rows));
  };
  if (form == kFew16x8)
    launch(mx_few_kernel<X, T, 1, 8>);
  else if (form == kFew32x8)
    launch(mx_few_kernel<X, T, 2, 8>);
  else
    launch(mx_few_kernel<X, T, 2, 4>);
}

// The kernel that multiplies two operands: a form of mx_few_kernel, a kernel of
// tiles, or, with neither, mx_product_kernel, which takes every size.
struct ProductChoice {
  int few = -1;
  const ProductKernel* tiles = nullptr;
  uint32_t grid = 0;  // of tiles
  const char* name;
};

// By the rule for these sizes or, with `wanted`, the kernel of that name; false
// if that one does not take them.
bool choose_product(int dtype, uint32_t rows, uint32_t n, uint32_t k, uint32_t experts, const char* wanted,
                    ProductChoice& out) {
  auto is_wanted = [&](const char* name) { return wanted == nullptr || strcmp(wanted, name) == 0; };
  if (wanted == nullptr ? few_rows(rows, k, experts) : few_fits(rows, k)) {
    for (int form = 0; form < kFewForms; ++form) {
      if (wanted == nullptr ? form != few_form(rows, n, experts) : !is_wanted(kProductFewNames[form][dtype])) continue;
      out.few = form;
      out.name = kProductFewNames[form][dtype];
      return true;
    }
  }
  // The ring addresses a matrix's scales, and a tile's rows, with 32-bit offsets.
  const uint64_t scale_rows = rows > n ? rows : n;
  const uint32_t steps = (k + 255) / 256;
  if (steps * scale_rows * 8 <= 0x7fffffffu) {
    double best_cost = 0;
    const bool ragged = uint64_t{n} * elem_bytes(dtype) % 16 != 0;
    for (const ProductKernel& kernel : kProductKernels) {
      const uint64_t tiles = most_row_tiles(rows, experts, kernel.rows) * ((n + kernel.features - 1) / kernel.features);
      const uint64_t grid = (tiles + kXcds - 1) / kXcds * kXcds;
      if (grid > 0xffffff) continue;
      if (kernel.persistent && experts > kStreamExperts) continue;
      if (!is_wanted(kernel.name[dtype])) continue;
      const double cost = product_cost(kernel, rows, n, steps, experts, ragged);
      if (out.tiles && cost >= best_cost) continue;
      best_cost = cost;
      out.tiles = &kernel;
      out.grid = static_cast<uint32_t>(grid);
      out.name = kernel.name[dtype];
    }
    if (out.tiles) return true;
  }
  out.name = kPlainNames[dtype];
  return is_wanted(out.name);
}

int launch_product(int dtype, const void* x_codes, const void* sx, const void* w_codes, const void* sw, void* y,
                   uint32_t rows, uint32_t n, uint32_t k, const int32_t* offsets, uint32_t experts,
                   const char* wanted, hipStream_t stream) {
  const uint8_t *x = static_cast<const uint8_t*>(x_codes), *w = static_cast<const uint8_t*>(w_codes);
  const uint8_t *sxb = static_cast<const uint8_t*>(sx), *swb = static_cast<const uint8_t*>(sw);
  ProductChoice choice;
  if (!choose_product(dtype, rows, n, k, experts, wanted, choice))
    return fail(MB_ERR_UNSUPPORTED, "mx_product: no kernel %s that takes %u x %u x %u and %u experts", wanted, rows, n,
                k, experts);
  if (choice.few >= 0) {
    MB_FOR_DTYPE(dtype, (launch_few<uint8_t, T>(static_cast<FewForm>(choice.few), x, 0, sx, w, sw, y, rows, n, k,
                                                offsets, nullptr, 1, rows, experts, stream)));
  } else if (choice.tiles) {
    const int padded = static_cast<int>((k + 31) / 32 * 32);
    choice.tiles->launch[dtype](x, sxb, w, swb, y, static_cast<int>(rows), static_cast<int>(n), padded, offsets,
                                static_cast<int>(experts), choice.grid, choice.tiles->band, stream);
  } else {
    const uint32_t tiles = (rows / experts + 15) / 16;
    const dim3 grid((n + 63) / 64, experts, tiles < 1 ? 1 : tiles < 256 ? tiles : 256);
    MB_FOR_DTYPE(dtype, (mx_product_kernel<T><<<grid, dim3(256), 0, stream>>>(
                            x, sxb, w, swb, static_cast<T*>(y), static_cast<int>(rows), static_cast<int>(n),
                            static_cast<int>(k), offsets)));
  }
  return launch_status(choice.name);
}

int run_product(const char* entry, const char* wanted, int dtype, const void* a, uint64_t a_bytes, const void* scale_a,
                uint64_t scale_a_bytes, const void* b, uint64_t b_bytes, const void* scale_b, uint64_t scale_b_bytes,
                void* c, uint64_t c_bytes, uint32_t rows, uint32_t n, uint32_t k, const int32_t* offsets,
                uint64_t offsets_bytes, uint32_t experts, void* stream) {
  if (int rc = check_shape(entry, dtype, rows, n, k, experts)) return rc;
  if (int rc = check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (int rc = check_operand(entry, "a", rows, k, 1, a, a_bytes, scale_a, scale_a_bytes)) return rc;
  if (int rc = check_operand(entry, "b", n, k, experts, b, b_bytes, scale_b, scale_b_bytes)) return rc;
  if (int rc = check_output(entry, dtype, c, c_bytes, rows, n)) return rc;
  return launch_product(dtype, a, scale_a, b, scale_b, c, rows, n, k, offsets, experts, wanted,
                        static_cast<hipStream_t>(stream));
}

}  // namespace
}  // namespace mb

extern "C" {

int mb_mx_product(int dtype, const void* a, uint64_t a_bytes, const void* scale_a, uint64_t scale_a_bytes,
                  const void* b, uint64_t b_bytes, const void* scale_b, uint64_t scale_b_bytes, void* c,
                  uint64_t c_bytes, uint32_t rows, uint32_t n, uint32_t k, const int32_t* offsets,
                  uint64_t offsets_bytes, uint32_t experts, void* stream) {
  return mb::run_product("mb_mx_product", nullptr, dtype, a, a_bytes, scale_a, scale_a_bytes, b, b_bytes, scale_b,
                         scale_b_bytes, c, c_bytes, rows, n, k, offsets, offsets_bytes, experts, stream);
}

int mb_mx_product_exact(const char* kernel, int dtype, const void* a, uint64_t a_bytes, const void* scale_a,
                        uint64_t scale_a_bytes, const void* b, uint64_t b_bytes, const void* scale_b,
                        uint64_t scale_b_bytes, void* c, uint64_t c_bytes, uint32_t rows, uint32_t n, uint32_t k,
                        const int32_t* offsets, uint64_t offsets_bytes, uint32_t experts, void* stream) {
  if (kernel == nullptr) return mb::fail(MB_ERR_INVALID, "mb_mx_product_exact: the kernel's name is NULL");
  return mb::run_product("mb_mx_product_exact", kernel, dtype, a, a_bytes, scale_a, scale_a_bytes, b, b_bytes, scale_b,
                         scale_b_bytes, c, c_bytes, rows, n, k, offsets, offsets_bytes, experts, stream);
}

const char* mb_mx_product_kernel(int dtype, uint32_t rows, uint32_t n, uint32_t k, uint32_t experts, uint32_t linear) {
  const char* entry = "mb_mx_product_kernel";
  if (mb::check_shape(entry, dtype, rows, n, k, experts)) return nullptr;
  if (rows == 0 || n == 0 || k == 0) {
    mb::fail(MB_ERR_INVALID, "%s: empty product %u x %u x %u", entry, rows, n, k);
    return nullptr;
  }
  mb::ProductChoice choice;
  mb::choose_product(dtype, rows, n, k, experts, nullptr, choice);
  return linear && choice.few >= 0 ? mb::kLinearFewNames[choice.few][dtype] : choice.name;
}

uint64_t mb_mx_linear_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  (void)n;
  return (mb::mx_code_bytes(rows, k) + 15) / 16 * 16 + mb::mx_scale_bytes(rows, k);
}

int mb_mx_linear(int dtype, const void* x, uint64_t x_bytes, uint32_t tokens, uint64_t row_stride, const void* w,
                 uint64_t w_bytes, const void* scale_w, uint64_t scale_w_bytes, void* y, uint64_t y_bytes, uint32_t n,
                 uint32_t k, const int32_t* offsets, uint64_t offsets_bytes, const int32_t* order,
                 const int32_t* slots, uint64_t slots_bytes, uint32_t copies, uint32_t experts, void* workspace,
                 uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_mx_linear";
  const bool gathered = slots != nullptr;
  if (gathered && (copies == 0 || copies > 64))
    return mb::fail(MB_ERR_INVALID, "%s: %u slots a token outside 1..64", entry, copies);
  const uint64_t rows = uint64_t{tokens} * (gathered ? copies : 1);
  if (int rc = mb::check_shape(entry, dtype, rows, n, k, experts)) return rc;
  if (int rc = mb::check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (gathered && (offsets == nullptr || order == nullptr || slots_bytes < rows * 4))
    return mb::fail(MB_ERR_INVALID, "%s: slots need offsets, order and, in both, an entry for each of %llu rows", entry,
                    (unsigned long long)rows);
  if (!mb::aligned(slots, 4) || !mb::aligned(order, 4))
    return mb::fail(MB_ERR_ALIGNMENT, "%s: order and slots must lie on 4 bytes", entry);
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return mb::fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (int rc = mb::check_rows(entry, dtype, x, x_bytes, tokens, k, row_stride)) return rc;
  if (int rc = mb::check_operand(entry, "the weight", n, k, experts, w, w_bytes, scale_w, scale_w_bytes)) return rc;
  if (int rc = mb::check_output(entry, dtype, y, y_bytes, rows, n)) return rc;
  const uint64_t codes_bytes = (mb::mx_code_bytes(rows, k) + 15) / 16 * 16;
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  if (codes == nullptr || workspace_bytes < codes_bytes + mb::mx_scale_bytes(rows, k))
    return mb::fail(MB_ERR_INVALID, "%s: the workspace is NULL or too small: %llu bytes needed", entry,
                    (unsigned long long)(codes_bytes + mb::mx_scale_bytes(rows, k)));
  if (!mb::aligned(codes, 16)) return mb::fail(MB_ERR_ALIGNMENT, "%s: the workspace must lie on 16 bytes", entry);
  uint8_t* scales = codes + codes_bytes;
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (mb::few_rows(rows, k, experts)) {
    const mb::FewForm form = mb::few_form(static_cast<uint32_t>(rows), n, experts);
    MB_FOR_DTYPE(dtype, (mb::launch_few<T, T>(form, x, row_stride, nullptr, w, scale_w, y, static_cast<uint32_t>(rows),
                                              n, k, offsets, gathered ? order : nullptr, copies, tokens, experts, on)));
    return mb::launch_status(mb::kLinearFewNames[form][dtype]);
  }
  if (int rc = mb::launch_quantize(dtype, x, tokens, k, row_stride, slots, gathered ? copies : 1,
                                   static_cast<uint32_t>(rows), codes, scales, on))
    return rc;
  return mb::launch_product(dtype, codes, scales, w, scale_w, y, static_cast<uint32_t>(rows), n, k, offsets, experts,
                            nullptr, on);
}

// Operands of mb_mx_linear_backward in its workspace: Q(d_out) [rows][n], and the
// columns of d_out [n][rows] and of x [k][rows].
static uint64_t place_operand(uint64_t at, uint64_t rows, uint64_t k, uint64_t* codes, uint64_t* scales) {
  *codes = at;
  *scales = at + (mb::mx_code_bytes(rows, k) + 15) / 16 * 16;
  return *scales + (mb::mx_scale_bytes(rows, k) + 15) / 16 * 16;
}

// K of d_w's operands: whole blocks of 256 past the first, so that their rows'
// 128-byte pieces lie on lines. 5000x3000 of K 4112 47.4 us, of 4352 (as many
// steps) 44.3.
static uint32_t gradient_depth(uint32_t rows) { return rows > 256 ? (rows + 255) / 256 * 256 : (rows + 31) / 32 * 32; }

uint64_t mb_mx_linear_backward_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  const uint64_t depth = gradient_depth(rows < mb::kMxMostRows ? rows : mb::kMxMostRows);
  uint64_t codes, scales, end = place_operand(0, rows, n, &codes, &scales);
  end = place_operand(end, n, depth, &codes, &scales);
  return place_operand(end, k, depth, &codes, &scales);
}

int mb_mx_linear_backward(int dtype, const void* d_out, uint64_t d_out_bytes, uint64_t d_out_stride, const void* x,
                          uint64_t x_bytes, uint64_t x_stride, const void* w_columns, uint64_t w_columns_bytes,
                          const void* scale_w, uint64_t scale_w_bytes, void* d_x, uint64_t d_x_bytes, void* d_w,
                          uint64_t d_w_bytes, uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_mx_linear_backward";
  if (int rc = mb::check_shape(entry, dtype, rows, n, k, 1)) return rc;
  if (rows == 0 || n == 0 || k == 0) return mb::fail(MB_ERR_INVALID, "%s: rows, n and K must be positive", entry);
  if (rows > mb::kMxMostK)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: at most %u rows, which d_w sums over", entry, mb::kMxMostK);
  if (int rc = mb::check_rows(entry, dtype, d_out, d_out_bytes, rows, n, d_out_stride)) return rc;
  if (int rc = mb::check_rows(entry, dtype, x, x_bytes, rows, k, x_stride)) return rc;
  if (int rc = mb::check_operand(entry, "the weight's columns", k, n, 1, w_columns, w_columns_bytes, scale_w,
                                 scale_w_bytes))
    return rc;
  if (int rc = mb::check_output(entry, dtype, d_x, d_x_bytes, rows, k)) return rc;
  if (int rc = mb::check_output(entry, dtype, d_w, d_w_bytes, n, k)) return rc;
  uint64_t codes[3], scales[3], end = place_operand(0, rows, n, &codes[0], &scales[0]);
  const uint32_t depth = gradient_depth(rows);
  end = place_operand(end, n, depth, &codes[1], &scales[1]);
  end = place_operand(end, k, depth, &codes[2], &scales[2]);
  uint8_t* const space = static_cast<uint8_t*>(workspace);
  if (space == nullptr || workspace_bytes < end)
    return mb::fail(MB_ERR_INVALID, "%s: the workspace is NULL or too small: %llu bytes needed", entry,
                    (unsigned long long)end);
  if (!mb::aligned(space, 16)) return mb::fail(MB_ERR_ALIGNMENT, "%s: the workspace must lie on 16 bytes", entry);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (int rc = mb::launch_quantize_gradient(dtype, d_out, d_out_stride, x, x_stride, rows, n, k, depth,
                                            space + codes[0], space + scales[0], space + codes[1], space + scales[1],
                                            space + codes[2], space + scales[2], on))
    return rc;
  if (int rc = mb::launch_product(dtype, space + codes[0], space + scales[0], w_columns, scale_w, d_x, rows, k, n,
                                  nullptr, 1, nullptr, on))
    return rc;
  return mb::launch_product(dtype, space + codes[1], space + scales[1], space + codes[2], space + scales[2], d_w, n, k,
                            depth, nullptr, 1, nullptr, on);
}

}  // extern "C"
