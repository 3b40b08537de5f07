// FP8 operands with block scales: tensors to E4M3 codes, and back.
//
// A block along K of 128 elements of one row, or of 128 rows, shares a
// power-of-two scale 2^e, e the smallest integer with max|x| <= 448 * 2^e, at least
// -127 (the scale byte is e + 127, 0 for zeros), and holds every element as the
// E4M3 value nearest to x / 2^e, ties to the even code. A power of two because E4M3
// is a floating format: another scale would gain no precision, cost the product a
// multiplication for each of its sums, and round the quotient. A block that holds an
// infinity or a NaN gets the byte 255, the scale format's NaN, and codes 0.
//
// Codes are [rows][k rounded up to 16] bytes, zero past k; scales
// [ceil(k / 512)][ceil(rows / block)][4]: a dword of a row's (or 128 rows') next
// four blocks, 127 for blocks past k.
#include "mb_fp8.h"

#include "mb_fp8_device.h"

namespace mb {
namespace {

constexpr uint32_t kBlock = kFp8Block;

// Rows of x to codes and scales, a scale for each row's 128. A lane takes eight
// elements, 16 lanes a block, a wave U * 512 elements of one row: whole dwords of
// scales. With `slots` [rows][copies], row r goes to the operand's rows slots[r][0 ..
// copies), those outside 0 .. out_rows - 1 left out; without, to row r.
//
// Bound by memory: 8192 x 8192 of bf16 take 45 us cold (4.5 TB/s), 5000 x 4112 14.5,
// where a launch's start and end are a fifth; 4096 rows of 4096 to eight places each 34.
template <class T, int U, bool STREAM>
__global__ void __launch_bounds__(256)
    fp8_quantize_kernel(const T* __restrict__ x, uint32_t rows, uint32_t k, uint64_t row_stride,
                        const int32_t* __restrict__ slots, uint32_t copies, uint32_t out_rows,
                        uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t chunks = (k + U * 512 - 1) / (U * 512);
  const uint32_t row = __builtin_amdgcn_readfirstlane(blockIdx.x / chunks * 4 + (threadIdx.x >> 6));
  if (row >= rows) return;
  const uint32_t start = blockIdx.x % chunks * (U * 512) + lane * 8;
  const uint32_t pitch = (k + 15) / 16 * 16;
  Raw8<T> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t k0 = start + u * 512;
    raw[u].load(x + row * row_stride + k0, static_cast<int>(k > k0 ? k - k0 : 0));
  }
  elem_u32x2 word[U];
  uint32_t four[U];  // scales of the 512 elements
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t scale = fp8_scale_byte(magnitude_bits<T>(row16_magnitude<T>(raw_magnitude(raw[u]))));
    word[u] = fp8_encode8(raw[u], scale);
    const uint32_t k0 = start + u * 512;
    const uint32_t kept = k0 - lane % 16 * 8 < k ? scale : 127;
    four[u] = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b) four[u] |= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(kept), 16 * b)) << (8 * b);
  }
  for (uint32_t c = 0; c < copies; ++c) {
    const uint32_t out = slots ? static_cast<uint32_t>(slots[static_cast<uint64_t>(row) * copies + c]) : row;
    if (out >= out_rows) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t k0 = start + u * 512;
      if (k0 < pitch) {
        elem_u32x2* to = reinterpret_cast<elem_u32x2*>(codes + static_cast<uint64_t>(out) * pitch + k0);
        if constexpr (STREAM)
          __builtin_nontemporal_store(word[u], to);
        else
          *to = word[u];
      }
      if (lane == 0 && k0 < k)
        *reinterpret_cast<uint32_t*>(scales + (k0 / 512 * uint64_t{out_rows} + out) * 4) = four[u];
    }
  }
}

// ---- tiles: rows and columns at once -------------------------------------------

constexpr uint32_t kTileThreads = 256;

// Where a tile's codes go: an operand of `rows` rows of `pitch` bytes and `blocks`
// blocks of K, as many as its tiles cover.
struct TileOut {
  uint8_t *codes, *scales;
  uint32_t rows, pitch, blocks;
};

struct TileShared {
  uint32_t largest[kTileThreads / 64][kBlock];
  __attribute__((aligned(16))) uint8_t codes[kBlock * kBlock];
};

__device__ __forceinline__ void put_scale(const TileOut& out, uint32_t scale_row, uint32_t scale_rows, uint32_t block,
                                          uint32_t scale) {
  uint8_t* to = out.scales + (block / 4 * uint64_t{scale_rows} + scale_row) * 4;
  to[block % 4] = static_cast<uint8_t>(scale);
  if (block + 1 == out.blocks)
    for (uint32_t b = block % 4 + 1; b < 4; ++b) to[b] = 127;
}

// A tile of 128 x 128 elements to codes of its rows, of its columns (transposed), or
// both. Thread t holds columns 8 (t % 16) .. + 7 of rows 8 (t / 16) .. + 7, so that a
// row's block is a row of 16 lanes, and the eight codes of a column are eight bytes of
// the transposed operand; those cross LDS (chunks of eight XORed with the column's
// group, so that neither side meets its banks), and leave a column's 128 bytes
// together. SQUARE: one scale for the whole tile, the same both ways.
//
// Bound by memory, the tile read once for both: a weight of 6000 x 4112 in bf16 both ways
// takes 25 us (3.9 TB/s).
template <class T, bool SQUARE>
__device__ __forceinline__ void quantize_tile(const Raw8<T> (&at)[8], uint32_t row_tile, uint32_t column_tile,
                                              const TileOut& by_rows, const TileOut& by_columns, TileShared& shared) {
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t piece = threadIdx.x % 16, group = threadIdx.x / 16;  // columns 8 piece .., rows 8 group ..
  const uint32_t row0 = row_tile * kBlock + group * 8, column0 = column_tile * kBlock + piece * 8;
  uint32_t square = 0;
  if constexpr (SQUARE) {
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = join_magnitudes(T(), largest, raw_magnitude(at[i]));
    largest = row16_magnitude<T>(largest);
    largest = join_magnitudes(T(), largest, __shfl_xor(largest, 16, 64));
    largest = join_magnitudes(T(), largest, __shfl_xor(largest, 32, 64));
    if (lane == 0) shared.largest[wave][0] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < static_cast<int>(kTileThreads / 64); ++w)
      largest = join_magnitudes(T(), largest, shared.largest[w][0]);
    square = fp8_scale_byte(magnitude_bits<T>(largest));
    if (threadIdx.x == 0) {
      if (by_rows.codes) put_scale(by_rows, row_tile, (by_rows.rows + kBlock - 1) / kBlock, column_tile, square);
      if (by_columns.codes) put_scale(by_columns, column_tile, (by_columns.rows + kBlock - 1) / kBlock, row_tile, square);
    }
  }
  if (by_rows.codes) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t scale = square;
      if constexpr (!SQUARE) scale = fp8_scale_byte(magnitude_bits<T>(row16_magnitude<T>(raw_magnitude(at[i]))));
      const uint32_t row = row0 + i;
      if (row < by_rows.rows) {
        if (column0 < by_rows.pitch)
          *reinterpret_cast<elem_u32x2*>(by_rows.codes + static_cast<uint64_t>(row) * by_rows.pitch + column0) =
              fp8_encode8(at[i], scale);
        if (!SQUARE && piece == 0) put_scale(by_rows, row, by_rows.rows, column_tile, scale);
      }
    }
  }
  if (!by_columns.codes) return;
  uint32_t scales[8];  // of the eight columns
  if constexpr (SQUARE) {
#pragma unroll
    for (int c = 0; c < 8; ++c) scales[c] = square;
  } else {
    // Over the thread's rows as they are stored (pairs of 16-bit columns stay packed),
    // then over the wave's four threads of a column, then over the waves.
    constexpr int WORDS = 2 * sizeof(T);
    constexpr uint32_t kMask = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
    uint32_t largest[WORDS];
#pragma unroll
    for (int c = 0; c < WORDS; ++c) {
      largest[c] = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) largest[c] = join_magnitudes(T(), largest[c], at[i].part[c / 4][c % 4] & kMask);
      largest[c] = join_magnitudes(T(), largest[c], __shfl_xor(largest[c], 16, 64));
      largest[c] = join_magnitudes(T(), largest[c], __shfl_xor(largest[c], 32, 64));
      if (lane < 16) shared.largest[wave][piece * WORDS + c] = largest[c];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < WORDS; ++c)
#pragma unroll
      for (int w = 0; w < static_cast<int>(kTileThreads / 64); ++w)
        largest[c] = join_magnitudes(T(), largest[c], shared.largest[w][piece * WORDS + c]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint32_t one = largest[c * WORDS / 8];
      if constexpr (sizeof(T) == 2) one = c % 2 ? one >> 16 : one & 0xffffu;
      scales[c] = fp8_scale_byte(magnitude_bits<T>(one));
    }
    if (group == 0) {
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (column0 + c < by_columns.rows) put_scale(by_columns, column0 + c, by_columns.rows, row_tile, scales[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    Raw8<T> column;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (sizeof(T) == 4)
        column.part[i / 4][i % 4] = at[i].part[c / 4][c % 4];
      else if (i % 2 == 0)  // one half of each of two rows
        column.part[0][i / 2] = __builtin_amdgcn_perm(at[i + 1].part[0][c / 2], at[i].part[0][c / 2],
                                                      c % 2 ? 0x07060302u : 0x05040100u);
    }
    const uint32_t chunk = group ^ piece;
    *reinterpret_cast<elem_u32x2*>(shared.codes + (piece * 8 + c) * kBlock + chunk * 8) =
        fp8_encode8(column, scales[c]);
  }
  __syncthreads();
  const uint32_t k0 = row_tile * kBlock + piece * 8;
  if (k0 < by_columns.pitch) {
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const uint32_t column = c * 16 + group, row = column_tile * kBlock + column;
      if (row < by_columns.rows)
        *reinterpret_cast<elem_u32x2*>(by_columns.codes + static_cast<uint64_t>(row) * by_columns.pitch + k0) =
            *reinterpret_cast<const elem_u32x2*>(shared.codes + column * kBlock + ((piece ^ (column / 8)) * 8));
    }
  }
}

// Rows row0 .. + 7 of columns column0 .. + 7 of x, zeros outside.
template <class T>
__device__ __forceinline__ void load_tile(Raw8<T> (&at)[8], const T* __restrict__ x, uint32_t rows, uint32_t columns,
                                          uint64_t row_stride, uint32_t row0, uint32_t column0) {
  const int live = static_cast<int>(columns > column0 ? columns - column0 : 0);
#pragma unroll
  for (int i = 0; i < 8; ++i)
    at[i].load(x + (row0 + i) * row_stride + column0, row0 + i < rows ? live : 0);
}

// Workgroup `index` of `count`: XCD c (c, c + 8, ..) takes neighbouring ones, whose
// pieces of a row share lines.
__device__ __forceinline__ uint32_t xcd_first(uint32_t index, uint32_t count) {
  const uint32_t xcd = index % 8;
  return xcd * (count / 8) + min(xcd, count % 8) + index / 8;
}

template <class T, bool SQUARE>
__global__ void __launch_bounds__(kTileThreads)
    fp8_quantize_tiles_kernel(const T* __restrict__ x, uint32_t rows, uint32_t columns, uint64_t row_stride,
                              TileOut by_rows, TileOut by_columns) {
  __shared__ TileShared shared;
  const uint32_t across = (columns + kBlock - 1) / kBlock, pid = xcd_first(blockIdx.x, gridDim.x);
  const uint32_t row_tile = pid / across, column_tile = pid % across;
  Raw8<T> at[8];
  load_tile(at, x, rows, columns, row_stride, row_tile * kBlock + threadIdx.x / 16 * 8,
            column_tile * kBlock + threadIdx.x % 16 * 8);
  quantize_tile<T, SQUARE>(at, row_tile, column_tile, by_rows, by_columns, shared);
}

// Eight columns from column0 on of 2 * half of [gate | up] and of the gradient of
// silu(gate) * up, as they are stored.
template <class T>
struct GatePiece {
  Raw8<T> gate, up, d;

  // All of them of one half, j their first column in it.
  __device__ __forceinline__ void load(const T* gate_up, const T* d_row, uint32_t half, uint32_t j) {
    gate.load(gate_up + j);
    up.load(gate_up + half + j);
    d.load(d_row + j);
  }
  // Across the end of a half; zeros past the second.
  __device__ __forceinline__ void load_across(const T* gate_up, const T* d_row, uint32_t half, uint32_t column0) {
    T g[8], u[8], v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // (Not a choice between c and min(c - half, ..): the compiler drops it for the minimum of a difference that wraps.)
      const uint32_t c = column0 + i, j = min(c - (c < half ? 0 : half), half - 1);
      g[i] = gate_up[j];
      u[i] = gate_up[half + j];
      v[i] = c < 2 * half ? d_row[j] : T(0);
    }
    __builtin_memcpy(&gate, g, sizeof(gate));
    __builtin_memcpy(&up, u, sizeof(up));
    __builtin_memcpy(&d, v, sizeof(d));
  }
  // The gradient of [gate | up] in fp32:
  //   d_up = d gate s,  d_gate = d up s (1 + gate (1 - s)),  s = 1 / (1 + e^-gate).
  __device__ __forceinline__ Raw8<float> gradient(uint32_t half, uint32_t column0) const {
    Raw8<float> out;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float g = gate[i], by = d[i];
      const Sigmoid s = sigmoid(g);
      const float at_up = by * (g * s.value);
      const float at_gate = by * up[i] * (s.value * fmaf(g, s.complement, 1.0f));
      out.part[i / 4][i % 4] = float_bits(column0 + i >= half ? at_up : at_gate);
    }
    return out;
  }
};

// The operands of a product's gradients in one launch: d's rows and columns, tile by
// tile, and x's columns. With gate_up, d is computed on the way: a tile of d_up follows
// the tile of d_gate that reads the same, which it then finds in the XCD's L2.
//
// d 5000 x 3000 and x 5000 x 4112 in bf16 take 26 us, by memory (4.7 TB/s). With gate_up
// 67, for 42 of memory at that rate, by instructions: about 30 us of sigmoids and scales
// do not lie under the loads. Tiles of one side that leave out the other's half of the
// gradient, and four rows' loads in flight at a time, changed nothing (66 to 76).
template <class T, bool GATED>
__global__ void __launch_bounds__(kTileThreads)
    fp8_gradient_kernel(const T* __restrict__ d, uint64_t d_stride, const T* __restrict__ gate_up,
                        const T* __restrict__ x, uint64_t x_stride, uint32_t rows, uint32_t n, uint32_t k,
                        uint32_t d_tiles, TileOut d_rows, TileOut d_columns, TileOut x_columns) {
  __shared__ TileShared shared;
  const uint32_t group = threadIdx.x / 16 * 8, piece = threadIdx.x % 16 * 8;
  if (blockIdx.x >= d_tiles) {
    const uint32_t across = (k + kBlock - 1) / kBlock, pid = xcd_first(blockIdx.x - d_tiles, gridDim.x - d_tiles);
    const uint32_t row_tile = pid / across, column_tile = pid % across;
    Raw8<T> at[8];
    load_tile(at, x, rows, k, x_stride, row_tile * kBlock + group, column_tile * kBlock + piece);
    quantize_tile<T, false>(at, row_tile, column_tile, TileOut{}, x_columns, shared);
    return;
  }
  const uint32_t across = (n + kBlock - 1) / kBlock, pid = xcd_first(blockIdx.x, d_tiles);
  const uint32_t row_tile = pid / across;
  uint32_t column_tile = pid % across;
  if constexpr (GATED) {
    const uint32_t first = (across + 1) / 2;  // 0, first, 1, first + 1, ..
    column_tile = column_tile % 2 ? first + column_tile / 2 : column_tile / 2;
    const uint32_t half = n / 2, tile0 = column_tile * kBlock, column0 = tile0 + piece;
    const bool whole = tile0 + kBlock <= half || (tile0 >= half && tile0 + kBlock <= n);
    Raw8<float> at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t row = row_tile * kBlock + group + i;
      at[i] = Raw8<float>{};
      if (row < rows && column0 < n) {
        GatePiece<T> values;
        const T* pair = gate_up + static_cast<uint64_t>(row) * n;
        if (whole)
          values.load(pair, d + row * d_stride, half, column0 < half ? column0 : column0 - half);
        else
          values.load_across(pair, d + row * d_stride, half, column0);
        at[i] = values.gradient(half, column0);
      }
    }
    quantize_tile<float, false>(at, row_tile, column_tile, d_rows, d_columns, shared);
  } else {
    Raw8<T> at[8];
    load_tile(at, d, rows, n, d_stride, row_tile * kBlock + group, column_tile * kBlock + piece);
    quantize_tile<T, false>(at, row_tile, column_tile, d_rows, d_columns, shared);
  }
}

// Codes and scales to values, rounded once to T (exact in fp32, and in bf16 from 2^-133
// to its largest). A lane takes eight. 16384 x 8192 to bf16 take 74 us (5.4 TB/s).
template <class T, bool STREAM>
__global__ void __launch_bounds__(256)
    fp8_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
                          uint32_t rows, uint32_t k, uint32_t block) {
  const uint32_t per_row = (k + 7) / 8;
  const uint64_t index = blockIdx.x * uint64_t{256} + threadIdx.x;
  const uint64_t row = index / per_row;
  if (row >= rows) return;
  const uint32_t k0 = static_cast<uint32_t>(index % per_row) * 8;
  const elem_u32x2 word = *reinterpret_cast<const elem_u32x2*>(codes + row * ((k + 15) / 16 * 16) + k0);
  const uint32_t scale =
      scales[(k0 / 512 * uint64_t{(rows + block - 1) / block} + row / block) * 4 + k0 / kBlock % 4];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; i += 4) {
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word[i / 4]), false);
    const auto high = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word[i / 4]), true);
    v[i] = low[0], v[i + 1] = low[1], v[i + 2] = high[0], v[i + 3] = high[1];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    v[i] = scale == 255 ? __builtin_bit_cast(float, 0x7fc00000u)
                        : __builtin_amdgcn_ldexpf(v[i], static_cast<int>(scale) - 127);
  store8<STREAM>(out + row * k + k0, v, static_cast<int>(min(8u, k - k0)));
}

#define MB_FP8_REGISTER(T, NAME)                                                                \
  MB_REGISTER_KERNEL("fp8_quantize_" NAME "_512", (fp8_quantize_kernel<T, 1, false>));          \
  MB_REGISTER_KERNEL("fp8_quantize_" NAME "_1024", (fp8_quantize_kernel<T, 2, false>));         \
  MB_REGISTER_KERNEL("fp8_quantize_" NAME "_1024_stream", (fp8_quantize_kernel<T, 2, true>));   \
  MB_REGISTER_KERNEL("fp8_quantize_tiles_" NAME, (fp8_quantize_tiles_kernel<T, false>));        \
  MB_REGISTER_KERNEL("fp8_quantize_tiles_" NAME "_square", (fp8_quantize_tiles_kernel<T, true>)); \
  MB_REGISTER_KERNEL("fp8_gradient_" NAME, (fp8_gradient_kernel<T, false>));                    \
  MB_REGISTER_KERNEL("fp8_gradient_" NAME "_gated", (fp8_gradient_kernel<T, true>));            \
  MB_REGISTER_KERNEL("fp8_dequantize_" NAME, (fp8_dequantize_kernel<T, false>));                \
  MB_REGISTER_KERNEL("fp8_dequantize_" NAME "_stream", (fp8_dequantize_kernel<T, true>))
MB_FP8_REGISTER(float, "f32");
MB_FP8_REGISTER(_Float16, "f16");
MB_FP8_REGISTER(__bf16, "bf16");

TileOut tile_out(Fp8Out out, uint32_t rows, uint32_t k) {
  return TileOut{out.codes, out.scales, rows, static_cast<uint32_t>(fp8_pitch(k)), (k + kBlock - 1) / kBlock};
}

uint64_t tile_count_of(uint64_t rows, uint64_t columns) {
  return (rows + kBlock - 1) / kBlock * ((columns + kBlock - 1) / kBlock);
}

constexpr uint64_t kMostTiles = 0xffffff;

}  // namespace

int fp8_check_operand(const char* entry, const char* what, uint64_t rows, uint64_t k, uint64_t copies, uint32_t block,
                      const void* codes, uint64_t codes_bytes, const void* scales, uint64_t scales_bytes) {
  if (block != 1 && block != kFp8Block)
    return fail(MB_ERR_INVALID, "%s: a scale of %s stands for 1 or 128 rows, not %u", entry, what, block);
  if (codes == nullptr || scales == nullptr) return fail(MB_ERR_INVALID, "%s: %s codes or scales are NULL", entry, what);
  if (!aligned(codes, 16) || !aligned(scales, 4))
    return fail(MB_ERR_ALIGNMENT, "%s: %s codes must lie on 16 bytes and scales on 4", entry, what);
  if (codes_bytes < copies * fp8_code_bytes(rows, k) || scales_bytes < copies * fp8_scale_bytes(rows, k, block))
    return fail(MB_ERR_INVALID, "%s: %s of %llu x %llu x %llu needs %llu code and %llu scale bytes; too small", entry,
                what, (unsigned long long)copies, (unsigned long long)rows, (unsigned long long)k,
                (unsigned long long)(copies * fp8_code_bytes(rows, k)),
                (unsigned long long)(copies * fp8_scale_bytes(rows, k, block)));
  return MB_OK;
}

int fp8_check_rows(const char* entry, const char* what, int dtype, const void* x, uint64_t x_bytes, uint64_t rows,
                   uint64_t k, uint64_t row_stride) {
  const uint32_t item = elem_bytes(dtype);
  if (!item) return fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (x == nullptr) return fail(MB_ERR_INVALID, "%s: %s is NULL", entry, what);
  if (!aligned(x, item))
    return fail(MB_ERR_ALIGNMENT, "%s: %s must lie on its elements' %u bytes", entry, what, item);
  if (rows > kFp8MostRows || k > kFp8MostK)
    return fail(MB_ERR_UNSUPPORTED, "%s: %s of %llu x %llu: at most %u rows of at most %u elements", entry, what,
                (unsigned long long)rows, (unsigned long long)k, kFp8MostRows, kFp8MostK);
  if (row_stride > UINT64_MAX / 8 / (rows ? rows : 1) || strided_bytes(rows, k, row_stride, item) > x_bytes)
    return fail(MB_ERR_INVALID, "%s: %s is too small for %llu rows of %llu elements at a stride of %llu", entry, what,
                (unsigned long long)rows, (unsigned long long)k, (unsigned long long)row_stride);
  return MB_OK;
}

int fp8_check_output(const char* entry, const char* what, int dtype, const void* y, uint64_t y_bytes, uint64_t rows,
                     uint64_t n) {
  const uint32_t item = elem_bytes(dtype);
  if (!item) return fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (y == nullptr || y_bytes < rows * n * item)
    return fail(MB_ERR_INVALID, "%s: %s is NULL or too small for %llu x %llu", entry, what, (unsigned long long)rows,
                (unsigned long long)n);
  if (!aligned(y, item))
    return fail(MB_ERR_ALIGNMENT, "%s: %s must lie on its elements' %u bytes", entry, what, item);
  return MB_OK;
}

int fp8_launch_quantize(int dtype, const void* x, uint32_t rows, uint32_t k, uint64_t row_stride, const int32_t* slots,
                        uint32_t copies, uint32_t out_rows, void* codes, void* scales, hipStream_t stream) {
  const uint32_t elements = k > 512 ? 1024 : 512;  // of a row and wave
  const uint64_t grid = (rows + uint64_t{3}) / 4 * ((k + elements - 1) / elements);
  if (grid > 0xffffffu) return fail(MB_ERR_UNSUPPORTED, "fp8_quantize: %u x %u exceeds one launch", rows, k);
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(256), 0, stream>>>(
        static_cast<const decltype(t)*>(x), rows, k, row_stride, slots, copies, out_rows,
        static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
  };
  const bool streamed = streams(fp8_code_bytes(uint64_t{rows} * copies, k));
  MB_FOR_DTYPE(dtype, {
    if (k <= 512)
      launch(fp8_quantize_kernel<T, 1, false>, T());
    else if (streamed)
      launch(fp8_quantize_kernel<T, 2, true>, T());
    else
      launch(fp8_quantize_kernel<T, 2, false>, T());
  });
  return launch_status("fp8_quantize");
}

int fp8_launch_gradient(int dtype, const void* d_out, uint64_t d_stride, const void* gate_up, const void* x,
                        uint64_t x_stride, uint32_t rows, uint32_t n, uint32_t k, uint32_t depth, Fp8Out d_rows,
                        Fp8Out d_columns, Fp8Out x_columns, hipStream_t stream) {
  const uint64_t d_tiles = tile_count_of(depth, n), x_tiles = tile_count_of(depth, k);
  if (d_tiles + x_tiles > kMostTiles)
    return fail(MB_ERR_UNSUPPORTED, "fp8_gradient: %u x %u x %u exceeds one launch", rows, n, k);
  auto launch = [&](auto kernel, auto t) {
    using T = decltype(t);
    kernel<<<dim3(static_cast<uint32_t>(d_tiles + x_tiles)), dim3(kTileThreads), 0, stream>>>(
        static_cast<const T*>(d_out), d_stride, static_cast<const T*>(gate_up), static_cast<const T*>(x), x_stride,
        rows, n, k, static_cast<uint32_t>(d_tiles), tile_out(d_rows, rows, n), tile_out(d_columns, n, depth),
        tile_out(x_columns, k, depth));
  };
  MB_FOR_DTYPE(dtype, {
    if (gate_up)
      launch(fp8_gradient_kernel<T, true>, T());
    else
      launch(fp8_gradient_kernel<T, false>, T());
  });
  return launch_status("fp8_gradient");
}

}  // namespace mb

extern "C" {

int mb_fp8_quantize(int dtype, const void* x, uint64_t x_bytes, uint32_t rows, uint32_t k, uint64_t row_stride,
                    const int32_t* slots, uint64_t slots_bytes, uint32_t copies, uint32_t out_rows, void* codes,
                    uint64_t codes_bytes, void* scales, uint64_t scales_bytes, void* stream) {
  const char* entry = "mb_fp8_quantize";
  if (!mb::elem_bytes(dtype)) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (rows == 0 || k == 0) return MB_OK;
  if (int rc = mb::fp8_check_rows(entry, "x", dtype, x, x_bytes, rows, k, row_stride)) return rc;
  if (slots == nullptr) {
    copies = 1;
    out_rows = rows;
  } else if (copies == 0 || copies > 64 || slots_bytes < uint64_t{rows} * copies * 4) {
    return mb::fail(MB_ERR_INVALID, "%s: slots must hold 1 to 64 entries for each of %u rows", entry, rows);
  } else if (!mb::aligned(slots, 4)) {
    return mb::fail(MB_ERR_ALIGNMENT, "%s: slots must lie on 4 bytes", entry);
  }
  if (out_rows > mb::kFp8MostRows)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: at most %u operand rows", entry, mb::kFp8MostRows);
  if (int rc = mb::fp8_check_operand(entry, "the operand", out_rows, k, 1, 1, codes, codes_bytes, scales, scales_bytes))
    return rc;
  return mb::fp8_launch_quantize(dtype, x, rows, k, row_stride, slots, copies, out_rows, codes, scales,
                                 static_cast<hipStream_t>(stream));
}

int mb_fp8_quantize_both(int dtype, const void* x, uint64_t x_bytes, uint32_t rows, uint32_t columns,
                         uint64_t row_stride, uint32_t block, void* codes, uint64_t codes_bytes, void* scales,
                         uint64_t scales_bytes, void* column_codes, uint64_t column_codes_bytes, void* column_scales,
                         uint64_t column_scales_bytes, void* stream) {
  const char* entry = "mb_fp8_quantize_both";
  if (!mb::elem_bytes(dtype)) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (block != 1 && block != mb::kFp8Block)
    return mb::fail(MB_ERR_INVALID, "%s: a scale stands for 1 or 128 rows, not %u", entry, block);
  if (rows == 0 || columns == 0 || (codes == nullptr && column_codes == nullptr)) return MB_OK;
  if (int rc = mb::fp8_check_rows(entry, "x", dtype, x, x_bytes, rows, columns, row_stride)) return rc;
  if (codes)
    if (int rc = mb::fp8_check_operand(entry, "the rows'", rows, columns, 1, block, codes, codes_bytes, scales,
                                       scales_bytes))
      return rc;
  if (column_codes) {
    if (columns > mb::kFp8MostRows || rows > mb::kFp8MostK)
      return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u: at most %u rows", entry, rows, columns, mb::kFp8MostK);
    if (int rc = mb::fp8_check_operand(entry, "the columns'", columns, rows, 1, block, column_codes,
                                       column_codes_bytes, column_scales, column_scales_bytes))
      return rc;
  }
  const uint64_t grid = mb::tile_count_of(rows, columns);
  if (grid > mb::kMostTiles)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u exceeds one launch", entry, rows, columns);
  const mb::Fp8Out by_rows{static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)};
  const mb::Fp8Out by_columns{static_cast<uint8_t*>(column_codes), static_cast<uint8_t*>(column_scales)};
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(mb::kTileThreads), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const decltype(t)*>(x), rows, columns, row_stride, mb::tile_out(by_rows, rows, columns),
        mb::tile_out(by_columns, columns, rows));
  };
  MB_FOR_DTYPE(dtype, {
    if (block == 1)
      launch(mb::fp8_quantize_tiles_kernel<T, false>, T());
    else
      launch(mb::fp8_quantize_tiles_kernel<T, true>, T());
  });
  return mb::launch_status("fp8_quantize_tiles");
}

int mb_fp8_dequantize(int dtype, const void* codes, uint64_t codes_bytes, const void* scales, uint64_t scales_bytes,
                      uint32_t block, void* out, uint64_t out_bytes, uint32_t rows, uint32_t k, void* stream) {
  const char* entry = "mb_fp8_dequantize";
  const uint32_t item = mb::elem_bytes(dtype);
  if (!item) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (rows == 0 || k == 0) return MB_OK;
  if (rows > mb::kFp8MostRows || k > mb::kFp8MostK)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u: at most %u rows of at most %u elements", entry, rows, k,
                    mb::kFp8MostRows, mb::kFp8MostK);
  if (int rc = mb::fp8_check_operand(entry, "the operand", rows, k, 1, block, codes, codes_bytes, scales,
                                     scales_bytes))
    return rc;
  if (int rc = mb::fp8_check_output(entry, "out", dtype, out, out_bytes, rows, k)) return rc;
  const uint64_t grid = (uint64_t{rows} * ((k + 7) / 8) + 255) / 256;
  if (grid > 0xffffffu) return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u exceeds one launch", entry, rows, k);
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<decltype(t)*>(out), rows,
        k, block);
  };
  const bool streamed = mb::streams(uint64_t{rows} * k * item);
  MB_FOR_DTYPE(dtype, {
    if (streamed)
      launch(mb::fp8_dequantize_kernel<T, true>, T());
    else
      launch(mb::fp8_dequantize_kernel<T, false>, T());
  });
  return mb::launch_status("fp8_dequantize");
}

}  // extern "C"
