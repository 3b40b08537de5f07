// MX quantisation: tensors to MXFP4 operands of the GEMMs, and back.
//
// A group of 32 elements along K shares a power-of-two scale 2^e,
//   e = clamp(floor(log2 max|x|) - 2, -127, 127)   (-127 for a group of zeros),
// and holds every element as the E2M1 value nearest to x / 2^e (ties to the even
// code, saturating at 6). floor(log2) - 2 puts the largest element into [4, 8),
// E2M1's top binade. The scale byte is S = e + 127; with the fp32 exponent field
// f of max|x| it is max(f - 2, 0). A group that holds an infinity or a NaN has no
// such scale: S = 255, the format's NaN, codes 0.
//
// Codes are [rows][ceil(k / 32) * 16] bytes, even k in the low nibble, zero past
// k; scales [ceil(k / 256)][rows][8], 127 for groups past k: mb_gemm's operands.
#include "mb_mx.h"
#include "mb_mx_device.h"

namespace mb {
namespace {

constexpr uint32_t kGroup = 32;   // elements sharing a scale
constexpr uint32_t kBlock = 256;  // elements along K whose 8 scales a row holds together

__device__ __forceinline__ float bits_float(uint32_t v) { return __builtin_bit_cast(float, v); }

// Rows of x to codes and scales. A lane takes eight elements, four lanes a
// group, a wave U * 512 elements of one row, a workgroup WAVES rows. With `slots`
// [rows][copies], row r goes to the operand's rows slots[r][0 .. copies), those
// outside 0 .. out_rows - 1 left out; without, to row r. STREAM as in store8.
//
// Bound by HBM: 8192x8192 bf16 29.0 us (5.9 TB/s; streamed 28.8), 8192x4096 to
// four rows each 28.0 streamed (4.9 TB/s), not 30.7. Two loads a lane: with one
// 30.8 and 29.0, with four 31.4 and 32.0; one where a row has no more (16384x512
// 5.4 us, with two 6.2). Half a wave a row, whose operand rows are written in
// pieces of 128 bytes, took 29.7 and 33.6.
template <class T, int U, bool STREAM, int WAVES>
__device__ __forceinline__ void quantize_rows(const T* __restrict__ x, uint32_t rows, uint32_t k, uint64_t row_stride,
                                              const int32_t* __restrict__ slots, uint32_t copies, uint32_t out_rows,
                                              uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                              uint32_t index) {
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t chunks = (k + U * 512 - 1) / (U * 512);
  const uint32_t row = __builtin_amdgcn_readfirstlane(index / chunks * WAVES + (threadIdx.x >> 6));
  if (row >= rows) return;
  const uint32_t start = index % chunks * (U * 512) + lane * 8;
  const uint32_t code_bytes = (k + kGroup - 1) / kGroup * 16, blocks = (k + kBlock - 1) / kBlock;
  Raw8<T> raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t k0 = start + u * 512;
    raw[u].load(x + row * row_stride + k0, static_cast<int>(k > k0 ? k - k0 : 0));
  }
  uint32_t word[U], scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint32_t largest = raw_magnitude(raw[u]);
    largest = join_magnitudes(T(), largest, quad_swap<kQuadXor1>(largest));
    largest = join_magnitudes(T(), largest, quad_swap<kQuadXor2>(largest));
    scale[u] = scale_byte(magnitude_bits<T>(largest));
    word[u] = encode8(raw[u], scale[u]);
    if (start + u * 512 >= k) scale[u] = 127;  // groups past K
  }
  for (uint32_t c = 0; c < copies; ++c) {
    const uint32_t out = slots ? static_cast<uint32_t>(slots[static_cast<uint64_t>(row) * copies + c]) : row;
    if (out >= out_rows) continue;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t k0 = start + u * 512;
      if (k0 / 2 < code_bytes) {
        uint32_t* to = reinterpret_cast<uint32_t*>(codes + static_cast<uint64_t>(out) * code_bytes + k0 / 2);
        if constexpr (STREAM)
          __builtin_nontemporal_store(word[u], to);
        else
          *to = word[u];
      }
      if (lane % 4 == 0 && k0 / kBlock < blocks)
        scales[(static_cast<uint64_t>(k0 / kBlock) * out_rows + out) * 8 + k0 % kBlock / kGroup] =
            static_cast<uint8_t>(scale[u]);
    }
  }
}

template <class T, int U, bool STREAM>
__global__ void __launch_bounds__(256)
    mx_quantize_kernel(const T* __restrict__ x, uint32_t rows, uint32_t k, uint64_t row_stride,
                       const int32_t* __restrict__ slots, uint32_t copies, uint32_t out_rows,
                       uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  quantize_rows<T, U, STREAM, 4>(x, rows, k, row_stride, slots, copies, out_rows, codes, scales, blockIdx.x);
}

// Columns of x to the rows of the transposed operand: groups of 32 run along
// x's rows. A workgroup takes 256 rows of 128 columns, a wave a group of 32
// rows, a lane two neighbouring columns, so that a group's largest magnitude
// needs no other lane and stays packed; the codes cross LDS, so that an operand
// row's 128 bytes leave together. An operand row holds `groups` groups, as many as
// the rows fill or, of zeros, up to the end of their block of 256.
//
// Bound by the memory's rate for 256 bytes a row: 8192x8192 bf16 36.9 us from HBM
// (4.6 TB/s; with 512 bytes a row 37.5), 25.0 from the memory-side cache (6.8).
// Rows off the lines lose if neighbouring strips run on different XCDs (8192x8190
// 48.9 us, so 39.0). A column at a time and unpacked took 20 instructions an
// element and 54 us from the cache.
constexpr int kTileColumns = 128, kTilePitch = 128 + 16;  // LDS bytes of a column, a bank group apart

// 32 rows of two columns, a pair a row as it is stored.
template <class T>
struct ColumnPairs {
  typedef uint32_t Pair __attribute__((ext_vector_type(sizeof(T) / 2), aligned(sizeof(T))));
  typedef uint32_t Word __attribute__((ext_vector_type(sizeof(T) / 2)));
  Word at[32];

  // Largest magnitudes of the columns, in the form of magnitude_bits.
  __device__ __forceinline__ void largest(uint32_t (&out)[2]) const {
    if constexpr (sizeof(T) == 4) {
      out[0] = out[1] = 0;
#pragma unroll
      for (int r = 0; r < 32; ++r) {
        out[0] = max(out[0], at[r][0] & 0x7fffffffu);
        out[1] = max(out[1], at[r][1] & 0x7fffffffu);
      }
    } else {
      uint32_t both = 0;
#pragma unroll
      for (int r = 0; r < 32; ++r) both = join_magnitudes(T(), both, word(r) & 0x7fff7fffu);
      out[0] = both & 0xffffu;
      out[1] = both >> 16;
    }
  }
  // Rows 8q .. 8q + 7 of a column.
  template <int COLUMN>
  __device__ __forceinline__ Raw8<T> piece(int q) const {
    Raw8<T> raw;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 8 * q + i;
      if constexpr (sizeof(T) == 4)
        raw.part[i / 4][i % 4] = at[r][COLUMN];
      else if (i % 2 == 0)  // one 16-bit half of each of two rows
        raw.part[0][i / 2] =
            __builtin_amdgcn_perm(word(r + 1), word(r), COLUMN ? 0x07060302u : 0x05040100u);
    }
    return raw;
  }

 private:
  __device__ __forceinline__ uint32_t word(int r) const { return at[r][0]; }
};

template <class T, int COLUMN>
__device__ __forceinline__ void quantize_column(const ColumnPairs<T>& values, uint32_t largest, uint8_t* codes,
                                                uint8_t* scale_at) {
  const uint32_t scale = scale_byte(magnitude_bits<T>(largest));
  elem_u32x4 word;
#pragma unroll
  for (int q = 0; q < 4; ++q) word[q] = encode8(values.template piece<COLUMN>(q), scale);
  *reinterpret_cast<elem_u32x4*>(codes) = word;
  *scale_at = static_cast<uint8_t>(scale);
}

template <class T, bool STREAM>
__device__ __forceinline__ void quantize_columns(const T* __restrict__ x, uint32_t rows, uint32_t columns,
                                                 uint64_t row_stride, uint32_t groups, uint8_t* __restrict__ codes,
                                                 uint8_t* __restrict__ scales, uint32_t index, uint32_t count) {
  __shared__ __attribute__((aligned(16))) uint8_t tile[kTileColumns * kTilePitch];
  __shared__ __attribute__((aligned(8))) uint8_t tile_scales[kTileColumns * 8];
  using Pair = typename ColumnPairs<T>::Pair;
  const uint32_t strips = (columns + kTileColumns - 1) / kTileColumns;
  // XCD c (workgroups c, c + 8, ..) takes neighbouring strips, whose pieces of a row share lines.
  const uint32_t xcd = index % 8;
  const uint32_t pid = xcd * (count / 8) + min(xcd, count % 8) + index / 8;
  const uint32_t strip = pid % strips, block = pid / strips;
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t local = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t group = block * 8 + local, column = lane * 2;
  const uint32_t live = min(static_cast<uint32_t>(kTileColumns), columns - strip * kTileColumns);
  if (group < groups) {
    const uint32_t row0 = group * kGroup;
    const T* from = x + row0 * row_stride + strip * kTileColumns;
    ColumnPairs<T> values;
    if (row0 + kGroup <= rows && live == kTileColumns) {
#pragma unroll
      for (int r = 0; r < 32; ++r, from += row_stride) {
        const Pair* pair = reinterpret_cast<const Pair*>(from + column);
        values.at[r] = STREAM ? __builtin_nontemporal_load(pair) : *pair;
      }
    } else {
#pragma unroll
      for (int r = 0; r < 32; ++r, from += row_stride) {
        T pair[2] = {T(0), T(0)};
        if (row0 + r < rows) {
          if (column < live) pair[0] = from[column];
          if (column + 1 < live) pair[1] = from[column + 1];
        }
        __builtin_memcpy(&values.at[r], pair, sizeof(pair));
      }
    }
    uint32_t largest[2];
    values.largest(largest);
    quantize_column<T, 0>(values, largest[0], tile + column * kTilePitch + local * 16, tile_scales + column * 8 + local);
    quantize_column<T, 1>(values, largest[1], tile + (column + 1) * kTilePitch + local * 16,
                          tile_scales + (column + 1) * 8 + local);
  } else {
    tile_scales[column * 8 + local] = tile_scales[(column + 1) * 8 + local] = 127;
  }
  __syncthreads();
  const uint64_t first = strip * uint64_t{kTileColumns};
  for (uint32_t i = threadIdx.x; i < live * 8; i += 512) {
    const uint32_t c = i / 8, chunk = i % 8;
    if (block * 8 + chunk >= groups) continue;
    elem_u32x4* to = reinterpret_cast<elem_u32x4*>(codes + ((first + c) * groups + block * 8 + chunk) * 16);
    const elem_u32x4 word = *reinterpret_cast<const elem_u32x4*>(tile + c * kTilePitch + chunk * 16);
    if constexpr (STREAM)
      __builtin_nontemporal_store(word, to);
    else
      *to = word;
  }
  if (threadIdx.x < live)
    *reinterpret_cast<elem_u32x2*>(scales + (block * uint64_t{columns} + first + threadIdx.x) * 8) =
        *reinterpret_cast<const elem_u32x2*>(tile_scales + threadIdx.x * 8);
}

template <class T, bool STREAM>
__global__ void __launch_bounds__(512)
    mx_quantize_columns_kernel(const T* __restrict__ x, uint32_t rows, uint32_t columns, uint64_t row_stride,
                               uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  quantize_columns<T, STREAM>(x, rows, columns, row_stride, (rows + kGroup - 1) / kGroup, codes, scales, blockIdx.x,
                              gridDim.x);
}

// The operands of a linear layer's gradient in one launch: the rows and the
// columns of d [rows][n] and the columns of x [rows][k]. The tails of the three
// run beside each other: 5000x3000 and 5000x4112 bf16 21.7 us, in three launches
// 28.5; the gradient of a small layer (64x256x256), which the launches bound,
// 14.2 for 19.6. The columns' operands have `depth` >= rows elements of K, zeros
// past the rows.
template <class T, bool STREAM>
__global__ void __launch_bounds__(512)
    mx_quantize_gradient_kernel(const T* __restrict__ d, uint64_t d_stride, const T* __restrict__ x, uint64_t x_stride,
                                uint32_t rows, uint32_t n, uint32_t k, uint32_t depth, uint8_t* __restrict__ d_codes,
                                uint8_t* __restrict__ d_scales, uint8_t* __restrict__ d_columns,
                                uint8_t* __restrict__ d_column_scales, uint8_t* __restrict__ x_columns,
                                uint8_t* __restrict__ x_column_scales, uint32_t d_tiles, uint32_t x_tiles) {
  const uint32_t index = blockIdx.x;
  if (index < d_tiles + x_tiles) {
    const bool first = index < d_tiles;
    quantize_columns<T, STREAM>(first ? d : x, rows, first ? n : k, first ? d_stride : x_stride,
                                depth / kGroup, first ? d_columns : x_columns, first ? d_column_scales : x_column_scales,
                                first ? index : index - d_tiles, first ? d_tiles : x_tiles);
  } else {
    quantize_rows<T, 2, STREAM, 8>(d, rows, n, d_stride, nullptr, 1, rows, d_codes, d_scales,
                                   index - d_tiles - x_tiles);
  }
}

// Codes and scales to values, rounded once to T (exact in fp32 and bf16).
template <class T, bool STREAM>
__global__ void __launch_bounds__(256)
    mx_dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
                         uint32_t rows, uint32_t k) {
  const uint32_t per_row = (k + 7) / 8;
  const uint64_t index = blockIdx.x * uint64_t{256} + threadIdx.x;
  const uint64_t row = index / per_row;
  if (row >= rows) return;
  const uint32_t k0 = static_cast<uint32_t>(index % per_row) * 8;
  const uint32_t code_bytes = (k + kGroup - 1) / kGroup * 16;
  const uint32_t word = *reinterpret_cast<const uint32_t*>(codes + row * code_bytes + k0 / 2);
  const uint32_t scale = scales[(k0 / kBlock * uint64_t{rows} + row) * 8 + k0 % kBlock / kGroup];
  float v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t code = word >> (4 * i) & 15u;
    const float unit = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.0f, 0)[0];
    v[i] = scale == 255 ? bits_float(0x7fc00000u) : __builtin_amdgcn_ldexpf(unit, static_cast<int>(scale) - 127);
  }
  store8<STREAM>(out + row * k + k0, v, static_cast<int>(min(8u, k - k0)));
}

#define MB_MX_REGISTER(T, NAME)                                      \
  MB_REGISTER_KERNEL("mx_quantize_" NAME "_512", (mx_quantize_kernel<T, 1, false>));           \
  MB_REGISTER_KERNEL("mx_quantize_" NAME "_1024", (mx_quantize_kernel<T, 2, false>));          \
  MB_REGISTER_KERNEL("mx_quantize_" NAME "_1024_stream", (mx_quantize_kernel<T, 2, true>));    \
  MB_REGISTER_KERNEL("mx_quantize_columns_" NAME, (mx_quantize_columns_kernel<T, false>));     \
  MB_REGISTER_KERNEL("mx_quantize_columns_" NAME "_stream", (mx_quantize_columns_kernel<T, true>)); \
  MB_REGISTER_KERNEL("mx_quantize_gradient_" NAME, (mx_quantize_gradient_kernel<T, false>));   \
  MB_REGISTER_KERNEL("mx_quantize_gradient_" NAME "_stream", (mx_quantize_gradient_kernel<T, true>)); \
  MB_REGISTER_KERNEL("mx_dequantize_" NAME, (mx_dequantize_kernel<T, false>)); \
  MB_REGISTER_KERNEL("mx_dequantize_" NAME "_stream", (mx_dequantize_kernel<T, true>))
MB_MX_REGISTER(float, "f32");
MB_MX_REGISTER(_Float16, "f16");
MB_MX_REGISTER(__bf16, "bf16");

}  // namespace

int check_operand(const char* entry, const char* what, uint64_t rows, uint64_t k, uint64_t copies, const void* codes,
                  uint64_t codes_bytes, const void* scales, uint64_t scales_bytes) {
  if (codes == nullptr || scales == nullptr) return fail(MB_ERR_INVALID, "%s: %s codes or scales are NULL", entry, what);
  if (!aligned(codes, 16) || !aligned(scales, 8))
    return fail(MB_ERR_ALIGNMENT, "%s: %s codes must lie on 16 bytes and scales on 8", entry, what);
  if (codes_bytes < copies * mx_code_bytes(rows, k) || scales_bytes < copies * mx_scale_bytes(rows, k))
    return fail(MB_ERR_INVALID, "%s: %s of %llu x %llu x %llu needs %llu code and %llu scale bytes; too small", entry,
                what, (unsigned long long)copies, (unsigned long long)rows, (unsigned long long)k,
                (unsigned long long)(copies * mx_code_bytes(rows, k)),
                (unsigned long long)(copies * mx_scale_bytes(rows, k)));
  return MB_OK;
}

int check_rows(const char* entry, int dtype, const void* x, uint64_t x_bytes, uint64_t rows, uint64_t k,
               uint64_t row_stride) {
  const uint32_t item = elem_bytes(dtype);
  if (!item) return fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (x == nullptr) return fail(MB_ERR_INVALID, "%s: x is NULL", entry);
  if (!aligned(x, item)) return fail(MB_ERR_ALIGNMENT, "%s: x must lie on its elements' %u bytes", entry, item);
  if (rows > kMxMostRows || k > kMxMostK)
    return fail(MB_ERR_UNSUPPORTED, "%s: %llu x %llu: at most %u rows of at most %u elements", entry,
                (unsigned long long)rows, (unsigned long long)k, kMxMostRows, kMxMostK);
  if (row_stride > UINT64_MAX / 8 / (rows ? rows : 1) || strided_bytes(rows, k, row_stride, item) > x_bytes)
    return fail(MB_ERR_INVALID, "%s: x is too small for %llu rows of %llu elements at a stride of %llu", entry,
                (unsigned long long)rows, (unsigned long long)k, (unsigned long long)row_stride);
  return MB_OK;
}

int launch_quantize(int dtype, const void* x, uint32_t rows, uint32_t k, uint64_t row_stride, const int32_t* slots,
                    uint32_t copies, uint32_t out_rows, void* codes, void* scales, hipStream_t stream) {
  const uint32_t elements = k > 512 ? 1024 : 512;  // of a row and wave
  const uint64_t grid = (rows + uint64_t{3}) / 4 * ((k + elements - 1) / elements);
  if (grid > 0xffffffu) return fail(MB_ERR_UNSUPPORTED, "mx_quantize: %u x %u exceeds one launch", rows, k);
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(256), 0, stream>>>(
        static_cast<const decltype(t)*>(x), rows, k, row_stride, slots, copies, out_rows,
        static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales));
  };
  const bool streamed = streams(mx_code_bytes(uint64_t{rows} * copies, k));
  MB_FOR_DTYPE(dtype, {
    if (k <= 512)
      launch(mx_quantize_kernel<T, 1, false>, T());
    else if (streamed)
      launch(mx_quantize_kernel<T, 2, true>, T());
    else
      launch(mx_quantize_kernel<T, 2, false>, T());
  });
  return launch_status("mx_quantize");
}

static uint64_t column_tiles(uint32_t rows, uint32_t columns) {
  return (columns + uint64_t{kTileColumns} - 1) / kTileColumns * ((rows + uint64_t{kBlock} - 1) / kBlock);
}

static int launch_quantize_columns(int dtype, const void* x, uint32_t rows, uint32_t columns, uint64_t row_stride,
                                   void* codes, void* scales, hipStream_t stream) {
  const uint64_t grid = column_tiles(rows, columns);
  if (grid > 0x7fffffu)
    return fail(MB_ERR_UNSUPPORTED, "mx_quantize_columns: %u x %u exceeds one launch", rows, columns);
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(512), 0, stream>>>(
        static_cast<const decltype(t)*>(x), rows, columns, row_stride, static_cast<uint8_t*>(codes),
        static_cast<uint8_t*>(scales));
  };
  const bool streamed = streams(mx_code_bytes(columns, rows));
  MB_FOR_DTYPE(dtype, {
    if (streamed)
      launch(mx_quantize_columns_kernel<T, true>, T());
    else
      launch(mx_quantize_columns_kernel<T, false>, T());
  });
  return launch_status("mx_quantize_columns");
}

int launch_quantize_gradient(int dtype, const void* d, uint64_t d_stride, const void* x, uint64_t x_stride,
                             uint32_t rows, uint32_t n, uint32_t k, uint32_t depth, void* d_codes, void* d_scales,
                             void* d_columns, void* d_column_scales, void* x_columns, void* x_column_scales,
                             hipStream_t stream) {
  const uint64_t d_tiles = column_tiles(rows, n), x_tiles = column_tiles(rows, k);
  const uint64_t grid = d_tiles + x_tiles + (rows + uint64_t{7}) / 8 * ((n + uint64_t{1023}) / 1024);
  if (grid > 0x7fffffu)
    return fail(MB_ERR_UNSUPPORTED, "mx_quantize_gradient: %u x %u x %u exceeds one launch", rows, n, k);
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(512), 0, stream>>>(
        static_cast<const decltype(t)*>(d), d_stride, static_cast<const decltype(t)*>(x), x_stride, rows, n, k, depth,
        static_cast<uint8_t*>(d_codes), static_cast<uint8_t*>(d_scales), static_cast<uint8_t*>(d_columns),
        static_cast<uint8_t*>(d_column_scales), static_cast<uint8_t*>(x_columns),
        static_cast<uint8_t*>(x_column_scales), static_cast<uint32_t>(d_tiles), static_cast<uint32_t>(x_tiles));
  };
  const bool streamed = streams(mx_code_bytes(rows, n) + mx_code_bytes(n, depth) + mx_code_bytes(k, depth));
  MB_FOR_DTYPE(dtype, {
    if (streamed)
      launch(mx_quantize_gradient_kernel<T, true>, T());
    else
      launch(mx_quantize_gradient_kernel<T, false>, T());
  });
  return launch_status("mx_quantize_gradient");
}

}  // namespace mb

extern "C" {

int mb_mx_quantize(int dtype, const void* x, uint64_t x_bytes, uint32_t rows, uint32_t k, uint64_t row_stride,
                   const int32_t* slots, uint64_t slots_bytes, uint32_t copies, uint32_t out_rows, void* codes,
                   uint64_t codes_bytes, void* scales, uint64_t scales_bytes, void* stream) {
  const char* entry = "mb_mx_quantize";
  if (rows == 0 || k == 0) return mb::elem_bytes(dtype) ? MB_OK
                                                        : mb::fail(MB_ERR_INVALID, "%s: unknown element type %d",
                                                                   entry, dtype);
  if (int rc = mb::check_rows(entry, dtype, x, x_bytes, rows, k, row_stride)) return rc;
  if (slots == nullptr) {
    copies = 1;
    out_rows = rows;
  } else if (copies == 0 || copies > 64 || slots_bytes < uint64_t{rows} * copies * 4) {
    return mb::fail(MB_ERR_INVALID, "%s: slots must hold 1 to 64 entries for each of %u rows", entry, rows);
  } else if (!mb::aligned(slots, 4)) {
    return mb::fail(MB_ERR_ALIGNMENT, "%s: slots must lie on 4 bytes", entry);
  }
  if (out_rows > mb::kMxMostRows)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: at most %u operand rows", entry, mb::kMxMostRows);
  if (int rc = mb::check_operand(entry, "the operand", out_rows, k, 1, codes, codes_bytes, scales, scales_bytes))
    return rc;
  return mb::launch_quantize(dtype, x, rows, k, row_stride, slots, copies, out_rows, codes, scales,
                             static_cast<hipStream_t>(stream));
}

int mb_mx_quantize_columns(int dtype, const void* x, uint64_t x_bytes, uint32_t rows, uint32_t columns,
                           uint64_t row_stride, void* codes, uint64_t codes_bytes, void* scales,
                           uint64_t scales_bytes, void* stream) {
  const char* entry = "mb_mx_quantize_columns";
  if (rows == 0 || columns == 0) return mb::elem_bytes(dtype) ? MB_OK
                                                              : mb::fail(MB_ERR_INVALID, "%s: unknown element type %d",
                                                                         entry, dtype);
  if (int rc = mb::check_rows(entry, dtype, x, x_bytes, rows, columns, row_stride)) return rc;
  if (columns > mb::kMxMostRows || rows > mb::kMxMostK)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u: at most %u rows", entry, rows, columns, mb::kMxMostK);
  if (int rc = mb::check_operand(entry, "the operand", columns, rows, 1, codes, codes_bytes, scales, scales_bytes))
    return rc;
  return mb::launch_quantize_columns(dtype, x, rows, columns, row_stride, codes, scales,
                                     static_cast<hipStream_t>(stream));
}

int mb_mx_dequantize(int dtype, const void* codes, uint64_t codes_bytes, const void* scales, uint64_t scales_bytes,
                     void* out, uint64_t out_bytes, uint32_t rows, uint32_t k, void* stream) {
  const char* entry = "mb_mx_dequantize";
  const uint32_t item = mb::elem_bytes(dtype);
  if (!item) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (rows == 0 || k == 0) return MB_OK;
  if (rows > mb::kMxMostRows || k > mb::kMxMostK)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u: at most %u rows of at most %u elements", entry, rows, k,
                    mb::kMxMostRows, mb::kMxMostK);
  if (int rc = mb::check_operand(entry, "the operand", rows, k, 1, codes, codes_bytes, scales, scales_bytes))
    return rc;
  if (out == nullptr || out_bytes < uint64_t{rows} * k * item)
    return mb::fail(MB_ERR_INVALID, "%s: out is NULL or too small for %u x %u", entry, rows, k);
  if (!mb::aligned(out, item)) return mb::fail(MB_ERR_ALIGNMENT, "%s: out must lie on its elements' %u bytes", entry, item);
  const uint64_t grid = (uint64_t{rows} * ((k + 7) / 8) + 255) / 256;
  if (grid > 0xffffffu) return mb::fail(MB_ERR_UNSUPPORTED, "%s: %u x %u exceeds one launch", entry, rows, k);
  auto launch = [&](auto kernel, auto t) {
    kernel<<<dim3(static_cast<uint32_t>(grid)), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
        static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), static_cast<decltype(t)*>(out), rows,
        k);
  };
  const bool streamed = mb::streams(uint64_t{rows} * k * item);
  MB_FOR_DTYPE(dtype, {
    if (streamed)
      launch(mb::mx_dequantize_kernel<T, true>, T());
    else
      launch(mb::mx_dequantize_kernel<T, false>, T());
  });
  return mb::launch_status("mx_dequantize");
}

}  // extern "C"
