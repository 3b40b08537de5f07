// Products of MXFP4 operands for linear layers: Y = X . W^T, each row of X with
// the weight of its expert where there are several.
#include "mb_elem.h"
#include "mb_mfma.h"
#include "mb_mx.h"

namespace mb {
namespace {

// Rows first .. last - 1 of expert `e`; all of them without offsets. Clamped, so
// that whatever `offsets` holds, no row outside 0 .. rows - 1 is touched.
__device__ __forceinline__ void expert_rows(const int32_t* __restrict__ offsets, uint32_t e, int rows, int& first,
                                            int& last) {
  first = offsets ? max(0, min(offsets[e], rows)) : 0;
  last = offsets ? max(first, min(offsets[e + 1], rows)) : rows;
}

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

#define MB_PRODUCT_REGISTER(T, NAME) MB_REGISTER_KERNEL("mx_product_" NAME, mx_product_kernel<T>)
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

int launch_product(int dtype, const void* x, const void* sx, const void* w, const void* sw, void* y, uint32_t rows,
                   uint32_t n, uint32_t k, const int32_t* offsets, uint32_t experts, hipStream_t stream) {
  const uint32_t tiles = (rows / experts + 15) / 16;
  const dim3 grid((n + 63) / 64, experts, tiles < 1 ? 1 : tiles < 256 ? tiles : 256);
  MB_FOR_DTYPE(dtype, (mx_product_kernel<T><<<grid, dim3(256), 0, stream>>>(
                          static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(sx),
                          static_cast<const uint8_t*>(w), static_cast<const uint8_t*>(sw), static_cast<T*>(y),
                          static_cast<int>(rows), static_cast<int>(n), static_cast<int>(k), offsets)));
  return launch_status("mx_product");
}

}  // namespace
}  // namespace mb

extern "C" {

int mb_mx_product(int dtype, const void* a, uint64_t a_bytes, const void* scale_a, uint64_t scale_a_bytes,
                  const void* b, uint64_t b_bytes, const void* scale_b, uint64_t scale_b_bytes, void* c,
                  uint64_t c_bytes, uint32_t rows, uint32_t n, uint32_t k, const int32_t* offsets,
                  uint64_t offsets_bytes, uint32_t experts, void* stream) {
  const char* entry = "mb_mx_product";
  if (int rc = mb::check_shape(entry, dtype, rows, n, k, experts)) return rc;
  if (int rc = mb::check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return mb::fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (int rc = mb::check_operand(entry, "a", rows, k, 1, a, a_bytes, scale_a, scale_a_bytes)) return rc;
  if (int rc = mb::check_operand(entry, "b", n, k, experts, b, b_bytes, scale_b, scale_b_bytes)) return rc;
  if (int rc = mb::check_output(entry, dtype, c, c_bytes, rows, n)) return rc;
  return mb::launch_product(dtype, a, scale_a, b, scale_b, c, rows, n, k, offsets, experts,
                            static_cast<hipStream_t>(stream));
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
    return mb::fail(MB_ERR_INVALID, "%s: slots need offsets, order and an entry for each of %llu rows", entry,
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
  if (int rc = mb::launch_quantize(dtype, x, tokens, k, row_stride, slots, gathered ? copies : 1,
                                   static_cast<uint32_t>(rows), codes, scales, on))
    return rc;
  return mb::launch_product(dtype, codes, scales, w, scale_w, y, static_cast<uint32_t>(rows), n, k, offsets, experts,
                            on);
}

}  // extern "C"
