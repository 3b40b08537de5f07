// Sizes, checks and launches of FP8 operands with block scales, shared by the
// quantiser (mb_fp8.hip), the products (mb_fp8_product.hip) and the norm
// (mb_norm.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mb_internal.h"

namespace mb {

constexpr uint32_t kFp8Block = 128;  // elements of K, and rows of a weight, that share a scale
// Row numbers are 31-bit and K offsets inside a row fit 24 bits and more; a grid
// holds at most 2^24 - 1 workgroups of 256.
constexpr uint32_t kFp8MostRows = 1u << 24, kFp8MostK = 1u << 20;

// Codes are [rows][pitch] bytes, zero past k, and scales
// [ceil(k / 512)][ceil(rows / block)][4].
constexpr uint64_t fp8_pitch(uint64_t k) { return (k + 15) / 16 * 16; }
constexpr uint64_t fp8_code_bytes(uint64_t rows, uint64_t k) { return rows * fp8_pitch(k); }
constexpr uint64_t fp8_scale_bytes(uint64_t rows, uint64_t k, uint32_t block) {
  return (k + 511) / 512 * ((rows + block - 1) / block) * 4;
}

// An operand of `copies` matrices [rows][k] whose scales stand for `block` rows, 1 or 128.
int fp8_check_operand(const char* entry, const char* what, uint64_t rows, uint64_t k, uint64_t copies, uint32_t block,
                      const void* codes, uint64_t codes_bytes, const void* scales, uint64_t scales_bytes);

// A strided tensor of rows of k elements.
int fp8_check_rows(const char* entry, const char* what, int dtype, const void* x, uint64_t x_bytes, uint64_t rows,
                   uint64_t k, uint64_t row_stride);

// A contiguous output [rows][n].
int fp8_check_output(const char* entry, const char* what, int dtype, const void* y, uint64_t y_bytes, uint64_t rows,
                     uint64_t n);

int fp8_launch_quantize(int dtype, const void* x, uint32_t rows, uint32_t k, uint64_t row_stride, const int32_t* slots,
                        uint32_t copies, uint32_t out_rows, void* codes, void* scales, hipStream_t stream);

// An operand that a kernel writes; codes NULL: none.
struct Fp8Out {
  uint8_t* codes;
  uint8_t* scales;
};

// The operands of a product's gradients: the rows of d [rows][n] with K = n and its
// columns with K = depth >= rows, and the columns of x [rows][k], likewise. With
// gate_up, d is the gradient of [rows][2 * half], half = n / 2, that d_out
// [rows][half] is for silu(gate) * up.
int fp8_launch_gradient(int dtype, const void* d_out, uint64_t d_stride, const void* gate_up, const void* x,
                        uint64_t x_stride, uint32_t rows, uint32_t n, uint32_t k, uint32_t depth, Fp8Out d_rows,
                        Fp8Out d_columns, Fp8Out x_columns, hipStream_t stream);

}  // namespace mb
