// Sizes, checks and launches of MXFP4 operands shared by the quantiser
// (mb_mx.hip) and the linear layer (mb_mx_linear.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "mb_internal.h"

namespace mb {

// Row numbers are 31-bit, K offsets inside a row fit 24 bits and more; a grid
// holds at most 2^24 - 1 workgroups of 256.
constexpr uint32_t kMxMostRows = 1u << 24, kMxMostK = 1u << 20;

constexpr uint64_t mx_code_bytes(uint64_t rows, uint64_t k) { return rows * ((k + 31) / 32 * 16); }
constexpr uint64_t mx_scale_bytes(uint64_t rows, uint64_t k) { return (k + 255) / 256 * rows * 8; }

// An operand of `copies` matrices [rows][k].
int check_operand(const char* entry, const char* what, uint64_t rows, uint64_t k, uint64_t copies, const void* codes,
                  uint64_t codes_bytes, const void* scales, uint64_t scales_bytes);

// A strided tensor of rows of k elements.
int check_rows(const char* entry, int dtype, const void* x, uint64_t x_bytes, uint64_t rows, uint64_t k,
               uint64_t row_stride);

int launch_quantize(int dtype, const void* x, uint32_t rows, uint32_t k, uint64_t row_stride, const int32_t* slots,
                    uint32_t copies, uint32_t out_rows, void* codes, void* scales, hipStream_t stream);
// The rows and the columns of d [rows][n] and the columns of x [rows][k]; the
// columns with K = depth: rows, rounded up to 32 or to 256.
int launch_quantize_gradient(int dtype, const void* d, uint64_t d_stride, const void* x, uint64_t x_stride,
                             uint32_t rows, uint32_t n, uint32_t k, uint32_t depth, void* d_codes, void* d_scales,
                             void* d_columns, void* d_column_scales, void* x_columns, void* x_column_scales,
                             hipStream_t stream);

}  // namespace mb
