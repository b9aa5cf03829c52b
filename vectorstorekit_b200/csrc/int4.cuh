// Products with rows in four bits: what int4.cu (checks, entry points) asks of int4_product.cu.
#pragma once
#include "common.cuh"

namespace vsk {

// y[q * y_stride + r] = sum over columns of (value of row r) x[q * x_stride + column]; arguments checked by the caller.
int32_t q4_product(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                   int32_t y_dtype, int64_t y_stride);

// The same in whole numbers, for a few vectors (int4_digits.cu).
int32_t q4_product_digits(Ctx* ctx, const vsk_q4_rows& rows, const void* x, int32_t x_dtype, int64_t nq, int64_t x_stride, void* y,
                          int32_t y_dtype, int64_t y_stride);

}  // namespace vsk
