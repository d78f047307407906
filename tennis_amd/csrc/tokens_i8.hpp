// Rows to int8 tokens (tokens_i8.hip), for the entry point and for the product that quantizes its rows first.
#pragma once
#include "elements.hpp"

namespace tsx {

// tsx_quantize_tokens without its checks; columns from cols up to cols_out of a row of q are zeros
int quantize_rows(int64_t rows, int cols, int cols_out, const void *x, int type, int64_t x_stride, int8_t *q, int64_t q_stride, float *scales,
                  hipStream_t stream);

}  // namespace tsx
