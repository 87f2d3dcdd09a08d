// lm_linear8.h -- products with INT8 weights, one scale a row of the weight:
// entries that lm_linear and lm_linear_input_grad call after their checks.
#pragma once
#include "lm_linear.h"

// products of codes, at most 127 * 128 each, add up in 32 bits
constexpr int LIN8_MAX_SUM = 0x7fffffff / (127 * 128);

// half: rows of fp16, as far as it matters to the input gradient
size_t lin8_workspace(int op, int64_t T, int64_t lda, int64_t N, int64_t K, int64_t E, bool quant, bool aligned, bool half);
int lin8_forward(LinArgs& a, int dtype, bool quant, void* workspace, size_t workspace_bytes, hipStream_t st);
int lin8_input_grad(LinArgs& a, int dtype, void* workspace, size_t workspace_bytes, hipStream_t st);
