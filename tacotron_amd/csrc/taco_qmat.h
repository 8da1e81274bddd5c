// The kernel of matrix-vector products with 4-bit weights; every type of vectors has a translation unit of its own
// (taco_qmat_f32.hip, taco_qmat_f16.hip, taco_qmat_bf16.hip), the layout is described in taco_qmat.hip.
#pragma once

#include "taco_step.h"

struct taco_qmat_multiply_params {
  const char *packed, *x;
  char* y;
  const float* bias;
  int64_t x_stride, y_stride;          // bytes
  int64_t col_blocks, groups, scales_at, zeros_at;
  int32_t n_rows, n_cols, n_vectors, per_block, scale_dtype;   // per_block: groups of a block's 128 columns
};

int taco_qmat_multiply_f32(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s);
int taco_qmat_multiply_f16(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s);
int taco_qmat_multiply_bf16(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s);
