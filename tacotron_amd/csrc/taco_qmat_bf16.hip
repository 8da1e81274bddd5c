#include "taco_qmat_kernel.h"

int taco_qmat_multiply_bf16(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s) { return launch<TACO_BF16>(a, n_cu, s); }
