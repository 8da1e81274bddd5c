#include "taco_qmat_kernel.h"

int taco_qmat_multiply_f32(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s) { return launch<TACO_F32>(a, n_cu, s); }
