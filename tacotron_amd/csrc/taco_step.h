// Shared by the kernels of the self-attention step (taco_paged.hip, taco_qmat.hip): element types, 16-byte loads and
// the matrix-core operand types.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "taco_internal.h"

typedef float taco_f2 __attribute__((ext_vector_type(2)));
typedef float taco_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 taco_bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 taco_bf2 __attribute__((ext_vector_type(2)));
typedef _Float16 taco_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 taco_h2 __attribute__((ext_vector_type(2)));
typedef uint32_t taco_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t taco_u2 __attribute__((ext_vector_type(2)));

template <int T>
constexpr int taco_size_of = T == TACO_F32 ? 4 : T == TACO_E4M3 ? 1 : 2;

// Two floats as one word of two 16-bit values, `a` in the low half, rounded to nearest.
template <int T>
__device__ __forceinline__ uint32_t taco_pack2(float a, float b) {
  static_assert(T == TACO_F16 || T == TACO_BF16, "16-bit types only");
  if constexpr (T == TACO_BF16) {
    const taco_bf2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, v);
  } else {
    const taco_h2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(uint32_t, v);
  }
}
// The two values of such a word.
template <int T>
__device__ __forceinline__ float taco_low(uint32_t w) {
  if constexpr (T == TACO_BF16) return __builtin_bit_cast(float, w << 16);
  else return (float)__builtin_bit_cast(taco_h2, w)[0];
}
template <int T>
__device__ __forceinline__ float taco_high(uint32_t w) {
  if constexpr (T == TACO_BF16) return __builtin_bit_cast(float, w & 0xffff0000u);
  else return (float)__builtin_bit_cast(taco_h2, w)[1];
}

// Eight consecutive elements of a 16-byte aligned row (32 bytes for fp32) as floats, and back.
template <int T>
__device__ __forceinline__ void taco_load8(const void* p, float (&x)[8]) {
  if constexpr (T == TACO_F32) {
    const taco_f4 a = ((const taco_f4*)p)[0], b = ((const taco_f4*)p)[1];
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[i] = a[i]; x[4 + i] = b[i]; }
  } else {
    const taco_u4 a = *(const taco_u4*)p;
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = taco_low<T>(a[i]); x[2 * i + 1] = taco_high<T>(a[i]); }
  }
}
template <int T>
__device__ __forceinline__ void taco_store8(void* p, const float (&x)[8]) {
  if constexpr (T == TACO_F32) {
    ((taco_f4*)p)[0] = taco_f4{x[0], x[1], x[2], x[3]};
    ((taco_f4*)p)[1] = taco_f4{x[4], x[5], x[6], x[7]};
  } else if constexpr (T == TACO_E4M3) {
    taco_u2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h], x[4 * h + 1], 0, false);
      w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2], x[4 * h + 3], v, true);
    }
    *(taco_u2*)p = w;
  } else {
    *(taco_u4*)p = taco_u4{taco_pack2<T>(x[0], x[1]), taco_pack2<T>(x[2], x[3]), taco_pack2<T>(x[4], x[5]),
                           taco_pack2<T>(x[6], x[7])};
  }
}

// One matrix-core product of 16 x 32 by 32 x 16 16-bit elements (v_mfma_f32_16x16x32): lane l holds row / column l & 15,
// elements 8 * (l >> 4) .. + 7 of the contraction; the result holds column l & 15, rows 4 * (l >> 4) .. + 3.
template <int T>
__device__ __forceinline__ taco_f4 taco_mfma32(taco_u4 a, taco_u4 b, taco_f4 c) {
  if constexpr (T == TACO_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(taco_bf8, a), __builtin_bit_cast(taco_bf8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(taco_h8, a), __builtin_bit_cast(taco_h8, b), c, 0, 0, 0);
}

// Maximum / sum over the four lanes l & 15, + 16, + 32, + 48 (v_permlane16_swap / v_permlane32_swap exchange rows of 16
// and halves between two registers, so a register swapped with its own copy leaves both partners side by side).
__device__ __forceinline__ float taco_max_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float taco_sum_rows(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
