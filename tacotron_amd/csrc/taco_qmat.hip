// Matrix-vector products with 4-bit weights (taco_qmat_* in include/taco.h): y = x W^T + bias for a few vectors x, W held as
// 4-bit codes with a scale (and optionally a zero point) per group of 32, 64 or 128 columns of a row.  A product of up to
// about a hundred vectors is bound by reading the codes once.
#include "taco_step.h"

namespace {

// ---- layout -----------------------------------------------------------------------------------------------------------
// Codes: blocks of 16 rows x 128 columns, 1 KiB each, a row block's blocks side by side.  Lane l of a wave reads 16 bytes of
// a block: word j holds row l & 15, columns 32 j + 8 (l >> 4) .. + 7 - the operand of one 16 x 32 matrix-core product - with
// column 2 i in nibble i and column 2 i + 1 in nibble 4 + i, so that (word >> 4 i) & 0x000f000f is a pair of neighbours.
// Scales (and zero points, a byte each): [row block][group][16 rows].  What lies outside the matrix is zero.
struct Layout {
  int64_t row_blocks, col_blocks, groups, scales_at, zeros_at, bytes;
};
__host__ __device__ inline int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
__host__ __device__ inline Layout layout_of(int32_t n_rows, int32_t n_cols, int32_t group, int32_t scale_size, bool zeros) {
  Layout l;
  l.row_blocks = ((int64_t)n_rows + 15) / 16;
  l.col_blocks = ((int64_t)n_cols + 127) / 128;
  l.groups = l.col_blocks * (128 / group);
  l.scales_at = l.row_blocks * l.col_blocks * 1024;
  l.zeros_at = l.scales_at + round16(l.row_blocks * l.groups * 16 * scale_size);
  l.bytes = l.zeros_at + (zeros ? l.row_blocks * l.groups * 16 : 0);
  return l;
}

// ---- packing ----------------------------------------------------------------------------------------------------------

struct PackParams {
  const uint8_t *codes, *zeros;
  const char* scales;
  char* packed;
  int64_t code_stride, scale_stride, zero_stride;      // bytes
  Layout l;
  int32_t n_rows, n_cols, group, scale_size;
};

__global__ __launch_bounds__(256) void taco_qmat_pack_kernel(const PackParams a) {
  const int64_t words = a.l.row_blocks * a.l.col_blocks * 256, stats = a.l.row_blocks * a.l.groups * 16;
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < words; i += step) {
    const int64_t block = i / 256, row_block = block / a.l.col_blocks, col_block = block % a.l.col_blocks;
    const int lane = (int)(i % 256) / 4, j = (int)(i % 4);
    const int64_t row = row_block * 16 + (lane & 15), col = col_block * 128 + 32 * j + 8 * (lane >> 4);
    uint32_t w = 0;
    if (row < a.n_rows) {
      const uint8_t* p = a.codes + row * a.code_stride;
      for (int e = 0; e < 8; ++e)
        if (col + e < a.n_cols) {
          const uint32_t byte = p[(col + e) / 2];
          w |= (((col + e) & 1) ? byte >> 4 : byte & 15) << (4 * ((e >> 1) + 4 * (e & 1)));
        }
    }
    ((uint32_t*)a.packed)[i] = w;
  }
  const int64_t given = ((int64_t)a.n_cols + a.group - 1) / a.group;     // groups that the caller's scales have
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < stats; i += step) {
    const int64_t row = i / 16 / a.l.groups * 16 + i % 16, group = i / 16 % a.l.groups;
    const bool have = row < a.n_rows && group < given;
    if (a.scale_size == 4) ((uint32_t*)(a.packed + a.l.scales_at))[i] = have ? *(const uint32_t*)(a.scales + row * a.scale_stride + group * 4) : 0;
    else ((uint16_t*)(a.packed + a.l.scales_at))[i] = have ? *(const uint16_t*)(a.scales + row * a.scale_stride + group * 2) : 0;
    if (a.zeros) ((uint8_t*)(a.packed + a.l.zeros_at))[i] = have ? a.zeros[row * a.zero_stride + group] & 15 : 0;
  }
}

__device__ __forceinline__ float load_as_float(const void* p, int dtype) {
  if (dtype == TACO_F32) return *(const float*)p;
  if (dtype == TACO_F16) return (float)*(const _Float16*)p;
  return (float)*(const __bf16*)p;
}

struct QuantizeParams {
  const char* weights;
  uint8_t *codes, *zeros;
  char* scales;
  int64_t weight_stride, code_stride, scale_stride, zero_stride;   // bytes
  int32_t n_rows, n_cols, group, dtype, scale_dtype;
};

// One wave per group of a row, two columns per lane.
__global__ __launch_bounds__(64) void taco_qmat_quantize_kernel(const QuantizeParams a) {
  const int64_t row = blockIdx.x;
  const int group = blockIdx.y, lane = threadIdx.x;
  const int64_t col = (int64_t)group * a.group + 2 * lane;
  const bool mine = 2 * lane < a.group;
  const int size = a.dtype == TACO_F32 ? 4 : 2;
  float w[2] = {0.0f, 0.0f};
  for (int e = 0; e < 2; ++e)
    if (mine && col + e < a.n_cols) w[e] = load_as_float(a.weights + row * a.weight_stride + (col + e) * size, a.dtype);
  float lo = fminf(0.0f, fminf(w[0], w[1])), hi = fmaxf(0.0f, fmaxf(w[0], w[1]));
  for (int m = 32; m >= 1; m >>= 1) {
    lo = fminf(lo, __shfl_xor(lo, m, 64));
    hi = fmaxf(hi, __shfl_xor(hi, m, 64));
  }
  // without zero points the codes 1 .. 15 stand for -7 .. 7 scales; with them 0 .. 15 span lo .. hi
  float scale = a.zeros ? (hi - lo) / 15.0f : fmaxf(hi, -lo) / 7.0f;
  if (a.scale_dtype == TACO_F16) scale = (float)(_Float16)scale;
  else if (a.scale_dtype == TACO_BF16) scale = (float)(__bf16)scale;
  const float zero = a.zeros ? (scale > 0.0f ? fminf(fmaxf(rintf(-lo / scale), 0.0f), 15.0f) : 0.0f) : 8.0f;
  uint32_t byte = 0;
  for (int e = 0; e < 2; ++e) {
    const float q = scale > 0.0f ? fminf(fmaxf(rintf(w[e] / scale) + zero, 0.0f), 15.0f) : zero;
    byte |= (uint32_t)q << (4 * e);
  }
  if (mine && col < a.n_cols) a.codes[row * a.code_stride + col / 2] = (uint8_t)byte;
  if (lane == 0) {
    char* s = a.scales + row * a.scale_stride;
    if (a.scale_dtype == TACO_F32) ((float*)s)[group] = scale;
    else if (a.scale_dtype == TACO_F16) ((_Float16*)s)[group] = (_Float16)scale;
    else ((__bf16*)s)[group] = (__bf16)scale;
    if (a.zeros) a.zeros[row * a.zero_stride + group] = (uint8_t)zero;
  }
}

// ---- multiplying --------------------------------------------------------------------------------------------------------

struct MultiplyParams {
  const char *packed, *x;
  char* y;
  const float* bias;
  int64_t x_stride, y_stride;          // bytes
  int64_t col_blocks, groups, scales_at, zeros_at;
  int32_t n_rows, n_cols, n_vectors, per_block, scale_dtype;   // per_block: groups of a block's 128 columns
};

typedef taco_u4 taco_u4_any __attribute__((aligned(2)));       // 16 bytes at any element's address
typedef taco_f4 taco_f4_any __attribute__((aligned(4)));

// Eight elements of vector row `x` from column `col`: as the product's operand (16-bit types) or as floats; what lies
// behind the row is zero.
template <int T>
struct Operand {
  taco_u4 v;
  __device__ __forceinline__ void load(const char* x, int col, int n_cols, bool have) {
    v = taco_u4{0, 0, 0, 0};
    if (!have) return;
    if (col + 8 <= n_cols) {
      v = *(const taco_u4_any*)(x + (int64_t)col * 2);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < n_cols) v[e / 2] |= (uint32_t)((const uint16_t*)x)[col + e] << (16 * (e & 1));
    }
  }
};
template <>
struct Operand<TACO_F32> {
  float v[8];
  __device__ __forceinline__ void load(const char* x, int col, int n_cols, bool have) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.0f;
    if (!have) return;
    if (col + 8 <= n_cols) {
      const taco_f4 a = *(const taco_f4_any*)(x + (int64_t)col * 4), b = *(const taco_f4_any*)(x + (int64_t)col * 4 + 16);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (col + e < n_cols) v[e] = ((const float*)x)[col + e];
    }
  }
};

__device__ __forceinline__ taco_f4 load_scales(const char* p, int dtype) {
  if (dtype == TACO_F32) return *(const taco_f4*)p;
  const taco_u2 w = *(const taco_u2*)p;
  if (dtype == TACO_F16) return taco_f4{taco_low<TACO_F16>(w[0]), taco_high<TACO_F16>(w[0]), taco_low<TACO_F16>(w[1]), taco_high<TACO_F16>(w[1])};
  return taco_f4{taco_low<TACO_BF16>(w[0]), taco_high<TACO_BF16>(w[0]), taco_low<TACO_BF16>(w[1]), taco_high<TACO_BF16>(w[1])};
}

// One workgroup per 16 rows of W and 16 * MT vectors; its NW waves take the row block's 128-column blocks in turn and
// are summed through LDS in their order.
//   16-bit x: a pair of nibbles becomes a pair of operands without a conversion.
//     bfloat16: 0x4300 | code is 128 + code.  That offset and the zero point come off per group: sum (c - z) x = sum (128 + c) x -
//     (128 + z) sum x, sum x from a product with ones (v_mfma_f32_16x16x32 is not what bounds this).
//     float16: 0x6400 | code is 1024 + code; one packed subtraction leaves c - z, exactly.  (The code alone, the subnormal
//     c * 2^-24, would save it, but the matrix cores lose bits of sums of such products: 2^-15 of the result measured.)
//   fp32 x: codes are converted (a byte at a time) and lose their zero point there, exactly; v_mfma_f32_16x16x4_f32.
template <int T, int MT, int NW>
__global__ __launch_bounds__(64 * NW) void taco_qmat_multiply_kernel(const MultiplyParams a) {
  __shared__ float part[NW][MT][16][17];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int64_t row_block = blockIdx.x;
  const int v0 = blockIdx.y * (16 * MT);
  const char* codes = a.packed + row_block * a.col_blocks * 1024 + lane * 16;
  const int ssize = a.scale_dtype == TACO_F32 ? 4 : 2;
  const char* scales = a.packed + a.scales_at + row_block * a.groups * 16 * ssize + g * 4 * ssize;
  const char* zeros = a.zeros_at ? a.packed + a.zeros_at + row_block * a.groups * 16 : nullptr;
  const char* xr[MT];
  bool have[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int v = v0 + m * 16 + r;
    have[m] = v < a.n_vectors;
    xr[m] = a.x + (have[m] ? (int64_t)v * a.x_stride : 0);
  }
  taco_f4 y[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) y[m] = taco_f4{0, 0, 0, 0};

  for (int kb = wave; kb < (int)a.col_blocks; kb += NW) {
    const taco_u4 w = *(const taco_u4*)(codes + (int64_t)kb * 1024);
    taco_f4 acc[MT], sum[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = sum[m] = taco_f4{0, 0, 0, 0};
    int group = kb * a.per_block;
    const int last = 4 / a.per_block - 1;       // a group's last product of 32 columns
    float zr = 8.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      Operand<T> x[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m].load(xr[m], kb * 128 + 32 * j + 8 * g, a.n_cols, have[m]);
      if constexpr (T == TACO_F32) {
        if (zeros) zr = (float)(uint8_t)zeros[group * 16 + r];
        const uint32_t lo = w[j] & 0x0f0f0f0fu, hi = (w[j] >> 4) & 0x0f0f0f0fu;     // columns 0, 4, 1, 5 and 2, 6, 3, 7
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float c = (float)((((e & 2) ? hi : lo) >> (8 * ((e >> 2) + 2 * (e & 1)))) & 255u) - zr;
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m] = __builtin_amdgcn_mfma_f32_16x16x4f32(c, x[m].v[e], acc[m], 0, 0, 0);
        }
      } else {
        constexpr uint32_t over = T == TACO_BF16 ? 0x43004300u : 0x64006400u;
        taco_u4 c = {(w[j] & 0x000f000fu) | over, ((w[j] >> 4) & 0x000f000fu) | over, ((w[j] >> 8) & 0x000f000fu) | over,
                     ((w[j] >> 12) & 0x000f000fu) | over};
        if constexpr (T == TACO_F16) {
          _Float16 z = (_Float16)1032.0f;
          if (zeros) z = (_Float16)(1024.0f + (float)(uint8_t)zeros[group * 16 + r]);
          const taco_h2 zz = {z, z};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t pair = c[e];     // a copy: __builtin_bit_cast of a vector's element takes its first one here
            c[e] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(taco_h2, pair) - zz);
          }
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          acc[m] = taco_mfma32<T>(c, x[m].v, acc[m]);
          if constexpr (T == TACO_BF16) sum[m] = taco_mfma32<T>(taco_u4{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}, x[m].v, sum[m]);
        }
      }
      if ((j & last) == last) {
        const taco_f4 s = load_scales(scales + (int64_t)group * 16 * ssize, a.scale_dtype);
        if constexpr (T != TACO_BF16) {
#pragma unroll
          for (int m = 0; m < MT; ++m) y[m] += s * acc[m];
        } else {
          taco_f4 off = taco_f4{136, 136, 136, 136};
          if (zeros) {
            const uint32_t z = *(const uint32_t*)(zeros + group * 16 + g * 4);
            off = taco_f4{(float)(z & 255), (float)((z >> 8) & 255), (float)((z >> 16) & 255), (float)(z >> 24)} + 128.0f;
          }
#pragma unroll
          for (int m = 0; m < MT; ++m) y[m] += s * (acc[m] - off * sum[m]);
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = sum[m] = taco_f4{0, 0, 0, 0};
        ++group;
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][m][r][4 * g + i] = y[m][i];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 256; i += 64 * NW) {
    const int row = i % 16, v = i / 16;
    float total = 0.0f;
#pragma unroll
    for (int n = 0; n < NW; ++n) total += part[n][v / 16][v % 16][row];
    const int64_t n = row_block * 16 + row;
    if (n < a.n_rows && v0 + v < a.n_vectors) {
      if (a.bias) total += a.bias[n];
      char* out = a.y + (int64_t)(v0 + v) * a.y_stride;
      if constexpr (T == TACO_F32) ((float*)out)[n] = total;
      else if constexpr (T == TACO_F16) ((_Float16*)out)[n] = (_Float16)total;
      else ((__bf16*)out)[n] = (__bf16)total;
    }
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------------

int check_qmat(const taco_qmat* m, const char* who) {
  if (!m) TACO_FAIL(TACO_EINVAL, "%s: NULL matrix", who);
  if (m->n_rows < 1 || m->n_cols < 1 || m->n_rows > (1 << 28) || m->n_cols > (1 << 28)) TACO_FAIL(TACO_EINVAL, "%s: %d rows, %d columns", who, m->n_rows, m->n_cols);
  if (m->group != 32 && m->group != 64 && m->group != 128) TACO_FAIL(TACO_EINVAL, "%s: group %d is not 32, 64 or 128", who, m->group);
  if (m->scale_dtype != TACO_F32 && m->scale_dtype != TACO_F16 && m->scale_dtype != TACO_BF16) TACO_FAIL(TACO_EINVAL, "%s: scale_dtype %d", who, m->scale_dtype);
  return TACO_OK;
}
int size_of(int dtype) { return dtype == TACO_F32 ? 4 : 2; }
Layout layout_of(const taco_qmat* m) { return layout_of(m->n_rows, m->n_cols, m->group, size_of(m->scale_dtype), m->has_zeros != 0); }

template <int T, int MT>
int launch(const MultiplyParams& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.n_rows + 15) / 16), (unsigned)((a.n_vectors + 16 * MT - 1) / (16 * MT)));
  taco_qmat_multiply_kernel<T, MT, 8><<<grid, dim3(64 * 8), 0, s>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}
template <int T>
int launch(const MultiplyParams& a, hipStream_t s) {
  if (a.n_vectors <= 16) return launch<T, 1>(a, s);
  if (a.n_vectors <= 32) return launch<T, 2>(a, s);
  return launch<T, 4>(a, s);
}

}  // namespace

extern "C" int64_t taco_qmat_bytes(const taco_qmat* m) {
  const int rc = check_qmat(m, "taco_qmat_bytes");
  return rc == TACO_OK ? layout_of(m).bytes : rc;
}

extern "C" int taco_qmat_pack(const taco_qmat* m, const uint8_t* codes, int64_t code_stride, const void* scales, int64_t scale_stride,
                              const uint8_t* zeros, int64_t zero_stride, void* packed, void* stream) {
  const char* who = "taco_qmat_pack";
  int rc = check_qmat(m, who);
  if (rc != TACO_OK) return rc;
  if (!codes || !scales || !packed || ((uintptr_t)packed & 15)) TACO_FAIL(TACO_EINVAL, "%s: codes, scales and a 16-byte aligned packed buffer are needed", who);
  if ((zeros != nullptr) != (m->has_zeros != 0)) TACO_FAIL(TACO_EINVAL, "%s: has_zeros %d does not go with the zero points given", who, m->has_zeros);
  const int64_t groups = ((int64_t)m->n_cols + m->group - 1) / m->group;
  if (code_stride < ((int64_t)m->n_cols + 1) / 2 || scale_stride < groups || (zeros && zero_stride < groups)) TACO_FAIL(TACO_EINVAL, "%s: strides shorter than a row", who);
  int n_cu;
  DeviceScope on_device(m->device);
  TACO_HIP(on_device.status);
  rc = taco_device_check(m->device, &n_cu);
  if (rc != TACO_OK) return rc;
  const int size = size_of(m->scale_dtype);
  const PackParams a = {codes, zeros, (const char*)scales, (char*)packed, code_stride, scale_stride * size, zero_stride, layout_of(m),
                        m->n_rows, m->n_cols, m->group, size};
  taco_qmat_pack_kernel<<<dim3((unsigned)(8 * n_cu)), dim3(256), 0, (hipStream_t)stream>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}

extern "C" int taco_qmat_quantize(const taco_qmat* m, const void* weights, int64_t weight_stride, int32_t dtype, uint8_t* codes,
                                  int64_t code_stride, void* scales, int64_t scale_stride, uint8_t* zeros, int64_t zero_stride,
                                  void* stream) {
  const char* who = "taco_qmat_quantize";
  int rc = check_qmat(m, who);
  if (rc != TACO_OK) return rc;
  if (dtype != TACO_F32 && dtype != TACO_F16 && dtype != TACO_BF16) TACO_FAIL(TACO_EINVAL, "%s: dtype %d", who, dtype);
  if (!weights || !codes || !scales) TACO_FAIL(TACO_EINVAL, "%s: NULL argument", who);
  if ((zeros != nullptr) != (m->has_zeros != 0)) TACO_FAIL(TACO_EINVAL, "%s: has_zeros %d does not go with the zero points given", who, m->has_zeros);
  const int64_t groups = ((int64_t)m->n_cols + m->group - 1) / m->group;
  if (weight_stride < m->n_cols || code_stride < ((int64_t)m->n_cols + 1) / 2 || scale_stride < groups || (zeros && zero_stride < groups)) TACO_FAIL(TACO_EINVAL, "%s: strides shorter than a row", who);
  if (groups > 65535) TACO_FAIL(TACO_EINVAL, "%s: %lld groups in a row", who, (long long)groups);
  int n_cu;
  DeviceScope on_device(m->device);
  TACO_HIP(on_device.status);
  rc = taco_device_check(m->device, &n_cu);
  if (rc != TACO_OK) return rc;
  const QuantizeParams a = {(const char*)weights, codes, zeros, (char*)scales, weight_stride * size_of(dtype), code_stride,
                            scale_stride * size_of(m->scale_dtype), zero_stride, m->n_rows, m->n_cols, m->group, dtype, m->scale_dtype};
  taco_qmat_quantize_kernel<<<dim3((unsigned)m->n_rows, (unsigned)groups), dim3(64), 0, (hipStream_t)stream>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}

extern "C" int taco_qmat_multiply(const taco_qmat* m, const void* x, int64_t x_stride, void* y, int64_t y_stride, int32_t n_vectors,
                                  int32_t dtype, void* stream) {
  const char* who = "taco_qmat_multiply";
  int rc = check_qmat(m, who);
  if (rc != TACO_OK) return rc;
  if (dtype != TACO_F32 && dtype != TACO_F16 && dtype != TACO_BF16) TACO_FAIL(TACO_EINVAL, "%s: dtype %d", who, dtype);
  if (n_vectors < 0 || n_vectors > (1 << 20)) TACO_FAIL(TACO_EINVAL, "%s: %d vectors", who, n_vectors);
  if (n_vectors == 0) return TACO_OK;
  if (!m->packed || ((uintptr_t)m->packed & 15)) TACO_FAIL(TACO_EINVAL, "%s: packed must be 16-byte aligned (and not NULL)", who);
  const int size = size_of(dtype);
  if (!x || !y || (uintptr_t)x % size || (uintptr_t)y % size) TACO_FAIL(TACO_EINVAL, "%s: x and y must be aligned to their elements (and not NULL)", who);
  if (n_vectors > 1 && (x_stride < m->n_cols || y_stride < m->n_rows)) TACO_FAIL(TACO_EINVAL, "%s: strides shorter than a vector", who);
  int n_cu;
  DeviceScope on_device(m->device);
  TACO_HIP(on_device.status);
  rc = taco_device_check(m->device, &n_cu);
  if (rc != TACO_OK) return rc;
  const Layout l = layout_of(m);
  const MultiplyParams a = {(const char*)m->packed, (const char*)x, (char*)y, m->bias, x_stride * size, y_stride * size, l.col_blocks,
                            l.groups, l.scales_at, m->has_zeros ? l.zeros_at : 0, m->n_rows, m->n_cols, n_vectors, 128 / m->group,
                            m->scale_dtype};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TACO_F32) return launch<TACO_F32>(a, s);
  if (dtype == TACO_F16) return launch<TACO_F16>(a, s);
  return launch<TACO_BF16>(a, s);
}
