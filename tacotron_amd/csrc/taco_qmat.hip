// Matrix-vector products with 4-bit weights (taco_qmat_* in include/taco.h): y = x W^T + bias for a few vectors x, W held as
// 4-bit codes with a scale (and optionally a zero point) per group of 32, 64 or 128 columns of a row.  Reading the codes is what bounds
// a large matrix with up to 16 vectors; its figures stand at the kernel (taco_qmat_kernel.h).
#include "taco_qmat.h"

namespace {

// ---- layout -----------------------------------------------------------------------------------------------------------
// Codes: blocks of 16 rows x 128 columns, 1 KiB each, a row block's blocks side by side.  Lane l of a wave reads 16 bytes of
// a block: word j holds row l & 15, columns 32 j + 8 (l >> 4) .. + 7 - the operand of one 16 x 32 matrix-core product - with
// column 2 i in nibble i and column 2 i + 1 in nibble 4 + i, so that (word >> 4 i) & 0x000f000f is a pair of neighbours.
// Scales (and zero points, a byte each): four row blocks together, [group][64], row 16 t + 4 g + i at 16 g + 4 t + i: what lane
// quarter g needs of one row block or of all four lies side by side.  What lies outside the matrix is zero.
struct Layout {
  int64_t row_blocks, col_blocks, groups, scales_at, zeros_at, bytes;
};
__host__ __device__ inline int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
__host__ __device__ inline Layout layout_of(int32_t n_rows, int32_t n_cols, int32_t group, int32_t scale_size, bool zeros) {
  Layout l;
  l.row_blocks = ((int64_t)n_rows + 63) / 64 * 4;
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
  // Bound by moving the codes: 28672 x 8192, 240 MB in and out with its scales, takes 89 us = 2.7 TB/s; done once per matrix.
  // A thread per lane of a block: four words of eight neighbouring columns each, in 16 bytes
  const int64_t lanes = a.l.row_blocks * a.l.col_blocks * 64, stats = a.l.row_blocks * a.l.groups * 16;
  const int64_t step = (int64_t)gridDim.x * 256;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < lanes; i += step) {
    const int64_t block = i / 64, row_block = block / a.l.col_blocks, col_block = block % a.l.col_blocks;
    const int lane = (int)(i % 64);
    const int64_t row = row_block * 16 + (lane & 15), col = col_block * 128 + 8 * (lane >> 4);
    taco_u4 w = {0, 0, 0, 0};
    if (row < a.n_rows) {
      const uint8_t* p = a.codes + row * a.code_stride;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t c = col + 32 * j;
        uint32_t v = 0;       // columns c .. c + 7 in their order
        if (c + 8 <= a.n_cols) {
          __builtin_memcpy(&v, p + c / 2, 4);
        } else {
          for (int e = 0; e < 8; ++e)
            if (c + e < a.n_cols) v |= (((e & 1) ? p[(c + e) / 2] >> 4 : p[(c + e) / 2] & 15u) << (4 * e));
        }
        // even columns to the low half, odd ones to the high half
        uint32_t even = v & 0x0f0f0f0fu, odd = (v >> 4) & 0x0f0f0f0fu;
        even = (even | even >> 4) & 0x00ff00ffu;
        odd = (odd | odd >> 4) & 0x00ff00ffu;
        w[j] = ((even | even >> 8) & 0xffffu) | (odd | odd >> 8) << 16;
      }
    }
    ((taco_u4*)a.packed)[i] = w;
  }
  const int64_t given = ((int64_t)a.n_cols + a.group - 1) / a.group;     // groups that the caller's scales have
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < stats; i += step) {
    const int64_t row = i / 64 / a.l.groups * 64 + (i % 16 / 4) * 16 + i % 64 / 16 * 4 + i % 4, group = i / 64 % a.l.groups;
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

// One wave per group of a row, two columns per lane: the group's extremes by six exchanges, then every lane rounds its own.  Done
// once per matrix and kept simple: a wave has 64 to 512 bytes to read, and starting so many is the bound (28672 x 8192 from fp32 or bfloat16: 0.5 ms in
// groups of 128, 1.8 in groups of 32).
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
  if (scale == __builtin_inff()) scale = hi / 15.0f - lo / 15.0f;      // the range of finite weights may be infinite, a fifteenth is not
  if (a.scale_dtype == TACO_F16) scale = (float)(_Float16)fminf(scale, 65504.0f);      // codes at the ends stand for what is beyond
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

// ---- host ----------------------------------------------------------------------------------------------------------------

int check_qmat(const taco_qmat* m, const char* who) {
  if (!m) TACO_FAIL(TACO_EINVAL, "%s: NULL matrix", who);
  // (a grid's threads are counted in 32 bits, 64 to a row at most)
  if (m->n_rows < 1 || m->n_cols < 1 || m->n_rows >= (1 << 26) || m->n_cols > (1 << 28)) TACO_FAIL(TACO_EINVAL, "%s: %d rows, %d columns", who, m->n_rows, m->n_cols);
  if (m->group != 32 && m->group != 64 && m->group != 128) TACO_FAIL(TACO_EINVAL, "%s: group %d is not 32, 64 or 128", who, m->group);
  if (m->scale_dtype != TACO_F32 && m->scale_dtype != TACO_F16 && m->scale_dtype != TACO_BF16) TACO_FAIL(TACO_EINVAL, "%s: scale_dtype %d", who, m->scale_dtype);
  return TACO_OK;
}
int size_of(int dtype) { return dtype == TACO_F32 ? 4 : 2; }
Layout layout_of(const taco_qmat* m) { return layout_of(m->n_rows, m->n_cols, m->group, size_of(m->scale_dtype), m->has_zeros != 0); }

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
  const taco_qmat_multiply_params a = {(const char*)m->packed, (const char*)x, (char*)y, m->bias, x_stride * size, y_stride * size, l.col_blocks,
                            l.groups, l.scales_at, m->has_zeros ? l.zeros_at : 0, m->n_rows, m->n_cols, n_vectors, 128 / m->group,
                            m->scale_dtype};
  hipStream_t s = (hipStream_t)stream;
  if (dtype == TACO_F32) return taco_qmat_multiply_f32(a, n_cu, s);
  if (dtype == TACO_F16) return taco_qmat_multiply_f16(a, n_cu, s);
  return taco_qmat_multiply_bf16(a, n_cu, s);
}
