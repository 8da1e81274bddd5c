// Matrix-vector products with 4-bit weights (taco_qmat_* in include/taco.h): y = x W^T + bias for a few vectors x, W held as
// 4-bit codes with a scale (and optionally a zero point) per group of 32, 64 or 128 columns of a row.  A product of up to
// about a hundred vectors is bound by reading the codes once.
#include "taco_step.h"


namespace {

// ---- layout -----------------------------------------------------------------------------------------------------------
// Codes: blocks of 16 rows x 128 columns, 1 KiB each, a row block's blocks side by side.  Lane l of a wave reads 16 bytes of
// a block: word j holds row l & 15, columns 32 j + 8 (l >> 4) .. + 7 - the operand of one 16 x 32 matrix-core product - with
// column 2 i in nibble i and column 2 i + 1 in nibble 4 + i, so that (word >> 4 i) & 0x000f000f is a pair of neighbours.
// Scales (and zero points, a byte each): four row blocks together, [group][64], row 16 t + 4 g + i at 16 g + 4 t + i: what lane
// quarter g needs of one row block or of all four lies side by side.  Zero points are stored with the 16 that the kernel's
// codes carry.  What lies outside the matrix is zero.
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
    const int64_t row = i / 64 / a.l.groups * 64 + (i % 16 / 4) * 16 + i % 64 / 16 * 4 + i % 4, group = i / 64 % a.l.groups;
    const bool have = row < a.n_rows && group < given;
    if (a.scale_size == 4) ((uint32_t*)(a.packed + a.l.scales_at))[i] = have ? *(const uint32_t*)(a.scales + row * a.scale_stride + group * 4) : 0;
    else ((uint16_t*)(a.packed + a.l.scales_at))[i] = have ? *(const uint16_t*)(a.scales + row * a.scale_stride + group * 2) : 0;
    if (a.zeros) ((uint8_t*)(a.packed + a.l.zeros_at))[i] = 16 + (have ? a.zeros[row * a.zero_stride + group] & 15 : 0);
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

// Eight elements of a vector from column `col` as operands of a product: one of a 16-bit type; three of bfloat16 for
// fp32, whose 24 bits they hold between them (each takes the leading 8 bits of what the ones before left, so every product with a
// code is exact).  At a vector's end the loads stay inside it and what lies behind is zero.
template <int T>
struct Operand {
  static constexpr int N = 1;
  taco_u4 v[1];
  __device__ __forceinline__ void load(const char* x, int col) { v[0] = *(const taco_u4_any*)(x + (int64_t)col * 2); }
  __device__ __forceinline__ void load_end(const char* x, int col, int n_cols) {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = ((const uint16_t*)x)[min(col + i, n_cols - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[0][i] = (col + 2 * i < n_cols ? e[2 * i] : 0) | (col + 2 * i + 1 < n_cols ? e[2 * i + 1] << 16 : 0);
  }
  __device__ __forceinline__ void split() {}
};
template <>
struct Operand<TACO_F32> {
  static constexpr int N = 3;
  float f[8];
  taco_u4 v[3];
  __device__ __forceinline__ void load(const char* x, int col) {
    const taco_f4 a = *(const taco_f4_any*)(x + (int64_t)col * 4), b = *(const taco_f4_any*)(x + (int64_t)col * 4 + 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
  }
  __device__ __forceinline__ void load_end(const char* x, int col, int n_cols) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = ((const float*)x)[min(col + e, n_cols - 1)];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = col + e < n_cols ? f[e] : 0.0f;
  }
  __device__ __forceinline__ void split() {
#pragma unroll
    for (int n = 0; n < 3; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // the upper halves of two floats side by side: two bfloat16, cut off
        v[n][i] = __builtin_amdgcn_perm(__float_as_uint(f[2 * i + 1]), __float_as_uint(f[2 * i]), 0x07060302u);
        if (n < 2) {
          f[2 * i] -= __uint_as_float(__float_as_uint(f[2 * i]) & 0xffff0000u);
          f[2 * i + 1] -= __uint_as_float(__float_as_uint(f[2 * i + 1]) & 0xffff0000u);
        }
      }
  }
};

// One workgroup per RT * 16 rows of W and MT * 16 vectors; its waves take the 128-column blocks in turn and are summed through
// LDS in their order.  GPB: groups in a block; S: type of the scales.
// A pair of nibbles becomes a pair of operands without a conversion: the code in the upper four bits of the mantissa of 16.0
// is 16 + code, in bfloat16 and float16 alike.  The 16 and the zero point come off per group, sum (c - z) x =
// sum (16 + c) x - (16 + z) sum x, with sum x from a product with ones, which the matrix cores have time for.  (A code in a
// float16's lowest bits, the subnormal c * 2^-24, would need nothing taken off, but the matrix cores lose bits of sums of
// such products: 2^-15 of the result measured.)
template <int T, int MT, int RT, int GPB, int S>
struct Multiply {
  static constexpr int SB = taco_size_of<S>;
  static constexpr int KIND = T == TACO_F16 ? TACO_F16 : TACO_BF16;       // of the products
  // A block's part of the matrix, which comes from far away: codes, scales and zero points of its rows.
  struct Block {
    taco_u4 w[RT];
    uint32_t s[GPB][RT * SB];       // four scales per row block
    uint32_t z[GPB][RT];
    __device__ __forceinline__ void load(const MultiplyParams& a, const char* codes, const char* scales, const char* zeros, int zero_step, int kb) {
#pragma unroll
      for (int t = 0; t < RT; ++t) w[t] = *(const taco_u4*)(codes + (t * a.col_blocks + kb) * 1024);
#pragma unroll
      for (int i = 0; i < GPB; ++i) {
        const int64_t group = (int64_t)kb * GPB + i;
        words<RT * SB>(s[i], scales + group * 64 * SB);
        words<RT>(z[i], zeros + group * zero_step);
        if (!zero_step) {
#pragma unroll
          for (int t = 0; t < RT; ++t) z[i][t] = 0x18181818u;
        }
      }
    }
    template <int N>
    static __device__ __forceinline__ void words(uint32_t (&to)[N], const char* p) {
      if constexpr (N % 4 == 0) {
#pragma unroll
        for (int n = 0; n < N; n += 4) {
          const taco_u4 v = *(const taco_u4*)(p + n * 4);
#pragma unroll
          for (int e = 0; e < 4; ++e) to[n + e] = v[e];
        }
      } else if constexpr (N == 2) {
        const taco_u2 v = *(const taco_u2*)p;
        to[0] = v[0];
        to[1] = v[1];
      } else {
        to[0] = *(const uint32_t*)p;
      }
    }
    __device__ __forceinline__ taco_f4 scale(int i, int t) const {
      if constexpr (S == TACO_F32) {
        return taco_f4{__uint_as_float(s[i][4 * t]), __uint_as_float(s[i][4 * t + 1]), __uint_as_float(s[i][4 * t + 2]), __uint_as_float(s[i][4 * t + 3])};
      } else {
        const uint32_t a = s[i][2 * t], b = s[i][2 * t + 1];
        return taco_f4{taco_low<S>(a), taco_high<S>(a), taco_low<S>(b), taco_high<S>(b)};
      }
    }
  };
  using Vectors = Operand<T>[4][MT];
  static __device__ __forceinline__ void load_x(Vectors& x, const char* const (&xr)[MT], int kb, int g) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m) x[j][m].load(xr[m], kb * 128 + 32 * j + 8 * g);
  }
  static __device__ __forceinline__ void load_x_end(Vectors& x, const char* const (&xr)[MT], int kb, int g, int n_cols) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int m = 0; m < MT; ++m) x[j][m].load_end(xr[m], kb * 128 + 32 * j + 8 * g, n_cols);
  }
  // Four words of codes: columns 0, 1, then 2, 3, ..
  static __device__ __forceinline__ taco_u4 widen(uint32_t w, uint32_t mask, uint32_t sixteen) {
    if constexpr (KIND == TACO_BF16) return taco_u4{((w << 3) & mask) | sixteen, ((w >> 1) & mask) | sixteen, ((w >> 5) & mask) | sixteen, ((w >> 9) & mask) | sixteen};
    else return taco_u4{((w << 6) & mask) | sixteen, ((w << 2) & mask) | sixteen, ((w >> 2) & mask) | sixteen, ((w >> 6) & mask) | sixteen};
  }
  static __device__ __forceinline__ void multiply(const Block& d, Vectors& x, uint32_t mask, uint32_t sixteen, taco_f4 (&y)[RT][MT]) {
    constexpr uint32_t one = KIND == TACO_BF16 ? 0x3f803f80u : 0x3c003c00u;
    constexpr int PER = 4 / GPB;        // products of 32 columns in a group
    taco_f4 acc[RT][MT], sum[MT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = j / PER;
      if (j % PER == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          sum[m] = taco_f4{0, 0, 0, 0};
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t][m] = taco_f4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        x[j][m].split();
#pragma unroll
        for (int n = Operand<T>::N - 1; n >= 0; --n) sum[m] = taco_mfma32<KIND>(taco_u4{one, one, one, one}, x[j][m].v[n], sum[m]);
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const taco_u4 c = widen(d.w[t][j], mask, sixteen);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = Operand<T>::N - 1; n >= 0; --n) acc[t][m] = taco_mfma32<KIND>(c, x[j][m].v[n], acc[t][m]);
      }
      if (j % PER == PER - 1) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const taco_f4 s = d.scale(i, t);
          const uint32_t z = d.z[i][t];
          const taco_f4 off = taco_f4{(float)(z & 255), (float)((z >> 8) & 255), (float)((z >> 16) & 255), (float)(z >> 24)};
#pragma unroll
          for (int m = 0; m < MT; ++m) y[t][m] += s * (acc[t][m] - off * sum[m]);
        }
      }
    }
  }
};

template <int T, int MT, int RT, int NW, int GPB, int S>
__global__ __launch_bounds__(64 * NW) void taco_qmat_multiply_kernel(const MultiplyParams a) {
  using K = Multiply<T, MT, RT, GPB, S>;
  constexpr int SB = K::SB;
  __shared__ float part[NW][MT * 16][RT * 16 + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int64_t row_block = (int64_t)blockIdx.x * RT;
  const int v0 = blockIdx.y * (16 * MT), whole = a.n_cols / 128;
  const char* codes = a.packed + row_block * a.col_blocks * 1024 + lane * 16;
  const int64_t side = row_block / 4 * a.groups * 64 + g * 16 + row_block % 4 * 4;      // of scales and zero points
  const char* scales = a.packed + a.scales_at + side * SB;
  // without zero points the same loads go to the first codes and are not looked at
  const char* zeros = a.zeros_at ? a.packed + a.zeros_at + side : a.packed;
  const int zero_step = a.zeros_at ? 64 : 0;
  const char* xr[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int v = v0 + m * 16 + r;
    xr[m] = a.x + (v < a.n_vectors ? (int64_t)v * a.x_stride : 0);      // columns without a vector repeat the first; nobody stores them
  }
  taco_f4 y[RT][MT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m) y[t][m] = taco_f4{0, 0, 0, 0};
  // constants the compiler does not know, so that it keeps them in registers: shift, v_and_or_b32 with both
  uint32_t mask, sixteen;
  if constexpr (K::KIND == TACO_BF16) asm("v_mov_b32 %0, 0x780078\n\tv_mov_b32 %1, 0x41804180" : "=&v"(mask), "=v"(sixteen));
  else asm("v_mov_b32 %0, 0x3c003c0\n\tv_mov_b32 %1, 0x4c004c00" : "=&v"(mask), "=v"(sixteen));
  if (wave < whole) {
    // The next block and its piece of the vectors come while this one is multiplied.  Every turn makes the same loads (the last
    // one again where there is no next block): a branch around them would leave the compiler with an unknown number of loads
    // in flight, and it would wait for all.
    typename K::Block block[2];
    typename K::Vectors x[2];
    block[0].load(a, codes, scales, zeros, zero_step, wave);
    K::load_x(x[0], xr, wave, g);
    for (int k0 = wave;; k0 += 2 * NW) {
      const int k1 = k0 + NW, k2 = k1 + NW;
      block[1].load(a, codes, scales, zeros, zero_step, min(k1, whole - 1));
      K::load_x(x[1], xr, min(k1, whole - 1), g);
      K::multiply(block[0], x[0], mask, sixteen, y);
      if (k1 >= whole) break;
      block[0].load(a, codes, scales, zeros, zero_step, min(k2, whole - 1));
      K::load_x(x[0], xr, min(k2, whole - 1), g);
      K::multiply(block[1], x[1], mask, sixteen, y);
      if (k2 >= whole) break;
    }
  }
  if (whole < (int)a.col_blocks && wave == whole % NW) {      // the last block's columns end inside it
    typename K::Block block;
    typename K::Vectors x;
    block.load(a, codes, scales, zeros, zero_step, whole);
    K::load_x_end(x, xr, whole, g, a.n_cols);
    K::multiply(block, x, mask, sixteen, y);
  }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 4; ++i) part[wave][m * 16 + r][t * 16 + 4 * g + i] = y[t][m][i];
  __syncthreads();
  for (int i = threadIdx.x; i < MT * 16 * RT * 16; i += 64 * NW) {
    const int row = i % (RT * 16), v = i / (RT * 16);
    float total = 0.0f;
#pragma unroll
    for (int n = 0; n < NW; ++n) total += part[n][v][row];
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

template <int T, int MT, int RT, int NW, int GPB, int S>
int launch(const MultiplyParams& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.n_rows + 16 * RT - 1) / (16 * RT)), (unsigned)((a.n_vectors + 16 * MT - 1) / (16 * MT)));
  taco_qmat_multiply_kernel<T, MT, RT, NW, GPB, S><<<grid, dim3(64 * NW), 0, s>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}

// How many row blocks a workgroup takes.  Few rows: one workgroup of 16 waves per CU, so that a row block's columns are read by as
// many waves as possible (bfloat16, one vector, us with 1 x 16 / 2 x 16 / 4 x 8 row blocks x waves: 4096 x 4096 4.6 / 6.6 / 7.1, 8192 x
// 8192 11.6 / 9.6 / 12.4).  Many rows: each piece of the vectors that is read serves four row blocks (14336 x 4096 with sixteen
// vectors 22 / 14 / 9.7, 28672 x 8192 with one 40 / 35 / 29).  Groups of 32 columns leave too few registers for four row blocks
// with fp32 scales, and for 16 waves with fp32 vectors.  More than 16 vectors take two tiles of 16 at a time (28672 x 8192
// with 32: 73 us with two row blocks, 110 with one).
template <int T, int GPB, int S>
int launch(const MultiplyParams& a, int n_cu, hipStream_t s) {
  constexpr bool FOUR = !(GPB == 4 && S == TACO_F32);
  constexpr int WAVES = T == TACO_F32 && GPB == 4 ? 8 : 16;
  const int row_blocks = (a.n_rows + 15) / 16;
  if (a.n_vectors > 16) return launch<T, 2, 2, 8, GPB, S>(a, s);
  if (row_blocks <= n_cu) return launch<T, 1, 1, 16, GPB, S>(a, s);
  if constexpr (FOUR)
    if (row_blocks > 2 * n_cu) return launch<T, 1, 4, 8, GPB, S>(a, s);
  return launch<T, 1, 2, WAVES, GPB, S>(a, s);
}
template <int T, int GPB>
int launch(const MultiplyParams& a, int n_cu, hipStream_t s) {
  if (a.scale_dtype == TACO_F32) return launch<T, GPB, TACO_F32>(a, n_cu, s);
  return a.scale_dtype == TACO_F16 ? launch<T, GPB, TACO_F16>(a, n_cu, s) : launch<T, GPB, TACO_BF16>(a, n_cu, s);
}
template <int T>
int launch(const MultiplyParams& a, int n_cu, hipStream_t s) {
  return a.per_block == 1 ? launch<T, 1>(a, n_cu, s) : a.per_block == 2 ? launch<T, 2>(a, n_cu, s) : launch<T, 4>(a, n_cu, s);
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
  if (dtype == TACO_F32) return launch<TACO_F32>(a, n_cu, s);
  if (dtype == TACO_F16) return launch<TACO_F16>(a, n_cu, s);
  return launch<TACO_BF16>(a, n_cu, s);
}
