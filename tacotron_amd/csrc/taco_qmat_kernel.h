// Matrix-vector products with 4-bit weights: the kernel and the choice of its form, included once per type of vectors.
#pragma once

#include "taco_qmat.h"

namespace {

typedef taco_u4 taco_u4_any __attribute__((aligned(4)));       // 16 bytes at any word's address
typedef taco_f4 taco_f4_any __attribute__((aligned(4)));

// Eight elements of a vector from column `col` as operands of a product: one of a 16-bit type; three of bfloat16 for
// fp32, whose 24 bits they hold between them (each takes the leading 8 bits of what the ones before left, so every product with a
// code is exact).  At a vector's end the loads stay inside it and what lies behind is zero.
// ODD: some vectors begin between two words.  A load there takes several times as long, so the words around are loaded and
// shifted (4096 x 4097 in groups of 32 for sixteen vectors 17.9 -> 13.1 us); what they hold beyond the vector shares a word with an element of it.
template <int T, bool ODD>
struct Operand {
  static constexpr int N = 1;
  taco_u4 v[1];
  __device__ __forceinline__ void load(const char* x, int col) {
    const char* p = x + (int64_t)col * 2;
    if constexpr (ODD) {
      const uint32_t off = (uint32_t)(uintptr_t)p & 2;
      const taco_u4 w = *(const taco_u4_any*)(p - off);
      const uint32_t next = *(const uint32_t*)(p - off + (off ? 16 : 12));
      v[0] = taco_u4{__builtin_amdgcn_alignbyte(w[1], w[0], off), __builtin_amdgcn_alignbyte(w[2], w[1], off),
                     __builtin_amdgcn_alignbyte(w[3], w[2], off), __builtin_amdgcn_alignbyte(next, w[3], off)};
    } else {
      v[0] = *(const taco_u4_any*)p;
    }
  }
  __device__ __forceinline__ void load_end(const char* x, int col, int n_cols) {
    uint32_t e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = ((const uint16_t*)x)[min(col + i, n_cols - 1)];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[0][i] = (col + 2 * i < n_cols ? e[2 * i] : 0) | (col + 2 * i + 1 < n_cols ? e[2 * i + 1] << 16 : 0);
  }
  __device__ __forceinline__ void split() {}
};
template <bool ODD>
struct Operand<TACO_F32, ODD> {
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
        // the upper halves of two floats side by side: two bfloat16, cut off (in the order in which the codes come, see widen)
        constexpr int FIRST[4] = {0, 2, 1, 3};
        float &a = f[FIRST[i]], &b = f[FIRST[i] + 4];
        v[n][i] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        if (n < 2) {
          a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
          b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        }
      }
  }
};

// One workgroup per RT * 16 rows of W and MT * 16 vectors; its waves take the 128-column blocks in turn and are summed through
// LDS in their order.  GPB: groups in a block; S: type of the scales.
// With 16-bit vectors a pair of nibbles becomes a pair of operands without a conversion: the code in the upper four bits of the mantissa of 16.0
// is 16 + code, in bfloat16 and float16 alike.  The 16 and the zero point come off per group, sum (c - z) x =
// sum (16 + c) x - 16 sum x - z sum x, with the sums from a product with constants, which the matrix cores have time for; without
// zero points all of it is one such product, of -24.  (A code in a
// float16's lowest bits, the subnormal c * 2^-24, would need nothing taken off, but the matrix cores lose bits of sums of
// such products: 2^-15 of the result measured.)
// A group's sums are formed before its scale makes them small: up to 31 * 128 times the largest element for bfloat16, 15 * 128 for
// fp32.  So that they stay below the largest fp32 number whatever the vectors, bfloat16 and fp32 codes are held 2^-12 times as large and
// the finished sum is multiplied by 2^12 (float16 vectors end at 65504).  Both are exact as long as sums are normal numbers: results
// below 2^-114 = 5e-35 are held to 2^-138 instead of 2^-149.
// Bound by reading the codes: 28672 x 8192 for one bfloat16 vector, 122 MB, takes 26.4 us = 4.6 TB/s (a large copy reaches 4.7; the
// same loads without any product 23.7 us); groups of 32 columns 35 us, where scaling the sums binds; an fp32 vector 45 us
// (groups of 64), where splitting it and converting the codes does (a byte at a time 54).  4096 x 4096 4.4 us, 4096 x 1558 for sixteen fp32 vectors 6.1 us, 80 x 1558 for one
// 5.1 us: the launch, one round trip to memory and, for the last two, a block's chain of products.
template <int T, int MT, int RT, int GPB, int S, bool ZEROS, bool ODD>
struct Multiply {
  static constexpr int SB = taco_size_of<S>;
  static constexpr int KIND = T == TACO_F16 ? TACO_F16 : TACO_BF16;       // of the products
  static constexpr float UNIT = T == TACO_F16 ? 1.0f : 0x1p-12f;          // what a code of 1 is held as
  struct Constants {
    uint32_t mask, sixteen, offset;
  };
  // A block's part of the matrix, which comes from far away: codes, scales and zero points of its rows.
  struct Block {
    taco_u4 w[RT];
    uint32_t s[GPB][RT * SB];       // four scales per row block
    uint32_t z[ZEROS ? GPB : 1][RT];
    __device__ __forceinline__ void load(const taco_qmat_multiply_params& a, const char* codes, const char* scales, const char* zeros, int kb) {
#pragma unroll
      for (int t = 0; t < RT; ++t) w[t] = *(const taco_u4*)(codes + (t * a.col_blocks + kb) * 1024);
#pragma unroll
      for (int i = 0; i < GPB; ++i) {
        const int64_t group = (int64_t)kb * GPB + i;
        words<RT * SB>(s[i], scales + group * 64 * SB);
        if constexpr (ZEROS) words<RT>(z[i], zeros + group * 64);
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
  using Vectors = Operand<T, ODD>[4][MT];
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
  // A word's codes as four words of operands: columns 0, 1, then 2, 3, ..  For fp32 vectors two at a time are converted from 8-bit
  // floats of 3 mantissa bits, whose smallest values, the bytes 0 .. 15, are that many times 2^-9: the 16 would triple the rounding
  // errors of the sums, which nothing hides there (8249 x 9077: 1.1e-6 of the result with it).  Those pairs are columns 0, 4, then 2, 6,
  // 1, 5 and 3, 7, and the vectors are taken in that order.
  template <int HALF>
  static __device__ __forceinline__ uint32_t bytes(uint32_t w) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 512.0f * UNIT, HALF));
  }
  static __device__ __forceinline__ taco_u4 widen(uint32_t w, uint32_t mask, uint32_t sixteen) {
    if constexpr (T == TACO_F32) {
      const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;     // columns 0, 4, 1, 5 and 2, 6, 3, 7
      return taco_u4{bytes<0>(lo), bytes<0>(hi), bytes<1>(lo), bytes<1>(hi)};
    } else if constexpr (T == TACO_BF16) {
      return taco_u4{((w << 3) & mask) | sixteen, ((w >> 1) & mask) | sixteen, ((w >> 5) & mask) | sixteen, ((w >> 9) & mask) | sixteen};
    } else {
      return taco_u4{((w << 6) & mask) | sixteen, ((w << 2) & mask) | sixteen, ((w >> 2) & mask) | sixteen, ((w >> 6) & mask) | sixteen};
    }
  }
  // `offset` is an operand of all the same numbers: what every code is too large by, negated (the 16, and the 8 that stands for a
  // zero point where there are none), or -1 for fp32 with zero points.  Its product with the vectors goes in front of the codes'
  // products of a group of 32 columns, or behind those of a longer one.
  static __device__ __forceinline__ void multiply(const Block& d, Vectors& x, const Constants& k, taco_f4 (&y)[RT][MT]) {
    constexpr int PER = 4 / GPB;        // products of 32 columns in a group
    taco_f4 acc[RT][MT], sum[MT];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = j / PER;
      if (j % PER == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m) sum[m] = taco_f4{0, 0, 0, 0};
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        x[j][m].split();
#pragma unroll
        for (int n = Operand<T, ODD>::N - 1; n >= 0; --n) sum[m] = taco_mfma32<KIND>(taco_u4{k.offset, k.offset, k.offset, k.offset}, x[j][m].v[n], sum[m]);
      }
      taco_f4 whole[MT];                // what comes off regardless of zero points
#pragma unroll
      for (int m = 0; m < MT; ++m) whole[m] = T == TACO_F32 && ZEROS ? taco_f4{0, 0, 0, 0} : sum[m];
      if (j % PER == 0) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int t = 0; t < RT; ++t) acc[t][m] = PER == 1 ? whole[m] : taco_f4{0, 0, 0, 0};
      }
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const taco_u4 c = widen(d.w[t][j], k.mask, k.sixteen);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = Operand<T, ODD>::N - 1; n >= 0; --n) acc[t][m] = taco_mfma32<KIND>(c, x[j][m].v[n], acc[t][m]);
      }
      if (j % PER == PER - 1) {
        if (PER > 1) {
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[t][m] += whole[m];
        }
        if constexpr (ZEROS) {
          float less[MT];               // minus the vectors' sums
#pragma unroll
          for (int m = 0; m < MT; ++m) less[m] = T == TACO_F32 ? sum[m][0] : sum[m][0] * 0.0625f;
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            const uint32_t z = d.z[i][t];
            const taco_f4 zero = taco_f4{(float)(z & 255), (float)((z >> 8) & 255), (float)((z >> 16) & 255), (float)(z >> 24)};
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[t][m] += zero * less[m];
          }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const taco_f4 s = d.scale(i, t);
#pragma unroll
          for (int m = 0; m < MT; ++m) y[t][m] += s * acc[t][m];
        }
      }
    }
  }
};

template <int T, int MT, int RT, int NW, int GPB, int S, bool ZEROS, bool ODD>
__global__ __launch_bounds__(64 * NW) void taco_qmat_multiply_kernel(const taco_qmat_multiply_params a) {
  using K = Multiply<T, MT, RT, GPB, S, ZEROS, ODD>;
  constexpr int SB = K::SB;
  __shared__ float part[NW][MT * 16][RT * 16 + 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int64_t row_block = (int64_t)blockIdx.x * RT;
  const int v0 = blockIdx.y * (16 * MT), whole = a.n_cols / 128;
  const char* codes = a.packed + row_block * a.col_blocks * 1024 + lane * 16;
  const int64_t side = row_block / 4 * a.groups * 64 + g * 16 + row_block % 4 * 4;      // of scales and zero points
  const char* scales = a.packed + a.scales_at + side * SB;
  const char* zeros = a.packed + a.zeros_at + side;
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
  typename K::Constants k;
  if constexpr (K::KIND == TACO_BF16) asm("v_mov_b32 %0, 0x780078\n\tv_mov_b32 %1, 0x3b803b80" : "=&v"(k.mask), "=v"(k.sixteen));
  else asm("v_mov_b32 %0, 0x3c003c0\n\tv_mov_b32 %1, 0x4c004c00" : "=&v"(k.mask), "=v"(k.sixteen));
  if constexpr (T == TACO_F32) k.offset = ZEROS ? 0xb980b980u : 0xbb00bb00u;               // -1, -8 (times UNIT)
  else if constexpr (T == TACO_BF16) k.offset = ZEROS ? 0xbb80bb80u : 0xbbc0bbc0u;         // -16, -24
  else k.offset = ZEROS ? 0xcc00cc00u : 0xce00ce00u;
  if (wave < whole) {
    // The next block and its piece of the vectors come while this one is multiplied.  Every turn makes the same loads (the last
    // one again where there is no next block): behind a branch around them the compiler would not know how many are in flight, and
    // would wait for all.  The empty statements keep it from moving them behind the products (28672 x 8192
    // with zero points 39 -> 30 us); with one row block, 16 waves do without, and better (4096 x 1558 for sixteen fp32 vectors 6.4
    // against 7.8).
    typename K::Block block[2];
    typename K::Vectors x[2];
    block[0].load(a, codes, scales, zeros, wave);
    K::load_x(x[0], xr, wave, g);
    for (int k0 = wave;; k0 += 2 * NW) {
      const int k1 = k0 + NW, k2 = k1 + NW;
      block[1].load(a, codes, scales, zeros, min(k1, whole - 1));
      K::load_x(x[1], xr, min(k1, whole - 1), g);
      if constexpr (RT > 1) asm volatile("" ::: "memory");
      K::multiply(block[0], x[0], k, y);
      if (k1 >= whole) break;
      block[0].load(a, codes, scales, zeros, min(k2, whole - 1));
      K::load_x(x[0], xr, min(k2, whole - 1), g);
      if constexpr (RT > 1) asm volatile("" ::: "memory");
      K::multiply(block[1], x[1], k, y);
      if (k2 >= whole) break;
    }
  }
  if (whole < (int)a.col_blocks && wave == whole % NW) {      // the last block's columns end inside it
    typename K::Block block;
    typename K::Vectors x;
    block.load(a, codes, scales, zeros, whole);
    K::load_x_end(x, xr, whole, g, a.n_cols);
    K::multiply(block, x, k, y);
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
    total *= 1.0f / K::UNIT;
    if (n < a.n_rows && v0 + v < a.n_vectors) {
      if (a.bias) total += a.bias[n];
      char* out = a.y + (int64_t)(v0 + v) * a.y_stride;
      if constexpr (T == TACO_F32) ((float*)out)[n] = total;
      else if constexpr (T == TACO_F16) ((_Float16*)out)[n] = (_Float16)total;
      else ((__bf16*)out)[n] = (__bf16)total;
    }
  }
}

template <int T, int MT, int RT, int NW, int GPB, int S>
int launch(const taco_qmat_multiply_params& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.n_rows + 16 * RT - 1) / (16 * RT)), (unsigned)((a.n_vectors + 16 * MT - 1) / (16 * MT))), block(64 * NW);
  const bool zeros = a.zeros_at != 0;
  if constexpr (T != TACO_F32)
    if (((uintptr_t)a.x | (a.n_vectors > 1 ? a.x_stride : 0)) & 2) {
      if (zeros) taco_qmat_multiply_kernel<T, MT, RT, NW, GPB, S, true, true><<<grid, block, 0, s>>>(a);
      else taco_qmat_multiply_kernel<T, MT, RT, NW, GPB, S, false, true><<<grid, block, 0, s>>>(a);
      TACO_HIP(hipGetLastError());
      return TACO_OK;
    }
  if (zeros) taco_qmat_multiply_kernel<T, MT, RT, NW, GPB, S, true, false><<<grid, block, 0, s>>>(a);
  else taco_qmat_multiply_kernel<T, MT, RT, NW, GPB, S, false, false><<<grid, block, 0, s>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}

// How many row blocks a workgroup takes, and whether one or two tiles of 16 vectors.  Blocks of rows times tiles that have a CU each:
// one workgroup of 16 waves per CU, so that a row block's columns are read by as many waves as possible (bfloat16, one vector, us with
// 1 x 16 / 2 x 16 / 4 x 8 row blocks x waves: 4096 x 4096 4.6 / 6.6 / 7.1, 8192 x 8192 11.6 / 9.6 / 12.4).  More than two to a CU: each
// piece of the vectors that is read serves four row blocks (14336 x 4096 with sixteen vectors 22 / 14 / 9.7, 28672 x 8192 with one 40 /
// 35 / 29).  Groups of 32 columns leave too few registers for four row blocks with fp32 scales, and for 16 waves with two.
// More than 16 vectors of a 16-bit type take two tiles at a time: with two row blocks reading the vectors would bind (28672 x 4096 with
// 32: 43 us, with four 26; 9000 x 4096 21.7 and 13.5), with one every CU is busy sooner (4096 x 4096 with 32: 11.6 with two, 10.2 with
// one; not in groups of 32, 4096 x 4097 19.5 and 22.1).  fp32 vectors need three times the registers and take a tile at a time (28672 x
// 4096 with 32: 50 us, two tiles and two row blocks 80), two only where four row blocks have no room (groups of 32, 28672 x 4096
// with 17: 73 and 81).
// Some of these have too few registers by a handful.  Two tiles with four row blocks (fp32 scales in groups of 64 5 to 13 short, other
// scales of vectors at odd addresses up to 12) win all the same: 28672 x 4096 with 32 bfloat16 vectors in groups of 64 with fp32 scales 32 us, with
// two row blocks 48, at odd addresses with zero points 42 and 60.  Sixteen waves with two row blocks in groups of 64 with fp32 scales (5 to 9 short)
// do not: eight would take 13.8 us instead of 17.7 for 4160 x 4096 with sixteen fp32 vectors, 9.3 instead of 10.5 with bfloat16 ones, 16.9 and
// 17.1 for 8192 x 8192 with one; with 16-bit scales one vector takes 8.9 and 8.7, 15.9 and 16.0.
template <int T, int GPB, int S>
int launch(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s) {
  constexpr bool FOUR = !(GPB == 4 && S == TACO_F32);
  constexpr int WAVES = GPB == 4 ? 8 : 16;
  const int64_t row_blocks = (a.n_rows + 15) / 16;
  int64_t blocks = row_blocks * ((a.n_vectors + 15) / 16);
  if (blocks <= n_cu) return launch<T, 1, 1, 16, GPB, S>(a, s);
  if constexpr (T != TACO_F32)
    if (a.n_vectors > 16) {
      blocks = row_blocks * ((a.n_vectors + 31) / 32);
      if constexpr (GPB < 4)
        if (blocks <= n_cu) return launch<T, 2, 1, 8, GPB, S>(a, s);
      if constexpr (FOUR)
        if (blocks > 2 * n_cu) return launch<T, 2, 4, 8, GPB, S>(a, s);
      return launch<T, 2, 2, 8, GPB, S>(a, s);
    }
  if (blocks > 2 * n_cu) {
    if constexpr (FOUR) return launch<T, 1, 4, 8, GPB, S>(a, s);
    else if (T == TACO_F32 && a.n_vectors > 16) return launch<T, 2, 2, 8, GPB, S>(a, s);
  }
  return launch<T, 1, 2, WAVES, GPB, S>(a, s);
}
template <int T, int GPB>
int launch(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s) {
  if (a.scale_dtype == TACO_F32) return launch<T, GPB, TACO_F32>(a, n_cu, s);
  return a.scale_dtype == TACO_F16 ? launch<T, GPB, TACO_F16>(a, n_cu, s) : launch<T, GPB, TACO_BF16>(a, n_cu, s);
}
template <int T>
int launch(const taco_qmat_multiply_params& a, int n_cu, hipStream_t s) {
  return a.per_block == 1 ? launch<T, 1>(a, n_cu, s) : a.per_block == 2 ? launch<T, 2>(a, n_cu, s) : launch<T, 4>(a, n_cu, s);
}

}  // namespace
