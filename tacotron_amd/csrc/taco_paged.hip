// A paged cache of keys and values and the attention of one new token over it (taco_kv_* in include/taco.h): the step of
// a decoder with self-attention.  Both kernels move every byte of their operands once and are bound by that.
#include "taco_place.h"
#include "taco_step.h"

#include <atomic>
#include <type_traits>

namespace {

// ---- append ---------------------------------------------------------------------------------------------------------

struct AppendParams {
  const char *k, *v, *q;
  char *q_out, *k_pages, *v_pages;
  int64_t k_st[2], v_st[2], q_st[2], qo_st[2], kp_st[3], vp_st[3];   // bytes
  const float *k_scale, *v_scale;
  const int32_t *table, *past, *offsets;
  const double* inv_freq;
  uint32_t* flags;
  int64_t table_stride;
  taco_divisor page;
  int32_t n_tokens, n_seqs, table_width, n_pages, n_heads, n_q_heads, head_dim, rot_dim, interleaved;
};

// sin and cos of pos * freq.  The angle is reduced in 64 bits (fp32 would lose an angle of 1e5 rad to 8e-3), the rest
// |r| <= pi/4 goes through the Taylor polynomials of degree 9 and 10, whose first omitted terms are 1.8e-9 and 1.2e-10.
__device__ __forceinline__ void sin_cos(double angle, float& s, float& c) {
  const double n = rint(angle * 0.63661977236758134308);            // 2 / pi
  double r = fma(-n, 1.57079632679489655800, angle);                // pi / 2 in two parts
  r = fma(-n, 6.12323399573676603587e-17, r);
  const float x = (float)r, z = x * x;
  const float ps = x + x * z * (-1.0f / 6 + z * (1.0f / 120 + z * (-1.0f / 5040 + z * (1.0f / 362880))));
  const float pc = 1.0f + z * (-0.5f + z * (1.0f / 24 + z * (-1.0f / 720 + z * (1.0f / 40320 + z * (-1.0f / 3628800)))));
  const int quadrant = (int)(long long)n & 3;
  s = (quadrant & 1) ? pc : ps;
  c = (quadrant & 1) ? ps : pc;
  if (quadrant & 2) s = -s;
  if (quadrant == 1 || quadrant == 2) c = -c;
}

// Rounds to the cache's type: 8-bit caches hold x / scale, held inside the type's range (a NaN stays one).
template <int C>
__device__ __forceinline__ void store_cache(char* p, float (&x)[8], float scale) {
  if constexpr (C == TACO_E4M3) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = x[i] / scale;
      x[i] = y != y ? y : __builtin_amdgcn_fmed3f(y, -448.0f, 448.0f);
    }
  }
  taco_store8<C>(p, x);
}

// One workgroup per token.  Its first rot_dim / 2 threads compute the token's sines and cosines once for all heads; then
// every thread takes pieces of 16 elements of a head: both halves of 8 pairs, or 16 elements that are only copied.
// Bound by moving the rows: 6200 tokens of ragged prompts, 32 + 2 x 8 heads of 128 from bfloat16 into an 8-bit cache, 144 MB, take
// 29.8 us = 4.8 TB/s, what a large copy reaches; one token of 64 utterances 4.1 us, mostly the launch and one round trip to memory.
// Beyond 256 pieces a token takes turns, a round trip each: 128 + 2 x 8 heads of 128 5.9 us, 384 + 2 x 16 heads of 256 (26 turns) 20.7.
template <int T, int C>
__global__ __launch_bounds__(256) void taco_kv_append_kernel(const AppendParams a) {
  __shared__ float cs[128], sn[128];
  const int n = blockIdx.x, tid = threadIdx.x;
  int b = n, j = 0;
  if (a.offsets) {
    // the utterance: how many of offsets[1 .. n_seqs] are at or below this row (64 at a time, every wave for itself)
    b = 0;
    for (int i = 0; i < a.n_seqs; i += 64) {
      const int at = i + (tid & 63);
      b += __popcll(__ballot(at < a.n_seqs && a.offsets[at + 1] <= n));
    }
    if (b >= a.n_seqs) return;              // behind the last utterance
    j = n - a.offsets[b];
    if (j < 0) return;                      // in front of the first
  }
  const int past = a.past[b];
  const int64_t pos = (int64_t)past + j;
  const taco_place place = taco_find(a.table + (int64_t)b * a.table_stride, a.table_width, a.n_pages, pos, a.page);
  if (place.flag && tid == 0) atomicOr(a.flags, place.flag);
  const int64_t page = place.page, slot = place.unit;
  const int half = a.rot_dim / 2;
  if (tid < half) {
    float s, c;
    sin_cos((double)pos * a.inv_freq[tid], s, c);
    sn[tid] = s;
    cs[tid] = c;
  }
  __syncthreads();

  constexpr int TB = taco_size_of<T>, CB = taco_size_of<C>;
  const int per_head = a.head_dim / 16, rotated = a.rot_dim / 16;
  const int heads = (a.q ? a.n_q_heads : 0) + 2 * a.n_heads;
  for (int i = tid; i < heads * per_head; i += 256) {
    const int head = i / per_head, piece = i % per_head;
    // heads of k, then v, then q
    const bool is_k = head < a.n_heads, is_v = !is_k && head < 2 * a.n_heads;
    const int h = is_k ? head : is_v ? head - a.n_heads : head - 2 * a.n_heads;
    if ((is_k || is_v) && page < 0) continue;
    const bool turn = !is_v && piece < rotated;
    const bool split = turn && !a.interleaved;
    const int e0 = split ? piece * 8 : piece * 16, e1 = split ? half + piece * 8 : piece * 16 + 8;
    const char* src = is_k ? a.k + n * a.k_st[0] + h * a.k_st[1]
                    : is_v ? a.v + n * a.v_st[0] + h * a.v_st[1] : a.q + n * a.q_st[0] + h * a.q_st[1];
    float x[8], y[8];
    taco_load8<T>(src + e0 * TB, x);
    taco_load8<T>(src + e1 * TB, y);
    if (turn) {
      const float *c = cs + piece * 8, *s = sn + piece * 8;
      if (split) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float u = x[e], w = y[e];
          x[e] = u * c[e] - w * s[e];
          y[e] = w * c[e] + u * s[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float u = x[2 * e], w = x[2 * e + 1];
          x[2 * e] = u * c[e] - w * s[e];
          x[2 * e + 1] = w * c[e] + u * s[e];
          const float u2 = y[2 * e], w2 = y[2 * e + 1];
          y[2 * e] = u2 * c[4 + e] - w2 * s[4 + e];
          y[2 * e + 1] = w2 * c[4 + e] + u2 * s[4 + e];
        }
      }
    }
    if (is_k || is_v) {
      char* dst = is_k ? a.k_pages + page * a.kp_st[0] + slot * a.kp_st[1] + h * a.kp_st[2]
                       : a.v_pages + page * a.vp_st[0] + slot * a.vp_st[1] + h * a.vp_st[2];
      const float scale = C == TACO_E4M3 ? (is_k ? a.k_scale[h] : a.v_scale[h]) : 1.0f;
      store_cache<C>(dst + e0 * CB, x, scale);
      store_cache<C>(dst + e1 * CB, y, scale);
    } else {
      char* dst = a.q_out + n * a.qo_st[0] + h * a.qo_st[1];
      taco_store8<T>(dst + e0 * TB, x);
      taco_store8<T>(dst + e1 * TB, y);
    }
  }
}

// ---- attend ---------------------------------------------------------------------------------------------------------

struct AttendParams {
  const char *k_pages, *v_pages, *q;
  char* out;
  float* lse;
  int64_t kp_st[3], vp_st[3], q_st[2], o_st[2];      // bytes
  const float *k_scale, *v_scale;
  const int32_t *table, *lens;
  uint32_t* flags;
  int64_t table_stride;
  taco_divisor page16;                                    // 16-token blocks of a page
  char* workspace;                                   // see Partials
  float scale_log2;                                  // scale * log2(e)
  int32_t n_seqs, table_width, n_pages, n_heads, n_q_heads, group, q_tiles, head_dim, window;
  taco_divisor workgroups;                           // of the grid
};

constexpr int AT_WAVES = 4;
constexpr uint32_t PART = AT_WAVES;        // tiles of a part of a row: one for every wave
constexpr float NEG_INF = -__builtin_inff();

// The logarithm (base 2) of the weight of a score that equals the maximum.
template <int T>
constexpr float weight_shift = T == TACO_F16 ? 15.0f : 0.0f;

// What a wave holds of one (utterance, cache head, up to 16 query heads): the running maximum and sum of the softmax of
// query column l & 15 (base 2; the sum is this lane's own part of it) and the unnormalised output, transposed:
// o[blk][e][i] belongs to element blk * 16 * VE + (4 * (l >> 4) + i) * VE + e of that query's head.
template <int NB, int VE>
struct State {
  float m = NEG_INF, l = 0.0f;
  taco_f4 o[NB][VE];
};

// The attention works on tiles of TT tokens per wave (32 of 16- and 8-bit elements, 16 of fp32), straight from memory into
// the matrix cores' operand layout, so that nothing of the cache passes through LDS:
//   scores, transposed:  S^T[token][query] = K Q^T.  Lane l holds 16 bytes of row token l & 15 (contraction over head_dim).
//   output, transposed:  O^T[element][query] += V^T P^T.  The scores' layout - lane l has tokens 4 (l >> 4) + i of column
//     l & 15 - is the operand layout of P^T with the tokens taken in that order, so weights never change lanes.  A lane
//     loads VE neighbouring elements of each of its own tokens (16 lanes read one row end to end) and element e of all of
//     them is one operand: for 16-bit types a v_perm per word turns rows into operands.
// Weights are rounded to the operand type twice, p = hi + lo: one rounding alone would be as large as that of the
// output itself, and the second product costs nothing while memory is the bound.  For float16 they are relative to the maximum
// times 2^-15 (the largest weight is 32768, sums and outputs are fp32): float16 ends at 2^-24, and beside a weight of 1 many
// small ones, which may outweigh it, would be held to 2^-25 only.
// Measured (both kernels): 64 ragged sequences up to 8191 tokens, 32 query heads over 8 of 128 in bfloat16, 1.24 GB: 224 us = 5.5
// TB/s; one of 131075 tokens 100 us = 5.4 TB/s; 33 up to 20000 in 8 bits behind a window of 12000, 64 query heads, 0.68 GB: 137 us =
// 4.9 TB/s.  A large copy reaches 4.7 TB/s on this card.  Sixteen lines up to 3000 frames, 16 heads of 64 in float16, 0.11 GB: 30 us;
// a lone line of 777 frames in fp32 9.2 us, mostly two launches and five dependent round trips to memory.
// K and V serve 16 * QT query heads of a cache head; further ones read them again.  With more than 16, QT = 2 pays where reading
// is the bound (16 x 16384 tokens, 2 heads of 128 in bfloat16, 64 query heads: 82 us with QT = 1, 71 with 2; 16 x 60000 tokens
// of 64 elements, 64 query heads over one: 144 and 90), not for fp32, whose products are slower than its reading (48 query
// heads over 2 of 128: 78 and 86).  Heads of more than 128 elements take all 512 registers with QT = 2 and spill 19 of them in 16-bit caches,
// one workgroup to a CU; it still pays (16 x 16384 tokens, 2 heads of 256 in bfloat16, 34 / 128 query heads: 165 / 301 us with QT = 1, 125 / 186
// with 2; heads of 144 124 / 222 and 88 / 152; of 256 in 8 bits 103 / 183 and 74 / 137).
// Heads run in the next larger instance of 64, 128, 256 elements, whose products meet zeros behind the head: 16 x 16384 tokens, 8 query heads over
// 2 in bfloat16, heads of 64 / 80 / 96 / 128 / 192 / 256: 4.5 / 4.9 / 5.3 / 5.7 / 4.7 / 5.2 TB/s.
template <int T, int C, int DP, int QT>
struct Attend {
  static constexpr int CB = taco_size_of<C>;
  static constexpr int TT = C == TACO_F32 ? 16 : 32;           // tokens of a tile
  static constexpr int SUB = TT / 16;
  static constexpr int KE = 16 / CB;                           // elements of a 16-byte load of K
  static constexpr int NK = DP * CB / 64;                      // loads per row of K: four lanes read 64 bytes of it
  static constexpr int NQ = C == TACO_F32 ? DP / 16 : DP / 32; // operands of Q
  static constexpr int VE = C == TACO_F32 ? 4 : C == TACO_E4M3 ? DP / 16 : (DP < 128 ? DP / 16 : 8);   // elements of a load of V
  static constexpr int NB = DP / (16 * VE);
  static constexpr int VW = VE * CB / 4;                       // ... in words
  static constexpr float SHIFT = weight_shift<T>;
  using St = State<NB, VE>;

  // Query operands: for the K operand whose lane holds elements d0 .. of a row, the same elements of query column l & 15.
  using Queries = taco_u4[QT][NQ];
  static __device__ void load_q(const AttendParams& a, int b, int h, int qt, Queries& q) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const int nth = (qt * QT + t) * 16 + col;
      const bool have = nth < a.group;
      const char* row = a.q + (int64_t)b * a.q_st[0] + (int64_t)(h * a.group + (have ? nth : 0)) * a.q_st[1];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        int d;      // first element
        if constexpr (C == TACO_E4M3) d = (n >> 1) * 64 + g * 16 + (n & 1) * 8;
        else d = (n * 4 + g) * KE;
        q[t][n] = taco_u4{0, 0, 0, 0};
        if (have && d < a.head_dim) q[t][n] = *(const taco_u4*)(row + (int64_t)d * taco_size_of<T>);
      }
    }
  }

  static __device__ __forceinline__ void tile(const AttendParams& a, int b, int h, int t0, int low, int len, float factor,
                                              const Queries& q, St (&st)[QT]) {
    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    // the pages of the tile's 16-token blocks; a block behind the last token, or on a bad page, reads page 0 and is masked
    const int32_t* row = a.table + (int64_t)b * a.table_stride;
    int64_t page[SUB];
    int slot[SUB];
    bool ok[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int blk = t0 / 16 + s;
      taco_place place = {-1, 0, 0};
      if (blk * 16 < len && blk * 16 + 16 > low) place = taco_find(row, a.table_width, a.n_pages, blk, a.page16);
      if (place.flag && lane == 0) atomicOr(a.flags, place.flag);
      ok[s] = place.page >= 0;
      page[s] = ok[s] ? place.page : 0;
      slot[s] = (int)place.unit * 16;
    }
    taco_u4 kr[SUB][NK];
    uint32_t vr[SUB * 4][NB][VW];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const char* row = a.k_pages + page[s] * a.kp_st[0] + (int64_t)(slot[s] + col) * a.kp_st[1] + h * a.kp_st[2];
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        const int d = (n * 4 + g) * KE;
        kr[s][n] = taco_u4{0, 0, 0, 0};
        if (d < a.head_dim) kr[s][n] = *(const taco_u4*)(row + d * CB);
      }
    }
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const char* row = a.v_pages + page[s] * a.vp_st[0] + (int64_t)(slot[s] + g * 4 + i) * a.vp_st[1] + h * a.vp_st[2];
#pragma unroll
        for (int blk = 0; blk < NB; ++blk) {
          const int d = blk * 16 * VE + col * VE;
#pragma unroll
          for (int w = 0; w < VW; ++w) vr[s * 4 + i][blk][w] = 0;
          if (d < a.head_dim) {
            if constexpr (VW == 4) {
              const taco_u4 x = *(const taco_u4*)(row + d * CB);
#pragma unroll
              for (int w = 0; w < 4; ++w) vr[s * 4 + i][blk][w] = x[w];
            } else if constexpr (VW == 2) {
              const taco_u2 x = *(const taco_u2*)(row + d * CB);
              vr[s * 4 + i][blk][0] = x[0];
              vr[s * 4 + i][blk][1] = x[1];
            } else {
              vr[s * 4 + i][blk][0] = *(const uint32_t*)(row + d * CB);
            }
          }
        }
      }
    // scores
    float p[QT][SUB * 4];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      taco_f4 acc[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) acc[t] = taco_f4{0, 0, 0, 0};
#pragma unroll
      for (int n = 0; n < NK; ++n) {
        if constexpr (C == TACO_F32) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[s][n][e]), __uint_as_float(q[t][n][e]), acc[t], 0, 0, 0);
        } else if constexpr (C == TACO_E4M3) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const taco_u4 x = {widen<0>(kr[s][n][2 * e]), widen<1>(kr[s][n][2 * e]), widen<0>(kr[s][n][2 * e + 1]), widen<1>(kr[s][n][2 * e + 1])};
#pragma unroll
            for (int t = 0; t < QT; ++t) acc[t] = taco_mfma32<T>(x, q[t][2 * n + e], acc[t]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < QT; ++t) acc[t] = taco_mfma32<T>(kr[s][n], q[t][n], acc[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[t][s * 4 + i] = acc[t][i] * factor;
    }
    // masked tokens: their weight is 0, and what lies in their V rows must not meet it (0 * NaN)
    bool whole = t0 >= low && t0 + TT <= len;
#pragma unroll
    for (int s = 0; s < SUB; ++s) whole = whole && ok[s];
    if (!whole) {
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = t0 + s * 16 + g * 4 + i;
          if (!(ok[s] && at >= low && at < len)) {
#pragma unroll
            for (int t = 0; t < QT; ++t) p[t][s * 4 + i] = NEG_INF;
#pragma unroll
            for (int blk = 0; blk < NB; ++blk)
#pragma unroll
              for (int w = 0; w < VW; ++w) vr[s * 4 + i][blk][w] = 0;
          }
        }
    }
    // running maximum; the outputs are rescaled only in the tiles that raise it
    taco_u4 hi[QT], lo[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      St& own = st[t];
      float top = p[t][0];
#pragma unroll
      for (int i = 1; i < SUB * 4; ++i) top = fmaxf(top, p[t][i]);
      top = taco_max_rows(top);
      if (__any(top > own.m)) {
        const float m = fmaxf(own.m, top);
        const float f = m == NEG_INF ? 1.0f : __builtin_amdgcn_exp2f(own.m - m);
        own.m = m;
        own.l *= f;
#pragma unroll
        for (int blk = 0; blk < NB; ++blk)
#pragma unroll
          for (int e = 0; e < VE; ++e) own.o[blk][e] *= f;
      }
      const float m = (own.m == NEG_INF ? 0.0f : own.m) - SHIFT;
#pragma unroll
      for (int i = 0; i < SUB * 4; ++i) {
        p[t][i] = __builtin_amdgcn_exp2f(p[t][i] - m);
        own.l += p[t][i];
      }
      if constexpr (C != TACO_F32) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          hi[t][w] = taco_pack2<T>(p[t][2 * w], p[t][2 * w + 1]);
          const uint32_t both = hi[t][w];
          lo[t][w] = taco_pack2<T>(p[t][2 * w] - taco_low<T>(both), p[t][2 * w + 1] - taco_high<T>(both));
        }
      }
    }
    // output
    if constexpr (C == TACO_F32) {
#pragma unroll
      for (int blk = 0; blk < NB; ++blk)
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < QT; ++t)
              st[t].o[blk][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[i][blk][e]), p[t][i], st[t].o[blk][e], 0, 0, 0);
    } else {
#pragma unroll
      for (int blk = 0; blk < NB; ++blk)
#pragma unroll
        for (int w = 0; w < VE / 2; ++w) {       // elements 2w, 2w + 1
          uint32_t x[8];
#pragma unroll
          for (int t = 0; t < 8; ++t) {
            if constexpr (C == TACO_E4M3) x[t] = (w & 1) ? widen<1>(vr[t][blk][w / 2]) : widen<0>(vr[t][blk][w / 2]);
            else x[t] = vr[t][blk][w];
          }
          taco_u4 even, odd;
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            even[t] = __builtin_amdgcn_perm(x[2 * t + 1], x[2 * t], 0x05040100u);
            odd[t] = __builtin_amdgcn_perm(x[2 * t + 1], x[2 * t], 0x07060302u);
          }
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            taco_f4 &o0 = st[t].o[blk][2 * w], &o1 = st[t].o[blk][2 * w + 1];
            o0 = taco_mfma32<T>(even, hi[t], o0);
            o1 = taco_mfma32<T>(odd, hi[t], o1);
            o0 = taco_mfma32<T>(even, lo[t], o0);
            o1 = taco_mfma32<T>(odd, lo[t], o1);
          }
        }
    }
  }

  // Two 8-bit floats (the low or the high half of a word) as two 16-bit ones; exact in both 16-bit types.
  template <int HALF>
  static __device__ __forceinline__ uint32_t widen(uint32_t w) {
    if constexpr (T == TACO_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, HALF));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, HALF));
  }
};

// ---- who does what ----
// All tiles of a call stand in one line: utterance by utterance, within it row by row (a row: one cache head and up to 16 or
// 32 of its query heads), within a row from the first seen tile to the last, in parts of four tiles, one for each wave.  The line is cut
// into equal shares of whole parts, one per workgroup of a grid that fills the GPU once, whatever the lengths are: a long utterance alone
// is split over its length, a batch of short ones is packed, and no workgroup waits for the longest.  A row that lies within one share is
// finished by its workgroup; of a row that crosses a border every workgroup leaves a partial result (maximum, sum, output), which a
// second kernel joins in the order of the workgroups.  Shares of any number of tiles were slower where rows are short, because a
// workgroup's waves wait for each other at a row's end (64 utterances up to 255 tokens, 8 heads of 128: 27.5 us, with whole parts 17.8;
// up to 1023: 48 and 46.5).  Joining in the first kernel, by the last workgroup of a row, was slower: what the others wrote has to be
// stored through to memory and awaited (sixteen lines 35 against 31 us, with a fence 211).
__device__ __forceinline__ uint32_t lane_of(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }

// Inclusive sum over the lanes of a wave (DPP: shifts within rows of 16, then each row's last value to the next one's lanes,
// then that of the lower half to the upper).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t add_dpp(uint32_t v) {
  return v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
  v = add_dpp<0x111, 0xf>(v);      // row_shr:1, 2, 4, 8
  v = add_dpp<0x112, 0xf>(v);
  v = add_dpp<0x114, 0xf>(v);
  v = add_dpp<0x118, 0xf>(v);
  v = add_dpp<0x142, 0xa>(v);      // row_bcast:15
  return add_dpp<0x143, 0xc>(v);   // row_bcast:31
}

// 64 utterances, one per lane: what each sees and of how many parts its rows are.
template <int TT>
struct Utterances {
  int base;                  // the first of them
  uint32_t before;           // parts of a row of each utterance in front of them
  int low, len;              // seen tokens [low, len) of this lane's utterance
  uint32_t tiles;            // of its rows (one that sees nothing has a tile, so that somebody writes its zeros)
  uint32_t parts, scan;      // of PART tiles each; inclusive sum

  __device__ __forceinline__ void load(const AttendParams& a, int first, bool flag) {
    base = first;
    const int b = first + (threadIdx.x & 63);
    len = low = 0;
    tiles = 0;
    if (b < a.n_seqs) {
      len = a.lens[b];
      const int64_t room = (int64_t)a.table_width * a.page16.div * 16;
      low = a.window > 0 && len > a.window ? len - a.window : 0;      // the window ends at the length given, wherever the table does
      if (len < 0 || len > room) {
        if (flag) atomicOr(a.flags, TACO_KV_BAD_PLACE);
        len = len < 0 ? 0 : (int)room;
      }
      tiles = len > low ? (uint32_t)((len + TT - 1) / TT - low / TT) : 1;
    }
    parts = (tiles + PART - 1) / PART;
    scan = wave_scan(parts);
  }
  __device__ __forceinline__ uint32_t last() const { return lane_of(scan, 63); }
  // Loads the first 64 and counts all.
  __device__ __forceinline__ uint32_t load_all(const AttendParams& a, bool flag) {
    uint32_t sum = 0;
    for (int i = 64; i < a.n_seqs; i += 64) {
      load(a, i, flag);
      sum += last();
    }
    load(a, 0, flag);
    before = 0;
    return sum + last();
  }
  // Moves on to the 64 that utterance `b` is one of.
  __device__ __forceinline__ void move_to(const AttendParams& a, int b) {
    while (b >= base + 64) {
      before += last();
      load(a, base + 64, false);
    }
  }
  // Moves on to the 64 in which part `at` of all rows lies and returns its utterance; `at` becomes the part within it.
  __device__ __forceinline__ int find(const AttendParams& a, uint64_t& at, uint32_t rows_per) {
    while (at >= (uint64_t)(before + last()) * rows_per) move_to(a, base + 64);
    const int lane = __popcll(__ballot((uint64_t)(before + scan) * rows_per <= at));      // those that end at or before it
    at -= (uint64_t)(before + lane_of(scan, lane) - lane_of(parts, lane)) * rows_per;
    return base + lane;
  }
};

// Parts of a share (the division by the number of workgroups is a multiplication as long as it fits, see taco_divisor).
__device__ __forceinline__ uint64_t share_of(const AttendParams& a, uint64_t all) {
  const uint64_t n = all + a.workgroups.div - 1;
  return n < (1u << 30) ? taco_divide((uint32_t)n, a.workgroups) : n / a.workgroups.div;
}
__device__ __forceinline__ uint64_t div64(uint64_t n, uint64_t d) { return (n | d) >> 32 ? n / d : (uint64_t)((uint32_t)n / (uint32_t)d); }

// The workspace: for every row its first workgroup and how many it has, then the partial results' maxima and sums, [2 per
// workgroup][queries][2], then their outputs [2 per workgroup][queries][DP].
struct Partials {
  taco_u2* rows;
  float *ml, *o;
  __device__ __forceinline__ Partials(const AttendParams& a, uint32_t rows_per, int held)
      : rows((taco_u2*)a.workspace), ml((float*)(rows + (((size_t)a.n_seqs * rows_per + 1) & ~(size_t)1))), o(ml + (size_t)a.workgroups.div * held * 4) {}
};

template <int T>
__device__ __forceinline__ void store_out(char* row, int d, float o) {
  if constexpr (T == TACO_F32) ((float*)row)[d] = o;
  else if constexpr (T == TACO_BF16) ((__bf16*)row)[d] = (__bf16)o;
  else ((_Float16*)row)[d] = (_Float16)o;
}
// Element d of a finished row: o and `sum` are relative to the maximum m.
template <int T, int C>
__device__ __forceinline__ void finish(const AttendParams& a, int b, int head, int h, int d, float o, float sum, float m) {
  if (d >= a.head_dim) return;
  o = sum == 0.0f ? 0.0f : o / sum * (C == TACO_E4M3 ? a.v_scale[h] : 1.0f);
  store_out<T>(a.out + (int64_t)b * a.o_st[0] + (int64_t)head * a.o_st[1], d, o);
  if (d == 0 && a.lse) a.lse[(int64_t)b * a.n_q_heads + head] = sum == 0.0f ? NEG_INF : (m - weight_shift<T> + __builtin_amdgcn_logf(sum)) * 0.693147180559945309f;
}
// What a part counts for beside the common maximum.
__device__ __forceinline__ float weight_of(float m_part, float m) { return m_part == NEG_INF ? 0.0f : __builtin_amdgcn_exp2f(m_part - m); }

template <int T, int C, int DP, int QT>
__global__ __launch_bounds__(64 * AT_WAVES) void taco_kv_attend_kernel(const AttendParams a) {
  using A = Attend<T, C, DP, QT>;
  extern __shared__ float lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  const uint32_t rows_per = a.n_heads * a.q_tiles;         // rows of an utterance
  Utterances<A::TT> us;
  const uint64_t all = (uint64_t)us.load_all(a, blockIdx.x == 0 && threadIdx.x < 64) * rows_per;
  const uint64_t share = share_of(a, all);        // parts of a workgroup
  uint64_t at = share * blockIdx.x;               // where this one begins
  if (at >= all) return;
  uint64_t left = min(share, all - at);
  int b = us.find(a, at, rows_per);
  const uint32_t first_parts = lane_of(us.parts, b - us.base);
  uint32_t row = (uint32_t)div64(at, first_parts);
  uint32_t part0 = (uint32_t)(at - (uint64_t)row * first_parts);
  const int held = min(a.group, 16 * QT);            // queries of a row in LDS and in the partial results
  for (bool first = true; left; first = false) {
    us.move_to(a, b);
    const int low = (int)lane_of(us.low, b - us.base), len = (int)lane_of(us.len, b - us.base);
    const uint32_t tiles = lane_of(us.tiles, b - us.base), row_parts = lane_of(us.parts, b - us.base);
    const uint32_t taken = left < row_parts - part0 ? (uint32_t)left : row_parts - part0;
    const uint32_t tile0 = part0 * PART, n = min(taken * PART, tiles - tile0);
    const int h = a.q_tiles == 1 ? row : row / a.q_tiles, qt = row - h * a.q_tiles;
    typename A::Queries q;
    A::load_q(a, b, h, qt, q);
    float factor = a.scale_log2;
    if (C == TACO_E4M3) factor *= a.k_scale[h];
    typename A::St st[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int blk = 0; blk < A::NB; ++blk)
#pragma unroll
        for (int e = 0; e < A::VE; ++e) st[t].o[blk][e] = taco_f4{0, 0, 0, 0};
    const int base = (low / A::TT + (int)tile0) * A::TT;
    if (len > low)
      for (uint32_t t = wave; t < n; t += AT_WAVES) A::tile(a, b, h, base + (int)t * A::TT, low, len, factor, q, st);
    // join the waves: [wave][query][m, l, DP outputs]
    if (!first) __syncthreads();
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float l = taco_sum_rows(st[t].l);
      if (t * 16 + col < held) {
        float* mine = lds + (wave * held + t * 16 + col) * (DP + 2);
        if (g == 0) { mine[0] = st[t].m; mine[1] = l; }
#pragma unroll
        for (int blk = 0; blk < A::NB; ++blk)
#pragma unroll
          for (int e = 0; e < A::VE; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[2 + blk * 16 * A::VE + (4 * g + i) * A::VE + e] = st[t].o[blk][e][i];
      }
    }
    __syncthreads();
    const int rows = min(a.group - qt * 16 * QT, 16 * QT);
    // a row that began in an earlier share is this workgroup's first partial result, one that only ends later its second
    const Partials parts(a, rows_per, held);
    if (part0 == 0 && threadIdx.x == 0)      // of how many shares the row is, the next ones holding `share` parts each
      parts.rows[(size_t)b * rows_per + row] = taco_u2{blockIdx.x, 1 + (uint32_t)div64(row_parts - taken + share - 1, share)};
    const size_t slot = (size_t)(2 * blockIdx.x + (part0 ? 0 : 1)) * held;
    for (int i = threadIdx.x; i < rows * DP; i += 64 * AT_WAVES) {
      const int r = i / DP, d = i % DP;
      const float* p = lds + r * (DP + 2);
      float m = NEG_INF, sum = 0.0f, o = 0.0f;
#pragma unroll
      for (int w = 0; w < AT_WAVES; ++w) m = fmaxf(m, p[w * held * (DP + 2)]);
#pragma unroll
      for (int w = 0; w < AT_WAVES; ++w) {
        const float* x = p + w * held * (DP + 2);
        const float f = weight_of(x[0], m);
        sum += f * x[1];
        o += f * x[2 + d];
      }
      if (taken == row_parts) {
        finish<T, C>(a, b, h * a.group + qt * 16 * QT + r, h, d, o, sum, m);
      } else {
        if (d == 0) { parts.ml[(slot + r) * 2] = m; parts.ml[(slot + r) * 2 + 1] = sum; }
        parts.o[(slot + r) * DP + d] = o;
      }
    }
    left -= taken;
    part0 = 0;
    if (++row == rows_per) { row = 0; ++b; }
  }
}

// Joins the rows that cross a border of shares, one workgroup per row and query.  A long utterance alone leaves a hundred parts
// of a row, so the maxima are taken by 256 threads at a time and the outputs by as many groups of DP / 4 threads as there are,
// each with its own parts, in a fixed order.  What most rows need, 256 maxima and sums and four parts for each group, is loaded at once.
template <int T, int C, int DP, int QT>
__global__ __launch_bounds__(256) void taco_kv_join_kernel(const AttendParams a) {
  constexpr int GROUPS = 256 / (DP / 4), AHEAD = 4;
  __shared__ float red[2][4], weight[256];
  __shared__ taco_f4 outs[GROUPS][DP / 4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t rows_per = a.n_heads * a.q_tiles;
  const int held = min(a.group, 16 * QT);
  const Partials parts(a, rows_per, held);
  const uint32_t nth = blockIdx.x / held;
  const taco_u2 info = parts.rows[nth];
  const uint32_t w0 = info[0], n = info[1];
  if (n == 1) return;
  const uint32_t row = nth % rows_per;
  const int r = blockIdx.x % held, b = nth / rows_per, qt = row % a.q_tiles, h = row / a.q_tiles;
  if (qt * 16 * QT + r >= a.group) return;
  const auto at = [&](uint32_t k) { return (size_t)(2 * (w0 + k) + (k ? 0 : 1)) * held + r; };
  const int mine = tid / (DP / 4), piece = tid % (DP / 4);
  const auto ml_of = [&](uint32_t k) { return *(const taco_f2*)(parts.ml + at(k) * 2); };
  const auto o_of = [&](uint32_t k) { return *(const taco_f4*)(parts.o + at(k) * DP + piece * 4); };
  taco_f2 own = {NEG_INF, 0.0f};
  taco_f4 part[AHEAD];
  const auto load_ahead = [&](uint32_t k0) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) part[i] = o_of(min(k0 + mine + i * GROUPS, n - 1));       // behind the last: it again, without weight
  };
  if ((uint32_t)tid < n) own = ml_of(tid);
  load_ahead(0);
  float m = own[0];
  for (uint32_t k = tid + 256; k < n; k += 256) m = fmaxf(m, ml_of(k)[0]);
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float sum = 0.0f;
  taco_f4 o = {0, 0, 0, 0};
  for (uint32_t k0 = 0; k0 < n; k0 += 256) {
    if (k0) {
      __syncthreads();
      if (k0 + tid < n) own = ml_of(k0 + tid);
      load_ahead(k0);
    }
    if (k0 + tid < n) {
      weight[tid] = weight_of(own[0], m);
      sum += weight[tid] * own[1];
    }
    __syncthreads();
    const uint32_t here = n - k0 < 256 ? n - k0 : 256;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if ((uint32_t)(mine + i * GROUPS) < here) o += weight[mine + i * GROUPS] * part[i];
#pragma unroll 4
    for (uint32_t j = mine + AHEAD * GROUPS; j < here; j += GROUPS) o += weight[j] * o_of(k0 + j);
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if (lane == 0) red[1][wave] = sum;
  outs[mine][piece] = o;
  __syncthreads();
  sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  for (int d = tid; d < DP; d += 256) {
    float total = 0.0f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) total += outs[i][d / 4][d % 4];
    finish<T, C>(a, b, h * a.group + qt * 16 * QT + r, h, d, total, sum, m);
  }
}

// ---- host ----------------------------------------------------------------------------------------------------------

// Workgroups of 256 threads of one launch must be fewer: a grid's threads are counted in 32 bits.
constexpr int32_t MAX_GRID = 1 << 24;

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Addresses of rows: base and strides (elements) in multiples of 16 bytes; writes the strides in bytes.
template <int N>
bool row_strides(const void* base, const int64_t* stride, int size, int64_t (&bytes)[N]) {
  bool ok = base && aligned(base);
  for (int i = 0; i < N; ++i) {
    bytes[i] = stride[i] * size;
    ok = ok && bytes[i] % 16 == 0;
  }
  return ok;
}

int check_cache(const taco_kv_cache* c, const char* who, int dtype) {
  if (!c) TACO_FAIL(TACO_EINVAL, "%s: NULL cache", who);
  if (c->dtype < TACO_F32 || c->dtype > TACO_E4M3) TACO_FAIL(TACO_EINVAL, "%s: cache dtype %d", who, c->dtype);
  if (c->dtype == TACO_E4M3 ? dtype != TACO_F16 && dtype != TACO_BF16 : dtype != c->dtype)
    TACO_FAIL(TACO_EINVAL, "%s: dtype %d does not go with a cache of dtype %d", who, dtype, c->dtype);
  if (c->n_pages < 1 || c->n_heads < 1 || c->n_heads > 65535) TACO_FAIL(TACO_EINVAL, "%s: %d pages, %d heads", who, c->n_pages, c->n_heads);
  if (c->page_size < 16 || c->page_size % 16 || c->page_size > 65536) TACO_FAIL(TACO_EINVAL, "%s: page_size %d is not a multiple of 16 up to 65536", who, c->page_size);
  if (c->head_dim < 16 || c->head_dim % 16 || c->head_dim > 256) TACO_FAIL(TACO_EINVAL, "%s: head_dim %d is not a multiple of 16 up to 256", who, c->head_dim);
  if ((c->dtype == TACO_E4M3) != (c->k_scale && c->v_scale) || (c->k_scale == nullptr) != (c->v_scale == nullptr))
    TACO_FAIL(TACO_EINVAL, "%s: scales belong to 8-bit caches, and those need both", who);
  if (!c->flags) TACO_FAIL(TACO_EINVAL, "%s: NULL flags", who);
  return TACO_OK;
}

}  // namespace

int taco_device_check(int device, int* n_cu) {
  static std::atomic<int> known[64];       // CUs of a gfx950 device, 0 = not asked yet
  if (device < 0 || device >= 64) TACO_FAIL(TACO_EINVAL, "device %d", device);
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    hipDeviceProp_t prop;
    TACO_HIP(hipGetDeviceProperties(&prop, device));
    bool same = true;
    for (int i = 0; i < 6; ++i) same = same && prop.gcnArchName[i] == "gfx950"[i];
    if (!same) TACO_FAIL(TACO_EINVAL, "device %d is %s; this library is built for gfx950 only", device, prop.gcnArchName);
    n = prop.multiProcessorCount;
    known[device].store(n, std::memory_order_relaxed);
  }
  *n_cu = n;
  return TACO_OK;
}

extern "C" int taco_kv_append(const taco_kv_cache* c, const taco_kv_append_args* t, void* stream) {
  const char* who = "taco_kv_append";
  if (!t) TACO_FAIL(TACO_EINVAL, "%s: NULL argument", who);
  int rc = check_cache(c, who, t->dtype);
  if (rc != TACO_OK) return rc;
  if (t->n_tokens < 0 || t->n_seqs < 0 || t->table_width < 0) TACO_FAIL(TACO_EINVAL, "%s: %d tokens, %d utterances, table width %d", who, t->n_tokens, t->n_seqs, t->table_width);
  if (t->n_tokens >= MAX_GRID) TACO_FAIL(TACO_EINVAL, "%s: %d tokens at once, at most %d", who, t->n_tokens, MAX_GRID - 1);
  if (!t->offsets && t->n_tokens != t->n_seqs) TACO_FAIL(TACO_EINVAL, "%s: %d tokens for %d utterances without offsets", who, t->n_tokens, t->n_seqs);
  if (t->rot_dim < 0 || t->rot_dim % 16 || t->rot_dim > c->head_dim) TACO_FAIL(TACO_EINVAL, "%s: rot_dim %d is not a multiple of 16 up to head_dim %d", who, t->rot_dim, c->head_dim);
  if (t->rot_dim && !t->inv_freq) TACO_FAIL(TACO_EINVAL, "%s: rot_dim %d without frequencies", who, t->rot_dim);
  if ((t->q == nullptr) != (t->q_out == nullptr) || (t->q && (t->n_q_heads < 1 || t->n_q_heads > 65535))) TACO_FAIL(TACO_EINVAL, "%s: queries", who);
  if (t->n_tokens == 0 || t->n_seqs == 0) return TACO_OK;
  if (!t->table || !t->past) TACO_FAIL(TACO_EINVAL, "%s: NULL table or past", who);
  AppendParams a;
  const int size = t->dtype == TACO_F32 ? 4 : 2, held = c->dtype == TACO_F32 ? 4 : c->dtype == TACO_E4M3 ? 1 : 2;
  bool ok = row_strides(t->k, t->k_stride, size, a.k_st) && row_strides(t->v, t->v_stride, size, a.v_st) &&
            row_strides(c->k, c->k_stride, held, a.kp_st) && row_strides(c->v, c->v_stride, held, a.vp_st);
  a.q_st[0] = a.q_st[1] = a.qo_st[0] = a.qo_st[1] = 0;
  if (t->q) ok = ok && row_strides(t->q, t->q_stride, size, a.q_st) && row_strides(t->q_out, t->q_out_stride, size, a.qo_st);
  if (!ok) TACO_FAIL(TACO_EINVAL, "%s: rows must start at multiples of 16 bytes (and not be NULL)", who);
  int n_cu;
  DeviceScope on_device(c->device);
  TACO_HIP(on_device.status);
  rc = taco_device_check(c->device, &n_cu);
  if (rc != TACO_OK) return rc;
  a.k = (const char*)t->k; a.v = (const char*)t->v; a.q = (const char*)t->q; a.q_out = (char*)t->q_out;
  a.k_pages = (char*)c->k; a.v_pages = (char*)c->v; a.k_scale = c->k_scale; a.v_scale = c->v_scale;
  a.table = t->table; a.past = t->past; a.offsets = t->offsets; a.inv_freq = t->inv_freq; a.flags = c->flags;
  a.table_stride = t->table_stride; a.page = taco_make_divisor((uint32_t)c->page_size);
  a.n_tokens = t->n_tokens; a.n_seqs = t->n_seqs; a.table_width = t->table_width; a.n_pages = c->n_pages;
  a.n_heads = c->n_heads; a.n_q_heads = t->n_q_heads; a.head_dim = c->head_dim; a.rot_dim = t->rot_dim; a.interleaved = t->interleaved;
  const dim3 grid((unsigned)t->n_tokens), block(256);
  hipStream_t s = (hipStream_t)stream;
  if (c->dtype == TACO_F32) taco_kv_append_kernel<TACO_F32, TACO_F32><<<grid, block, 0, s>>>(a);
  else if (c->dtype == TACO_F16) taco_kv_append_kernel<TACO_F16, TACO_F16><<<grid, block, 0, s>>>(a);
  else if (c->dtype == TACO_BF16) taco_kv_append_kernel<TACO_BF16, TACO_BF16><<<grid, block, 0, s>>>(a);
  else if (t->dtype == TACO_F16) taco_kv_append_kernel<TACO_F16, TACO_E4M3><<<grid, block, 0, s>>>(a);
  else taco_kv_append_kernel<TACO_BF16, TACO_E4M3><<<grid, block, 0, s>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}

namespace {

// Everything about a call that its sizes decide.
struct Plan {
  int group, q_tiles, held, dp, tt;
  uint32_t workgroups;
  bool join;
  int64_t bytes;
};

template <int T, int C, int DP, int QT>
int plan_of(Plan& p, int device, int n_cu) {
  // workgroups of this kernel that a CU holds: a grid beyond that would end with a part-filled round
  static std::atomic<int> known[64][16 * QT + 1];
  p.tt = Attend<T, C, DP, QT>::TT;
  const size_t lds = (size_t)AT_WAVES * p.held * (DP + 2) * 4;
  int per_cu = known[device][p.held].load(std::memory_order_relaxed);
  if (!per_cu) {
    auto kernel = taco_kv_attend_kernel<T, C, DP, QT>;
    constexpr int MOST = AT_WAVES * 16 * QT * (DP + 2) * 4;
    static_assert(MOST <= 160 * 1024, "a CU's LDS");
    if (MOST > 65536) TACO_HIP(hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, MOST));
    TACO_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&per_cu, kernel, 64 * AT_WAVES, lds));
    if (per_cu < 1) TACO_FAIL(TACO_EINVAL, "taco_kv_attend: the kernel does not fit a CU");
    known[device][p.held].store(per_cu, std::memory_order_relaxed);
  }
  p.workgroups = (uint32_t)(per_cu * n_cu);
  return TACO_OK;
}
template <int T, int C, int DP, int QT>
int launch_attend(const AttendParams& a, const Plan& p, hipStream_t s) {
  const size_t lds = (size_t)AT_WAVES * p.held * (DP + 2) * 4;
  taco_kv_attend_kernel<T, C, DP, QT><<<dim3(p.workgroups), dim3(64 * AT_WAVES), lds, s>>>(a);
  if (p.join) taco_kv_join_kernel<T, C, DP, QT><<<dim3((unsigned)(a.n_seqs * a.n_heads * a.q_tiles * p.held)), dim3(256), 0, s>>>(a);
  TACO_HIP(hipGetLastError());
  return TACO_OK;
}

// The kernel for a call's types, head size and queries per cache head.
template <typename F>
int by_types(const taco_kv_cache* c, int dtype, int group, F&& f) {
  const auto by_group = [&](auto t, auto h, auto d) {
    if constexpr (h.value != TACO_F32)
      if (group > 16) return f(t, h, d, std::integral_constant<int, 2>());
    return f(t, h, d, std::integral_constant<int, 1>());
  };
  const auto by_dim = [&](auto t, auto h) {
    if (c->head_dim <= 64) return by_group(t, h, std::integral_constant<int, 64>());
    if (c->head_dim <= 128) return by_group(t, h, std::integral_constant<int, 128>());
    return by_group(t, h, std::integral_constant<int, 256>());
  };
  using F32 = std::integral_constant<int, TACO_F32>;
  using F16 = std::integral_constant<int, TACO_F16>;
  using BF16 = std::integral_constant<int, TACO_BF16>;
  using E4M3 = std::integral_constant<int, TACO_E4M3>;
  if (c->dtype == TACO_F32) return by_dim(F32(), F32());
  if (c->dtype == TACO_F16) return by_dim(F16(), F16());
  if (c->dtype == TACO_BF16) return by_dim(BF16(), BF16());
  if (dtype == TACO_F16) return by_dim(F16(), E4M3());
  return by_dim(BF16(), E4M3());
}

// The rest of a plan; the device is current.
int plan_attend(const taco_kv_cache* c, const taco_kv_attend_args* t, Plan& p) {
  p.dp = c->head_dim <= 64 ? 64 : c->head_dim <= 128 ? 128 : 256;
  int n_cu;
  int rc = taco_device_check(c->device, &n_cu);
  if (rc != TACO_OK) return rc;
  rc = by_types(c, t->dtype, p.group, [&](auto ty, auto ca, auto dp, auto qt) { return plan_of<ty.value, ca.value, dp.value, qt.value>(p, c->device, n_cu); });
  if (rc != TACO_OK) return rc;
  const int64_t rows = (int64_t)t->n_seqs * c->n_heads * p.q_tiles;
  const int64_t tiles = ((int64_t)t->table_width * c->page_size + p.tt - 1) / p.tt;       // of a row, at most
  // no more workgroups than there are parts when every row is cut on its own; shares are whole parts, so where a table has room for
  // one part of a row only, every row is finished by one workgroup and the second kernel is left out
  const int64_t parts = ((tiles < 1 ? 1 : tiles) + PART - 1) / PART, most = rows * parts;
  p.join = parts > 1;
  if (most < p.workgroups) p.workgroups = (uint32_t)most;
  p.bytes = (rows + 1) / 2 * 16 + (int64_t)2 * p.workgroups * p.held * (2 + p.dp) * 4;
  return TACO_OK;
}

// Checks the sizes and settles how the query heads are divided.
int check_attend(const taco_kv_cache* c, const taco_kv_attend_args* t, const char* who, Plan& p) {
  if (!t) TACO_FAIL(TACO_EINVAL, "%s: NULL argument", who);
  const int rc = check_cache(c, who, t->dtype);
  if (rc != TACO_OK) return rc;
  if (t->n_seqs < 0 || t->table_width < 0) TACO_FAIL(TACO_EINVAL, "%s: %d utterances, table width %d", who, t->n_seqs, t->table_width);
  if (t->n_q_heads < 1 || t->n_q_heads % c->n_heads) TACO_FAIL(TACO_EINVAL, "%s: %d query heads over %d cache heads", who, t->n_q_heads, c->n_heads);
  if ((int64_t)t->table_width * c->page_size >= TACO_KV_MAX_TOKENS) TACO_FAIL(TACO_EINVAL, "%s: %d pages of %d tokens per utterance", who, t->table_width, c->page_size);
  p.group = t->n_q_heads / c->n_heads;
  const int at_once = p.group <= 16 || c->dtype == TACO_F32 ? 16 : 32;
  p.q_tiles = (p.group + at_once - 1) / at_once;
  p.held = p.group < at_once ? p.group : at_once;
  // a workgroup joins each query head (of whole groups of `held`); 16-token tiles are counted in 32 bits
  if ((int64_t)t->n_seqs * c->n_heads * p.q_tiles * p.held >= MAX_GRID || ((int64_t)t->table_width * c->page_size / 16 + 1) * t->n_seqs >= (1ll << 32))
    TACO_FAIL(TACO_EINVAL, "%s: %d utterances of %d heads and up to %d pages", who, t->n_seqs, t->n_q_heads, t->table_width);
  return TACO_OK;
}

}  // namespace

extern "C" int64_t taco_kv_attend_workspace(const taco_kv_cache* c, const taco_kv_attend_args* t) {
  const char* who = "taco_kv_attend_workspace";
  Plan p;
  int rc = check_attend(c, t, who, p);
  if (rc != TACO_OK) return rc;
  if (t->n_seqs == 0) return 0;
  DeviceScope on_device(c->device);
  TACO_HIP(on_device.status);
  rc = plan_attend(c, t, p);
  return rc == TACO_OK ? p.bytes : rc;
}

extern "C" int taco_kv_attend(const taco_kv_cache* c, const taco_kv_attend_args* t, void* stream) {
  const char* who = "taco_kv_attend";
  Plan p;
  int rc = check_attend(c, t, who, p);
  if (rc != TACO_OK) return rc;
  if (t->window < 0) TACO_FAIL(TACO_EINVAL, "%s: window %d", who, t->window);
  if (!(t->scale - t->scale == 0.0f)) TACO_FAIL(TACO_EINVAL, "%s: scale is not finite", who);
  if (t->n_seqs == 0) return TACO_OK;
  if (!t->lens || (!t->table && t->table_width)) TACO_FAIL(TACO_EINVAL, "%s: NULL table or lens", who);
  AttendParams a;
  const int size = t->dtype == TACO_F32 ? 4 : 2, held = c->dtype == TACO_F32 ? 4 : c->dtype == TACO_E4M3 ? 1 : 2;
  if (!(row_strides(t->q, t->q_stride, size, a.q_st) && row_strides(t->out, t->out_stride, size, a.o_st) &&
        row_strides(c->k, c->k_stride, held, a.kp_st) && row_strides(c->v, c->v_stride, held, a.vp_st)))
    TACO_FAIL(TACO_EINVAL, "%s: rows must start at multiples of 16 bytes (and not be NULL)", who);
  DeviceScope on_device(c->device);
  TACO_HIP(on_device.status);
  rc = plan_attend(c, t, p);
  if (rc != TACO_OK) return rc;
  if ((!t->workspace || !aligned(t->workspace) || t->workspace_bytes < p.bytes)) TACO_FAIL(TACO_EINVAL, "%s: needs a 16-byte aligned workspace of %lld bytes, has %lld", who, (long long)p.bytes, (long long)t->workspace_bytes);
  a.k_pages = (const char*)c->k; a.v_pages = (const char*)c->v; a.k_scale = c->k_scale; a.v_scale = c->v_scale;
  a.q = (const char*)t->q; a.out = (char*)t->out; a.lse = t->lse; a.table = t->table; a.lens = t->lens; a.flags = c->flags;
  a.table_stride = t->table_stride; a.page16 = taco_make_divisor((uint32_t)c->page_size / 16);
  a.scale_log2 = t->scale * 1.44269504088896340736f;
  a.n_seqs = t->n_seqs; a.table_width = t->table_width; a.n_pages = c->n_pages; a.n_heads = c->n_heads;
  a.n_q_heads = t->n_q_heads; a.head_dim = c->head_dim; a.window = t->window;
  a.group = p.group; a.q_tiles = p.q_tiles; a.workspace = (char*)t->workspace;
  a.workgroups = taco_make_divisor(p.workgroups);
  return by_types(c, t->dtype, p.group, [&](auto ty, auto ca, auto dp, auto qt) { return launch_attend<ty.value, ca.value, dp.value, qt.value>(a, p, (hipStream_t)stream); });
}

namespace {

// Clears what has been reported and nothing else: a call on another stream may have set a bit since the flags were read.
__global__ void taco_kv_clear_flags_kernel(uint32_t* flags, uint32_t reported) { atomicAnd(flags, ~reported); }

}  // namespace

extern "C" int taco_kv_status(const taco_kv_cache* c, void* stream) {
  if (!c || !c->flags) TACO_FAIL(TACO_EINVAL, "taco_kv_status: NULL argument");
  DeviceScope on_device(c->device);
  TACO_HIP(on_device.status);
  hipStream_t s = (hipStream_t)stream;
  uint32_t flags = 0;
  TACO_HIP(hipMemcpyAsync(&flags, c->flags, 4, hipMemcpyDeviceToHost, s));
  TACO_HIP(hipStreamSynchronize(s));
  if (!flags) return TACO_OK;
  taco_kv_clear_flags_kernel<<<dim3(1), dim3(1), 0, s>>>(c->flags, flags);
  TACO_HIP(hipGetLastError());
  TACO_HIP(hipStreamSynchronize(s));
  TACO_FAIL(TACO_ERANGE, "%s%s%s", flags & TACO_KV_BAD_PAGE ? "a table entry is no page of the cache" : "",
            flags == (TACO_KV_BAD_PAGE | TACO_KV_BAD_PLACE) ? "; " : "", flags & TACO_KV_BAD_PLACE ? "a position or length lies outside the table" : "");
}
