// Matrix product with bias, activation and residual in its epilogue, and what its backward pass needs beside products.
//
//   z = x w^T + b (8-bit operands: z = sx_m sw_n (xq wq^T) + b)     y = f(z) + res        x [M, K], w [N, K], y [M, N]
//   backward: dz = dy f'(z),  dx = dz w,  dw = dz^T x,  db = sum_m dz,  dres = dy
//
// One tile kernel for every type and direction.  A tile step is 128 bytes of contraction (64 16-bit, 32 fp32 or 128 8-bit
// elements), and only the matrix instruction differs between types:
//   16-bit: 2 x v_mfma_f32_16x16x32,   fp32: 8 x v_mfma_f32_16x16x4_f32,   e4m3: 1 x v_mfma_f32_16x16x128_f8f6f4
// (a contraction may take its terms in any order, so each type reads 16-byte pieces lane group by lane group).
// The e4m3 instruction adds eight products at a time aligned to the largest of them and drops what is below 2^-13 of it
// (measured with powers of two; between the eights, and onto the accumulator, it adds in fp32): at most 2^-10 of the largest
// product, and 1e-5 of a whole result at K = 16 .. 4096, next to 2^-9 / 2^-12 that a 16-bit result is rounded by.  An fp32
// result would show it, so there the operands become bf16 (exactly: 4 significant bits) and 4 x v_mfma_f32_16x16x32_bf16 add
// them in fp32.
//
// An operand has the contraction along its rows, or (dx reads w, dw reads dz and x that way) down its columns; the tile in LDS
// keeps the operand's own order, and a transposed fragment is read by ds_read_b64_tr_b16 (16-bit) or as single floats (one
// matrix instruction takes one float a lane), so no transposed copy is ever made.
//
// Tiles go global -> LDS by DMA, two stages.  The DMA writes 64 consecutive 16-byte pieces, so the swizzle that keeps fragment
// reads off each other's banks is applied to the SOURCE address.  One barrier a step, placed before the step's last row of
// matrix instructions: by then every fragment of the stage is in registers and the next stage has landed, so behind the
// barrier the DMA of the step after next starts and the next step's first fragments are read while matrix instructions run.
//
// Measured (large library products reach 1 354 TFLOP/s in bf16, 2 748 in e4m3, 153 in fp32 here): 8 192^3 bf16 807 us =
// 1 362 TFLOP/s, 8 192^3 e4m3 389 us = 2 823; 16 384 x 4 096 x 1 024 bf16 129 us = 1 066 (with bias, gelu and slopes 190), its
// dx 111 us = 1 238, its dw 135 us = 1 018; 8 192 x 2 048 x 4 096 e4m3 62 us = 2 200; 4 096 x 4 096 x 1 024 fp32 254 us = 135.
//
// For training, 16-bit types keep f'(z) in a 16-bit code (la_slope_codes) whose half step stays below the type's for slopes
// down to 2^-15 (fp16) and 2^-58 (bf16), where z rounded to the type would add as much as dz's rounding and more as |z| grows,
// and the backward pass needs no transcendental.  fp32 keeps z.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "ffn.h"

namespace {

struct e4m3 {};                                    // operand tags: OCP e4m3, one byte, for 16-bit results
struct e4m3_wide {};                               // and for fp32 results

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int LA_SLOPE_NAN = -32768;
constexpr float LA_LEAK = 0.01f;
constexpr int LA_MAX_SPLIT = 16;
constexpr int64_t LA_MAX_GRID = 1 << 23;           // workgroups of up to 512 threads: a launch holds fewer than 2^32 threads

__device__ __align__(16) const uint32_t la_zeros[4] = {0, 0, 0, 0};   // what lies past the end of a contraction

// ---- activations: f(z) and f'(z) ---------------------------------------------------------------------------------------
// FAST (16-bit results): gelu from q = erfc(|z| / sqrt 2) / 2 = exp(-z^2 / 2) P(t), t = 1 / (1 + p |z|), whose exponential the slope
// shares; p and the sixth-degree P, without a constant, were fitted here (weighted least squares, weights by the last fit's
// error) so that q as computed is off by less than 3e-7 and less than 3e-5 of itself: the negative tail, z q, is as exact as the type
// holds it.  tanh and the logistic function from one exponential.  fp32 results: gelu by the Chebyshev fit of erfc in Press
// et al., Numerical Recipes, 6.2 (relative error below 1.2e-7, and 1.5 z^2 2^-24 from the exponent's own rounding; a third of
// the library function's time), else the math library.
// ACT: HOTK_ACT_RELU stands for all three that are linear on either side of zero, with `neg` the slope below it.
template <int ACT, bool FAST>
__device__ __forceinline__ float la_act(float z, float neg, float& slope) {
  if constexpr (ACT == HOTK_ACT_GELU) {
    float cdf, pdf;
    if (FAST) {
      const float t = __builtin_amdgcn_rcpf(fmaf(0.2958828887f, fabsf(z), 1.f));
      const float e = __builtin_amdgcn_exp2f(z * (-0.72134752f * z));
      const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.08316676316f, 0.2464154638f), -0.04891132795f), 0.1582405465f), 0.1087127227f),
                               0.1187092262f) * e;
      cdf = z < 0.f ? q : 1.f - q;       // (1/2 - (1/2 - q) would leave nothing of a small q)
      pdf = 0.39894228f * e;
    } else {
      const float x = 0.70710678f * fabsf(z), xx = 0.5f * z * z;
      const float t = 1.f / fmaf(0.5f, x, 1.f);
      const float p = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.17087277f, -0.82215223f), 1.48851587f), -1.13520398f),
                      0.27886807f), -0.18628806f), 0.09678418f), 0.37409196f), 1.00002368f), -1.26551223f);
      const float q = 0.5f * t * __builtin_amdgcn_exp2f(1.44269504f * (p - xx));
      cdf = z < 0.f ? q : 1.f - q;
      pdf = 0.39894228f * __builtin_amdgcn_exp2f(-1.44269504f * xx);
    }
    slope = fmaf(z, pdf, cdf);
    return z * cdf;
  } else if constexpr (ACT == HOTK_ACT_TANH) {
    // q = 1 - |tanh z| = 2 / (e^2|z| + 1): the slope 1 - tanh^2 is q (2 - q), which keeps its digits where tanh is next to one
    const float e = FAST ? __builtin_amdgcn_exp2f(2.88539008f * fabsf(z)) : expf(2.f * fabsf(z));
    const float q = FAST ? 2.f * __builtin_amdgcn_rcpf(e + 1.f) : 2.f / (e + 1.f);
    slope = q * (2.f - q);
    if (!FAST) return tanhf(z);
    const float s = z * z;
    const float series = z * fmaf(s, fmaf(s, fmaf(s, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);   // to z^7: |z| < 1/4
    return fabsf(z) < 0.25f ? series : copysignf(1.f - q, z);
  } else if constexpr (ACT == HOTK_ACT_SILU) {
    const float e = FAST ? __builtin_amdgcn_exp2f(-1.44269504f * z) : expf(-z);
    const float s = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
    slope = s * fmaf(z, 1.f - s, 1.f);
    return z * s;
  } else {
    slope = z > 0.f ? 1.f : neg;
    return z > 0.f ? z : neg == 0.f ? (z <= 0.f ? 0.f : z) : neg * z;      // (relu: no infinity times zero, and a NaN stays one)
  }
}
__device__ __forceinline__ float la_neg(int act) { return act == HOTK_ACT_RELU ? 0.f : act == HOTK_ACT_LEAKYRELU ? LA_LEAK : 1.f; }
// v times the slopes at z (fp32): the activation is chosen once for the piece
__device__ __forceinline__ void la_times_slope(f32x4& v, const f32x4& z, int act) {
  const float neg = la_neg(act);
  auto each = [&](auto which) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float d;
      la_act<decltype(which)::value, false>(z[k], neg, d);
      v[k] *= d;
    }
  };
  switch (act) {
    case HOTK_ACT_GELU: each(std::integral_constant<int, HOTK_ACT_GELU>{}); break;
    case HOTK_ACT_TANH: each(std::integral_constant<int, HOTK_ACT_TANH>{}); break;
    case HOTK_ACT_SILU: each(std::integral_constant<int, HOTK_ACT_SILU>{}); break;
    default: each(std::integral_constant<int, HOTK_ACT_RELU>{});
  }
}
// Codes of slopes, -0.13 < d < 1.13.  A code is sign(d) k - 8192: the codes below zero that negative slopes leave unused go to the
// positive ones.  From |d| = 1/16 up k goes in steps of 2^-14 (2^-11 of |d| at most); below, where a saturated unit's gradient
// lives, as a root of |d|, so that k's half step stays small against |d|:  k = 21504 (16 |d|)^(1/n).  fp16: n = 8, half a step is
// 2^-12.4 of |d| at 1/16, 2^-11.1 at 2^-14 (fp16's smallest normal number), 2^-10 at 2^-23; bf16: n = 16, 2^-11.4 at 1/16, 2^-10 at
// 2^-26, 2^-8 at 2^-58.  The types' own half steps are 2^-11 and 2^-8.  (With one step of 2^-14 for all, at the cost of two
// transcendentals less, gradients of tanh units were 9 % off at |z| = 5.5 and zero from 6 on.)  Piecewise linear activations
// need one bit.
typedef int16_t s16x8 __attribute__((ext_vector_type(8)));
constexpr float LA_CODE_EDGE = 0.0625f, LA_CODE_AT_EDGE = 21504.f, LA_CODE_SHIFT = 8192.f, LA_CODE_STEP = 0x1p-14f;
template <class OT> struct LaRoot;
template <> struct LaRoot<_Float16> {
  static constexpr int N = 8;
  static constexpr float LOG_EDGE = -0.10763855f;      // log2(21504 / 32767 * 16^(1/n)): the packed conversion's unit is 1 / 32767
  static constexpr float WEIGHT = 0.70710678f / LA_CODE_AT_EDGE;       // 16^(-1/n)
};
template <> struct LaRoot<__bf16> {
  static constexpr int N = 16;
  static constexpr float LOG_EDGE = -0.35763855f;
  static constexpr float WEIGHT = 0.84089642f / LA_CODE_AT_EDGE;
};
template <int ACT, class OT>
__device__ __forceinline__ s16x8 la_slope_codes(const float* d) {
  constexpr float UNIT = 1.f / 32767.f;
  s16x8 c;
  if constexpr (ACT == HOTK_ACT_RELU) {
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = d[k] == 1.f;
    return c;
  }
  float sum = 0.f, v[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = fabsf(d[k]);
    const float linear = fmaf(a, UNIT / LA_CODE_STEP, UNIT * (LA_CODE_AT_EDGE - LA_CODE_EDGE / LA_CODE_STEP));
    const float root = __builtin_amdgcn_exp2f(fmaf(__builtin_amdgcn_logf(a), 1.f / LaRoot<OT>::N, LaRoot<OT>::LOG_EDGE));
    v[k] = copysignf(a < LA_CODE_EDGE ? root : linear, d[k]) - UNIT * LA_CODE_SHIFT;
    sum += d[k];
  }
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    const auto p = __builtin_amdgcn_cvt_pknorm_i16(v[k], v[k + 1]);
    c[k] = p[0];
    c[k + 1] = p[1];
  }
  if (sum != sum) {                      // (a NaN among them is rare)
#pragma unroll
    for (int k = 0; k < 8; ++k) c[k] = d[k] != d[k] ? (int16_t)LA_SLOPE_NAN : c[k];
  }
  return c;
}
template <class OT>
__device__ __forceinline__ float la_slope(int16_t code, int act) {
  if (act == HOTK_ACT_RELU || act == HOTK_ACT_LEAKYRELU) return code ? 1.f : la_neg(act);
  const float c = (float)code + LA_CODE_SHIFT, a = fabsf(c);
  float root = a * LaRoot<OT>::WEIGHT;
#pragma unroll
  for (int n = LaRoot<OT>::N; n > 1; n /= 2) root *= root;
  const float linear = fmaf(a, LA_CODE_STEP, LA_CODE_EDGE - LA_CODE_AT_EDGE * LA_CODE_STEP);
  return code == LA_SLOPE_NAN ? __builtin_nanf("") : copysignf(a < LA_CODE_AT_EDGE ? root : linear, c);
}

// ---- epilogue ----------------------------------------------------------------------------------------------------------
template <class OT>
struct LaEpi {
  const OT *bias, *res;
  int64_t ld_res;
  OT* y;
  int64_t ld_y;
  void* save;                    // [M, N]: int16 slopes (16-bit types) or fp32 z, or null
  const float *xs, *ws;          // scales of 8-bit operands, or null
  int act;
};

// a piece of W values of a row as 16-byte accesses
template <int ACT, int W, class OT>
__device__ __forceinline__ void la_activate(const LaEpi<OT>& e, int64_t m, int64_t n0, int64_t N, int left, float (&z)[W]) {
  constexpr bool FAST = !std::is_same<OT, float>::value;
  const float neg = la_neg(e.act);
  float d[W];
  if (!FAST && e.save && e.act != HOTK_ACT_NONE) {
    float* row = (float*)e.save + m * N + n0;
#pragma unroll
    for (int i = 0; i < W; i += 4)
      if (i < left) ffn_store(row, i, left, f32x4{z[i], z[i + 1], z[i + 2], z[i + 3]});
  }
#pragma unroll
  for (int i = 0; i < W; ++i) z[i] = la_act<ACT, FAST>(z[i], neg, d[i]);
  if constexpr (FAST) {
    if (!e.save || e.act == HOTK_ACT_NONE) return;
    typedef int16_t s16x8u __attribute__((ext_vector_type(8), aligned(2)));
    int16_t* row = (int16_t*)e.save + m * N + n0;
#pragma unroll
    for (int i = 0; i < W; i += 8) {
      const s16x8 c = la_slope_codes<ACT, OT>(d + i);
      if (i + 8 <= left) {
        *reinterpret_cast<s16x8u*>(row + i) = c;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (i + k < left) row[i + k] = c[k];
      }
    }
  }
}

// W consecutive columns (a multiple of the 16-byte piece) of one row, from n0: z is the bare product.  The activation is chosen once per piece:
// W independent chains run side by side
template <int W, class OT>
__device__ __forceinline__ void la_finish(const LaEpi<OT>& e, int64_t m, int64_t n0, int64_t N, float (&z)[W]) {
  using E = Elem<OT>;
  const int left = (int)(N - n0 < W ? N - n0 : W);               // columns of this piece that exist
  if (left <= 0) return;
  if (e.xs) {
    const float xs = e.xs[m];
    const bool large = fabsf(xs) > 1.f;  // then w's scale goes first: nothing overflows on the way that the result holds
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const f32x4 s = ffn_load(e.ws + n0, i, left);
#pragma unroll
      for (int k = 0; k < 4; ++k) z[i + k] *= large ? s[k] : xs;
#pragma unroll
      for (int k = 0; k < 4; ++k) z[i + k] *= large ? xs : s[k];
    }
  }
  if (e.bias) {
#pragma unroll
    for (int i = 0; i < W; i += E::VEC) {
      const auto b = ffn_load(e.bias + n0, i, left);
#pragma unroll
      for (int k = 0; k < E::VEC; ++k) z[i + k] += b[k];
    }
  }
  switch (e.act) {
    case HOTK_ACT_NONE: break;
    case HOTK_ACT_GELU: la_activate<HOTK_ACT_GELU>(e, m, n0, N, left, z); break;
    case HOTK_ACT_TANH: la_activate<HOTK_ACT_TANH>(e, m, n0, N, left, z); break;
    case HOTK_ACT_SILU: la_activate<HOTK_ACT_SILU>(e, m, n0, N, left, z); break;
    default: la_activate<HOTK_ACT_RELU>(e, m, n0, N, left, z);
  }
#pragma unroll
  for (int i = 0; i < W; i += E::VEC) {
    typename E::fvec v;
#pragma unroll
    for (int k = 0; k < E::VEC; ++k) v[k] = z[i + k];
    if (e.res) v += ffn_load(e.res + m * e.ld_res + n0, i, left);
    if (i < left) ffn_store(e.y + m * e.ld_y + n0, i, left, v);
  }
}

// ---- the tile kernel ---------------------------------------------------------------------------------------------------
template <class OT>
struct LaTile {
  const char *a, *b;             // x [M, K] or [K, M], w [N, K] or [K, N]
  int64_t lda, ldb;              // bytes per row
  int64_t M, N, K;
  int ktiles, kper;              // 128-byte steps, and how many of them a split takes
  int wrap;                      // steps of the contraction: from here on x_lo, `low` bytes behind x, takes x's place
  int64_t low;
  int tiles_m, tiles_n;
  float* part;                   // [splits][M][N] bare products, where there is more than one split
  LaEpi<OT> e;
};

// 16 bytes per lane from a wave-uniform base plus a 32-bit offset per lane, or from a lane's own address, to LDS bytes
// dst + 16 * lane.  The compiler does not count these loads: every wait for them is written out.
__device__ __forceinline__ void la_dma(const void* base, uint32_t voff, uint32_t dst) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(voff), "s"(base), "s"(dst) : "memory");
}
__device__ __forceinline__ void la_dma_at(const void* src, uint32_t dst) {
  unsigned keep;
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep) : "v"(src), "s"(dst) : "memory");
}
template <int N>
__device__ __forceinline__ void la_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory"); }
// workgroup barrier behind this wave's LDS reads, silent about the loads in flight
__device__ __forceinline__ void la_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory"); }

// An operand tile in LDS: BLK columns by one step.  Along rows (T false): BLK rows of 8 pieces, piece p of row r holds chunk
// p ^ (r & 7).  Down columns (T true): a step's rows of BLK elements; blocks of 16 elements are exchanged by a key of the row,
// such that the rows which a fragment read touches at once lie in different banks.
template <class IT> struct LaBytes { static constexpr int E = 2; };
template <> struct LaBytes<float> { static constexpr int E = 4; };
template <> struct LaBytes<e4m3> { static constexpr int E = 1; };
template <> struct LaBytes<e4m3_wide> { static constexpr int E = 1; };

template <class IT, bool T, int BLK>
struct LaSide {
  static constexpr int E = LaBytes<IT>::E, STEP = 128 / E;       // elements of contraction a step
  static constexpr int PPR = T ? BLK * E / 16 : 8;               // pieces per row of the tile
  static constexpr int PPB = E;                                  // pieces per block of 16 elements (T)
  static __device__ __forceinline__ int key(int k) {
    return (E == 2 ? (k & 3) | ((k >> 1) & 4) : (k >> 2) & 3) & (BLK / 16 - 1);
  }
  // piece number `piece` of the tile: its row of the operand's tile, and which chunk of that row it holds
  static __device__ __forceinline__ void source(int piece, int& row, int& chunk) {
    row = piece / PPR;
    const int pos = piece % PPR;
    if (T) chunk = (((pos / PPB) ^ key(row)) * PPB) | (pos % PPB);
    else chunk = pos ^ (row & 7);
  }
  // 16 bytes of contraction of column col0 + lr, piece 4 h + lg
  static __device__ __forceinline__ u32x4 frag(const unsigned char* tile, int col0, int h, int lr, int lg) {
    u32x4 v;
    if constexpr (!T) {
      const int row = col0 + lr;
      v = *reinterpret_cast<const u32x4*>(tile + row * 128 + (((4 * h + lg) ^ (row & 7)) << 4));
    } else if constexpr (E == 2) {
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
      for (int q = 0; q < 2; ++q) {      // lane 4 r + c of a group brings columns 4 c .. of row r and leaves with a column of four rows
        const int k = 32 * h + 8 * lg + 4 * q + (lr >> 2), col = col0 + 4 * (lr & 3);
        const unsigned char* at = tile + k * (BLK * 2) + (((col >> 4) ^ key(k)) << 5) + (col & 15) * 2;
        const u32x2 t = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at));
        v[2 * q] = t[0];
        v[2 * q + 1] = t[1];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 16 * h + 4 * lg + i, col = col0 + lr;
        v[i] = *reinterpret_cast<const uint32_t*>(tile + k * (BLK * 4) + (((col >> 4) ^ key(k)) << 6) + (col & 15) * 4);
      }
    }
    return v;
  }
};

// what a lane holds of a fragment: two 16-byte pieces, or their elements in bf16
template <class IT>
struct LaFrag {
  u32x4 h[2];
  __device__ __forceinline__ void set(int i, u32x4 v) { h[i] = v; }
};
template <>
struct LaFrag<e4m3_wide> {
  bf16x8 b[4];
  __device__ __forceinline__ void set(int i, u32x4 v) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const auto lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[k], 1.f, false), hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(v[k], 1.f, true);
      b[2 * i + k / 2][4 * (k & 1)] = lo[0];
      b[2 * i + k / 2][4 * (k & 1) + 1] = lo[1];
      b[2 * i + k / 2][4 * (k & 1) + 2] = hi[0];
      b[2 * i + k / 2][4 * (k & 1) + 3] = hi[1];
    }
  }
};

// matrix instructions of one fragment pair, in parts of one instruction each
template <class IT> struct LaParts { static constexpr int N = 2; };
template <> struct LaParts<float> { static constexpr int N = 8; };
template <> struct LaParts<e4m3> { static constexpr int N = 1; };
template <> struct LaParts<e4m3_wide> { static constexpr int N = 4; };
template <class IT>
__device__ __forceinline__ void la_mma(int p, f32x4& c, const LaFrag<IT>& w, const LaFrag<IT>& x) {
  if constexpr (std::is_same<IT, __bf16>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.h[p]), __builtin_bit_cast(bf16x8, x.h[p]), c, 0, 0, 0);
  } else if constexpr (std::is_same<IT, _Float16>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w.h[p]), __builtin_bit_cast(f16x8, x.h[p]), c, 0, 0, 0);
  } else if constexpr (std::is_same<IT, float>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.h[p >> 2][p & 3]), __uint_as_float(x.h[p >> 2][p & 3]), c, 0, 0, 0);
  } else if constexpr (std::is_same<IT, e4m3_wide>::value) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.b[p], x.b[p], c, 0, 0, 0);
  } else {
    const i32x8 wv = {(int)w.h[0][0], (int)w.h[0][1], (int)w.h[0][2], (int)w.h[0][3], (int)w.h[1][0], (int)w.h[1][1], (int)w.h[1][2], (int)w.h[1][3]};
    const i32x8 xv = {(int)x.h[0][0], (int)x.h[0][1], (int)x.h[0][2], (int)x.h[0][3], (int)x.h[1][0], (int)x.h[1][1], (int)x.h[1][2], (int)x.h[1][3]};
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wv, xv, c, 0, 0, 0, 0, 0, 0);     // (scale operands 0: none)
  }
}

// which tile a workgroup takes: workgroups go round the eight dies, so each die is given a run of consecutive tiles, and
// runs walk down groups of eight tile rows: what a die reads at a time is a few tile rows of x and of w, in its own L2
__device__ __forceinline__ void la_tile_of(int pid, int tiles_m, int tiles_n, int& im, int& in) {
  const int total = tiles_m * tiles_n, per = total >> 3, rem = total & 7, die = pid & 7;
  pid = die * per + (die < rem ? die : rem) + (pid >> 3);
  const int span = 8 * tiles_n, first = pid / span * 8, in_group = pid % span;
  const int rows = tiles_m - first < 8 ? tiles_m - first : 8;
  im = first + in_group % rows;
  in = in_group / rows;
}

// one operand's part of the DMA: its pieces for this lane and where they come from
template <class IT, bool T, int BLK, int NW>
struct LaFeed {
  using S = LaSide<IT, T, BLK>;
  static constexpr int LOADS = BLK * 8 / 64 / NW;
  static_assert(BLK * 8 % (64 * NW) == 0, "whole DMA instructions per wave");
  const char* base;
  int64_t ld;
  uint32_t off[LOADS];
  int wave, lane;
  // columns past the operand's end repeat its last row (T: piece); their products are not stored
  __device__ __forceinline__ LaFeed(const char* p, int64_t ld_, int64_t col0, int64_t cols, int wave_, int lane_)
      : base(T ? p + col0 * S::E : p + col0 * ld_), ld(ld_), wave(wave_), lane(lane_) {
    const int64_t left = cols - col0;
    const int last = T ? (int)((left < BLK ? left : BLK) * S::E + 15) / 16 - 1 : (int)(left < BLK ? left : BLK) - 1;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int row, chunk;
      S::source((wave + NW * i) * 64 + lane, row, chunk);
      if (T) chunk = chunk < last ? chunk : last;
      else row = row < last ? row : last;
      off[i] = (uint32_t)(row * ld) + chunk * 16;
    }
  }
  __device__ __forceinline__ void issue(int kt, int64_t K, uint32_t dst, int64_t shift) const {
    const char* at = base + shift + (T ? (int64_t)kt * S::STEP * ld : (int64_t)kt * 128);
    if ((int64_t)(kt + 1) * S::STEP <= K) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) la_dma(at, off[i], dst + (wave + NW * i) * 1024);
    } else {                             // the last step: zeros where the contraction has ended
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        int row, chunk;
        S::source((wave + NW * i) * 64 + lane, row, chunk);
        const int64_t k = (int64_t)kt * S::STEP + (T ? row : chunk * (16 / S::E));
        la_dma_at(k < K ? at + off[i] : (const char*)la_zeros, dst + (wave + NW * i) * 1024);
      }
    }
  }
};

template <class IT, class OT, bool TA, bool TB, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_linact_tile(const LaTile<OT> g) {
  constexpr int NW = WM * WN, TM = BM / WM, MF = TM / 16, NF = 4, STAGE = (BM + BN) * 128;
  // (the two x stages side by side where both operands lie along rows: 2 % faster; where one is read across, stage by stage)
  constexpr int XS = TB ? STAGE : BM * 128, WS = TB ? STAGE : BN * 128, W0 = TB ? BM * 128 : 2 * BM * 128;
  static_assert(BN / WN == 64 && BM % (16 * WM) == 0, "a wave owns 64 columns");
  using SA = LaSide<IT, TA, BM>;
  using SB = LaSide<IT, TB, BN>;
  extern __shared__ __align__(16) unsigned char lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, lr = lane & 15, lg = lane >> 4;
  int im, in;
  la_tile_of(blockIdx.x, g.tiles_m, g.tiles_n, im, in);
  const int64_t m0 = (int64_t)im * BM, n0 = (int64_t)in * BN;
  const int k0 = blockIdx.y * g.kper, k1 = min(g.ktiles, k0 + g.kper);
  const LaFeed<IT, TA, BM, NW> fa(g.a, g.lda, m0, g.M, wave, lane);
  const LaFeed<IT, TB, BN, NW> fb(g.b, g.ldb, n0, g.N, wave, lane);
  auto issue = [&](int kt, int stage) {
    const bool lo = kt >= g.wrap;
    const int k = lo ? kt - g.wrap : kt;
    fa.issue(k, g.K, lds0 + stage * XS, lo ? g.low : 0);
    fb.issue(k, g.K, lds0 + W0 + stage * WS, 0);
  };

  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = 0.f;
  LaFrag<IT> wf[2][NF], xf[2];
  auto read_w = [&](int stage, LaFrag<IT>(&f)[NF]) {
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) f[j].set(h, SB::frag(lds + W0 + stage * WS, wn * 64 + 16 * j, h, lr, lg));
  };
  auto read_x = [&](int stage, int i, LaFrag<IT>& f) {
#pragma unroll
    for (int h = 0; h < 2; ++h) f.set(h, SA::frag(lds + stage * XS, wm * TM + 16 * i, h, lr, lg));
  };
  // step kt from stage S: fragments 0 are in registers.  Before the last row of matrix instructions the stage has been read
  // whole, and step kt + 1 has landed in the other
  auto step = [&](int kt, auto stage_tag) {
    constexpr int S = decltype(stage_tag)::value;
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      if (i + 1 < MF) {
        read_x(S, i + 1, xf[(i + 1) & 1]);
      } else if (kt + 1 < k1) {
        la_wait_vm<0>();
        la_barrier();
        if (kt + 2 < k1) issue(kt + 2, S);
        read_w(S ^ 1, wf[S ^ 1]);
        read_x(S ^ 1, 0, xf[MF > 1 ? 0 : 1]);
      }
      __builtin_amdgcn_sched_barrier(0);       // the reads are under way before the matrix instructions that hide them
#pragma unroll
      for (int p = 0; p < LaParts<IT>::N; ++p)
#pragma unroll
        for (int j = 0; j < NF; ++j) la_mma<IT>(p, acc[i][j], wf[S][j], xf[i & 1]);
    }
    if (MF == 1) xf[0] = xf[1];
  };
  static_assert(MF == 1 || MF % 2 == 0, "the first fragment of a step is in xf[0]");

  if (k0 < k1) {
    issue(k0, 0);
    la_wait_vm<0>();
    la_barrier();
    if (k0 + 1 < k1) issue(k0 + 1, 1);
    read_w(0, wf[0]);
    read_x(0, 0, xf[0]);
    for (int kt = k0; kt < k1; kt += 2) {
      step(kt, std::integral_constant<int, 0>{});
      if (kt + 1 < k1) step(kt + 1, std::integral_constant<int, 1>{});
    }
  }

  // Out: HALF * 16 rows of the wave at a time go through its own piece of LDS, after which a lane holds V consecutive columns and
  // neighbouring lanes whole lines of a row.  The activations are a loop over pieces with one copy of the code, kept small:
  // unrolled over the accumulators it was 40 KB that every tile ran once, and fetching it took longer than running it (a 256 x 256
  // tile's end: 35 us against 6)
  constexpr int V = Elem<OT>::VEC, PER_ROW = 64 / V, ROWS = 64 / PER_ROW, PITCH = 68;
  constexpr int HALF = MF > 4 ? 4 : MF;
  static_assert(NW * HALF * 16 * PITCH * 4 <= 160 * 1024 && MF % HALF == 0, "the waves' pieces fit LDS");
  la_barrier();                          // every wave has read the last stage
  float* box = reinterpret_cast<float*>(lds) + wave * HALF * 16 * PITCH;
  const int64_t n = n0 + wn * 64 + V * (lane % PER_ROW);
  const int left = (int)(g.N - n < V ? g.N - n : V);
#pragma unroll 1
  for (int half = 0; half < MF / HALF; ++half) {
#pragma unroll
    for (int s = 0; s < MF / HALF; ++s)
      if (s == half) {
#pragma unroll
        for (int i = 0; i < HALF; ++i)
#pragma unroll
          for (int j = 0; j < NF; ++j) *reinterpret_cast<f32x4*>(box + (16 * i + lr) * PITCH + 16 * j + 4 * lg) = acc[s * HALF + i][j];
      }
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int r = lane / PER_ROW; r < HALF * 16; r += ROWS) {
      const int64_t m = m0 + wm * TM + half * (HALF * 16) + r;
      float z[V];
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(box + r * PITCH + V * (lane % PER_ROW) + k);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[k + q] = v[q];
      }
      if (m >= g.M || left <= 0) continue;
      if (g.part) {
        float* row = g.part + ((int64_t)blockIdx.y * g.M + m) * g.N + n;
#pragma unroll
        for (int k = 0; k < V; k += 4)
          if (k < left) ffn_store(row, k, left, f32x4{z[k], z[k + 1], z[k + 2], z[k + 3]});
      } else {
        la_finish<V>(g.e, m, n, g.N, z);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// joins the splits and finishes: LANES threads a piece of V columns, each adding every LANES-th split in order; they meet in LDS,
// again in order.  One thread a piece for up to four splits, eight for more (4 096 x 1 024 of two splits: 8.6 us against 17;
// 256 x 256 fp32 of sixteen: 6.7 against 3.9)
template <class OT, int LANES>
__global__ __launch_bounds__(256) void k_linact_join(const float* __restrict__ part, int splits, int64_t M, int64_t N,
                                                     const LaEpi<OT> e) {
  constexpr int V = Elem<OT>::VEC, PIECES = 256 / LANES;
  __shared__ __align__(16) float sums[LANES > 1 ? LANES : 1][PIECES][V];
  const int64_t per_row = (N + V - 1) / V, total = M * per_row;
  const int piece = threadIdx.x % PIECES, lane = threadIdx.x / PIECES;
  for (int64_t t0 = (int64_t)blockIdx.x * PIECES; t0 < total; t0 += (int64_t)gridDim.x * PIECES) {
    const int64_t t = t0 + piece, m = t / per_row, n = t % per_row * V;
    const int left = (int)(N - n < V ? N - n : V);
    float z[V];
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = 0.f;
    if (t < total)
      for (int s = lane; s < splits; s += LANES) {
        const float* row = part + ((int64_t)s * M + m) * N + n;
#pragma unroll
        for (int i = 0; i < V; i += 4) {
          if (i >= left) continue;
          const f32x4 v = ffn_load(row, i, left);
#pragma unroll
          for (int k = 0; k < 4; ++k) z[i + k] += v[k];
        }
      }
    if (LANES > 1) {
#pragma unroll
      for (int i = 0; i < V; i += 4) *reinterpret_cast<f32x4*>(&sums[lane][piece][i]) = f32x4{z[i], z[i + 1], z[i + 2], z[i + 3]};
      __syncthreads();
      if (lane == 0)
        for (int s = 1; s < LANES; ++s)
#pragma unroll
          for (int k = 0; k < V; ++k) z[k] += sums[s][piece][k];
      __syncthreads();
    }
    if (lane == 0 && t < total) la_finish<V>(e, m, n, N, z);
  }
}

// ---- few rows: a weight read once ----------------------------------------------------------------------------------------
// 16 columns of the result a workgroup, MB blocks of 16 rows of x; the waves take the contraction's steps in turn, fragments
// come straight from global memory (U steps of them under way), the waves' sums meet in LDS and are finished there.  One
// launch where the tile kernel would need a split and a join: 3.5 us against 7.2 at 1 x 4 096 x 1 024 (bf16, 8 MB of weight).
// Every workgroup reads all of x, so with more rows or a long contraction the tiles win: la_shape.  (64 columns a workgroup
// were slower but for 16 x 16 384 x 4 096, where the tiles are as fast.)
template <class IT, class OT, int MB>
__global__ __launch_bounds__(512) void k_linact_few(const LaTile<OT> g) {
  constexpr int WAVES = 8, E = LaBytes<IT>::E, V = Elem<OT>::VEC, PITCH = 20;
  constexpr int U = MB == 1 ? 4 : MB == 2 ? 2 : 1;                 // (registers: 8 U (1 + MB) of them hold pieces under way)
  __shared__ __align__(16) float sums[WAVES][MB * 16][PITCH];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, lg = lane >> 4;
  const int64_t n0 = (int64_t)blockIdx.x * 16, bytes = g.K * E;
  const char* wrow = g.b + (n0 + lr < g.N ? n0 + lr : g.N - 1) * g.ldb;
  const char* xrow[MB];
  f32x4 acc[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) {
    xrow[b] = g.a + (16 * b + lr < g.M ? 16 * b + lr : g.M - 1) * g.lda;
    acc[b] = 0.f;
  }
  // rows may start anywhere and end inside a piece: what lies behind the end counts as zero.  Loads off a word's start are split
  // by the hardware (64 x 2 101 -> 128 bf16: 29 us): such rows are read by the words that hold them, and shifted (18 us)
  const bool off_word = E < 4 && (((uintptr_t)g.a | (uintptr_t)g.b | (uint64_t)g.lda | (uint64_t)g.ldb) & 3) != 0;
  auto piece = [&](const char* row, int64_t c) {
    typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(4)));
    u32x4 v = 0;
    const int64_t at = c * 16;
    if (at + 16 <= bytes) {
      if (!off_word) {
        v = *reinterpret_cast<const u32x4u*>(row + at);
      } else {
        const unsigned shift = (unsigned)((uintptr_t)(row + at) & 3);
        const uint32_t* word = reinterpret_cast<const uint32_t*>(row + at - shift);
        const u32x4 t = *reinterpret_cast<const u32x4u*>(word);
        const uint32_t next = word[shift ? 4 : 3];       // (at a word's start there is no fifth)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_alignbyte(i < 3 ? t[i + 1] : next, t[i], shift);
      }
    } else if (at < bytes) {
#pragma unroll
      for (int i = 0; i < 16; i += E)
        if (at + i < bytes) {
          if (E == 4) v[i / 4] = *reinterpret_cast<const uint32_t*>(row + at + i);
          else if (E == 2) v[i / 4] |= (uint32_t)*reinterpret_cast<const uint16_t*>(row + at + i) << (8 * (i & 3));
          else v[i / 4] |= (uint32_t)*reinterpret_cast<const uint8_t*>(row + at + i) << (8 * (i & 3));
        }
    }
    return v;
  };
  for (int k0 = wave; k0 < g.ktiles; k0 += WAVES * U) {
    u32x4 w[U][2], x[U][MB][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t c = (int64_t)(k0 + u * WAVES) * 8 + 4 * h + lg;
        w[u][h] = piece(wrow, c);
#pragma unroll
        for (int b = 0; b < MB; ++b) x[u][b][h] = piece(xrow[b], c);
      }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      LaFrag<IT> fw, fx[MB];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        fw.set(h, w[u][h]);
#pragma unroll
        for (int b = 0; b < MB; ++b) fx[b].set(h, x[u][b][h]);
      }
#pragma unroll
      for (int p = 0; p < LaParts<IT>::N; ++p)
#pragma unroll
        for (int b = 0; b < MB; ++b) la_mma<IT>(p, acc[b], fw, fx[b]);
    }
  }
#pragma unroll
  for (int b = 0; b < MB; ++b) *reinterpret_cast<f32x4*>(&sums[wave][16 * b + lr][4 * lg]) = acc[b];
  __syncthreads();
  constexpr int PER_ROW = 16 / V;
  for (int t = threadIdx.x; t < MB * 16 * PER_ROW; t += 64 * WAVES) {
    const int m = t / PER_ROW, c = t % PER_ROW * V;
    if (m >= g.M || n0 + c >= g.N) continue;
    float z[V];
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
#pragma unroll
      for (int k = 0; k < V; k += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(&sums[w][m][c + k]);
#pragma unroll
        for (int q = 0; q < 4; ++q) z[k + q] += v[q];
      }
    la_finish<V>(g.e, m, n0 + c, g.N, z);
  }
}

// ---- backward: dz and its column sums; rows padded to whole pieces ---------------------------------------------------------
// v = in * slope over a block of `rows` rows: out [R, ld_out] with zeros from C on, partial [block][C] the block's column sums, or
// total [C] where there is one block.  out_lo: what out's rounding left, so that out + out_lo is v to the square of a half step
// A thread owns one 16-byte piece of columns and every (256 / cg)th row of the block; cg (a power of two) pieces go side by side
template <class T>
__global__ __launch_bounds__(256) void k_linact_dz(const T* __restrict__ in, int64_t ld_in, const void* __restrict__ save, int act,
                                                   T* __restrict__ out, T* __restrict__ out_lo, int64_t ld_out,
                                                   float* __restrict__ partial, T* __restrict__ total, int64_t R, int64_t C, int rows, int cg_log, unsigned across) {
  using E = Elem<T>;
  using FV = typename E::fvec;
  __shared__ FV sums[256];
  const int cg = 1 << cg_log, piece = threadIdx.x & (cg - 1), rl = threadIdx.x >> cg_log, rstep = 256 >> cg_log;
  const int64_t block = blockIdx.x / across, c = ((int64_t)(blockIdx.x % across) * cg + piece) * E::VEC;
  const int64_t r1 = (block + 1) * rows < R ? (block + 1) * rows : R;
  const int left = (int)(C - c < E::VEC ? (C > c ? C - c : 0) : E::VEC), room = (int)(ld_out - c < E::VEC ? (ld_out > c ? ld_out - c : 0) : E::VEC);
  FV s = 0.f;
  // WHOLE: a whole piece on either side, no test between the loads, so that those of several rows are under way together
  const auto block_rows = [&](auto whole) {
    constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll 2
    for (int64_t r = block * rows + rl; r < r1; r += rstep) {
      FV v = 0.f;
      if (WHOLE || left > 0) {
        v = WHOLE ? ffn_load(in + r * ld_in + c, 0, E::VEC) : ffn_load(in + r * ld_in + c, 0, left);
        if (act != HOTK_ACT_NONE) {
          if constexpr (std::is_same<T, float>::value) {
            la_times_slope(v, ffn_load((const float*)save + r * C + c, 0, WHOLE ? E::VEC : left), act);
          } else {
            typedef int16_t s16x8u __attribute__((ext_vector_type(8), aligned(2)));
            const int16_t* codes = (const int16_t*)save + r * C + c;
            if (WHOLE) {
              const s16x8u d = *reinterpret_cast<const s16x8u*>(codes);
#pragma unroll
              for (int k = 0; k < E::VEC; ++k) v[k] *= la_slope<T>(d[k], act);
            } else {
#pragma unroll
              for (int k = 0; k < E::VEC; ++k)
                if (k < left) v[k] *= la_slope<T>(codes[k], act);
            }
          }
        }
        s += v;
      }
      if (out && (WHOLE || room > 0)) {
        ffn_store(out + r * ld_out + c, 0, WHOLE ? E::VEC : room, v);
        if (out_lo) {
          const FV hi = __builtin_convertvector(__builtin_convertvector(v, typename E::vec), FV);
          FV lo;
#pragma unroll
          for (int k = 0; k < E::VEC; ++k) lo[k] = hi[k] - hi[k] == 0.f ? v[k] - hi[k] : 0.f;     // (an infinity leaves nothing)
          ffn_store(out_lo + r * ld_out + c, 0, WHOLE ? E::VEC : room, lo);
        }
      }
    }
  };
  if (left == E::VEC && (!out || room == E::VEC)) block_rows(std::true_type{});
  else if (left > 0 || (out && room > 0)) block_rows(std::false_type{});
  if (partial || total) {
    sums[threadIdx.x] = s;
    for (int half = rstep / 2; half >= 1; half /= 2) {
      __syncthreads();
      if (rl < half) sums[threadIdx.x] += sums[threadIdx.x + (half << cg_log)];
    }
    if (rl == 0) {
      s = sums[threadIdx.x];
#pragma unroll
      for (int k = 0; k < E::VEC; ++k)
        if (k < left) {
          if (total) total[c + k] = (T)s[k];
          else partial[block * C + c + k] = s[k];
        }
    }
  }
}

// a copy of rows of `bytes` bytes with zeros behind them up to ld_out, 16 bytes a thread
__global__ __launch_bounds__(256) void k_pad_rows(const uint8_t* __restrict__ in, int64_t ld_in, uint8_t* __restrict__ out, int64_t ld_out,
                                                  int64_t R, int64_t bytes) {
  typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(1)));
  const int64_t per_row = ld_out / 16, total = R * per_row;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t r = t / per_row, c = t % per_row * 16;
    const uint8_t* src = in + r * ld_in + c;
    u32x4 v = 0;
    if (c + 16 <= bytes) {
      v = *reinterpret_cast<const u32x4u*>(src);
    } else {
      for (int i = 0; i < 16; ++i)
        if (c + i < bytes) v[i / 4] |= (uint32_t)src[i] << (8 * (i % 4));
    }
    *reinterpret_cast<u32x4*>(out + r * ld_out + c) = v;
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------
int64_t la_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Which kernel, tile and split a product takes: the least of their times by a model of what was measured (us, bf16: 128-byte
// steps; sweeps of all tiles and splits over M, N of 1 .. 16 384 and K of 256 .. 16 384).  A workgroup's step takes `lat` alone, and
// `sat` for each of those that share a compute unit where that is more; `end` is its start and end.  The matrix work of a step
// is 8 times a 16-bit type's in fp32, twice with 8-bit operands and an fp32 result.
struct LaShape { int bm, bn, splits; };      // bn 16: k_linact_few, bm / 16 blocks of rows
struct LaCost { int bm, bn; float sat, lat, end; };
const LaCost LA_COSTS[] = {{256, 256, 1.58f, 1.58f, 6.f}, {128, 128, 0.42f, 0.69f, 3.f}, {64, 128, 0.26f, 0.39f, 1.2f}, {64, 64, 0.16f, 0.32f, 0.7f}};
LaShape la_shape(int64_t M, int64_t N, int64_t K, int type, int out_type, int flags, bool whole, bool off_word, int parts) {
  const int64_t ktiles = la_div(K * ffn_bytes(type), 128) * parts;
  const bool wide = type == HOTK_E4M3 && out_type == HOTK_F32;
  const float mfma = type == HOTK_F32 ? 8.f : wide ? 2.f : 1.f;
  LaShape best{64, 64, 1};
  float least = 1e30f;
  if (M <= 64 && flags == 0 && parts == 1) {     // k_linact_few: 8.6 TB/s in all, 50 GB/s a compute unit, its matrix work beside that
    const int mb = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const float wgs = (float)la_div(N, 16), bytes = ktiles * 128.f * 16 * (1 + mb);
    // (rows in no whole pieces: the tiles would need two copies first; off a word's start the loads take 1.7 times as long)
    least = -(whole ? 0.f : 8.f) + std::max((off_word ? 1.7f : 1.f) * std::max(wgs * bytes / 8.6e6f, std::ceil(wgs / 256.f) * bytes / 50e3f),
                     std::ceil(wgs / 256.f) * ktiles * 0.89f * mfma * mb / 256.f);
    best = {16 * mb, 16, 1};
  }
  for (const LaCost& c : LA_COSTS) {
    // (256 x 256 spills registers with bf16 copies of 8-bit operands; with both operands transposed a step takes 3.7)
    if (c.bm == 256 && wide) continue;
    const float flop = 0.89f * mfma * (c.bm * c.bn) / 65536.f;              // a step's matrix work at the clock's rate
    const float sat = std::max(c.bm == 256 && flags == (HOTK_LINEAR_X_DOWN | HOTK_LINEAR_W_DOWN) ? 3.7f : c.sat, 1.12f * flop);
    const float lat = mfma > 1.f ? c.lat + 0.9f * flop : c.lat;
    const double tiles = (double)la_div(M, c.bm) * la_div(N, c.bn);
    for (int64_t s = 1; s <= LA_MAX_SPLIT && s <= ktiles; s *= 2) {
      const int64_t kper = la_div(ktiles, s), splits = la_div(ktiles, kper);
      const float q = (float)std::ceil(tiles * splits / 256.);
      float t = q * c.end + kper * std::max(lat, sat * q);
      if (splits > 1) t += 6.f + splits * (float)M * N * 4.f / 3e6f;       // the join: a launch on either side, and the parts written and read
      if (t < least) {
        least = t;
        best = {c.bm, c.bn, (int)splits};
      }
    }
  }
  return best;
}

LaShape la_shape(const hotk_linear_args& a);

template <class IT, class OT, int MB>
int la_run_few(const LaTile<OT>& g, hipStream_t st) {
  if (la_div(g.N, 16) >= LA_MAX_GRID) return HOTK_ETOOLARGE;
  hipLaunchKernelGGL((k_linact_few<IT, OT, MB>), dim3((unsigned)la_div(g.N, 16)), dim3(512), 0, st, g);
  return hotk_launch_status();
}

template <class IT, class OT, bool TA, bool TB, int BM, int BN, int WM, int WN>
int la_run(LaTile<OT>& g, int splits, hipStream_t st) {
  // two stages, or the waves' pieces of the result where those are larger
  constexpr int BOX = WM * WN * (BM / WM < 64 ? BM / WM : 64) * 68 * 4, STAGES = 2 * (BM + BN) * 128, LDS = BOX > STAGES ? BOX : STAGES;
  auto kernel = k_linact_tile<IT, OT, TA, TB, BM, BN, WM, WN>;
  if (LDS > 64 * 1024) {                 // more LDS than a kernel gets without asking: asked for once per device
    static std::atomic<uint64_t> asked{0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return HOTK_ELAUNCH;
    const uint64_t bit = 1ull << (dev & 63);
    if (!(asked.load(std::memory_order_relaxed) & bit)) {
      if (hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, LDS) != hipSuccess) return HOTK_ELAUNCH;
      asked.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  if (la_div(g.M, BM) * la_div(g.N, BN) >= LA_MAX_GRID) return HOTK_ETOOLARGE;
  g.tiles_m = (int)la_div(g.M, BM);
  g.tiles_n = (int)la_div(g.N, BN);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n), (unsigned)splits), dim3(64 * WM * WN), LDS, st, g);
  return hotk_launch_status();
}

template <class IT, class OT, bool TA, bool TB>
int la_product(const hotk_linear_args& a, void* ws, size_t nws, hipStream_t st) {
  const int e = ffn_bytes(a.type);
  const int64_t steps = la_div(a.K * e, 128), ktiles = a.x_lo ? 2 * steps : steps;
  const LaShape s = la_shape(a);
  const size_t need = s.splits > 1 ? (size_t)s.splits * a.M * a.N * 4 : 0;
  if (nws < need || (need && !ws)) return HOTK_EWORKSPACE;
  LaTile<OT> g{};
  g.a = (const char*)a.x; g.b = (const char*)a.w;
  g.lda = a.ld_x * e; g.ldb = a.ld_w * e;
  g.M = a.M; g.N = a.N; g.K = a.K;
  g.wrap = (int)steps;
  g.low = a.x_lo ? (const char*)a.x_lo - (const char*)a.x : 0;
  g.ktiles = (int)ktiles; g.kper = (int)la_div(ktiles, s.splits);
  g.part = need ? (float*)ws : nullptr;
  g.e = {(const OT*)a.bias, (const OT*)a.res, a.ld_res, (OT*)a.y, a.ld_y, a.save, a.x_scale, a.w_scale, a.act};
  if constexpr (!TA && !TB)
    if (s.bn == 16) return s.bm == 16 ? la_run_few<IT, OT, 1>(g, st) : s.bm == 32 ? la_run_few<IT, OT, 2>(g, st) : la_run_few<IT, OT, 4>(g, st);
  int rc = s.bm == 256 ? la_run<IT, OT, TA, TB, 256, 256, 2, 4>(g, s.splits, st)
         : s.bm == 128 ? la_run<IT, OT, TA, TB, 128, 128, 2, 2>(g, s.splits, st)
         : s.bn == 128 ? la_run<IT, OT, TA, TB, 64, 128, 2, 2>(g, s.splits, st)
                       : la_run<IT, OT, TA, TB, 64, 64, 4, 1>(g, s.splits, st);
  if (rc == HOTK_OK && need) {
    const int64_t work = a.M * la_div(a.N, Elem<OT>::VEC);
    if (s.splits <= 4)
      hipLaunchKernelGGL((k_linact_join<OT, 1>), dim3(hotk_grid(work, 256)), dim3(256), 0, st, (const float*)ws, s.splits, a.M, a.N, g.e);
    else
      hipLaunchKernelGGL((k_linact_join<OT, 8>), dim3(hotk_grid(work, 32, 256 * 32)), dim3(256), 0, st, (const float*)ws, s.splits, a.M, a.N, g.e);
    rc = hotk_launch_status();
  }
  return rc;
}

// rows of x and w in whole, aligned 16-byte pieces, with zeros behind the contraction's end
bool la_whole(const hotk_linear_args& a) {
  const int e = ffn_bytes(a.type), m = 16 / e;
  const int64_t row_x = a.flags & HOTK_LINEAR_X_DOWN ? a.M : a.K, row_w = a.flags & HOTK_LINEAR_W_DOWN ? a.N : a.K;
  if (a.K % m && !(a.flags & (HOTK_LINEAR_PADDED | HOTK_LINEAR_X_DOWN))) return false;
  return a.ld_x >= la_div(row_x, m) * m && a.ld_w >= la_div(row_w, m) * m && (a.ld_x * e) % 16 == 0 && (a.ld_w * e) % 16 == 0 &&
         hotk_aligned16(a.x) && hotk_aligned16(a.w);
}
LaShape la_shape(const hotk_linear_args& a) {
  const int64_t e = ffn_bytes(a.type);
  const bool off_word = (((uintptr_t)a.x | (uintptr_t)a.w | (uint64_t)(a.ld_x * e) | (uint64_t)(a.ld_w * e)) & 3) != 0;
  return la_shape(a.M, a.N, a.K, a.type, a.out_type, a.flags & (HOTK_LINEAR_X_DOWN | HOTK_LINEAR_W_DOWN), la_whole(a), off_word, a.x_lo ? 2 : 1);
}

int la_check(const hotk_linear_args& a) {
  HOTK_CHECK_ARG(a.M >= 0 && a.N > 0 && a.K > 0);
  if (!(ffn_type_ok(a.type) || a.type == HOTK_E4M3) || !ffn_type_ok(a.out_type)) return HOTK_EUNSUPPORTED;
  if (a.type != HOTK_E4M3 && a.out_type != a.type) return HOTK_EUNSUPPORTED;
  HOTK_CHECK_ARG((a.flags & ~(HOTK_LINEAR_X_DOWN | HOTK_LINEAR_W_DOWN | HOTK_LINEAR_PADDED)) == 0);
  const int down = a.flags & (HOTK_LINEAR_X_DOWN | HOTK_LINEAR_W_DOWN);
  if (down == HOTK_LINEAR_X_DOWN || (down && a.type == HOTK_E4M3)) return HOTK_EUNSUPPORTED;
  HOTK_CHECK_ARG(a.act >= HOTK_ACT_NONE && a.act <= HOTK_ACT_SILU);
  HOTK_CHECK_ARG((a.type == HOTK_E4M3) == (a.x_scale != nullptr) && (a.x_scale != nullptr) == (a.w_scale != nullptr));
  HOTK_CHECK_ARG(a.type != HOTK_E4M3 || !a.save);
  const int e = ffn_bytes(a.type);
  const int64_t row_x = a.flags & HOTK_LINEAR_X_DOWN ? a.M : a.K, row_w = a.flags & HOTK_LINEAR_W_DOWN ? a.N : a.K;
  HOTK_CHECK_ARG(a.ld_x >= row_x && a.ld_w >= row_w && a.ld_y >= a.N && (!a.res || a.ld_res >= a.N));
  if (a.M > 0) {
    HOTK_CHECK_ARG(a.x && a.w && a.y);
    HOTK_CHECK_ARG(ffn_elem_aligned(a.x, a.type) && ffn_elem_aligned(a.w, a.type));
    // the tiles read rows in whole, aligned 16-byte pieces (the caller pads others: hotk_pad_rows)
    if (!la_whole(a) && la_shape(a).bn != 16) return HOTK_EUNSUPPORTED;
    if (a.x_lo && (!hotk_aligned16(a.x_lo) || a.type == HOTK_E4M3)) return HOTK_EUNSUPPORTED;
    HOTK_CHECK_ARG(ffn_elem_aligned(a.y, a.out_type) && ffn_elem_aligned(a.bias, a.out_type) && ffn_elem_aligned(a.res, a.out_type));
    HOTK_CHECK_ARG(((uintptr_t)a.save) % (a.out_type == HOTK_F32 ? 4 : 2) == 0);
    HOTK_CHECK_ARG(((uintptr_t)a.x_scale) % 4 == 0 && ((uintptr_t)a.w_scale) % 4 == 0);
  }
  // 32-bit offsets inside a tile, 32-bit tile and step counts
  if (a.ld_x * e > (1 << 23) || a.ld_w * e > (1 << 23) || la_div(a.M, 64) * la_div(a.N, 64) > (1ll << 30) || la_div(a.K * e, 128) > (1ll << 30))
    return HOTK_ETOOLARGE;
  return HOTK_OK;
}

// rows of a block of hotk_linear_dz: all of up to 1024 (one block: its sums are the result, and a launch is saved), else 16, and
// more where that would be over 512 blocks
int64_t la_dz_rows(int64_t R) { return R <= 1024 ? 1024 : la_div(la_div(R, 512), 16) * 16; }

}  // namespace

extern "C" int hotk_linear_workspace_bytes(const hotk_linear_args* args, size_t* bytes) {
  HOTK_CHECK_ARG(args && bytes);
  if (const int rc = la_check(*args)) return rc;
  const LaShape s = la_shape(*args);
  *bytes = s.splits > 1 ? (size_t)s.splits * args->M * args->N * 4 : 0;
  return HOTK_OK;
}

extern "C" int hotk_linear_act(const hotk_linear_args* args, void* workspace, size_t ws_bytes, void* stream) {
  HOTK_CHECK_ARG(args);
  if (const int rc = la_check(*args)) return rc;
  if (args->M == 0) return HOTK_OK;
  hipStream_t st = (hipStream_t)stream;
  int rc = HOTK_EUNSUPPORTED;
  ffn_dispatch(args->out_type, [&](auto* tag) {
    using OT = std::remove_pointer_t<decltype(tag)>;
    using T8 = std::conditional_t<std::is_same<OT, float>::value, e4m3_wide, e4m3>;
    rc = args->type == HOTK_E4M3 ? la_product<T8, OT, false, false>(*args, workspace, ws_bytes, st)
       : !(args->flags & HOTK_LINEAR_W_DOWN) ? la_product<OT, OT, false, false>(*args, workspace, ws_bytes, st)
       : !(args->flags & HOTK_LINEAR_X_DOWN) ? la_product<OT, OT, false, true>(*args, workspace, ws_bytes, st)
                                           : la_product<OT, OT, true, true>(*args, workspace, ws_bytes, st);
  });
  return rc;
}

extern "C" int hotk_linear_dz_partials(int64_t R, int64_t* n_partials) {
  HOTK_CHECK_ARG(n_partials && R >= 0);
  *n_partials = R ? la_div(R, la_dz_rows(R)) : 0;
  return HOTK_OK;
}

extern "C" int hotk_linear_dz(const void* in, int64_t ld_in, const void* save, int act, void* out, void* out_lo, int64_t ld_out,
                              float* partial, void* total, int64_t R, int64_t C, int type, void* stream) {
  HOTK_CHECK_ARG(R >= 0 && C > 0 && ld_in >= C && (!out || ld_out >= C) && (out || partial || total));
  HOTK_CHECK_ARG(!out_lo || out);
  HOTK_CHECK_ARG(!total || (!partial && R <= la_dz_rows(R)));
  HOTK_CHECK_ARG(act >= HOTK_ACT_NONE && act <= HOTK_ACT_SILU && (act == HOTK_ACT_NONE || save || R == 0));
  if (!ffn_type_ok(type)) return HOTK_EUNSUPPORTED;
  HOTK_CHECK_ARG(ffn_elem_aligned(in, type) && ffn_elem_aligned(out, type) && ffn_elem_aligned(out_lo, type) && ffn_elem_aligned(total, type) && ((uintptr_t)save) % (type == HOTK_F32 ? 4 : 2) == 0 &&
                 ((uintptr_t)partial) % 4 == 0);
  if (R == 0) return HOTK_OK;
  HOTK_CHECK_ARG(in);
  const int64_t pieces = la_div(out ? ld_out : C, 16 / ffn_bytes(type)), rows = la_dz_rows(R), down = la_div(R, rows);
  // 32 pieces side by side (16 384 x 4 096 bf16 76 us; 4 of them 153), 16 where a block has many rows (700 000 x 256: 223 and 292); one
  // block of up to 1 024 rows has few workgroups and goes by its rows' time: 2 pieces (1 000 x 4 096: 15 us, 4 of them 19, 32 of them
  // 76), 4 of up to 64 rows (64 x 4 096: 3.7 and 7.4 with 32)
  const int most = down == 1 ? (R > 64 ? 1 : 2) : rows >= 1024 ? 4 : 5;
  int cg_log = 0;
  while (cg_log < most && (1 << cg_log) < pieces) ++cg_log;
  const int64_t across = la_div(pieces, 1 << cg_log);
  if (across * down >= 2 * LA_MAX_GRID || rows > (1 << 30)) return HOTK_ETOOLARGE;
  ffn_dispatch(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(k_linact_dz<T>, dim3((unsigned)(across * down)), dim3(256), 0, (hipStream_t)stream, (const T*)in, ld_in, save, act,
                       (T*)out, (T*)out_lo, ld_out, partial, (T*)total, R, C, (int)rows, cg_log, (unsigned)across);
  });
  return hotk_launch_status();
}

extern "C" int hotk_pad_rows(const void* in, int64_t ld_in, void* out, int64_t ld_out, int64_t R, int64_t bytes, void* stream) {
  HOTK_CHECK_ARG(R >= 0 && bytes > 0 && ld_in >= bytes && ld_out >= bytes && ld_out % 16 == 0);
  if (R == 0) return HOTK_OK;
  HOTK_CHECK_ARG(in && out && hotk_aligned16(out));
  hipLaunchKernelGGL(k_pad_rows, dim3(hotk_grid(R * (ld_out / 16), 256)), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)in, ld_in,
                     (uint8_t*)out, ld_out, R, bytes);
  return hotk_launch_status();
}
