// Matrix product with bias, activation and residual in its epilogue, and what its backward pass needs beside products.
//
//   z = x w^T + b (8-bit operands: z = sx_m sw_n (xq wq^T) + b)     y = f(z) + res        x [M, K], w [N, K], y [M, N]
//   backward: dz = dy f'(z),  dx = dz w,  dw = dz^T x,  db = sum_m dz,  dres = dy
//
// One tile kernel for every type.  All operands have the contraction along their rows (dx and dw take transposed copies), a
// tile row is 128 bytes of it = 64 16-bit, 32 fp32 or 128 8-bit elements, so loads, LDS image and fragment addresses are the
// same bytes for all types and only the matrix instruction differs:
//   16-bit: 2 x v_mfma_f32_16x16x32,   fp32: 8 x v_mfma_f32_16x16x4_f32,   e4m3: 1 x v_mfma_f32_16x16x128_f8f6f4
// (a contraction may take its terms in any order, so each type reads 16-byte pieces lane group by lane group).
// The e4m3 instruction adds eight products at a time aligned to the largest of them and drops what is below 2^-13 of it
// (measured with powers of two; between the eights, and onto the accumulator, it adds in fp32): at most 2^-10 of the largest
// product, and 1e-5 of a whole result at K = 16 .. 4096, next to 2^-9 / 2^-12 that a 16-bit result is rounded by.  An fp32
// result would show it, so there the operands become bf16 (exactly: 4 significant bits) and 4 x v_mfma_f32_16x16x32_bf16 add
// them in fp32.
//
// Tiles go global -> LDS by DMA, two stages, one barrier per step.  The DMA writes 64 consecutive 16-byte pieces, so the
// swizzle that keeps fragment reads off each other's banks is applied to the SOURCE address: piece p of row r holds chunk
// p ^ key(r).  The weight is the matrix instruction's row operand, its rows dealt to fragments so that a lane ends with 16
// CONSECUTIVE output columns: bias, residual, y and the saved slope move in 16-byte accesses without a pass through LDS.
//
// For training, 16-bit types keep f'(z) as a 16-bit fixed-point number in steps of 2^-14 (|f'| < 1.13): its error of 2^-15
// is far below the rounding of dz, where z rounded to the type would add as much as that rounding again, and the backward
// pass needs no transcendental.  fp32 keeps z.
#include <atomic>
#include <type_traits>

#include "ffn.h"

namespace {

struct e4m3 {};                                    // operand tags: OCP e4m3, one byte, for 16-bit results
struct e4m3_wide {};                               // and for fp32 results

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr float LA_SLOPE_STEP = 0x1p-14f;
constexpr int LA_SLOPE_NAN = -32768;
constexpr float LA_LEAK = 0.01f;
constexpr int LA_MAX_SPLIT = 16;

__device__ __align__(16) const uint32_t la_zeros[4] = {0, 0, 0, 0};   // what lies past the end of a contraction

// ---- activations: f(z) and f'(z) ---------------------------------------------------------------------------------------
// FAST (16-bit results): gelu by Abramowitz & Stegun 7.1.26 (|error of erf| <= 1.5e-7), whose exponential the slope shares;
// tanh and the logistic function from one exponential.  fp32 results: the math library's functions.
template <bool FAST>
__device__ __forceinline__ float la_act(float z, int act, float& slope) {
  switch (act) {
    case HOTK_ACT_RELU: slope = z > 0.f ? 1.f : 0.f; return z < 0.f ? 0.f : z;       // (a NaN stays one)
    case HOTK_ACT_LEAKYRELU: slope = z > 0.f ? 1.f : LA_LEAK; return z > 0.f ? z : LA_LEAK * z;
    case HOTK_ACT_GELU: {
      float cdf, pdf;
      if (FAST) {
        const float x = fabsf(z) * 0.70710678f;
        const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f, x, 1.f));
        const float e = __builtin_amdgcn_exp2f(-1.44269504f * x * x);
        const float q = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, 1.061405429f, -1.453152027f), 1.421413741f), -0.284496736f), 0.254829592f) * e;
        cdf = z < 0.f ? 0.5f * q : fmaf(-0.5f, q, 1.f);
        pdf = 0.39894228f * e;
      } else {
        cdf = 0.5f * erfcf(-0.70710678f * z);
        pdf = 0.39894228f * expf(-0.5f * z * z);
      }
      slope = fmaf(z, pdf, cdf);
      return z * cdf;
    }
    case HOTK_ACT_TANH: {
      float t;
      if (FAST) {
        const float s = z * z;
        const float series = z * fmaf(s, fmaf(s, fmaf(s, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);   // to z^7: |z| < 1/4
        const float e = __builtin_amdgcn_exp2f(2.88539008f * z);
        const float quot = fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
        t = fabsf(z) < 0.25f ? series : quot;
      } else {
        t = tanhf(z);
      }
      slope = fmaf(-t, t, 1.f);
      return t;
    }
    case HOTK_ACT_SILU: {
      const float e = FAST ? __builtin_amdgcn_exp2f(-1.44269504f * z) : expf(-z);
      const float s = FAST ? __builtin_amdgcn_rcpf(1.f + e) : 1.f / (1.f + e);
      slope = s * fmaf(z, 1.f - s, 1.f);
      return z * s;
    }
    default: slope = 1.f; return z;
  }
}
__device__ __forceinline__ int16_t la_slope_code(float d) {
  const int c = (int)rintf(d * (1.f / LA_SLOPE_STEP));
  return (int16_t)(d != d ? LA_SLOPE_NAN : c);
}
__device__ __forceinline__ float la_slope(int16_t code, int act) {
  if (act == HOTK_ACT_LEAKYRELU) return code > 8192 ? 1.f : LA_LEAK;
  return code == LA_SLOPE_NAN ? __builtin_nanf("") : (float)code * LA_SLOPE_STEP;
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

// W consecutive columns (a multiple of 8) of one row, from n0: z is the bare product
template <int W, class OT>
__device__ __forceinline__ void la_finish(const LaEpi<OT>& e, int64_t m, int64_t n0, int64_t N, float (&z)[W]) {
  using E = Elem<OT>;
  constexpr bool FAST = !std::is_same<OT, float>::value;
  const int left = (int)(N - n0 < W ? N - n0 : W);               // columns of this piece that exist
  if (left <= 0) return;
  if (e.xs) {
    const float xs = e.xs[m];
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const f32x4 s = ffn_load(e.ws + n0, i, left);
#pragma unroll
      for (int k = 0; k < 4; ++k) z[i + k] = z[i + k] * xs * s[k];
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
  if (e.act != HOTK_ACT_NONE) {
    if (e.save) {
      if (FAST) {
        int16_t* row = (int16_t*)e.save + m * N + n0;
        typedef int16_t s16x8 __attribute__((ext_vector_type(8)));
        typedef int16_t s16x8u __attribute__((ext_vector_type(8), aligned(2)));
#pragma unroll
        for (int i = 0; i < W; i += 8) {
          s16x8 c;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            float d;
            z[i + k] = la_act<FAST>(z[i + k], e.act, d);
            c[k] = la_slope_code(d);
          }
          if (i + 8 <= left) {
            *reinterpret_cast<s16x8u*>(row + i) = c;
          } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (i + k < left) row[i + k] = c[k];
          }
        }
      } else {
        float* row = (float*)e.save + m * N + n0;
#pragma unroll
        for (int i = 0; i < W; i += 4) {
          f32x4 c;
#pragma unroll
          for (int k = 0; k < 4; ++k) c[k] = z[i + k];
          if (i < left) ffn_store(row, i, left, c);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float d;
            z[i + k] = la_act<FAST>(z[i + k], e.act, d);
          }
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) {
        float d;
        z[i] = la_act<FAST>(z[i], e.act, d);
      }
    }
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
  const char *a, *b;             // x [M, K], w [N, K]
  int64_t lda, ldb;              // bytes per row
  int64_t M, N;
  int chunks;                    // 16-byte pieces of a row
  int ktiles, kper;              // 128-byte steps, and how many of them a split takes
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

// chunk p ^ key of a row sits at piece p.  x fragments read 16 consecutive rows, w fragments rows {0..3} + 16 {0..3}
__device__ __forceinline__ int la_key_x(int row) { return row & 7; }
__device__ __forceinline__ int la_key_w(int row) { return (row & 3) | ((row >> 2) & 4); }

__device__ __forceinline__ u32x4 la_frag(const unsigned char* tile, int row, int chunk, int key) {
  return *reinterpret_cast<const u32x4*>(tile + row * 128 + ((chunk ^ key) << 4));
}

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

template <class IT>
__device__ __forceinline__ void la_mma(f32x4& c, const LaFrag<IT>& w, const LaFrag<IT>& x) {
  if constexpr (std::is_same<IT, __bf16>::value) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w.h[h]), __builtin_bit_cast(bf16x8, x.h[h]), c, 0, 0, 0);
  } else if constexpr (std::is_same<IT, _Float16>::value) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      c = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, w.h[h]), __builtin_bit_cast(f16x8, x.h[h]), c, 0, 0, 0);
  } else if constexpr (std::is_same<IT, float>::value) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w.h[h][k]), __uint_as_float(x.h[h][k]), c, 0, 0, 0);
  } else if constexpr (std::is_same<IT, e4m3_wide>::value) {
#pragma unroll
    for (int h = 0; h < 4; ++h) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.b[h], x.b[h], c, 0, 0, 0);
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

template <class IT, class OT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void k_linact_tile(const LaTile<OT> g) {
  constexpr int NW = WM * WN, TM = BM / WM, MF = TM / 16, NF = 4, STAGE = (BM + BN) * 128;
  constexpr int PIECES = (BM + BN) / 8, LOADS = PIECES / NW;     // a wave's DMA instructions per step: 8 rows each
  static_assert(BN / WN == 64 && PIECES % NW == 0 && BM % (16 * WM) == 0, "a wave owns 64 columns");
  extern __shared__ __align__(16) unsigned char lds[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / WN, wn = wave % WN, lr = lane & 15, lg = lane >> 4;
  int im, in;
  la_tile_of(blockIdx.x, g.tiles_m, g.tiles_n, im, in);
  const int64_t m0 = (int64_t)im * BM, n0 = (int64_t)in * BN;
  const int k0 = blockIdx.y * g.kper, k1 = min(g.ktiles, k0 + g.kper);
  const char* abase = g.a + m0 * g.lda;
  const char* bbase = g.b + n0 * g.ldb;

  // this lane's source offsets: piece group i of the wave = rows 8 (wave + NW i) .. + 8 of [x tile | w tile]; rows past the
  // end repeat the last one (their products are not stored)
  uint32_t off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int p = wave + NW * i;
    const bool is_x = p < BM / 8;
    const int row = (is_x ? p : p - BM / 8) * 8 + (lane >> 3);
    const int chunk = (lane & 7) ^ (is_x ? la_key_x(row) : la_key_w(row));
    const int64_t last = (is_x ? g.M - m0 : g.N - n0) - 1;
    off[i] = (uint32_t)((row < last ? row : last) * (is_x ? g.lda : g.ldb)) + chunk * 16;
  }
  auto issue = [&](int kt, int stage) {
    const bool whole = kt * 8 + 8 <= g.chunks;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int p = wave + NW * i;
      const bool is_x = p < BM / 8;
      const char* base = (is_x ? abase : bbase) + (int64_t)kt * 128;
      const uint32_t dst = lds0 + stage * STAGE + p * 1024;
      if (whole) {
        la_dma(base, off[i], dst);
      } else {
        const int row = (is_x ? p : p - BM / 8) * 8 + (lane >> 3);
        const int chunk = (lane & 7) ^ (is_x ? la_key_x(row) : la_key_w(row));
        la_dma_at(kt * 8 + chunk < g.chunks ? base + off[i] : (const char*)la_zeros, dst);
      }
    }
  };

  f32x4 acc[MF][NF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) acc[i][j] = 0.f;

  if (k0 < k1) issue(k0, 0);
  for (int kt = k0; kt < k1; ++kt) {
    const int stage = (kt - k0) & 1;
    la_wait_vm<0>();       // this wave's part of the step has landed,
    la_barrier();          // everyone's has, and everyone has read the other stage
    if (kt + 1 < k1) issue(kt + 1, stage ^ 1);
    const unsigned char* xt = lds + stage * STAGE;
    const unsigned char* wt = xt + BM * 128;
    LaFrag<IT> wf[NF];
#pragma unroll
    for (int j = 0; j < NF; ++j) {
      const int row = wn * 64 + 16 * (lr >> 2) + 4 * j + (lr & 3);
#pragma unroll
      for (int h = 0; h < 2; ++h) wf[j].set(h, la_frag(wt, row, 4 * h + lg, la_key_w(row)));
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int row = wm * TM + 16 * i + lr;
      LaFrag<IT> xf;
#pragma unroll
      for (int h = 0; h < 2; ++h) xf.set(h, la_frag(xt, row, 4 * h + lg, la_key_x(row)));
#pragma unroll
      for (int j = 0; j < NF; ++j) la_mma<IT>(acc[i][j], wf[j], xf);
    }
  }

  const int64_t n = n0 + wn * 64 + 16 * lg;
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int64_t m = m0 + wm * TM + 16 * i + lr;
    float z[16];
#pragma unroll
    for (int j = 0; j < NF; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) z[4 * j + k] = acc[i][j][k];
    if (m >= g.M) continue;
    if (g.part) {
      float* row = g.part + ((int64_t)blockIdx.y * g.M + m) * g.N + n;
      const int left = (int)(g.N - n < 16 ? g.N - n : 16);
#pragma unroll
      for (int j = 0; j < 16; j += 4) {
        const f32x4 v = {z[j], z[j + 1], z[j + 2], z[j + 3]};
        if (j < left) ffn_store(row, j, left, v);
      }
    } else {
      la_finish<16>(g.e, m, n, g.N, z);
    }
  }
}

// joins the splits in order and finishes: eight columns a thread
template <class OT>
__global__ __launch_bounds__(256) void k_linact_join(const float* __restrict__ part, int splits, int64_t M, int64_t N,
                                                     const LaEpi<OT> e) {
  const int64_t per_row = (N + 7) / 8, total = M * per_row;
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < total; t += (int64_t)gridDim.x * 256) {
    const int64_t m = t / per_row, n = t % per_row * 8;
    const int left = (int)(N - n < 8 ? N - n : 8);
    float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < splits; ++s) {
      const float* row = part + ((int64_t)s * M + m) * N + n;
#pragma unroll
      for (int i = 0; i < 8; i += 4) {
        const f32x4 v = ffn_load(row, i, left);
#pragma unroll
        for (int k = 0; k < 4; ++k) z[i + k] += v[k];
      }
    }
    la_finish<8>(e, m, n, N, z);
  }
}

// ---- backward: dz and its transpose, transposed and padded copies --------------------------------------------------------
// 64 x 64 tiles through LDS.  in [R, C] -> (MODE >= 1: times the saved slope) -> out [R, ld_out] and / or out_t [C, ld_t], both
// with zeros up to their row length, and column sums of each tile, partial [tile row][C]
template <class T, bool DZ>
__global__ __launch_bounds__(256) void k_linact_turn(const T* __restrict__ in, int64_t ld_in, const void* __restrict__ save, int act,
                                                     T* __restrict__ out, int64_t ld_out, T* __restrict__ out_t, int64_t ld_t,
                                                     float* __restrict__ partial, int64_t R, int64_t C, unsigned across) {
  __shared__ T tile[64][65];
  __shared__ float sums[4][64];
  const int64_t down = blockIdx.x / across, r0 = down * 64, c0 = (int64_t)(blockIdx.x % across) * 64;
  const int cx = threadIdx.x & 63, ry = threadIdx.x >> 6;
  float s = 0.f;
  for (int i = ry; i < 64; i += 4) {
    const int64_t r = r0 + i, c = c0 + cx;
    float v = 0.f;
    if (r < R && c < C) {
      v = (float)in[r * ld_in + c];
      if (DZ && act != HOTK_ACT_NONE) {
        if (std::is_same<T, float>::value) {
          float d;
          la_act<false>(((const float*)save)[r * C + c], act, d);
          v *= d;
        } else {
          v *= la_slope(((const int16_t*)save)[r * C + c], act);
        }
      }
    }
    const T t = (T)v;
    s += v;
    if (out && r < R && c < ld_out) out[r * ld_out + c] = t;
    tile[i][cx] = t;
  }
  if (partial) sums[ry][cx] = s;
  __syncthreads();
  if (partial && ry == 0 && r0 < R && c0 + cx < C) partial[down * C + c0 + cx] = (sums[0][cx] + sums[1][cx]) + (sums[2][cx] + sums[3][cx]);
  if (out_t)
    for (int i = ry; i < 64; i += 4) {
      const int64_t c = c0 + i, r = r0 + cx;
      if (c < C && r < ld_t) out_t[c * ld_t + r] = tile[cx][i];
    }
}

// ---- host --------------------------------------------------------------------------------------------------------------
int64_t la_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// tile and split of a product
struct LaShape { int bm, bn, splits; };
LaShape la_shape(int64_t M, int64_t N, int64_t ktiles) {
  LaShape s{256, 256, 1};
  if (la_div(M, 256) * la_div(N, 256) < 192) s = {128, 128, 1};
  if (M <= 64) s = {32, 128, 1};
  const int64_t tiles = la_div(M, s.bm) * la_div(N, s.bn);
  // fewer tiles than compute units: the contraction is split until there is one workgroup each, four steps or more a split
  if (tiles < 192) {
    int64_t want = 256 / (tiles < 1 ? 1 : tiles);
    if (want > ktiles / 4) want = ktiles / 4;
    if (want > LA_MAX_SPLIT) want = LA_MAX_SPLIT;
    if (want > 1) s.splits = (int)la_div(ktiles, la_div(ktiles, want));
  }
  return s;
}

template <class IT, class OT, int BM, int BN, int WM, int WN>
int la_run(LaTile<OT>& g, int splits, hipStream_t st) {
  constexpr int LDS = 2 * (BM + BN) * 128;
  auto kernel = k_linact_tile<IT, OT, BM, BN, WM, WN>;
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
  g.tiles_m = (int)la_div(g.M, BM);
  g.tiles_n = (int)la_div(g.N, BN);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(g.tiles_m * g.tiles_n), (unsigned)splits), dim3(64 * WM * WN), LDS, st, g);
  return hotk_launch_status();
}

template <class IT, class OT>
int la_product(const hotk_linear_args& a, void* ws, size_t nws, hipStream_t st) {
  const int e = ffn_bytes(a.type);
  const int64_t chunks = a.K * e / 16, ktiles = la_div(chunks, 8);
  const LaShape s = la_shape(a.M, a.N, ktiles);
  const size_t need = s.splits > 1 ? (size_t)s.splits * a.M * a.N * 4 : 0;
  if (nws < need || (need && !ws)) return HOTK_EWORKSPACE;
  LaTile<OT> g{};
  g.a = (const char*)a.x; g.b = (const char*)a.w;
  g.lda = a.ld_x * e; g.ldb = a.ld_w * e;
  g.M = a.M; g.N = a.N;
  g.chunks = (int)chunks; g.ktiles = (int)ktiles; g.kper = (int)la_div(ktiles, s.splits);
  g.part = need ? (float*)ws : nullptr;
  g.e = {(const OT*)a.bias, (const OT*)a.res, a.ld_res, (OT*)a.y, a.ld_y, a.save, a.x_scale, a.w_scale, a.act};
  int rc = s.bm == 256 ? la_run<IT, OT, 256, 256, 2, 4>(g, s.splits, st)
         : s.bm == 128 ? la_run<IT, OT, 128, 128, 2, 2>(g, s.splits, st)
                       : la_run<IT, OT, 32, 128, 2, 2>(g, s.splits, st);
  if (rc == HOTK_OK && need) {
    const int64_t work = a.M * la_div(a.N, 8);
    hipLaunchKernelGGL(k_linact_join<OT>, dim3(hotk_grid(work, 256)), dim3(256), 0, st, (const float*)ws, s.splits, a.M, a.N, g.e);
    rc = hotk_launch_status();
  }
  return rc;
}

int la_check(const hotk_linear_args& a) {
  HOTK_CHECK_ARG(a.M >= 0 && a.N > 0 && a.K > 0);
  if (!(ffn_type_ok(a.type) || a.type == HOTK_E4M3) || !ffn_type_ok(a.out_type)) return HOTK_EUNSUPPORTED;
  if (a.type != HOTK_E4M3 && a.out_type != a.type) return HOTK_EUNSUPPORTED;
  HOTK_CHECK_ARG(a.act >= HOTK_ACT_NONE && a.act <= HOTK_ACT_SILU);
  HOTK_CHECK_ARG((a.type == HOTK_E4M3) == (a.x_scale != nullptr) && (a.x_scale != nullptr) == (a.w_scale != nullptr));
  HOTK_CHECK_ARG(a.type != HOTK_E4M3 || !a.save);
  const int e = ffn_bytes(a.type);
  HOTK_CHECK_ARG(a.ld_x >= a.K && a.ld_w >= a.K && a.ld_y >= a.N && (!a.res || a.ld_res >= a.N));
  // contraction rows in whole, aligned 16-byte pieces (the caller pads others: hotk_linear_turn)
  if ((a.K * e) % 16 || (a.ld_x * e) % 16 || (a.ld_w * e) % 16) return HOTK_EUNSUPPORTED;
  if (a.M > 0) {
    HOTK_CHECK_ARG(a.x && a.w && a.y);
    if (!hotk_aligned16(a.x) || !hotk_aligned16(a.w)) return HOTK_EUNSUPPORTED;
    HOTK_CHECK_ARG(ffn_elem_aligned(a.y, a.out_type) && ffn_elem_aligned(a.bias, a.out_type) && ffn_elem_aligned(a.res, a.out_type));
    HOTK_CHECK_ARG(((uintptr_t)a.save) % 4 == 0 || a.out_type != HOTK_F32);
  }
  // 32-bit offsets inside a tile, 32-bit tile counts
  if (a.ld_x * e > (1 << 23) || a.ld_w * e > (1 << 23) || la_div(a.M, 32) * la_div(a.N, 128) > (1ll << 30)) return HOTK_ETOOLARGE;
  return HOTK_OK;
}

}  // namespace

extern "C" int hotk_linear_workspace_bytes(int64_t M, int64_t N, int64_t K, int type, size_t* bytes) {
  HOTK_CHECK_ARG(bytes && M >= 0 && N > 0 && K > 0);
  if (!(ffn_type_ok(type) || type == HOTK_E4M3)) return HOTK_EUNSUPPORTED;
  const LaShape s = la_shape(M, N, la_div(K * ffn_bytes(type), 128));
  *bytes = s.splits > 1 ? (size_t)s.splits * M * N * 4 : 0;
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
    rc = args->type == HOTK_E4M3 ? la_product<T8, OT>(*args, workspace, ws_bytes, st)
                                 : la_product<OT, OT>(*args, workspace, ws_bytes, st);
  });
  return rc;
}

extern "C" int hotk_linear_turn(const void* in, int64_t ld_in, const void* save, int act, void* out, int64_t ld_out, void* out_t,
                                int64_t ld_t, float* partial, int64_t R, int64_t C, int type, void* stream) {
  HOTK_CHECK_ARG(R >= 0 && C > 0 && ld_in >= C && (!out || ld_out >= C) && (!out_t || ld_t >= R));
  HOTK_CHECK_ARG(act >= HOTK_ACT_NONE && act <= HOTK_ACT_SILU && (act == HOTK_ACT_NONE || save || R == 0));
  HOTK_CHECK_ARG(out || out_t || partial);
  if (!ffn_type_ok(type) && type != HOTK_E4M3) return HOTK_EUNSUPPORTED;
  HOTK_CHECK_ARG(type != HOTK_E4M3 || (act == HOTK_ACT_NONE && !partial));      // (bytes are copied, not added)
  if (R == 0) return HOTK_OK;
  HOTK_CHECK_ARG(in);
  const int64_t across = la_div(out && ld_out > C ? ld_out : C, 64), down = la_div(out_t && ld_t > R ? ld_t : R, 64);
  if (across > (1 << 20) || down > (1ll << 30) / across) return HOTK_ETOOLARGE;
  const dim3 grid((unsigned)(across * down)), block(256);
  hipStream_t st = (hipStream_t)stream;
  if (type == HOTK_E4M3)
    hipLaunchKernelGGL((k_linact_turn<uint8_t, false>), grid, block, 0, st, (const uint8_t*)in, ld_in, save, act, (uint8_t*)out,
                       ld_out, (uint8_t*)out_t, ld_t, partial, R, C, (unsigned)across);
  else
    ffn_dispatch(type, [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      hipLaunchKernelGGL((k_linact_turn<T, true>), grid, block, 0, st, (const T*)in, ld_in, save, act, (T*)out, ld_out, (T*)out_t,
                         ld_t, partial, R, C, (unsigned)across);
    });
  return hotk_launch_status();
}
