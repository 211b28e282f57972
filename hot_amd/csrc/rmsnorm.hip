// Root-mean-square norm of a residual stream, its 8-bit form, and rows to 8 bits (the norm and the operand makers of the
// feed-forward block; the product that reads them is in linact.hip).
//
//   h = round(x + r)                   the stream as it is stored; without a residual h = x
//   rstd = (mean_c h^2 + eps)^(-1/2)   y = h * rstd * w
//   backward, u = h * rstd, g = dy * w:   dx = dr = rstd * (g - u * mean_c(g u)) + dh,   dw = sum_r dy * u
//   8 bits:  scale = max(max_c |y| / 448, 2^-126),   q = e4m3(y / scale)
//   rows that `keep` leaves out: h, y, q and dx are zero and nothing of the row is read
//
// Everything between the load and the one rounding at the store is in 32 bits; the norm reads the ROUNDED h, so that the
// backward pass, which finds h and not x and r, differentiates what the forward pass computed.
//
// A group of LPR lanes (8 to 64 of a wave, or 4, 8 or 16 waves) owns a row and holds it in registers, VEC elements (16 bytes) a
// lane and NV of them, so a row is read once.  Sums cross lanes by shuffles and waves through LDS.  HBM-bound.  A row that is no multiple of VEC has no tail: the
// last piece starts VEC before its end, overlapping its neighbour (and so do the lanes past the end); the sums count each
// element in one lane only, the stores write the same values twice.  Rows shorter than VEC go element by element (SMALL).
//
// Measured (a large copy reads and writes 5.0 TB/s here): 16 384 x 4 096 bf16 with a residual 88 us forward (6.1 TB/s of x, r, h, y)
// and 98 to 112 + 5 backward (5.5 to 4.8 TB/s); 8 192 x 2 048 bf16 to 8 bits 25 us (4.7 TB/s); rows of 8 192 x 4 096 bf16 to 8 bits 18 us (5.5);
// one row of 4 096: 2.5 us, a launch.
#include <algorithm>

#include "ffn.h"

namespace {

constexpr int RN_MAX_D = 32768;
constexpr float RN_E4M3_MAX = 448.f;
constexpr float RN_SCALE_MIN = 0x1p-126f;

template <int N>
__device__ __forceinline__ float rn_lane_sum(float v) {
#pragma unroll
  for (int o = N / 2; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
// the largest magnitude as the bits of a non-negative float: integer order is float order there, and a NaN is above infinity
template <int N>
__device__ __forceinline__ uint32_t rn_lane_max(uint32_t v) {
#pragma unroll
  for (int o = N / 2; o >= 1; o >>= 1) {
    const uint32_t t = (uint32_t)__shfl_xor((int)v, o, 64);
    v = t > v ? t : v;
  }
  return v;
}
// over the LPR lanes of a row's group.  `slot` alternates between calls: one barrier per call is enough, since a wave that
// writes a slot again has passed the barrier of the call in between, which every reader reached after its reads.
template <int LPR>
__device__ __forceinline__ float rn_group_sum(float v, float (*box)[16], int& slot) {
  if (LPR <= 64) return rn_lane_sum<LPR>(v);
  v = rn_lane_sum<64>(v);
  if ((threadIdx.x & 63) == 0) box[slot][threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < LPR / 64; ++i) t += box[slot][i];
  slot ^= 1;
  return t;
}
template <int LPR>
__device__ __forceinline__ uint32_t rn_group_max(uint32_t v, float (*box)[16], int& slot) {
  if (LPR <= 64) return rn_lane_max<LPR>(v);
  v = rn_lane_max<64>(v);
  if ((threadIdx.x & 63) == 0) box[slot][threadIdx.x >> 6] = __uint_as_float(v);
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < LPR / 64; ++i) {
    const uint32_t u = __float_as_uint(box[slot][i]);
    t = u > t ? u : t;
  }
  slot ^= 1;
  return t;
}

// ---- a lane's piece of a row --------------------------------------------------------------------------------------------
template <class T, bool SMALL>
struct Piece {
  using E = Elem<T>;
  using FV = typename E::fvec;
  int c;          // first column
  int skip;       // leading elements that belong to a neighbour (VEC: the whole piece); SMALL: unused
  __device__ __forceinline__ Piece(int lane, int D) {
    const int want = E::VEC * lane;
    if (SMALL) {
      c = want;
      skip = 0;
    } else {
      c = want < D - E::VEC ? want : D - E::VEC;
      skip = want < D ? want - c : E::VEC;
    }
  }
  __device__ __forceinline__ bool mine(int k, int D) const { return SMALL ? c + k < D : k >= skip; }
  __device__ __forceinline__ FV load(const T* __restrict__ row, int D) const {
    if (SMALL) return ffn_load(row, c, D);
    return __builtin_convertvector((typename E::vec)(*reinterpret_cast<const typename E::uvec*>(row + c)), FV);
  }
  __device__ __forceinline__ bool any(int D) const { return SMALL ? c < D : skip < E::VEC; }
  __device__ __forceinline__ void store(T* __restrict__ row, int D, FV v) const {
    if (!any(D)) return;
    if (SMALL) ffn_store(row, c, D, v);
    else *reinterpret_cast<typename E::uvec*>(row + c) = __builtin_convertvector(v, typename E::vec);
  }
  // rounded to e4m3
  __device__ __forceinline__ void store8(uint8_t* __restrict__ row, int D, FV v) const {
    if (!any(D)) return;
    uint32_t b[E::VEC / 4];
#pragma unroll
    for (int i = 0; i < E::VEC / 4; ++i) {
      const int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i], v[4 * i + 1], 0, false);
      b[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * i + 2], v[4 * i + 3], t, true);
    }
    if (SMALL) {
#pragma unroll
      for (int i = 0; i < E::VEC; ++i)
        if (c + i < D) row[c + i] = (uint8_t)(b[i / 4] >> (8 * (i % 4)));
    } else {
      __builtin_memcpy(row + c, b, E::VEC);
    }
  }
};

template <class T>
struct RnFwd {
  const T *x, *r, *w;
  int64_t ld_x, ld_r;
  const uint8_t* kind;
  unsigned keep;
  float eps;
  T *y, *h;
  float* rstd;
  uint8_t* q;
  float* scale;
  int64_t R;
  int D;
};

enum { RN_NORM = 0, RN_NORM8 = 1, RN_QUANT = 2 };

// 256 threads a workgroup, or the LPR of one row where that is more (its barriers are then the whole workgroup's)
template <class T, int MODE, int NV, int LPR, bool SMALL>
__global__ __launch_bounds__(LPR > 64 ? LPR : 256) void k_rmsnorm_fwd(const RnFwd<T> a) {
  using E = Elem<T>;
  using FV = typename E::fvec;
  constexpr int VEC = E::VEC, GROUPS = LPR > 64 ? 1 : 256 / LPR;
  __shared__ float box[2][16];
  int slot = 0;
  const int t = threadIdx.x % LPR, D = a.D;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPR; row < a.R; row += (int64_t)gridDim.x * GROUPS) {
    const bool kept = !a.kind || hotk_keep(a.keep, a.kind[row]);
    FV v[NV];
    if (kept) {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = Piece<T, SMALL>(t + LPR * i, D).load(a.x + row * a.ld_x, D);
      if (MODE != RN_QUANT && a.r) {
        FV r[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) r[i] = Piece<T, SMALL>(t + LPR * i, D).load(a.r + row * a.ld_r, D);
#pragma unroll
        for (int i = 0; i < NV; ++i)      // what the norm reads is what is stored
          v[i] = __builtin_convertvector(__builtin_convertvector(v[i] + r[i], typename E::vec), FV);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i) v[i] = 0.f;
    }
    if (MODE != RN_QUANT) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Piece<T, SMALL> p(t + LPR * i, D);
        if (a.r) p.store(a.h + row * D, D, v[i]);
#pragma unroll
        for (int k = 0; k < VEC; ++k) s += p.mine(k, D) ? v[i][k] * v[i][k] : 0.f;
      }
      const float rstd = rsqrtf(rn_group_sum<LPR>(s, box, slot) / (float)D + a.eps);
      if (a.rstd && t == 0) a.rstd[row] = rstd;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const Piece<T, SMALL> p(t + LPR * i, D);
        v[i] = v[i] * rstd * p.load(a.w, D);
        if (!kept) v[i] = 0.f;            // (an infinite weight times zero)
        if (MODE == RN_NORM) p.store(a.y + row * D, D, v[i]);
      }
    }
    if (MODE != RN_NORM) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {   // (SMALL: the elements past the end are zeros; else a lane past the end repeats others)
          const uint32_t u = __float_as_uint(v[i][k]) & 0x7fffffffu;
          m = u > m ? u : m;
        }
      float scale = __uint_as_float(rn_group_max<LPR>(m, box, slot)) / RN_E4M3_MAX;
      scale = scale < RN_SCALE_MIN ? RN_SCALE_MIN : scale;     // (a NaN stays one)
      if (t == 0) a.scale[row] = scale;
#pragma unroll
      for (int i = 0; i < NV; ++i) Piece<T, SMALL>(t + LPR * i, D).store8(a.q + row * D, D, v[i] / scale);
    }
  }
}

template <class T>
struct RnBwd {
  const T *dy, *dh, *h, *w;
  int64_t ld_dy, ld_dh, ld_h;
  const float* rstd;
  const uint8_t* kind;
  unsigned keep;
  T *dx, *dw;
  float* partial;
  int64_t R;
  int D;
};

// dw of few rows: a workgroup takes four pieces of columns, its row lanes every (THREADS / 4)th row each; LDS joins them by halves
template <class T, int THREADS, bool SMALL>
__device__ __forceinline__ void rn_columns(const RnBwd<T>& a, typename Elem<T>::fvec* sums) {
  using FV = typename Elem<T>::fvec;
  constexpr int LANES = THREADS / 4;
  if ((int64_t)blockIdx.x * 4 * Elem<T>::VEC >= a.D) return;
  const Piece<T, SMALL> p(blockIdx.x * 4 + (threadIdx.x & 3), a.D);
  FV s = 0.f;
  for (int64_t row = threadIdx.x >> 2; row < a.R; row += LANES) {
    if (a.kind && !hotk_keep(a.keep, a.kind[row])) continue;
    s += p.load(a.dy + row * a.ld_dy, a.D) * (p.load(a.h + row * a.ld_h, a.D) * a.rstd[row]);
  }
  sums[threadIdx.x] = s;
  for (int half = LANES / 2; half >= 1; half >>= 1) {
    __syncthreads();
    if ((int)(threadIdx.x >> 2) < half) sums[threadIdx.x] += sums[threadIdx.x + 4 * half];
  }
  if (threadIdx.x < 4) p.store(a.dw, a.D, sums[threadIdx.x]);
}

// FEW: few rows, dw wanted.  (An instance of its own: with the branch in all of them 16 384 x 4 096 bf16 took 107 us instead of 98.)
template <class T, int NV, int LPR, bool SMALL, bool FEW>
__global__ __launch_bounds__(LPR > 64 ? LPR : 256) void k_rmsnorm_bwd(const RnBwd<T> a) {
  using E = Elem<T>;
  using FV = typename E::fvec;
  constexpr int VEC = E::VEC, GROUPS = LPR > 64 ? 1 : 256 / LPR;
  constexpr int THREADS = LPR > 64 ? LPR : 256;
  constexpr bool LATE = NV * VEC >= 32;      // the widest rows: dh is read where it is added, so that what a lane holds stays in registers
  __shared__ float box[2][16];
  __shared__ FV fold[THREADS];
  if (FEW && blockIdx.y) return rn_columns<T, THREADS, SMALL>(a, fold);
  int slot = 0;
  const int t = threadIdx.x % LPR, D = a.D;
  const float inv_d = 1.f / (float)D;
  FV dw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) dw[i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * GROUPS + threadIdx.x / LPR; row < a.R; row += (int64_t)gridDim.x * GROUPS) {
    if (a.kind && !hotk_keep(a.keep, a.kind[row])) {
#pragma unroll
      for (int i = 0; i < NV; ++i) Piece<T, SMALL>(t + LPR * i, D).store(a.dx + row * D, D, (FV)0.f);
      continue;
    }
    const float rstd = a.rstd[row];
    FV g[NV], u[NV], o[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Piece<T, SMALL> p(t + LPR * i, D);
      g[i] = p.load(a.dy + row * a.ld_dy, D);
      u[i] = p.load(a.h + row * a.ld_h, D);
      if (!LATE) o[i] = a.dh ? p.load(a.dh + row * a.ld_dh, D) : (FV)0.f;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Piece<T, SMALL> p(t + LPR * i, D);
      u[i] *= rstd;
      dw[i] += g[i] * u[i];
      g[i] *= p.load(a.w, D);
#pragma unroll
      for (int k = 0; k < VEC; ++k) s += p.mine(k, D) ? g[i][k] * u[i][k] : 0.f;
    }
    const float m = rn_group_sum<LPR>(s, box, slot) * inv_d;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const Piece<T, SMALL> p(t + LPR * i, D);
      if (LATE) o[i] = a.dh ? p.load(a.dh + row * a.ld_dh, D) : (FV)0.f;
      p.store(a.dx + row * D, D, o[i] + rstd * (g[i] - u[i] * m));
    }
  }
  if (FEW || !a.partial) return;      // few rows: the grid's second line writes dw, or nobody wants it
  // one partial row of dw per workgroup: rows side by side in a wave are added across lanes, the waves in order through LDS
  float* out = a.partial + (int64_t)blockIdx.x * D;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const Piece<T, SMALL> p(t + LPR * i, D);
    FV o = dw[i];
    if (GROUPS > 1) {
#pragma unroll
      for (int k = 0; k < VEC; ++k)
#pragma unroll
        for (int d = 32; d >= LPR; d >>= 1) o[k] += __shfl_xor(o[k], d, 64);
      __syncthreads();
      fold[threadIdx.x] = o;
      __syncthreads();
      if (threadIdx.x >= LPR) continue;
#pragma unroll
      for (int w = 1; w < 4; ++w) o += fold[64 * w + t];
    }
#pragma unroll
    for (int k = 0; k < VEC; ++k)
      if (p.mine(k, D)) out[p.c + k] = o[k];
  }
}

// out[c] = sum over b of partial[b][c], in an order that the sizes alone set: 16 columns a workgroup, its 64 row lanes add every
// 64th row each (eight loads under way), LDS joins them by halves
template <class T>
__global__ __launch_bounds__(1024) void k_sum_partials(const float* __restrict__ partial, int64_t n, int64_t D, T* __restrict__ out) {
  __shared__ float part[64][17];
  const int col = threadIdx.x & 15, row = threadIdx.x >> 4;
  const int64_t c = (int64_t)blockIdx.x * 16 + col;
  float s = 0.f;
  if (c < D) {
#pragma unroll 8
    for (int64_t b = row; b < n; b += 64) s += partial[b * D + c];
  }
  part[row][col] = s;
  for (int half = 32; half >= 1; half >>= 1) {
    __syncthreads();
    if (row < half) part[row][col] += part[row + half][col];
  }
  if (row == 0 && c < D) out[c] = (T)part[0][col];
}

unsigned rn_grid(int64_t rows, int groups, unsigned cap) {
  const int64_t g = (rows + groups - 1) / groups;
  return (unsigned)(g < 1 ? 1 : (g > cap ? cap : g));
}

// lanes per row and pieces per lane for a row of D: as few lanes as hold it in one or two pieces.  Measured at 16 384 rows of 4 096
// bf16: the norm with a residual 93 us with 8 waves and one piece, 94 / 98 with 4 and two / four, its backward pass 98 / 102 / 124;
// rows to 8 bits, with two sums to wait for and less to move, 48 / 38 / 43, so there a lane holds more.
struct RnShape { int lpr, nv; };
RnShape rn_shape(int64_t D, int vec, bool quant) {
  if (D < vec) return {8, 0};                       // SMALL
  const int64_t v = (D + vec - 1) / vec;
  if (v <= 64) return {v <= 8 ? 8 : v <= 16 ? 16 : v <= 32 ? 32 : 64, 1};
  if (v <= 128) return {64, 2};
  if (v <= 256) return quant ? RnShape{64, 4} : RnShape{256, 1};
  if (v <= 512) return quant ? RnShape{256, 2} : RnShape{512, 1};
  if (v <= 1024) return quant ? RnShape{256, 4} : RnShape{512, 2};
  return {1024, v <= 2048 ? 2 : v <= 4096 ? 4 : 8};
}
int rn_rows_per_group(int lpr) { return lpr > 64 ? 1 : 256 / lpr; }

template <class T, int MODE>
int rn_launch_fwd(const RnFwd<T>& a, hipStream_t st) {
  const RnShape sh = rn_shape(a.D, Elem<T>::VEC, MODE == RN_QUANT);
  const dim3 grid(rn_grid(a.R, rn_rows_per_group(sh.lpr), 8192)), block(sh.lpr > 64 ? sh.lpr : 256);
#define RN_F(LPR, NV, SMALL) hipLaunchKernelGGL((k_rmsnorm_fwd<T, MODE, NV, LPR, SMALL>), grid, block, 0, st, a)
  constexpr bool Q = MODE == RN_QUANT;
  switch (sh.lpr * 16 + sh.nv) {
    case 8 * 16: RN_F(8, 1, true); break;
    case 8 * 16 + 1: RN_F(8, 1, false); break;
    case 16 * 16 + 1: RN_F(16, 1, false); break;
    case 32 * 16 + 1: RN_F(32, 1, false); break;
    case 64 * 16 + 1: RN_F(64, 1, false); break;
    case 64 * 16 + 2: RN_F(64, 2, false); break;
    case 64 * 16 + 4: if constexpr (Q) RN_F(64, 4, false); break;
    case 256 * 16 + 1: if constexpr (!Q) RN_F(256, 1, false); break;
    case 256 * 16 + 2: if constexpr (Q) RN_F(256, 2, false); break;
    case 256 * 16 + 4: if constexpr (Q) RN_F(256, 4, false); break;
    case 512 * 16 + 1: if constexpr (!Q) RN_F(512, 1, false); break;
    case 512 * 16 + 2: if constexpr (!Q) RN_F(512, 2, false); break;
    case 1024 * 16 + 2: RN_F(1024, 2, false); break;
    case 1024 * 16 + 4: RN_F(1024, 4, false); break;
    default: if constexpr (Elem<T>::VEC == 4) RN_F(1024, 8, false);
  }
#undef RN_F
  return hotk_launch_status();
}

// few rows: dw is written by a second line of workgroups of the same launch, which read dy and h once more.  Measured at 1 024 rows
// against a launch for the partial sums: fp32 of 1 024 columns 5.9 and 10.2 us, 2 048 10.8 and 10.5, 4 096 19.7 and 16.6; bf16 of 2 048 6.8
// and 11.9, 4 096 10.9 and 17.1.  A workgroup reads its columns of all rows, which bounds the rows whatever their size.
bool rn_few(int64_t R, int64_t D, int bytes) { return R <= 1024 && R * D * bytes <= 8 << 20; }
// workgroups of the backward pass, each with one partial row of dw: enough to fill the chip, few enough that the partial sums
// stay a few percent of the traffic.  Rows of 16 waves: as many as fit at once (16 384 columns of bf16, 1 025 rows: 35 us; 512 of
// them 50); rows of 4 waves, few of them: 1 025 x 2 048 bf16 11.9 us with 512 and 16.3 with 1 024, 8 192 x 2 048 30.3 and 28.8.
unsigned rn_bwd_grid(int64_t R, int lpr) {
  return rn_grid(R, rn_rows_per_group(lpr), lpr > 512 ? 256 : lpr > 256 || (lpr > 64 && R < 8192) ? 512 : 1024);
}

template <class T>
int rn_launch_bwd(const RnBwd<T>& a, hipStream_t st) {
  const RnShape sh = rn_shape(a.D, Elem<T>::VEC, false);
  // few rows: a second line of workgroups writes dw
  const unsigned blocks = rn_bwd_grid(a.R, sh.lpr), columns = (unsigned)((a.D + 4 * Elem<T>::VEC - 1) / (4 * Elem<T>::VEC));
  const dim3 grid(a.dw ? std::max(blocks, columns) : blocks, a.dw ? 2 : 1), block(sh.lpr > 64 ? sh.lpr : 256);
#define RN_B(LPR, NV, SMALL)                                                                    \
  if (a.dw) hipLaunchKernelGGL((k_rmsnorm_bwd<T, NV, LPR, SMALL, true>), grid, block, 0, st, a); \
  else hipLaunchKernelGGL((k_rmsnorm_bwd<T, NV, LPR, SMALL, false>), grid, block, 0, st, a)
  switch (sh.lpr * 16 + sh.nv) {
    case 8 * 16: RN_B(8, 1, true); break;
    case 8 * 16 + 1: RN_B(8, 1, false); break;
    case 16 * 16 + 1: RN_B(16, 1, false); break;
    case 32 * 16 + 1: RN_B(32, 1, false); break;
    case 64 * 16 + 1: RN_B(64, 1, false); break;
    case 64 * 16 + 2: RN_B(64, 2, false); break;
    case 256 * 16 + 1: RN_B(256, 1, false); break;
    case 512 * 16 + 1: RN_B(512, 1, false); break;
    case 512 * 16 + 2: RN_B(512, 2, false); break;
    case 1024 * 16 + 2: RN_B(1024, 2, false); break;
    case 1024 * 16 + 4: RN_B(1024, 4, false); break;
    default: if constexpr (Elem<T>::VEC == 4) { RN_B(1024, 8, false); }
  }
#undef RN_B
  return hotk_launch_status();
}

bool rn_rows_ok(const void* p, int64_t ld, int64_t D, int type) { return p && ld >= D && ffn_elem_aligned(p, type); }

}  // namespace

extern "C" int hotk_rmsnorm_supported(int64_t D, int type) { return (D > 0 && D <= RN_MAX_D && ffn_type_ok(type)) ? 1 : 0; }

extern "C" int hotk_rmsnorm_fwd(const void* x, int64_t ld_x, const void* res, int64_t ld_res, const void* w, const uint8_t* kind,
                                unsigned keep, float eps, void* y, void* h, float* rstd, int64_t R, int64_t D, int type,
                                void* stream) {
  HOTK_CHECK_ARG(R >= 0);
  if (!hotk_rmsnorm_supported(D, type)) return HOTK_EUNSUPPORTED;
  if (R == 0) return HOTK_OK;
  HOTK_CHECK_ARG(rn_rows_ok(x, ld_x, D, type) && rn_rows_ok(w, D, D, type) && rn_rows_ok(y, D, D, type));
  HOTK_CHECK_ARG(!res || (rn_rows_ok(res, ld_res, D, type) && rn_rows_ok(h, D, D, type)));
  int rc = HOTK_OK;
  ffn_dispatch(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const RnFwd<T> a{(const T*)x, (const T*)res, (const T*)w, ld_x, ld_res, kind, keep, eps, (T*)y, (T*)h, rstd, nullptr,
                     nullptr, R, (int)D};
    rc = rn_launch_fwd<T, RN_NORM>(a, (hipStream_t)stream);
  });
  return rc;
}

extern "C" int hotk_rmsnorm_quant(const void* x, int64_t ld_x, const void* res, int64_t ld_res, const void* w,
                                  const uint8_t* kind, unsigned keep, float eps, uint8_t* q, float* scale, void* h, int64_t R,
                                  int64_t D, int type, void* stream) {
  HOTK_CHECK_ARG(R >= 0);
  if (!hotk_rmsnorm_supported(D, type)) return HOTK_EUNSUPPORTED;
  if (R == 0) return HOTK_OK;
  HOTK_CHECK_ARG(rn_rows_ok(x, ld_x, D, type) && rn_rows_ok(w, D, D, type) && q && scale);
  HOTK_CHECK_ARG(!res || (rn_rows_ok(res, ld_res, D, type) && rn_rows_ok(h, D, D, type)));
  int rc = HOTK_OK;
  ffn_dispatch(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const RnFwd<T> a{(const T*)x, (const T*)res, (const T*)w, ld_x, ld_res, kind, keep, eps, nullptr, (T*)h, nullptr, q,
                     scale, R, (int)D};
    rc = rn_launch_fwd<T, RN_NORM8>(a, (hipStream_t)stream);
  });
  return rc;
}

extern "C" int hotk_quantize_rows(const void* x, int64_t ld_x, uint8_t* q, float* scale, int64_t R, int64_t D, int type,
                                  void* stream) {
  HOTK_CHECK_ARG(R >= 0);
  if (!hotk_rmsnorm_supported(D, type)) return HOTK_EUNSUPPORTED;
  if (R == 0) return HOTK_OK;
  HOTK_CHECK_ARG(rn_rows_ok(x, ld_x, D, type) && q && scale);
  int rc = HOTK_OK;
  ffn_dispatch(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const RnFwd<T> a{(const T*)x, nullptr, nullptr, ld_x, 0, nullptr, 0, 0.f, nullptr, nullptr, nullptr, q, scale, R, (int)D};
    rc = rn_launch_fwd<T, RN_QUANT>(a, (hipStream_t)stream);
  });
  return rc;
}

extern "C" int hotk_rmsnorm_partials(int64_t R, int64_t D, int type, int64_t* n_partials) {
  HOTK_CHECK_ARG(n_partials && R >= 0);
  if (!hotk_rmsnorm_supported(D, type)) return HOTK_EUNSUPPORTED;
  *n_partials = rn_few(R, D, ffn_bytes(type)) ? 0 : (int64_t)rn_bwd_grid(R, rn_shape(D, 16 / ffn_bytes(type), false).lpr);
  return HOTK_OK;
}

extern "C" int hotk_rmsnorm_bwd(const void* dy, int64_t ld_dy, const void* dh, int64_t ld_dh, const void* h, int64_t ld_h,
                                const float* rstd, const void* w, const uint8_t* kind, unsigned keep, void* dx, float* partial,
                                void* dw, int64_t R, int64_t D, int type, void* stream) {
  HOTK_CHECK_ARG(R >= 0);
  if (!hotk_rmsnorm_supported(D, type)) return HOTK_EUNSUPPORTED;
  HOTK_CHECK_ARG(rn_few(R, D, ffn_bytes(type)) ? !partial : !dw);
  HOTK_CHECK_ARG(!dw || ffn_elem_aligned(dw, type));
  HOTK_CHECK_ARG(R == 0 || (rn_rows_ok(dy, ld_dy, D, type) && rn_rows_ok(h, ld_h, D, type) && rstd && rn_rows_ok(dx, D, D, type)));
  HOTK_CHECK_ARG(rn_rows_ok(w, D, D, type) && (!dh || rn_rows_ok(dh, ld_dh, D, type)));
  int rc = HOTK_OK;
  ffn_dispatch(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const RnBwd<T> a{(const T*)dy, (const T*)dh, (const T*)h, (const T*)w, ld_dy, ld_dh, ld_h, rstd, kind, keep, (T*)dx, (T*)dw,
                     partial, R, (int)D};
    rc = rn_launch_bwd<T>(a, (hipStream_t)stream);
  });
  return rc;
}

extern "C" int hotk_sum_partials(const float* partial, int64_t n, int64_t D, void* out, int type, void* stream) {
  HOTK_CHECK_ARG(n >= 0 && D >= 0);
  if (!ffn_type_ok(type)) return HOTK_EUNSUPPORTED;
  if (D == 0) return HOTK_OK;
  if (D > (1 << 25)) return HOTK_ETOOLARGE;      // (a launch holds fewer than 2^32 threads)
  HOTK_CHECK_ARG(out && (partial || n == 0) && ffn_elem_aligned(out, type));
  const dim3 grid((unsigned)((D + 15) / 16)), block(1024);
  ffn_dispatch(type, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    hipLaunchKernelGGL(k_sum_partials<T>, grid, block, 0, (hipStream_t)stream, partial, n, D, (T*)out);
  });
  return hotk_launch_status();
}
