// Shared by the feed-forward operators (rmsnorm.hip, linact.hip): element types and 16-byte row access.
#pragma once
#include "common.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Rows start wherever the caller's stride puts them, so 16-byte accesses promise no more than the element's alignment:
// global memory takes a 16-byte access at any address on gfx950 (one instruction, slower only where it crosses a line).
template <class T> struct Elem;
template <> struct Elem<float> {
  static constexpr int VEC = 4;
  typedef float vec __attribute__((ext_vector_type(4)));
  typedef float uvec __attribute__((ext_vector_type(4), aligned(4)));
  typedef float fvec __attribute__((ext_vector_type(4)));
};
template <> struct Elem<__bf16> {
  static constexpr int VEC = 8;
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
  typedef __bf16 uvec __attribute__((ext_vector_type(8), aligned(2)));
  typedef float fvec __attribute__((ext_vector_type(8)));
};
template <> struct Elem<_Float16> {
  static constexpr int VEC = 8;
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
  typedef _Float16 uvec __attribute__((ext_vector_type(8), aligned(2)));
  typedef float fvec __attribute__((ext_vector_type(8)));
};

// VEC elements of a row of n at column c, in 32 bits; beyond the row's end: zeros (nothing is read there)
template <class T>
__device__ __forceinline__ typename Elem<T>::fvec ffn_load(const T* __restrict__ row, int c, int n) {
  using E = Elem<T>;
  if (c + E::VEC <= n) return __builtin_convertvector((typename E::vec)(*reinterpret_cast<const typename E::uvec*>(row + c)), typename E::fvec);
  typename E::fvec v = 0.f;
#pragma unroll
  for (int i = 0; i < E::VEC; ++i)
    if (c + i < n) v[i] = (float)row[c + i];
  return v;
}

// the same, rounded to the element's type (nearest, ties to even) and stored
template <class T>
__device__ __forceinline__ void ffn_store(T* __restrict__ row, int c, int n, typename Elem<T>::fvec v) {
  using E = Elem<T>;
  const typename E::vec t = __builtin_convertvector(v, typename E::vec);
  if (c + E::VEC <= n) {
    *reinterpret_cast<typename E::uvec*>(row + c) = t;
  } else {
#pragma unroll
    for (int i = 0; i < E::VEC; ++i)
      if (c + i < n) row[c + i] = t[i];
  }
}

// calls f with a null pointer of the element type that the code names; false where it names none
template <class F>
static inline bool ffn_dispatch(int type, F&& f) {
  switch (type) {
    case HOTK_F32: f((float*)nullptr); return true;
    case HOTK_BF16: f((__bf16*)nullptr); return true;
    case HOTK_F16: f((_Float16*)nullptr); return true;
    default: return false;
  }
}

static inline int ffn_bytes(int type) { return type == HOTK_F32 ? 4 : type == HOTK_E4M3 ? 1 : 2; }
static inline bool ffn_type_ok(int type) { return type == HOTK_F32 || type == HOTK_BF16 || type == HOTK_F16; }
static inline bool ffn_elem_aligned(const void* p, int type) { return ((uintptr_t)p) % (uintptr_t)ffn_bytes(type) == 0; }
