// Element types and matrix-instruction fragments of the attention-block operators (gfx950).
#pragma once
#include "common.h"

namespace trace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32v8 __attribute__((ext_vector_type(8), aligned(16)));
typedef float f32v4 __attribute__((ext_vector_type(4)));
typedef float f32v2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16v8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16v4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16v2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16v8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16v4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16v2 __attribute__((ext_vector_type(2)));

// V8 / V4: eight / four consecutive elements.  V8 is also one lane's share of an operand of mma32: lane l holds row (A)
// or column (B) l & 31 and the contraction slots 8 (l >> 5) .. + 7 of 16.  The 16-bit types use the 32x32x16 instruction; float
// runs eight 32x32x2 ones, instruction i contracting slot i of both lane halves, so all types share one layout.
// The result of mma32: lane l holds column l & 31 and, in register r, row 8 (r / 4) + 4 (l >> 5) + r % 4.
template <typename T> struct Elem;
template <> struct Elem<float> {
  typedef f32v8 V8;
  typedef f32v4 V4;
  static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};
template <> struct Elem<__bf16> {
  typedef bf16v8 V8;
  typedef bf16v4 V4;
  static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Elem<_Float16> {
  typedef f16v8 V8;
  typedef f16v4 V4;
  static __device__ __forceinline__ f32x16 mma32(V8 a, V8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};

// Eight elements at p, of which the first n exist; the others are zero.  vec: p is 16-byte aligned, and n a multiple of 8.
template <typename T>
__device__ __forceinline__ typename Elem<T>::V8 load8(const T* p, int n, bool vec) {
  typename Elem<T>::V8 v = {};
  if (vec) {
    if (n > 0) v = *reinterpret_cast<const typename Elem<T>::V8*>(p);
    return v;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : (T)0.f;
  return v;
}

// Stores the first n (<= 4) of four elements.  vec: p is aligned to four elements.
template <typename T>
__device__ __forceinline__ void store4(T* p, f32v4 v, int n, bool vec) {
  typename Elem<T>::V4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = (T)v[i];
  if (vec && n >= 4) {
    *reinterpret_cast<typename Elem<T>::V4*>(p) = o;
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) p[i] = o[i];
}

// Workgroups are handed to the eight XCDs in turn; item() gives each XCD a contiguous range of the n work items, so that
// items that read the same data meet in one L2.  Launch xcd_grid(n) workgroups; item() >= n: nothing to do.
constexpr long MAX_GRID_THREADS = 0xffffffffL;              // of one launch
constexpr long XCDS = 8;
inline long xcd_grid(long n) { return (n + XCDS - 1) / XCDS * XCDS; }
__device__ __forceinline__ long xcd_item(long n) {
  const long each = (n + XCDS - 1) / XCDS;
  return (long)(blockIdx.x % XCDS) * each + blockIdx.x / XCDS;
}

}  // namespace trace
