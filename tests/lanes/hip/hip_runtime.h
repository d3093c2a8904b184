// Runs the library's HIP kernels on the CPU, lane by lane, for tests: what the attention sources need of the HIP runtime, of the
// gfx950 builtins and of a launch.  Every lane of a workgroup is a fiber; it runs until it meets a barrier or an operation of its
// wave (matrix instruction, shuffle, ballot, wave barrier) and goes on when the others have got there.  A launch is over when
// hipLaunchKernelGGL returns.  Memory is the process's own, so a read out of range ends on a guard page (lanes.cpp).
#pragma once
#include <immintrin.h>

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)

typedef int hipError_t;
typedef void* hipStream_t;
enum { hipSuccess = 0, hipFuncAttributeMaxDynamicSharedMemorySize = 0 };
inline const char* hipGetErrorString(hipError_t) { return ""; }
inline hipError_t hipGetDevice(int* d) { return *d = 0; }
inline hipError_t hipFuncSetAttribute(const void*, int, int) { return hipSuccess; }
inline hipError_t hipGetLastError() { return hipSuccess; }

struct dim3 {
  unsigned x;
  explicit dim3(unsigned n) : x(n) {}
};
struct LaneIndex {
  unsigned x;
};
extern LaneIndex threadIdx, blockIdx;

namespace lanes {
// Puts `in` (of `bytes`) beside those of the other lanes of the wave, and waits for them; lane l's is at the result + l * 128.
const char* wave_all(const void* in, size_t bytes);
void workgroup_barrier();
void run(unsigned grid, unsigned block, size_t lds, void (*body)(const void*), const void* args);

template <typename A>
struct Launch {
  void (*kernel)(A);
  const A* args;
  static void body(const void* p) { static_cast<const Launch*>(p)->kernel(*static_cast<const Launch*>(p)->args); }
};
template <typename A>
void launch(void (*kernel)(A), dim3 grid, dim3 block, size_t lds, hipStream_t, const A& a) {
  const Launch<A> l{kernel, &a};
  run(grid.x, block.x, lds, &Launch<A>::body, &l);
}
template <typename V>
const V& of_lane(const char* all, int lane) {
  static_assert(sizeof(V) <= 128, "a lane's place");
  return *reinterpret_cast<const V*>(all + 128 * lane);
}

typedef float Result __attribute__((ext_vector_type(16)));
// 32x32 result: lane l holds column l & 31, register r row 8 (r / 4) + 4 (l >> 5) + r % 4; K slots a lane half.
template <int K, typename V, typename At>
Result mfma(V a, V b, Result c, At at) {
  struct Pair {
    V a, b;
  };
  const int lane = threadIdx.x & 63;
  const Pair mine{a, b};
  const char* all = wave_all(&mine, sizeof mine);
  for (int r = 0; r < 16; ++r) {
    const int row = 8 * (r / 4) + 4 * (lane >> 5) + r % 4;
    float t = c[r];
    for (int h = 0; h < 2; ++h)
      for (int s = 0; s < K; ++s)
        t = fmaf(at(of_lane<Pair>(all, row + 32 * h).a, s), at(of_lane<Pair>(all, (lane & 31) + 32 * h).b, s), t);
    c[r] = t;
  }
  return c;
}
template <typename V>
Result mfma16(V a, V b, Result c) {
  return mfma<8>(a, b, c, [](const V& v, int s) { return (float)v[s]; });
}
typedef _Float16 Halves __attribute__((ext_vector_type(2)));
inline Halves halves_towards_zero(float a, float b) {
  const unsigned short h[2] = {_cvtss_sh(a, _MM_FROUND_TO_ZERO), _cvtss_sh(b, _MM_FROUND_TO_ZERO)};
  return __builtin_bit_cast(Halves, h);
}
inline uint64_t ballot(bool on) {
  const char* all = wave_all(&on, sizeof on);
  uint64_t bits = 0;
  for (int l = 0; l < 64; ++l) bits |= (uint64_t)of_lane<bool>(all, l) << l;
  return bits;
}
}  // namespace lanes

#define hipLaunchKernelGGL(kernel, ...) lanes::launch(kernel, __VA_ARGS__)
#define __syncthreads lanes::workgroup_barrier
#define __builtin_amdgcn_wave_barrier() (void)lanes::wave_all("", 1)
#define __builtin_amdgcn_fence(...)
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_logf log2f
#define __builtin_amdgcn_rcpf(x) (1.f / (x))
#define __builtin_amdgcn_cvt_pkrtz lanes::halves_towards_zero
#define __builtin_amdgcn_readfirstlane(x) (x)                  // of values that are the same in every lane
#define __builtin_amdgcn_inverse_ballot_w64(bits) ((((bits) >> (threadIdx.x & 63)) & 1) != 0)
#define __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, ...) lanes::mfma<1>(a, b, c, [](float v, int) { return v; })
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, ...) lanes::mfma16(a, b, c)
#define __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, ...) lanes::mfma16(a, b, c)

inline float __shfl_xor(float v, int mask, int) {
  return lanes::of_lane<float>(lanes::wave_all(&v, sizeof v), (threadIdx.x & 63) ^ mask);
}
inline uint64_t __ballot(bool on) { return lanes::ballot(on); }
inline bool __any(bool on) { return lanes::ballot(on) != 0; }
inline bool __all(bool on) { return lanes::ballot(on) == ~0ull; }
inline int min(int a, int b) { return a < b ? a : b; }
inline int max(int a, int b) { return a > b ? a : b; }
inline long min(long a, long b) { return a < b ? a : b; }
inline long max(long a, long b) { return a > b ? a : b; }
