// Launches of the attention kernels for one element type; a translation unit each (attn_f32.hip, attn_bf16.hip, attn_f16.hip)
// instantiates attn_run.
#pragma once
#include "attn_kernels.h"

namespace trace {
namespace {

template <typename K>
int launch(K kernel, unsigned long long* attr, size_t lds, int threads, const AttnArgs& a, hipStream_t st, const char* what) {
  const long grid = xcd_grid(a.items);
  TRACE_REQUIRE(grid * threads <= MAX_GRID_THREADS, "%s: grid of %ld workgroups", what, grid);
  if (lds > 64 * 1024) TRACE_CHECK_HIP(ensure_dynamic_lds(attr, reinterpret_cast<const void*>(kernel), (int)lds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, a);
  return launch_status(what);
}

template <typename T, int DP>
int join(const AttnArgs& a, hipStream_t st) {
  if (a.splits == 1) return TRACE_OK;
  const int64_t rows = (int64_t)a.B * a.Hq * a.Lq;
  if (a.splits <= ATTN_ROW_SPLITS && rows > 512) {         // 256 rows in 16 ranges: 5.4 us, against 4.4 with a workgroup a row
    const int64_t grid = (rows * (DP / 4) + 255) / 256;
    TRACE_REQUIRE(grid * 256 <= MAX_GRID_THREADS, "attn_join_rows_kernel: grid of %lld workgroups", (long long)grid);
    hipLaunchKernelGGL((attn_join_rows_kernel<T, DP>), dim3((unsigned)grid), dim3(256), 0, st, a);
    return launch_status("attn_join_rows_kernel");
  }
  TRACE_REQUIRE(rows * 256 <= MAX_GRID_THREADS, "attn_join_kernel: grid of %lld workgroups", (long long)rows);
  hipLaunchKernelGGL((attn_join_kernel<T, DP>), dim3((unsigned)rows), dim3(256), 0, st, a);
  return launch_status("attn_join_kernel");
}

template <typename T, int DP, int NW>
int fwd(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)((a.Lq + 32 * NW - 1) / (32 * NW)) * a.Hq * a.B * a.splits;
  const size_t lds = sizeof(T) * (KEY_TILE<T> * TileR<T, DP>::S + DP * TileX<T, KEY_TILE<T>>::S);
  const int r = launch(&attn_fwd_kernel<T, DP, NW>, &attr, lds, NW * 64, a, st, "attn_fwd_kernel");
  return r != TRACE_OK ? r : join<T, DP>(a, st);
}

template <typename T, int DP>
int few(const AttnArgs& a, hipStream_t st) {
  const int r = launch(&attn_few_kernel<T, DP>, nullptr, 0, 64, a, st, "attn_few_kernel");
  return r != TRACE_OK ? r : join<T, DP>(a, st);
}

template <typename T, int DP, int NW>
int dq(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)((a.Lq + 32 * NW - 1) / (32 * NW)) * a.Hq * a.B * a.splits_q;
  const size_t lds = sizeof(T) * (2 * KEY_TILE<T> * TileR<T, DP>::S + DP * TileX<T, KEY_TILE<T>>::S);
  const int r = launch(&attn_dq_kernel<T, DP, NW>, &attr, lds, NW * 64, a, st, "attn_dq_kernel");
  if (r != TRACE_OK || a.splits_q == 1) return r;
  const long grid = ((long)a.B * a.Hq * a.Lq * (DP / 4) + 255) / 256;
  TRACE_REQUIRE(grid * 256 <= MAX_GRID_THREADS, "attn_sum_q_kernel: grid of %ld workgroups", grid);
  hipLaunchKernelGGL((attn_sum_q_kernel<T, DP>), dim3((unsigned)grid), dim3(256), 0, st, a);
  return launch_status("attn_sum_q_kernel");
}

template <typename T, int DP, int NW>
int dkv(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)((a.Lk + 32 * NW - 1) / (32 * NW)) * a.Hk * a.B * a.splits;
  const size_t lds = sizeof(T) * 2 * (32 * TileR<T, DP>::S + DP * TileX<T, 32>::S) + 2 * 32 * sizeof(float) +
                     (DKV_V_LDS<T, DP> ? sizeof(T) * 32 * NW * TileR<T, DP>::S : 0);
  const int r = launch(&attn_dkv_kernel<T, DP, NW>, &attr, lds, NW * 64, a, st, "attn_dkv_kernel");
  if (r != TRACE_OK || a.splits == 1) return r;
  const long grid = ((long)a.B * a.Hk * a.Lk * (DP / 4) + 255) / 256;
  TRACE_REQUIRE(grid * 256 <= MAX_GRID_THREADS, "attn_sum_kernel: grid of %ld workgroups", grid);
  hipLaunchKernelGGL((attn_sum_kernel<T, DP>), dim3((unsigned)grid), dim3(256), 0, st, a);
  return launch_status("attn_sum_kernel");
}

template <typename T, int DP, int QB, int KB, bool MANY>
int short_heads(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)a.Hk * a.B;
  const size_t lds = sizeof(T) * (2 * QB + KB) * 32 * TileN<T, DP>::S + sizeof(float) * 32 * QB * TileN<float, 32 * KB>::S +
                     (FIT<T> ? sizeof(float) * QB * KB : 0);
  return launch(&attn_short_backward_kernel<T, DP, QB, KB, MANY>, &attr, lds, QB * KB * 64, a, st, "attn_short_backward_kernel");
}
template <typename T, int DP, int QB, int KB>
int short_backward(const AttnArgs& a, hipStream_t st) {
  return FIT<T> && a.G > 1 ? short_heads<T, DP, QB, KB, FIT<T>>(a, st) : short_heads<T, DP, QB, KB, false>(a, st);
}
template <typename T, int DP>
int short_blocks(const AttnArgs& a, hipStream_t st) {
  if (a.Lq <= 32) return a.Lk <= 32 ? short_backward<T, DP, 1, 1>(a, st) : short_backward<T, DP, 1, 2>(a, st);
  return a.Lk <= 32 ? short_backward<T, DP, 2, 1>(a, st) : short_backward<T, DP, 2, 2>(a, st);
}

#define TRACE_ATTN_NW(FN, T, DP, W) (W == 1 ? FN<T, DP, 1>(a, st) : W == 2 ? FN<T, DP, 2>(a, st) : FN<T, DP, 4>(a, st))
#define TRACE_ATTN_DP(FN, T, W)                                                        \
  (a.D <= 32   ? TRACE_ATTN_NW(FN, T, 32, W)                                           \
   : a.D <= 64 ? TRACE_ATTN_NW(FN, T, 64, W)                                           \
               : TRACE_ATTN_NW(FN, T, 128, W))

}  // namespace

template <typename T>
int attn_run(AttnPass pass, const AttnArgs& a, hipStream_t st) {
  switch (pass) {
    case AttnPass::forward: return TRACE_ATTN_DP(fwd, T, a.waves_q);
    case AttnPass::few: return a.D <= 32 ? few<T, 32>(a, st) : a.D <= 64 ? few<T, 64>(a, st) : few<T, 128>(a, st);
    case AttnPass::short_backward:
      return a.D <= 32 ? short_blocks<T, 32>(a, st) : a.D <= 64 ? short_blocks<T, 64>(a, st) : short_blocks<T, 128>(a, st);
    case AttnPass::dq: return TRACE_ATTN_DP(dq, T, a.waves_q);
    default: return TRACE_ATTN_DP(dkv, T, a.waves_k);
  }
}

}  // namespace trace
