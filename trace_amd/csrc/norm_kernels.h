// The norms before and after a block, fused with the block's gate and the residual connection (gfx950):
//   u = N(y) p  (or y),   h = alpha x + g u,   z = N(h) w + b      N: layer or root-mean-square norm of a row
// and the gradient, recomputed from x and y.  HBM-bound: the forward reads x, y and writes h, z once, the backward
// reads x, y, dh, dz and writes dx, dy once; a row stays in the registers of its team of TPR lanes in between, as
// fp32.  Moments are exact two-pass ones (mean first, then the squares about it).  8192 x 4096 bf16, forward: 47 us with part of
// the inputs in the last-level cache, 60 without (4.5 TB/s); 532480 x 256 fp32, backward: 763 us (4.3 TB/s over six streams).
#pragma once
#include "layer_types.h"

namespace trace {

struct NormArgs {
  const void *x, *y, *dh, *dz;
  void *h, *z, *dx, *dy;
  const float *gate, *post, *weight, *bias;
  long xs, ys, dhs, dzs;             // row strides of the inputs; outputs are contiguous
  int R, C, rpc;                     // rows, columns, rows of a conditioning group
  long row0;                         // forward: first row of the launch
  int layer;                         // 1: layer norm, 0: rms
  int cond, gate_cond;               // weight and bias / gate: one row per conditioning group (1) or one for all (0)
  float alpha, eps;
  // backward
  float *dgate, *dweight, *dbias, *dpost;
  float *part_g, *part_s;            // per-chunk and per-workgroup partial column sums
  int nsub, rows_sub;                // chunks of a group, rows of a chunk
  int chunks, per_team;              // all chunks, chunks of a team
};

// The columns of a lane: K vectors of V elements, vector k at column (k TPR + lane) V.
template <typename T, int V>
__device__ __forceinline__ void row_load(float (&o)[V], const T* p, bool ok) {
  typedef T Vec __attribute__((ext_vector_type(V)));
  if (!ok) {
#pragma unroll
    for (int e = 0; e < V; ++e) o[e] = 0.f;
    return;
  }
  const Vec v = *reinterpret_cast<const Vec*>(p);
#pragma unroll
  for (int e = 0; e < V; ++e) o[e] = (float)v[e];
}
template <typename T, int V>
__device__ __forceinline__ void row_store(T* p, const float (&o)[V]) {
  typedef T Vec __attribute__((ext_vector_type(V)));
  Vec v;
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = (T)o[e];
  *reinterpret_cast<Vec*>(p) = v;
}

// Sum over the TPR lanes of a row's team; every lane gets it.  red: TPR / 64 floats of LDS, used alternately (two calls in
// a row take different halves, so one barrier a call is enough).
template <int TPR>
__device__ __forceinline__ float team_sum(float v, float* red, int& turn) {
  v = wave_sum(v);
  if (TPR == 64) return v;
  constexpr int W = TPR / 64;
  float* r = red + (turn & 1) * W;
  ++turn;
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = 0.f;
#pragma unroll
  for (int w = 0; w < W; ++w) t += r[w];
  return t;
}

// The team's number in the workgroup, in a scalar register: a row's addresses are then a uniform base and a lane's offset.
template <int TPR>
__device__ __forceinline__ int team_of() {
  return TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
}

template <int TPR, int V, int K>
struct RowStats {
  float mean, rstd;
  __device__ __forceinline__ void of(const float (&a)[K][V], int C, int lane, int layer, float eps, float* red, int& turn) {
    mean = 0.f;
    if (layer) {
      float s = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < V; ++e) s += a[k][e];            // columns beyond C hold zero
      mean = team_sum<TPR>(s, red, turn) / (float)C;
    }
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if ((k * TPR + lane) * V >= C) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = a[k][e] - mean;
        q = fmaf(d, d, q);
      }
    }
    rstd = 1.f / sqrtf(team_sum<TPR>(q, red, turn) / (float)C + eps);
  }
};

template <typename TX, typename TY, int TPR, int V, int K>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void residual_norm_kernel(NormArgs a) {
  constexpr int NT = TPR < 256 ? 256 : TPR;
  __shared__ float red[2 * (NT / 64)];
  const int lane = threadIdx.x % TPR;
  const long row = a.row0 + (long)blockIdx.x * (NT / TPR) + team_of<TPR>();
  if (row >= a.R) return;                                     // TPR > 64: a workgroup is one team
  int turn = 0;
  const int g = (int)(row / a.rpc);
  const long gtab = a.gate_cond ? (long)g * a.C : 0;
  float h[K][V], t[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * TPR + lane) * V;
    row_load<TX, V>(h[k], (const TX*)a.x + row * a.xs + c, c < a.C);
  }
  if (a.y) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * TPR + lane) * V;
      row_load<TY, V>(t[k], (const TY*)a.y + row * a.ys + c, c < a.C);
    }
    if (a.post) {
      RowStats<TPR, V, K> st;
      st.of(t, a.C, lane, a.layer, a.eps, red, turn);
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + lane) * V;
        float p[V];
        row_load<float, V>(p, a.post + c, c < a.C);
#pragma unroll
        for (int e = 0; e < V; ++e) t[k][e] = (t[k][e] - st.mean) * st.rstd * p[e];
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * TPR + lane) * V;
      float w[V];
      if (a.gate) row_load<float, V>(w, a.gate + gtab + c, c < a.C);
#pragma unroll
      for (int e = 0; e < V; ++e) h[k][e] = fmaf(a.alpha, h[k][e], a.gate ? w[e] * t[k][e] : t[k][e]);
      if (a.h && c < a.C) row_store<TX, V>((TX*)a.h + row * a.C + c, h[k]);
    }
  }
  if (!a.z) return;
  RowStats<TPR, V, K> st;
  st.of(h, a.C, lane, a.layer, a.eps, red, turn);
  const long tab = a.cond ? (long)g * a.C : 0;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * TPR + lane) * V;
    if (c >= a.C) continue;
    float w[V], b[V], z[V];
    if (a.weight) row_load<float, V>(w, a.weight + tab + c, true);
    if (a.bias) row_load<float, V>(b, a.bias + tab + c, true);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      z[e] = (h[k][e] - st.mean) * st.rstd;
      if (a.weight) z[e] *= w[e];
      if (a.bias) z[e] += b[e];
    }
    row_store<TY, V>((TY*)a.z + row * a.C + c, z);
  }
}

// Backward.  A team owns a run of chunks (a chunk: consecutive rows of one conditioning group) and its lanes own columns, so the
// column sums of gate, weight, bias and post weight stay in registers: sums of a group are flushed when its chunk ends,
// shared ones once at the end, added up over the workgroup's teams in order.  norm_reduce_kernel adds the partial rows in a
// fixed order: no atomics.
template <typename TX, typename TY, int TPR, int V, int K>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void residual_norm_backward_kernel(NormArgs a) {
  constexpr int NT = TPR < 256 ? 256 : TPR, TEAMS = NT / TPR;
  __shared__ float red[2 * (NT / 64)];
  __shared__ float comb[TEAMS > 1 ? (TEAMS - 1) * TPR * V * K : 1];
  const int lane = threadIdx.x % TPR;
  const int team = blockIdx.x * TEAMS + team_of<TPR>();
  int turn = 0;
  float sg[K][V] = {}, sw[K][V] = {}, sb[K][V] = {}, sp[K][V] = {};
  const long first = (long)team * a.per_team;
  const int last = (int)min((long)a.chunks, first + a.per_team);
  for (int chunk = (int)min(first, (long)a.chunks); chunk < last; ++chunk) {
    const int g = chunk / a.nsub, sub = chunk % a.nsub;
    const long base = (long)g * a.rpc;
    const int r0 = sub * a.rows_sub;
    const int r1 = (int)min(min((long)r0 + a.rows_sub, (long)a.rpc), a.R - base);
    const long tab = a.cond ? (long)g * a.C : 0, gtab = a.gate_cond ? (long)g * a.C : 0;
    for (int r = r0; r < r1; ++r) {
      const long row = base + r;
      float x[K][V], y[K][V], d[K][V];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + lane) * V;
        row_load<TX, V>(x[k], (const TX*)a.x + row * a.xs + c, c < a.C);
        if (a.y) row_load<TY, V>(y[k], (const TY*)a.y + row * a.ys + c, c < a.C);
        if (a.dz) row_load<TY, V>(d[k], (const TY*)a.dz + row * a.dzs + c, c < a.C);
      }
      // y becomes N(y), x becomes h
      RowStats<TPR, V, K> sy, sh;
      if (a.y) {
        if (a.post) sy.of(y, a.C, lane, a.layer, a.eps, red, turn);
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (k * TPR + lane) * V;
          float w[V], p[V];
          if (a.gate) row_load<float, V>(w, a.gate + gtab + c, c < a.C);
          if (a.post) row_load<float, V>(p, a.post + c, c < a.C);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (a.post) y[k][e] = (y[k][e] - sy.mean) * sy.rstd;
            const float u = a.post ? y[k][e] * p[e] : y[k][e];
            x[k][e] = fmaf(a.alpha, x[k][e], a.gate ? w[e] * u : u);
          }
        }
      }
      if (a.dz) {
        sh.of(x, a.C, lane, a.layer, a.eps, red, turn);
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
          const int c = (k * TPR + lane) * V;
          if (c >= a.C) continue;
          float w[V];
          if (a.weight) row_load<float, V>(w, a.weight + tab + c, true);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float n = (x[k][e] - sh.mean) * sh.rstd;
            sw[k][e] = fmaf(d[k][e], n, sw[k][e]);
            sb[k][e] += d[k][e];
            if (a.weight) d[k][e] *= w[e];
            s1 += d[k][e];
            s2 = fmaf(d[k][e], n, s2);
            x[k][e] = n;
          }
        }
        s1 = a.layer ? team_sum<TPR>(s1, red, turn) / (float)a.C : 0.f;
        s2 = team_sum<TPR>(s2, red, turn) / (float)a.C;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) d[k][e] = sh.rstd * (d[k][e] - s1 - x[k][e] * s2);
      }
      float s1 = 0.f, s2 = 0.f;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + lane) * V;
        if (c >= a.C) continue;
        float w[V], p[V], o[V];
        if (a.dh) {
          row_load<TX, V>(o, (const TX*)a.dh + row * a.dhs + c, true);
#pragma unroll
          for (int e = 0; e < V; ++e) d[k][e] = a.dz ? d[k][e] + o[e] : o[e];
        }
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = a.y ? a.alpha * d[k][e] : d[k][e];
        row_store<TX, V>((TX*)a.dx + row * a.C + c, o);
        if (!a.y) continue;
        if (a.gate) row_load<float, V>(w, a.gate + gtab + c, true);
        if (a.post) row_load<float, V>(p, a.post + c, true);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float u = a.post ? y[k][e] * p[e] : y[k][e];
          sg[k][e] = fmaf(d[k][e], u, sg[k][e]);
          if (a.gate) d[k][e] *= w[e];
          if (a.post) {
            sp[k][e] = fmaf(d[k][e], y[k][e], sp[k][e]);
            d[k][e] *= p[e];
            s1 += d[k][e];
            s2 = fmaf(d[k][e], y[k][e], s2);
          }
        }
      }
      if (!a.y) continue;
      if (a.post) {
        s1 = a.layer ? team_sum<TPR>(s1, red, turn) / (float)a.C : 0.f;
        s2 = team_sum<TPR>(s2, red, turn) / (float)a.C;
      }
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + lane) * V;
        if (c >= a.C) continue;
        if (a.post) {
#pragma unroll
          for (int e = 0; e < V; ++e) d[k][e] = sy.rstd * (d[k][e] - s1 - y[k][e] * s2);
        }
        row_store<TY, V>((TY*)a.dy + row * a.C + c, d[k]);
      }
    }
    // sums of the group: straight to the gradient where the chunk is the whole group, else to the chunk's partial rows
    auto flush = [&](float (&s)[K][V], float* to, int slot) {
      if (!to) return;
      float* p = a.nsub == 1 ? to + (long)g * a.C : a.part_g + ((long)slot * a.chunks + chunk) * a.C;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * TPR + lane) * V;
        if (c < a.C) row_store<float, V>(p + c, s[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) s[k][e] = 0.f;
      }
    };
    if (a.gate_cond) flush(sg, a.dgate, 0);
    if (a.cond) {
      flush(sw, a.dweight, 1);
      flush(sb, a.dbias, 2);
    }
  }
  auto total = [&](float (&s)[K][V], float* to, int slot) {
    if (!to) return;
    if (TEAMS > 1) {
      const int t = threadIdx.x / TPR;
      __syncthreads();
      if (t > 0) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) comb[((t - 1) * V * K + k * V + e) * TPR + lane] = s[k][e];
      }
      __syncthreads();
      if (t > 0) return;
#pragma unroll
      for (int w = 0; w + 1 < TEAMS; ++w)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < V; ++e) s[k][e] += comb[(w * V * K + k * V + e) * TPR + lane];
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * TPR + lane) * V;
      if (c < a.C) row_store<float, V>(a.part_s + ((long)slot * gridDim.x + blockIdx.x) * a.C + c, s[k]);
    }
  };
  total(sp, a.dpost, 3);
  if (!a.gate_cond) total(sg, a.dgate, 0);
  if (!a.cond) {
    total(sw, a.dweight, 1);
    total(sb, a.dbias, 2);
  }
}

// out[i][g][c] = sum of rows g n .. g n + n - 1 of part[i], in a fixed order: 16 row lanes, then their sums in order.  All of a
// call's sums of one kind in one launch.
struct NormReduceArgs {
  const float* part[4];
  float* out[4];
  int count, groups, n, C;
};
__global__ __launch_bounds__(1024) void norm_reduce_kernel(NormReduceArgs a) {
  __shared__ float s[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int blocks = (a.C + 63) / 64;
  const int at = blockIdx.x / blocks, i = at / a.groups;
  const long g = at % a.groups;
  const int c = (int)(blockIdx.x % blocks) * 64 + lane;
  const float* p = a.part[i] + g * a.n * a.C + c;
  float t = 0.f;
  if (c < a.C) {
#pragma unroll 8
    for (int r = w; r < a.n; r += 16) t += p[(long)r * a.C];
  }
  s[w][lane] = t;
  __syncthreads();
  if (w == 0 && c < a.C) {
#pragma unroll
    for (int k = 1; k < 16; ++k) t += s[k][lane];
    a.out[i][g * a.C + c] = t;
  }
}

}  // namespace trace
