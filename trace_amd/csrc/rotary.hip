// trace_rotary: rotary positions of queries and keys (gfx950).
//   pair (a, b) of a head at position t, pair index p:  scale (a cos w - b sin w, b cos w + a sin w),  w = t freqs[p]
// The angle is formed in turns in 64 bits and reduced to half a turn before it meets 32 bits: at position 10^6 the fp32
// product t freqs[0] would already be off by 0.03 rad.  A workgroup computes the sines of a few tokens once, into LDS, and
// applies them to all of their heads, queries and keys, in one launch: HBM-bound (each element read and written once).
// 2 x 8192 tokens, 32 + 8 heads of 128, bf16: 66 us, 5.1 TB/s; 532480 tokens, 4 + 4 heads of 64, fp32: 421 us, 5.2 TB/s.
#include "layer_types.h"

#include <algorithm>
#include <cmath>

namespace trace {
namespace {

struct RotaryArgs {
  const void *q, *k;
  void *oq, *ok;
  long qb, qt, qh, kb, kt, kh;            // strides of q, k (batch, token, head)
  long oqb, oqt, oqh, okb, okt, okh;      // of the results
  const void* positions;
  int wide;                               // positions are 64-bit
  long pos_batch;                         // stride of a batch in positions; 0: shared
  const double* freqs;
  int L, Hq, H, D, half;                  // H = Hq + Hk heads, half = rotated pairs
  long tokens;                            // B L
  int per_wg;                             // tokens of a workgroup
  float scale, sin_sign;
};

// One item = V pairs of one head, or V unrotated elements behind them.  INTER: pair p is elements 2p, 2p + 1; else
// p, p + half.
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  typedef T Vec __attribute__((ext_vector_type(V)));
  extern __shared__ float2 turn[];        // [per_wg][half]
  const long token0 = (long)blockIdx.x * a.per_wg;
  const int n = (int)min((long)a.per_wg, a.tokens - token0);
  for (int i = threadIdx.x; i < n * a.half; i += 256) {
    const int t = i / a.half, p = i - t * a.half;
    const long token = token0 + t;
    const long b = token / a.L, at = b * a.pos_batch + (token - b * a.L);
    const double pos = a.wide ? (double)static_cast<const long*>(a.positions)[at]
                              : (double)static_cast<const int*>(a.positions)[at];
    const double w = pos * a.freqs[p] * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(w - rint(w)), &s, &c);
    turn[i] = make_float2(c * a.scale, s * a.scale * a.sin_sign);
  }
  __syncthreads();
  const int pairs = a.half / V, tail = (a.D - 2 * a.half) / V;
  const int per_head = pairs + tail, per_token = per_head * a.H;
  for (int i = threadIdx.x; i < n * per_token; i += 256) {
    const int t = i / per_token, r = i - t * per_token;
    const int head = r / per_head, c = r - head * per_head;
    const long token = token0 + t, b = token / a.L, l = token - b * a.L;
    const T* x;
    T* o;
    if (head < a.Hq) {
      x = (const T*)a.q + b * a.qb + l * a.qt + head * a.qh;
      o = (T*)a.oq + b * a.oqb + l * a.oqt + head * a.oqh;
    } else {
      x = (const T*)a.k + b * a.kb + l * a.kt + (head - a.Hq) * a.kh;
      o = (T*)a.ok + b * a.okb + l * a.okt + (head - a.Hq) * a.okh;
    }
    if (c >= pairs) {
      const int d = 2 * a.half + (c - pairs) * V;
      *reinterpret_cast<Vec*>(o + d) = *reinterpret_cast<const Vec*>(x + d);
      continue;
    }
    const float2* w = turn + t * a.half + c * V;
    const int d0 = INTER ? 2 * c * V : c * V, d1 = INTER ? d0 + V : a.half + d0;
    const Vec u = *reinterpret_cast<const Vec*>(x + d0), v = *reinterpret_cast<const Vec*>(x + d1);
    Vec ru, rv;
    auto pair = [&](T xa, T xb, int p, T& ra, T& rb) {
      const float2 cs = w[p];
      const float fa = (float)xa, fb = (float)xb;
      ra = (T)(fa * cs.x - fb * cs.y);
      rb = (T)(fb * cs.x + fa * cs.y);
    };
#pragma unroll
    for (int p = 0; p < V; ++p) {
      T ra, rb;
      if (INTER) {
        const int e = 2 * p;               // element of the 2 V consecutive ones
        if (V == 1) {
          pair(u[0], v[0], p, ra, rb);
          ru[0] = ra;
          rv[0] = rb;
        } else if (e < V) {
          pair(u[e], u[(e + 1) % V], p, ra, rb);
          ru[e] = ra;
          ru[(e + 1) % V] = rb;
        } else {
          pair(v[e - V], v[(e - V + 1) % V], p, ra, rb);
          rv[e - V] = ra;
          rv[(e - V + 1) % V] = rb;
        }
      } else {
        pair(u[p], v[p], p, ra, rb);
        ru[p] = ra;
        rv[p] = rb;
      }
    }
    *reinterpret_cast<Vec*>(o + d0) = ru;
    *reinterpret_cast<Vec*>(o + d1) = rv;
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename T, int V>
int run_v(bool inter, const RotaryArgs& a, int grid, size_t lds, hipStream_t st) {
  if (inter)
    hipLaunchKernelGGL((rotary_kernel<T, V, true>), dim3(grid), dim3(256), lds, st, a);
  else
    hipLaunchKernelGGL((rotary_kernel<T, V, false>), dim3(grid), dim3(256), lds, st, a);
  return launch_status("rotary_kernel");
}

template <typename T>
int run(bool inter, bool vec, const RotaryArgs& a, int grid, size_t lds, hipStream_t st) {
  // 16-byte accesses where the pairs and the rest of a head divide, half of that (16-bit types) or single elements else
  constexpr int W = 16 / (int)sizeof(T);
  if (vec && a.half % W == 0 && a.D % W == 0) return run_v<T, W>(inter, a, grid, lds, st);
  if (W == 8 && vec && a.half % 4 == 0 && a.D % 4 == 0) return run_v<T, 4>(inter, a, grid, lds, st);
  return run_v<T, 1>(inter, a, grid, lds, st);
}

}  // namespace
}  // namespace trace

using namespace trace;

extern "C" int trace_rotary(const trace_rotary_desc* d, const void* q, const void* k, const void* positions,
                            const double* freqs, void* out_q, void* out_k, void* stream) {
  TRACE_REQUIRE(d, "trace_rotary: null descriptor");
  TRACE_REQUIRE(d->dtype >= TRACE_F32 && d->dtype <= TRACE_F16, "trace_rotary: unknown dtype %d", d->dtype);
  TRACE_REQUIRE(d->B >= 0 && d->L >= 0 && d->Hq >= 0 && d->Hk >= 0, "trace_rotary: bad sizes");
  TRACE_REQUIRE(d->D >= 1 && d->D <= 1024 && d->rot >= 2 && d->rot % 2 == 0 && d->rot <= d->D,
                "trace_rotary: %d rotated of %d head elements (an even number, at most 1024)", d->rot, d->D);
  TRACE_REQUIRE((int64_t)d->Hq + d->Hk <= 65536, "trace_rotary: more than 65536 heads");
  TRACE_REQUIRE(std::isfinite(d->scale), "trace_rotary: scale is not finite");
  if (d->B == 0 || d->L == 0 || d->Hq + d->Hk == 0) return TRACE_OK;
  TRACE_REQUIRE(positions && freqs && (d->Hq == 0 || (q && out_q)) && (d->Hk == 0 || (k && out_k)),
                "trace_rotary: null argument");
  const int es = d->dtype == TRACE_F32 ? 4 : 2;
  bool vec = true;
  for (const trace_heads* h : {&d->q, &d->out_q, &d->k, &d->out_k}) {
    if (d->Hk == 0 && (h == &d->k || h == &d->out_k)) continue;
    if (d->Hq == 0 && (h == &d->q || h == &d->out_q)) continue;
    vec = vec && h->batch * es % 16 == 0 && h->token * es % 16 == 0 && h->head * es % 16 == 0;
  }
  vec = vec && aligned16(q) && aligned16(k) && aligned16(out_q) && aligned16(out_k);
  RotaryArgs a{};
  a.q = q; a.k = k; a.oq = out_q; a.ok = out_k;
  a.qb = d->q.batch; a.qt = d->q.token; a.qh = d->q.head;
  a.kb = d->k.batch; a.kt = d->k.token; a.kh = d->k.head;
  a.oqb = d->out_q.batch; a.oqt = d->out_q.token; a.oqh = d->out_q.head;
  a.okb = d->out_k.batch; a.okt = d->out_k.token; a.okh = d->out_k.head;
  a.positions = positions; a.wide = d->wide_positions; a.pos_batch = d->position_batch_stride;
  a.freqs = freqs;
  a.L = d->L; a.Hq = d->Hq; a.H = d->Hq + d->Hk; a.D = d->D; a.half = d->rot / 2;
  a.tokens = (long)d->B * d->L;
  a.scale = d->scale;
  a.sin_sign = d->inverse ? -1.f : 1.f;
  // a sine for each lane, or one token; and no more elements than a workgroup's 32-bit index counts, 256 lanes further included
  const int64_t most = (1 << 30) / ((int64_t)a.H * d->D);         // 16 or more
  a.per_wg = a.half >= 256 ? 1 : (int)std::min<int64_t>(256 / a.half, most);
  const long grid = (a.tokens + a.per_wg - 1) / a.per_wg;
  TRACE_REQUIRE(grid * 256 <= MAX_GRID_THREADS, "trace_rotary: grid of %ld workgroups", grid);
  const size_t lds = (size_t)a.per_wg * a.half * sizeof(float2);
  const bool inter = d->interleaved != 0;
  hipStream_t st = (hipStream_t)stream;
  if (d->dtype == TRACE_F32) return run<float>(inter, vec, a, (int)grid, lds, st);
  if (d->dtype == TRACE_BF16) return run<__bf16>(inter, vec, a, (int)grid, lds, st);
  return run<_Float16>(inter, vec, a, (int)grid, lds, st);
}
