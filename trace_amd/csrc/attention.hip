// trace_attention / trace_attention_backward: argument checks, choice of the kernel instance, launches.
#include "attn_kernels.h"

#include <cmath>

namespace trace {
namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Check {
  const trace_attention_desc& d;
  int es;
  bool vec;
  // takes a tensor's strides over and notes whether 16-byte accesses reach all of it
  AttnView view(const trace_heads& h, const void* p) {
    vec = vec && aligned16(p) && h.batch * es % 16 == 0 && h.token * es % 16 == 0 && h.head * es % 16 == 0;
    return AttnView{(long)h.batch, (long)h.token, (long)h.head};
  }
};

int check_desc(const trace_attention_desc* d, const char* who) {
  TRACE_REQUIRE(d, "%s: null descriptor", who);
  TRACE_REQUIRE(d->dtype == TRACE_F32 || d->dtype == TRACE_BF16 || d->dtype == TRACE_F16, "%s: unknown dtype %d", who,
                d->dtype);
  TRACE_REQUIRE(d->B >= 0 && d->Lq >= 0 && d->Lk >= 0 && d->Hq >= 1 && d->Hk >= 1 && d->Hq % d->Hk == 0,
                "%s: bad sizes B %d, Lq %d, Lk %d, Hq %d, Hk %d (Hq must be a multiple of Hk)", who, d->B, d->Lq, d->Lk,
                d->Hq, d->Hk);
  TRACE_REQUIRE(d->D >= 1 && d->D <= 128, "%s: head dimension %d unsupported (1..128)", who, d->D);
  TRACE_REQUIRE(std::isfinite(d->scale) && d->scale > 0.f, "%s: scale %g must be positive and finite", who,
                (double)d->scale);
  // token indexes stay below this in the kernels' 32-bit arithmetic, tile overhang included
  TRACE_REQUIRE(d->Lq <= (1 << 30) && d->Lk <= (1 << 30), "%s: more than 2^30 tokens", who);
  return TRACE_OK;
}

AttnArgs common_args(const trace_attention_desc& d) {
  AttnArgs a{};
  a.B = d.B; a.Lq = d.Lq; a.Lk = d.Lk; a.Hq = d.Hq; a.Hk = d.Hk; a.G = d.Hq / d.Hk; a.D = d.D;
  a.scale = d.scale;
  a.scale_log2 = d.scale * LOG2E;
  a.causal = d.causal;
  a.query_start = d.query_start;
  a.key_lengths = d.key_lengths;
  a.key_mask = d.key_mask;
  a.mask_stride = (long)d.key_mask_stride;
  return a;
}

template <typename K>
int launch(K kernel, unsigned long long* attr, size_t lds, int threads, const AttnArgs& a, hipStream_t st, const char* what) {
  const long grid = xcd_grid(a.items);
  TRACE_REQUIRE(grid < 0x7fffffffL, "%s: grid of %ld workgroups", what, grid);
  if (lds > 64 * 1024) TRACE_CHECK_HIP(ensure_dynamic_lds(attr, reinterpret_cast<const void*>(kernel), (int)lds));
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(threads), lds, st, a);
  return launch_status(what);
}

// Waves of a workgroup: as many as the 32-row tiles that one (batch, head) has, up to four -- a sequence of 52 steps
// keeps two busy.
int waves_for(int rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }

template <typename T, int DP, int NW>
int fwd(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)((a.Lq + 32 * NW - 1) / (32 * NW)) * a.Hq * a.B;
  const size_t lds = sizeof(T) * (64 * TileR<T, DP>::S + DP * TileX<T, 64>::S);
  return launch(&attn_fwd_kernel<T, DP, NW>, &attr, lds, NW * 64, a, st, "attn_fwd_kernel");
}

template <typename T, int DP, int NW>
int dq(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)((a.Lq + 32 * NW - 1) / (32 * NW)) * a.Hq * a.B;
  const size_t lds = sizeof(T) * (2 * 64 * TileR<T, DP>::S + DP * TileX<T, 64>::S);
  return launch(&attn_dq_kernel<T, DP, NW>, &attr, lds, NW * 64, a, st, "attn_dq_kernel");
}

template <typename T, int DP, int NW>
int dkv(AttnArgs a, hipStream_t st) {
  static unsigned long long attr = 0;
  a.items = (long)((a.Lk + 32 * NW - 1) / (32 * NW)) * a.Hk * a.B;
  const size_t lds = sizeof(T) * 2 * (32 * TileR<T, DP>::S + DP * TileX<T, 32>::S) + 2 * 32 * sizeof(float);
  return launch(&attn_dkv_kernel<T, DP, NW>, &attr, lds, NW * 64, a, st, "attn_dkv_kernel");
}

#define TRACE_ATTN_NW(FN, T, DP, W) (W == 1 ? FN<T, DP, 1>(a, st) : W == 2 ? FN<T, DP, 2>(a, st) : FN<T, DP, 4>(a, st))
#define TRACE_ATTN_PICK(NAME, FN, LEN)                                                                     \
  template <typename T>                                                                                    \
  int NAME##_t(const AttnArgs& a, hipStream_t st) {                                                        \
    const int w = waves_for(LEN);                                                                          \
    return a.D <= 32 ? TRACE_ATTN_NW(FN, T, 32, w) : a.D <= 64 ? TRACE_ATTN_NW(FN, T, 64, w) : TRACE_ATTN_NW(FN, T, 128, w); \
  }                                                                                                        \
  int NAME(int dtype, const AttnArgs& a, hipStream_t st) {                                                 \
    return dtype == TRACE_F32 ? NAME##_t<float>(a, st) : dtype == TRACE_BF16 ? NAME##_t<__bf16>(a, st)     \
                                                                             : NAME##_t<_Float16>(a, st);  \
  }
TRACE_ATTN_PICK(run_fwd, fwd, a.Lq)
TRACE_ATTN_PICK(run_dq, dq, a.Lq)
TRACE_ATTN_PICK(run_dkv, dkv, a.Lk)

}  // namespace
}  // namespace trace

using namespace trace;

extern "C" int64_t trace_attention_workspace_bytes(const trace_attention_desc* d, int backward) {
  const int rc = check_desc(d, "trace_attention_workspace_bytes");
  if (rc != TRACE_OK) return rc;
  return backward ? (int64_t)d->B * d->Hq * d->Lq * (int64_t)sizeof(float) : 0;
}

extern "C" int trace_attention(const trace_attention_desc* d, const void* q, const void* k, const void* v, void* out,
                               float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_desc(d, "trace_attention");
  if (rc != TRACE_OK) return rc;
  if (d->B == 0 || d->Lq == 0) return TRACE_OK;
  TRACE_REQUIRE(q && out && lse && (d->Lk == 0 || (k && v)), "trace_attention: null argument");
  (void)workspace;
  (void)workspace_bytes;
  AttnArgs a = common_args(*d);
  Check c{*d, d->dtype == TRACE_F32 ? 4 : 2, d->D % 8 == 0};
  a.q = q; a.vq = c.view(d->q, q);
  a.k = k; a.vk = c.view(d->k, k);
  a.v = v; a.vv = c.view(d->v, v);
  a.out = out; a.vo = c.view(d->out, out);
  a.lse = lse;
  a.vec = c.vec;
  return run_fwd(d->dtype, a, (hipStream_t)stream);
}

extern "C" int trace_attention_backward(const trace_attention_desc* d, const void* dout, const void* q, const void* k,
                                        const void* v, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_desc(d, "trace_attention_backward");
  if (rc != TRACE_OK) return rc;
  if (d->B == 0) return TRACE_OK;
  TRACE_REQUIRE((d->Lq == 0 || (dout && q && out && lse && dq)) && (d->Lk == 0 || (k && v && dk && dv)),
                "trace_attention_backward: null argument");
  const int64_t need = trace_attention_workspace_bytes(d, 1);
  if (need > 0 && (!workspace || workspace_bytes < need)) {
    set_error("trace_attention_backward: workspace too small (%lld bytes, need %lld)", (long long)workspace_bytes,
              (long long)need);
    return TRACE_ENOMEM;
  }
  AttnArgs a = common_args(*d);
  Check c{*d, d->dtype == TRACE_F32 ? 4 : 2, d->D % 8 == 0};
  a.q = q; a.vq = c.view(d->q, q);
  a.k = k; a.vk = c.view(d->k, k);
  a.v = v; a.vv = c.view(d->v, v);
  a.out_in = out; a.vo = c.view(d->out, out);
  a.dout = dout; a.vdo = c.view(d->dout, dout);
  a.dq = dq; a.vdq = c.view(d->dq, dq);
  a.dk = dk; a.vdk = c.view(d->dk, dk);
  a.dv = dv; a.vdv = c.view(d->dv, dv);
  a.lse_in = lse;
  a.delta = static_cast<float*>(workspace);
  a.vec = c.vec;
  if (d->Lq > 0) {
    const int r = run_dq(d->dtype, a, (hipStream_t)stream);
    if (r != TRACE_OK) return r;
  }
  return d->Lk > 0 ? run_dkv(d->dtype, a, (hipStream_t)stream) : TRACE_OK;
}
