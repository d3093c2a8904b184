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

int check_back(const trace_attention_desc* d, const char* who) {
  const int rc = check_desc(d, who);
  if (rc != TRACE_OK) return rc;
  // attn_dkv_kernel counts the query tiles of the heads that share a key head in 32 bits
  TRACE_REQUIRE(((int64_t)d->Lq + 31) / 32 * (d->Hq / d->Hk) < (1ll << 31), "%s: more than 2^31 tiles of 32 queries to a key head", who);
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

// Waves of a workgroup over `rows` tokens: as many as there are 32-row tiles, up to four.
int waves_for(int rows) { return rows <= 32 ? 1 : rows <= 64 ? 2 : 4; }
int64_t items_of(int rows, int64_t heads) { return (rows + 32 * waves_for(rows) - 1) / (32 * waves_for(rows)) * heads; }

int padded_dim(int D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// Into how many shares the loop of a kernel with `items` workgroups is cut for `target` of them: at most 16, and `most`.
int shares(int64_t items, int64_t most, int target) {
  int64_t n = items > 0 ? (target + items - 1) / items : 1;
  n = n < most ? n : most;
  return (int)(n < 1 ? 1 : n < 16 ? n : 16);
}

// The forward pass.  Up to 16 queries the heads of a group share a tile (attn_few_kernel), with one wave a SIMD, which is what the
// registers of that kernel leave room for (1024 and 2048 waves measured alike, 1536 and 4096 a fifth slower: a second, partly filled
// round), in ranges of at least 64 keys.  Otherwise two workgroups a CU, in ranges of at least two tiles.
struct ForwardPlan {
  bool few;
  int splits;
  int64_t ml_bytes, bytes;           // of workspace
};
ForwardPlan forward_plan(const trace_attention_desc& d) {
  ForwardPlan p{};
  p.few = d.Lq <= 16;
  if (p.few) {
    const int64_t waves = ((int64_t)d.Lq * (d.Hq / d.Hk) + 31) / 32 * d.B * d.Hk;
    const int64_t n = waves > 0 ? (1024 + waves - 1) / waves : 1, most = (d.Lk + 63) / 64;
    p.splits = (int)(n < most ? n : most);
    p.splits = p.splits < 1 ? 1 : p.splits < ATTN_MAX_SPLITS ? p.splits : ATTN_MAX_SPLITS;
  } else {
    p.splits = shares(items_of(d.Lq, (int64_t)d.B * d.Hq), (d.Lk + 63) / 64 / 2, 512);
  }
  if (p.splits > 1) {
    const int64_t partial = (int64_t)d.B * d.Hq * d.Lq * p.splits;
    p.ml_bytes = (partial * 2 * (int64_t)sizeof(float) + 15) / 16 * 16;
    p.bytes = p.ml_bytes + partial * padded_dim(d.D) * (int64_t)sizeof(float);
  }
  return p;
}

// The backward pass: one kernel for short sequences, else the shares of its two kernels: four workgroups a CU, of at least two key
// tiles (dq) or four query tiles (dk / dv) each.
struct BackPlan {
  bool whole;                        // short sequences: no workspace
  int splits_q, splits;
  int64_t delta_bytes, q_bytes, bytes;
};
BackPlan back_plan(const trace_attention_desc& d) {
  BackPlan p{};
  p.whole = d.Lq >= 1 && d.Lk >= 1 && d.Lq <= 64 && d.Lk <= 64;
  if (p.whole) return p;
  const int64_t hq = (int64_t)d.B * d.Hq, hk = (int64_t)d.B * d.Hk, row = padded_dim(d.D) * (int64_t)sizeof(float);
  p.splits_q = shares(items_of(d.Lq, hq), (d.Lk + 63) / 64 / 2, 1024);
  p.splits = shares(items_of(d.Lk, hk), (int64_t)((d.Lq + 31) / 32) * (d.Hq / d.Hk) / 4, 1024);
  p.delta_bytes = (hq * d.Lq * (int64_t)sizeof(float) + 15) / 16 * 16;
  p.q_bytes = p.splits_q > 1 ? p.splits_q * hq * d.Lq * row : 0;
  p.bytes = p.delta_bytes + p.q_bytes + (p.splits > 1 ? p.splits * 2 * hk * d.Lk * row : 0);
  return p;
}

int by_type(int dtype, AttnPass pass, const AttnArgs& a, hipStream_t st) {
  return dtype == TRACE_F32    ? attn_run<float>(pass, a, st)
         : dtype == TRACE_BF16 ? attn_run<__bf16>(pass, a, st)
                               : attn_run<_Float16>(pass, a, st);
}

}  // namespace
}  // namespace trace

using namespace trace;

extern "C" int64_t trace_attention_workspace_bytes(const trace_attention_desc* d, int backward) {
  const int rc = backward ? check_back(d, "trace_attention_workspace_bytes") : check_desc(d, "trace_attention_workspace_bytes");
  if (rc != TRACE_OK) return rc;
  if (d->B == 0 || d->Lq == 0) return 0;
  return backward ? back_plan(*d).bytes : forward_plan(*d).bytes;
}

extern "C" int trace_attention(const trace_attention_desc* d, const void* q, const void* k, const void* v, void* out,
                               float* lse, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_desc(d, "trace_attention");
  if (rc != TRACE_OK) return rc;
  if (d->B == 0 || d->Lq == 0) return TRACE_OK;
  TRACE_REQUIRE(q && out && lse && (d->Lk == 0 || (k && v)), "trace_attention: null argument");
  const ForwardPlan plan = forward_plan(*d);
  if (plan.bytes > 0 && (!workspace || workspace_bytes < plan.bytes)) {
    set_error("trace_attention: workspace too small (%lld bytes, need %lld)", (long long)workspace_bytes,
              (long long)plan.bytes);
    return TRACE_ENOMEM;
  }
  TRACE_REQUIRE(plan.bytes == 0 || aligned16(workspace), "trace_attention: workspace must be 16-byte aligned");
  AttnArgs a = common_args(*d);
  Check c{*d, d->dtype == TRACE_F32 ? 4 : 2, d->D % 8 == 0};
  a.q = q; a.vq = c.view(d->q, q);
  a.k = k; a.vk = c.view(d->k, k);
  a.v = v; a.vv = c.view(d->v, v);
  a.out = out; a.vo = c.view(d->out, out);
  a.lse = lse;
  a.vec = c.vec;
  a.splits = plan.splits;
  a.part_ml = static_cast<float*>(workspace);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.ml_bytes);
  a.waves_q = waves_for(d->Lq);
  a.items = (int64_t)d->B * d->Hk * (((int64_t)d->Lq * a.G + 31) / 32) * plan.splits;        // of attn_few_kernel
  return by_type(d->dtype, plan.few ? AttnPass::few : AttnPass::forward, a, (hipStream_t)stream);
}

extern "C" int trace_attention_backward(const trace_attention_desc* d, const void* dout, const void* q, const void* k,
                                        const void* v, const void* out, const float* lse, void* dq, void* dk, void* dv,
                                        void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_back(d, "trace_attention_backward");
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
  TRACE_REQUIRE(need == 0 || aligned16(workspace), "trace_attention_backward: workspace must be 16-byte aligned");
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
  const BackPlan plan = back_plan(*d);
  a.delta = static_cast<float*>(workspace);
  a.waves_q = waves_for(d->Lq);
  a.waves_k = waves_for(d->Lk);
  a.splits_q = plan.splits_q;
  a.splits = plan.splits;
  a.part_q = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.delta_bytes);
  a.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.delta_bytes + plan.q_bytes);
  a.vec = c.vec;
  if (plan.whole) return by_type(d->dtype, AttnPass::short_backward, a, (hipStream_t)stream);
  if (d->Lq > 0) {
    const int r = by_type(d->dtype, AttnPass::dq, a, (hipStream_t)stream);
    if (r != TRACE_OK) return r;
  }
  return d->Lk > 0 ? by_type(d->dtype, AttnPass::dkv, a, (hipStream_t)stream) : TRACE_OK;
}
