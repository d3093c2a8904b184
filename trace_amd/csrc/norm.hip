// trace_residual_norm / trace_residual_norm_backward: argument checks, choice of the kernel instance, launches.
#include "norm_kernels.h"

#include <algorithm>
#include <cmath>

namespace trace {
namespace {

struct NormPlan {
  int tpr, v, k;          // lanes of a row, vector width, vectors of a lane
  int teams_wg;           // teams of a workgroup
};

// The narrowest team that holds a row in 16 elements a lane: a wave up to 1024 columns (no barrier in its sums), 256 lanes
// up to 4096, 1024 lanes up to 16384.  Vectors are 16 bytes where C and all addresses allow (8 of a 16-bit type beside an fp32
// stream), single elements else, as many as the row needs (20448 x 1637 fp32, backward: 501 us, 946 with 16 for every row).
bool plan_for(int C, int es_x, int es_y, bool vec, NormPlan* p) {
  const int wide = es_x == 2 && es_y == 2 ? 8 : 4;
  p->v = vec && C % wide == 0 ? wide : 1;
  p->tpr = C <= 1024 ? 64 : C <= 4096 ? 256 : 1024;
  p->teams_wg = p->tpr == 64 ? 4 : 1;
  if (p->v == 1) {
    p->k = p->tpr > 64 ? (C <= 8 * p->tpr ? 8 : 16) : C <= 64 ? 1 : C <= 256 ? 4 : 16;
  } else {
    p->k = 1;
    while (p->tpr * p->v * p->k < C) p->k *= 2;
  }
  return C <= 16384;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename TX, typename TY, int TPR, int V, int K>
int run(bool back, const NormArgs& a, int grid, hipStream_t st) {
  constexpr int NT = TPR < 256 ? 256 : TPR;
  if (back)
    hipLaunchKernelGGL((residual_norm_backward_kernel<TX, TY, TPR, V, K>), dim3(grid), dim3(NT), 0, st, a);
  else
    hipLaunchKernelGGL((residual_norm_kernel<TX, TY, TPR, V, K>), dim3(grid), dim3(NT), 0, st, a);
  return launch_status(back ? "residual_norm_backward_kernel" : "residual_norm_kernel");
}

template <typename TX, typename TY, int TPR>
int run_tpr(bool back, const NormPlan& p, const NormArgs& a, int grid, hipStream_t st) {
  constexpr int W = sizeof(TX) == 2 && sizeof(TY) == 2 ? 8 : 4, KM = 16 / W;
  if (p.v == 1) {
    if (p.k == 16) return run<TX, TY, TPR, 1, 16>(back, a, grid, st);
    if (TPR > 64) return run<TX, TY, TPR, 1, (TPR > 64 ? 8 : 16)>(back, a, grid, st);
    return p.k == 4 ? run<TX, TY, TPR, 1, (TPR > 64 ? 16 : 4)>(back, a, grid, st)
                    : run<TX, TY, TPR, 1, (TPR > 64 ? 16 : 1)>(back, a, grid, st);
  }
  if (p.k == KM) return run<TX, TY, TPR, W, KM>(back, a, grid, st);
  if (p.k == KM / 2) return run<TX, TY, TPR, W, KM / 2>(back, a, grid, st);
  return run<TX, TY, TPR, W, 1>(back, a, grid, st);
}

template <typename TX, typename TY>
int run_types(bool back, const NormPlan& p, const NormArgs& a, int grid, hipStream_t st) {
  if (p.tpr == 64) return run_tpr<TX, TY, 64>(back, p, a, grid, st);
  if (p.tpr == 256) return run_tpr<TX, TY, 256>(back, p, a, grid, st);
  return run_tpr<TX, TY, 1024>(back, p, a, grid, st);
}

int dispatch(bool back, const trace_norm_desc& d, const NormPlan& p, const NormArgs& a, int grid, hipStream_t st) {
  if (d.stream_dtype == TRACE_F32) {
    if (d.dtype == TRACE_F32) return run_types<float, float>(back, p, a, grid, st);
    if (d.dtype == TRACE_BF16) return run_types<float, __bf16>(back, p, a, grid, st);
    return run_types<float, _Float16>(back, p, a, grid, st);
  }
  if (d.dtype == TRACE_BF16) return run_types<__bf16, __bf16>(back, p, a, grid, st);
  return run_types<_Float16, _Float16>(back, p, a, grid, st);
}

int check_desc(const trace_norm_desc* d, const char* who) {
  TRACE_REQUIRE(d, "%s: null descriptor", who);
  TRACE_REQUIRE(d->dtype >= TRACE_F32 && d->dtype <= TRACE_F16 &&
                    (d->stream_dtype == TRACE_F32 || d->stream_dtype == d->dtype),
                "%s: dtype %d with a residual stream of dtype %d (the stream is fp32 or of the same type)", who, d->dtype,
                d->stream_dtype);
  TRACE_REQUIRE(d->rows >= 0 && d->C >= 1 && d->C <= 16384, "%s: %d rows of %d columns (1..16384 columns)", who, d->rows,
                d->C);
  TRACE_REQUIRE(d->rows_per_cond >= 1, "%s: rows_per_cond %d must be positive", who, d->rows_per_cond);
  TRACE_REQUIRE(d->kind == TRACE_NORM_RMS || d->kind == TRACE_NORM_LAYER, "%s: unknown norm %d", who, d->kind);
  TRACE_REQUIRE(std::isfinite(d->eps) && d->eps >= 0.f && std::isfinite(d->residual_scale),
                "%s: eps %g and residual_scale %g must be finite, eps not negative", who, (double)d->eps,
                (double)d->residual_scale);
  return TRACE_OK;
}

int elem_bytes(int dtype) { return dtype == TRACE_F32 ? 4 : 2; }

NormArgs common_args(const trace_norm_desc& d) {
  NormArgs a{};
  a.R = d.rows; a.C = d.C; a.rpc = d.rows_per_cond;
  a.layer = d.kind == TRACE_NORM_LAYER;
  a.cond = d.per_cond != 0;
  a.gate_cond = d.gate_per_cond != 0;
  a.alpha = d.residual_scale; a.eps = d.eps;
  a.xs = (long)d.x_stride; a.ys = (long)d.y_stride; a.dhs = (long)d.dh_stride; a.dzs = (long)d.dz_stride;
  return a;
}

struct BackPlan {
  int groups, nsub, rows_sub, chunks, teams, per_team, wgs;
  int64_t part_g, part_s;         // floats of one partial table
};

// Rows are cut into chunks of one conditioning group each, for the 16 waves a CU that the registers of the column sums leave room for
// (four a SIMD); rows of 1024 lanes for two workgroups a CU, of which one runs at a time.  Up to 4096 columns, four times as many
// measured 2 % faster for 10240 groups and leave four times as many partial rows to add up; twice as many were 15 % slower (a second,
// partly filled round).  A lane of a 1024-lane row has 128 registers, and 16 elements of every array do not fit: 4096 x 16384 fp32 take
// 971 us (1.7 TB/s, 380 .. 700 bytes of scratch a lane), where 8192 x 8192, eight a lane, take 407 (4.0 TB/s).
BackPlan back_plan(const trace_norm_desc& d, int tpr, int teams_wg) {
  BackPlan b;
  const int target = tpr == 64 ? 4096 : tpr == 256 ? 1024 : 512;
  const int64_t rpc = d.rows_per_cond < d.rows ? d.rows_per_cond : d.rows;         // up to 2^31 - 1, as the rows
  const int64_t groups = (d.rows + rpc - 1) / rpc;
  const int64_t most = (rpc + 1) / 2;                        // two rows at least: with few rows it is a team's rows one by one that take the time
  const int64_t cut = std::max<int64_t>(1, std::min(target / groups, most));
  const int64_t rows_sub = (rpc + cut - 1) / cut, nsub = (rpc + rows_sub - 1) / rows_sub;
  const int64_t chunks = groups * nsub, teams = std::min<int64_t>(chunks, target);
  const int64_t per_team = (chunks + teams - 1) / teams;
  b.groups = (int)groups;
  b.rows_sub = (int)rows_sub;
  b.nsub = (int)nsub;
  b.chunks = (int)chunks;
  b.per_team = (int)per_team;
  b.teams = (int)((chunks + per_team - 1) / per_team);
  b.wgs = (b.teams + teams_wg - 1) / teams_wg;
  b.part_g = b.nsub > 1 && (d.per_cond || d.gate_per_cond) ? (int64_t)b.chunks * d.C : 0;
  b.part_s = (int64_t)b.wgs * d.C;
  return b;
}

int reduce(const NormReduceArgs& a, hipStream_t st) {
  if (a.count == 0) return TRACE_OK;
  const long grid = (long)a.count * a.groups * ((a.C + 63) / 64);
  TRACE_REQUIRE(grid * 1024 <= MAX_GRID_THREADS, "norm_reduce_kernel: grid of %ld workgroups", grid);
  hipLaunchKernelGGL(norm_reduce_kernel, dim3((unsigned)grid), dim3(1024), 0, st, a);
  return launch_status("norm_reduce_kernel");
}

}  // namespace
}  // namespace trace

using namespace trace;

extern "C" int trace_residual_norm(const trace_norm_desc* d, const void* x, const void* y, const float* gate,
                                   const float* post_weight, const float* weight, const float* bias, void* h, void* z,
                                   void* stream) {
  const int rc = check_desc(d, "trace_residual_norm");
  if (rc != TRACE_OK) return rc;
  if (d->rows == 0) return TRACE_OK;
  TRACE_REQUIRE(y || (!gate && !post_weight && !h), "trace_residual_norm: gate, post_weight and h belong to a block output y");
  TRACE_REQUIRE(x && (h || z), "trace_residual_norm: null argument");
  const int ex = elem_bytes(d->stream_dtype), ey = elem_bytes(d->dtype);
  const bool vec = aligned16(x) && aligned16(y) && aligned16(gate) && aligned16(post_weight) && aligned16(weight) &&
                   aligned16(bias) && aligned16(h) && aligned16(z) && d->x_stride * ex % 16 == 0 &&
                   (!y || d->y_stride * ey % 16 == 0);
  NormPlan p;
  plan_for(d->C, ex, ey, vec, &p);
  NormArgs a = common_args(*d);
  a.x = x; a.y = y; a.gate = gate; a.post = post_weight; a.weight = weight; a.bias = bias; a.h = h; a.z = z;
  // a launch holds 2^32 - 1 threads: 2^21 workgroups of up to 1024 at a time
  const int per_launch = (1 << 21) * p.teams_wg;
  for (a.row0 = 0; a.row0 < d->rows; a.row0 += per_launch) {
    const long rows = std::min<long>(per_launch, d->rows - a.row0);
    const int rc2 = dispatch(false, *d, p, a, (int)((rows + p.teams_wg - 1) / p.teams_wg), (hipStream_t)stream);
    if (rc2 != TRACE_OK) return rc2;
  }
  return TRACE_OK;
}

extern "C" int64_t trace_residual_norm_workspace_bytes(const trace_norm_desc* d) {
  const int rc = check_desc(d, "trace_residual_norm_workspace_bytes");
  if (rc != TRACE_OK) return rc;
  if (d->rows == 0) return 0;
  const int tpr = d->C <= 1024 ? 64 : d->C <= 4096 ? 256 : 1024;
  const BackPlan b = back_plan(*d, tpr, tpr == 64 ? 4 : 1);
  return (3 * b.part_g + 4 * b.part_s) * (int64_t)sizeof(float);
}

extern "C" int trace_residual_norm_backward(const trace_norm_desc* d, const void* dh, const void* dz, const void* x,
                                            const void* y, const float* gate, const float* post_weight,
                                            const float* weight, void* dx, void* dy, float* dgate, float* dpost_weight,
                                            float* dweight, float* dbias, void* workspace, int64_t workspace_bytes,
                                            void* stream) {
  const int rc = check_desc(d, "trace_residual_norm_backward");
  if (rc != TRACE_OK) return rc;
  hipStream_t st = (hipStream_t)stream;
  TRACE_REQUIRE(y || (!gate && !post_weight && !dy && !dgate && !dpost_weight),
                "trace_residual_norm_backward: gate, post_weight and their gradients belong to a block output y");
  TRACE_REQUIRE((!dgate || gate) && (!dpost_weight || post_weight) && (dz || (!dweight && !dbias)),
                "trace_residual_norm_backward: a gradient of what the call does not have");
  TRACE_REQUIRE(d->rows > 0, "trace_residual_norm_backward: no rows");
  TRACE_REQUIRE(x && dx && (dh || dz) && (!y || dy), "trace_residual_norm_backward: null argument");
  const int ex = elem_bytes(d->stream_dtype), ey = elem_bytes(d->dtype);
  const bool vec = aligned16(x) && aligned16(y) && aligned16(gate) && aligned16(post_weight) && aligned16(weight) &&
                   aligned16(dh) && aligned16(dz) && aligned16(dx) && aligned16(dy) && aligned16(dgate) &&
                   aligned16(dpost_weight) && aligned16(dweight) && aligned16(dbias) && aligned16(workspace) &&
                   d->x_stride * ex % 16 == 0 && (!dh || d->dh_stride * ex % 16 == 0) &&
                   (!y || d->y_stride * ey % 16 == 0) && (!dz || d->dz_stride * ey % 16 == 0);
  NormPlan p;
  plan_for(d->C, ex, ey, vec, &p);
  const BackPlan b = back_plan(*d, p.tpr, p.teams_wg);
  const int64_t need = trace_residual_norm_workspace_bytes(d);
  if (!workspace || workspace_bytes < need) {
    set_error("trace_residual_norm_backward: workspace too small (%lld bytes, need %lld)", (long long)workspace_bytes,
              (long long)need);
    return TRACE_ENOMEM;
  }
  NormArgs a = common_args(*d);
  a.x = x; a.y = y; a.dh = dh; a.dz = dz; a.gate = gate; a.post = post_weight; a.weight = weight;
  a.dx = dx; a.dy = dy; a.dgate = dgate; a.dpost = dpost_weight; a.dweight = dweight; a.dbias = dbias;
  a.part_s = static_cast<float*>(workspace);
  a.part_g = a.part_s + 4 * b.part_s;
  a.nsub = b.nsub; a.rows_sub = b.rows_sub; a.chunks = b.chunks; a.per_team = b.per_team;
  int r = dispatch(true, *d, p, a, b.wgs, st);
  float* const grads[4] = {dgate, dweight, dbias, dpost_weight};
  NormReduceArgs shared{}, cond{};
  shared.groups = 1; shared.n = b.wgs; shared.C = d->C;
  cond.groups = b.groups; cond.n = b.nsub; cond.C = d->C;
  for (int i = 0; i < 4; ++i) {
    if (!grads[i]) continue;
    if (i == 3 || !(i > 0 ? a.cond : a.gate_cond)) {
      shared.part[shared.count] = a.part_s + i * b.part_s;
      shared.out[shared.count++] = grads[i];
    } else if (b.nsub > 1) {
      cond.part[cond.count] = a.part_g + i * b.part_g;
      cond.out[cond.count++] = grads[i];
    }
  }
  if (r == TRACE_OK) r = reduce(shared, st);
  return r == TRACE_OK ? reduce(cond, st) : r;
}
