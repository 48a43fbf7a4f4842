// The gradients of the norms before and after a block with its gate and
// residual scale (gfx950).  With xh, yh the normalised rows and r0, r1 their
// reciprocal deviations (from the forward pass), D = grad_sum and U = grad_normed:
//
//   dy = D + through(U * pre_weight, yh, r1)          grad_residual
//   dn = dy * scale * gate
//   grad_x = through(dn * post_weight, xh, r0)
//   through(v, h, r) = r (v - h mean(v h) [- mean(v)])
//   grad_gate = dy * scale * n * gate'                summed over shared rows
//   grad_scale = sum of dy * gate * n                 ... and the others below,
//   grad_post_weight = sum of dn * xh                 over all rows
//   grad_post_bias = sum of dn, grad_pre_weight = sum of U * yh,
//   grad_pre_bias = sum of U
//
// Bound by memory: as in the forward kernel rows stay in registers between
// their row sums, so every operand is read once.  Work-groups walk runs of rows
// and keep the sums over rows in registers, each lane for its channels; a second
// launch adds the work-groups' sums in their order.
#include <algorithm>

#include "residual_norm.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using norm::Rows;

enum { kScale, kPostWeight, kPostBias, kPreWeight, kPreBias, kSums };
static_assert(kSums == seq::kMaxSums, "outputs of a launch");

struct Grad {
  snn_hip_residual_norm_gradients g;
  // Runs of rows: a run belongs to one row of a shared gate, `per_gate` runs to
  // each; without one the rows are one such range.  Work-group w takes the
  // runs w, w + groups, ...
  int gate_span, per_gate, run_rows, runs, groups;
  float* sums;       // [groups][kSums][channels]
  float* gate_sums;  // [runs][channels] where per_gate > 1
};

template <typename T, int VEC, int PT, int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
    residual_norm_grad_kernel(Rows r, Grad d) {
  typedef norm::Slice<T, VEC, PT, WAVES> S;
  // (a wave that holds a row alone has its own sums; four of them are added
  // through LDS)
  constexpr int kTeams = WAVES == 1 ? 4 : 1;
  __shared__ float lds[WAVES == 1 ? 4 * 64 * PT : 4 * WAVES];
  int turn = 0;
  const int channels = r.channels;
  const float per = 1.f / static_cast<float>(channels);
  const int team = WAVES == 1 ? static_cast<int>(threadIdx.x >> 6) : 0;
  const bool shared_gate = r.gate != SNN_HIP_GATE_NONE && r.gate_rows > 1;
  auto tensor = [&](const void* p, long offset) {
    return static_cast<const void*>(static_cast<const T*>(p) + offset);
  };
  float sums[kSums][PT], gate_sum[PT];
#pragma unroll
  for (int s = 0; s < kSums; ++s)
#pragma unroll
    for (int i = 0; i < PT; ++i) sums[s][i] = 0.f;

  // The teams' sums together, in the first team's registers.
  auto gather = [&](float (&v)[PT]) {
    if constexpr (kTeams > 1) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < PT; ++i) lds[(team * PT + i) * 64 + S::lane()] = v[i];
      __syncthreads();
      if (team == 0) {
#pragma unroll
        for (int i = 0; i < PT; ++i)
          for (int t = 1; t < kTeams; ++t)
            v[i] += lds[(t * PT + i) * 64 + S::lane()];
      }
    }
  };
  auto store_floats = [&](float* to, const float (&v)[PT]) {
#pragma unroll
    for (int i = 0; i < PT; ++i)
      if (S::inside(i, channels)) to[S::channel(i, channels)] = v[i];
  };

  for (int run = blockIdx.x; run < d.runs; run += d.groups) {
    const int gate_row = run / d.per_gate;
    const long first = static_cast<long>(gate_row) * d.gate_span +
                       static_cast<long>(run - gate_row * d.per_gate) * d.run_rows;
    const long last = min(min(first + d.run_rows,
                              (gate_row + 1l) * d.gate_span),
                          static_cast<long>(r.rows));
#pragma unroll
    for (int i = 0; i < PT; ++i) gate_sum[i] = 0.f;
    for (long row = first + team; row < last; row += kTeams) {
      const long at = row * channels;
      float mean0 = 0.f, rstd0 = 0.f, mean1 = 0.f, rstd1 = 0.f;
      if (r.t.stats != nullptr) {
        const float* const s = r.t.stats + 4 * row;
        mean0 = s[0];
        rstd0 = s[1];
        mean1 = s[2];
        rstd1 = s[3];
      }
      float dy[PT], w[PT];
#pragma unroll
      for (int i = 0; i < PT; ++i) dy[i] = 0.f;
      if (d.g.grad_sum != nullptr)
        S::load(tensor(d.g.grad_sum, at), channels, dy);
      float xh[PT];
      S::load(tensor(r.t.x, row * r.x_stride), channels, xh);
      if (d.g.grad_normed != nullptr) {
        float u[PT], yh[PT];
        S::load(tensor(d.g.grad_normed, at), channels, u);
        S::load(tensor(r.t.sum, at), channels, yh);
#pragma unroll
        for (int i = 0; i < PT; ++i) {
          yh[i] = S::inside(i, channels) ? (yh[i] - mean1) * rstd1 : 0.f;
          sums[kPreWeight][i] += u[i] * yh[i];
          sums[kPreBias][i] += u[i];
        }
        if (r.t.pre_weight != nullptr) {
          S::load(r.t.pre_weight, channels, w);
#pragma unroll
          for (int i = 0; i < PT; ++i) u[i] *= w[i];
        }
        float m[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PT; ++i) {
          m[0] += u[i] * yh[i];
          m[1] += u[i];
        }
        norm::row_sums<WAVES>(m, lds, &turn);
        m[0] *= per;
        m[1] = r.pre == SNN_HIP_NORM_LAYER ? m[1] * per : 0.f;
#pragma unroll
        for (int i = 0; i < PT; ++i)
          if (S::inside(i, channels))
            dy[i] += rstd1 * (u[i] - yh[i] * m[0] - m[1]);
      }
      if (d.g.grad_residual != nullptr)
        S::store(static_cast<T*>(d.g.grad_residual) + at, channels, dy);

      // n, of which the gate and the scale have their gradients
      float n[PT], gate[PT], slope[PT];
      if (r.post != SNN_HIP_NORM_NONE) {
#pragma unroll
        for (int i = 0; i < PT; ++i)
          xh[i] = S::inside(i, channels) ? (xh[i] - mean0) * rstd0 : 0.f;
      }
#pragma unroll
      for (int i = 0; i < PT; ++i) n[i] = xh[i];
      if (r.t.post_weight != nullptr) {
        S::load(r.t.post_weight, channels, w);
#pragma unroll
        for (int i = 0; i < PT; ++i) n[i] *= w[i];
      } else {
#pragma unroll
        for (int i = 0; i < PT; ++i) w[i] = 1.f;
      }
      if (r.t.post_bias != nullptr) {
        float b[PT];
        S::load(r.t.post_bias, channels, b);
#pragma unroll
        for (int i = 0; i < PT; ++i) n[i] += b[i];
      }
      float scale[PT];
      if (r.t.scale != nullptr) {
        S::load(r.t.scale, channels, scale);
      } else {
#pragma unroll
        for (int i = 0; i < PT; ++i) scale[i] = 1.f;
      }
      if (r.gate != SNN_HIP_GATE_NONE) {
        const long gate_at = static_cast<long>(row / r.gate_rows);
        S::load(tensor(r.t.gate, gate_at * r.gate_stride), channels, gate);
#pragma unroll
        for (int i = 0; i < PT; ++i)
          norm::gate_of<T>(r.gate, gate[i], &gate[i], &slope[i]);
        float dg[PT];
#pragma unroll
        for (int i = 0; i < PT; ++i) dg[i] = dy[i] * scale[i] * n[i] * slope[i];
        if (shared_gate) {
#pragma unroll
          for (int i = 0; i < PT; ++i) gate_sum[i] += dg[i];
        } else if (d.g.grad_gate != nullptr) {
          S::store(static_cast<T*>(d.g.grad_gate) + at, channels, dg);
        }
#pragma unroll
        for (int i = 0; i < PT; ++i) dy[i] *= gate[i];
      }
      // dy is dy * gate from here on
      float m[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        sums[kScale][i] += dy[i] * n[i];
        dy[i] *= scale[i];
        sums[kPostWeight][i] += dy[i] * xh[i];
        sums[kPostBias][i] += dy[i];
        dy[i] *= w[i];
        m[0] += dy[i] * xh[i];
        m[1] += dy[i];
      }
      if (d.g.grad_x != nullptr) {
        if (r.post != SNN_HIP_NORM_NONE) {
          norm::row_sums<WAVES>(m, lds, &turn);
          m[0] *= per;
          m[1] = r.post == SNN_HIP_NORM_LAYER ? m[1] * per : 0.f;
#pragma unroll
          for (int i = 0; i < PT; ++i)
            dy[i] = rstd0 * (dy[i] - xh[i] * m[0] - m[1]);
        }
        S::store(static_cast<T*>(d.g.grad_x) + at, channels, dy);
      }
    }
    if (shared_gate && d.g.grad_gate != nullptr) {
      gather(gate_sum);
      if (team == 0) {
        if (d.per_gate > 1)
          store_floats(d.gate_sums + static_cast<long>(run) * channels,
                       gate_sum);
        else
          S::store(static_cast<T*>(d.g.grad_gate) +
                       static_cast<long>(gate_row) * channels,
                   channels, gate_sum);
      }
    }
  }
  if (d.sums == nullptr) return;
  float* const to =
      d.sums + static_cast<long>(blockIdx.x) * kSums * channels;
#pragma unroll
  for (int s = 0; s < kSums; ++s) {
    gather(sums[s]);
    if (team == 0) store_floats(to + static_cast<long>(s) * channels, sums[s]);
  }
}

// Work-groups that walk the rows, and the runs they take.
constexpr int kMaxGroups = 512;
constexpr int kLeastRows = 8;  // of a run, so that its sums cost little

void plan_runs(const snn_hip_residual_norm_params& p, Grad* d) {
  const bool shared = p.gate != SNN_HIP_GATE_NONE && p.gate_rows > 1;
  const int span = shared ? std::min(p.gate_rows, p.rows) : p.rows;
  const int gates = ceil_div(p.rows, span);
  const int teams = p.channels <= 512 ? 4 : 1;
  const int target = std::max(
      kLeastRows * teams, ceil_div(p.rows, kMaxGroups));
  d->gate_span = span;
  d->per_gate = ceil_div(span, target);
  d->run_rows = ceil_div(span, d->per_gate);
  d->runs = gates * d->per_gate;
  d->groups = std::min(d->runs, kMaxGroups);
}

size_t sum_floats(const snn_hip_residual_norm_params& p, const Grad& d) {
  return static_cast<size_t>(d.groups) * kSums * p.channels;
}
size_t gate_floats(const snn_hip_residual_norm_params& p, const Grad& d) {
  return p.gate != SNN_HIP_GATE_NONE && p.gate_rows > 1 && d.per_gate > 1
             ? static_cast<size_t>(d.runs) * p.channels
             : 0;
}

template <typename T, int VEC, int PT, int WAVES>
int launch_as(const Rows& r, const Grad& d, hipStream_t stream) {
  KernelTimer timer(stream);
  hipLaunchKernelGGL((residual_norm_grad_kernel<T, VEC, PT, WAVES>),
                     dim3(static_cast<unsigned>(d.groups)),
                     dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, stream, r, d);
  SNN_HIP_CHECK_LAUNCH();
  const unsigned columns = static_cast<unsigned>(ceil_div(r.channels, 64));
  if (d.sums != nullptr) {
    const seq::SumOutputs outputs = {{d.g.grad_scale, d.g.grad_post_weight,
                                 d.g.grad_post_bias, d.g.grad_pre_weight,
                                 d.g.grad_pre_bias}};
    hipLaunchKernelGGL(seq::add_rows_kernel<T>, dim3(columns, kSums), dim3(1024),
                       0, stream, d.sums, outputs, static_cast<T*>(nullptr),
                       r.channels, d.groups,
                       static_cast<long>(kSums) * r.channels,
                       static_cast<long>(r.channels));
    SNN_HIP_CHECK_LAUNCH();
  }
  if (d.gate_sums != nullptr) {
    hipLaunchKernelGGL(
        seq::add_rows_kernel<T>,
        dim3(columns, static_cast<unsigned>(d.runs / d.per_gate)), dim3(1024),
        0, stream, d.gate_sums, seq::SumOutputs{}, static_cast<T*>(d.g.grad_gate),
        r.channels, d.per_gate, static_cast<long>(r.channels),
        static_cast<long>(d.per_gate) * r.channels);
    SNN_HIP_CHECK_LAUNCH();
  }
  return SNN_HIP_OK;
}

template <typename T>
int residual_norm_grad(const snn_hip_residual_norm_tensors* tensors,
                       const snn_hip_residual_norm_gradients* gradients,
                       const snn_hip_residual_norm_params* params,
                       void* workspace, size_t elems, void* stream) {
  int v = norm::check_params(params);
  if (v == SNN_HIP_OK) v = norm::check_operands(tensors, *params);
  if (v != SNN_HIP_OK) return v;
  if (gradients == nullptr) return SNN_HIP_INVALID_PARAMETER;
  const snn_hip_residual_norm_tensors& t = *tensors;
  const snn_hip_residual_norm_gradients& g = *gradients;
  const bool pre = params->pre_norm != SNN_HIP_NORM_NONE;
  const bool post = params->post_norm != SNN_HIP_NORM_NONE;
  SNN_REQUIRE(g.grad_sum != nullptr || g.grad_normed != nullptr);
  SNN_REQUIRE(g.grad_normed == nullptr || (pre && t.sum != nullptr));
  SNN_REQUIRE(t.stats != nullptr || (!post && g.grad_normed == nullptr));
  SNN_REQUIRE(g.grad_gate == nullptr || t.gate != nullptr);
  SNN_REQUIRE(g.grad_scale == nullptr || t.scale != nullptr);
  SNN_REQUIRE(g.grad_post_weight == nullptr || t.post_weight != nullptr);
  SNN_REQUIRE(g.grad_post_bias == nullptr || t.post_bias != nullptr);
  SNN_REQUIRE(g.grad_pre_weight == nullptr || t.pre_weight != nullptr);
  SNN_REQUIRE(g.grad_pre_bias == nullptr || t.pre_bias != nullptr);
  SNN_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
  const Rows r = norm::rows_of(t, *params);
  Grad d = {};
  d.g = g;
  plan_runs(*params, &d);
  const size_t sums = g.grad_scale != nullptr || g.grad_post_weight != nullptr ||
                              g.grad_post_bias != nullptr ||
                              g.grad_pre_weight != nullptr ||
                              g.grad_pre_bias != nullptr
                          ? sum_floats(*params, d)
                          : 0;
  const size_t gates = g.grad_gate != nullptr ? gate_floats(*params, d) : 0;
  if (sums + gates > 0) {
    if (workspace == nullptr ||
        elems * sizeof(T) < (sums + gates) * sizeof(float))
      return SNN_HIP_INSUFFICIENT_WORKSPACE;
    float* const floats = static_cast<float*>(workspace);
    d.sums = sums > 0 ? floats : nullptr;
    d.gate_sums = gates > 0 ? floats + sums : nullptr;
  }
  if (d.runs / d.per_gate > 65535 && d.gate_sums != nullptr)
    return SNN_HIP_INDEX_EXCEEDED;  // (the grid of the gate's sums)
  constexpr int VEC = 16 / sizeof(T);
  if (r.channels < VEC) return launch_as<T, 1, 8, 1>(r, d, as_stream(stream));
  return norm::by_channels(r.channels, [&](auto waves, auto values) {
    return launch_as<T, VEC, decltype(values)::value, decltype(waves)::value>(
        r, d, as_stream(stream));
  });
}

}  // namespace
}  // namespace snn

extern "C" {

int snn_hip_residual_norm_grad_f32(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_gradients* gradients,
    const snn_hip_residual_norm_params* params, void* workspace,
    size_t workspace_elems, void* stream) {
  return snn::residual_norm_grad<float>(tensors, gradients, params, workspace,
                                        workspace_elems, stream);
}
int snn_hip_residual_norm_grad_f16(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_gradients* gradients,
    const snn_hip_residual_norm_params* params, void* workspace,
    size_t workspace_elems, void* stream) {
  return snn::residual_norm_grad<_Float16>(tensors, gradients, params,
                                           workspace, workspace_elems, stream);
}
int snn_hip_residual_norm_grad_bf16(
    const snn_hip_residual_norm_tensors* tensors,
    const snn_hip_residual_norm_gradients* gradients,
    const snn_hip_residual_norm_params* params, void* workspace,
    size_t workspace_elems, void* stream) {
  return snn::residual_norm_grad<__bf16>(tensors, gradients, params, workspace,
                                         workspace_elems, stream);
}

int snn_hip_residual_norm_grad_workspace_size(
    const snn_hip_residual_norm_params* params, int dtype,
    size_t* required_elems, size_t* recommended_elems) {
  const int v = snn::norm::check_params(params);
  if (v != SNN_HIP_OK) return v;
  if (required_elems == nullptr || recommended_elems == nullptr ||
      dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16)
    return SNN_HIP_INVALID_PARAMETER;
  snn::Grad d = {};
  snn::plan_runs(*params, &d);
  *required_elems = *recommended_elems =
      (snn::sum_floats(*params, d) + snn::gate_floats(*params, d)) *
      (dtype == SNN_HIP_DTYPE_F32 ? 1 : 2);
  return SNN_HIP_OK;
}

}  // extern "C"
