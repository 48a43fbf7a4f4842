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
// launch adds the work-groups' sums in their order.  A row's two sums are two
// waits for all its waves, so the next row is on its way meanwhile.  16384 x 2048
// bfloat16 with both norms, a gate and its weights' sums: 111-117 us, 537 MB at
// 4.6-4.8 TB/s, and 5 for the second launch.
#include <algorithm>

#include "residual_norm.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using norm::Rows;
enum { kScale, kPostWeight, kPreWeight, kPostBias, kPreBias, kSums };
// (... of which there are this many where no bias has a gradient)
constexpr int kWeightSums = 3;
static_assert(kSums == seq::kMaxSums, "outputs of a launch");

struct Grad {
  snn_hip_residual_norm_gradients g;
  // Runs of rows: a run belongs to one row of a shared gate, `per_gate` runs to
  // each; without one the rows are one such range.  Work-group w takes the
  // runs w, w + groups, ...
  int gate_span, per_gate, run_rows, runs, groups;
  float* sums;       // [groups][kSums or kWeightSums][channels]
  float* gate_sums;  // [runs][channels] where per_gate > 1
};

// BIASES: sums for the biases' gradients; SHARED: the gate is shared by rows.
template <typename T, int VEC, int PT, int WAVES, bool WHOLE, bool BIASES,
          bool SHARED>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
    __attribute__((amdgpu_waves_per_eu(WAVES == 16 ? 4 : 2)))
    residual_norm_grad_kernel(Rows r, Grad d) {
  typedef norm::Slice<T, VEC, PT, WAVES, WHOLE> S;
  typedef typename S::V V;
  constexpr int kOwn = BIASES ? kSums : kWeightSums;
  // (a wave that holds a row alone has its own sums; four of them are added
  // through LDS)
  constexpr int kTeams = WAVES == 1 ? 4 : 1;
  // (sixteen waves have 128 registers each: none for a row on its way and the
  // weights, and LDS holds as many of the sums as fit: 4096 x 8192 fp32 194 us,
  // with all in registers, of which 65 go to memory, 275)
  constexpr bool kLean = WAVES == 16;
  constexpr int kInLds = !kLean ? 0 : PT == 8 ? (kOwn < 4 ? kOwn : 4) : 2;
  __shared__ float own_sums[kLean ? kInLds * PT * 64 * WAVES : 1];
  __shared__ float lds[WAVES == 1 ? 4 * 64 * PT : 4 * WAVES];
  int turn = 0;
  const int channels = r.channels;
  const float per = 1.f / static_cast<float>(channels);
  const int team = WAVES == 1 ? static_cast<int>(threadIdx.x >> 6) : 0;
  const bool pre = d.g.grad_normed != nullptr;
  float sums[kOwn][PT], gate_sum[SHARED ? PT : 1];
  auto place = [&](int s, int i) -> float& {
    return own_sums[(s * PT + i) * (64 * WAVES) + threadIdx.x];
  };
#pragma unroll
  for (int s = 0; s < kOwn; ++s)
#pragma unroll
    for (int i = 0; i < PT; ++i) {
      if (s < kInLds)
        place(s, i) = 0.f;
      else
        sums[s][i] = 0.f;
    }
  auto add = [&](int s, int i, float v) {
    if (s < kInLds)
      place(s, i) += v;
    else
      sums[s][i] += v;
  };
  V pre_weight[S::kAccesses], post_weight[S::kAccesses],
      post_bias[S::kAccesses], scale[S::kAccesses];
  auto fetch_pre = [&]() { S::fetch(r.t.pre_weight, channels, pre_weight, 1.f); };
  auto fetch_post = [&]() {
    S::fetch(r.t.post_weight, channels, post_weight, 1.f);
    S::fetch(r.t.post_bias, channels, post_bias);
    S::fetch(r.t.scale, channels, scale, 1.f);
  };
  if constexpr (!kLean) {
    fetch_pre();
    fetch_post();
  }

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

  // A row's operands as they come from memory.
  V next_d[S::kAccesses], next_u[S::kAccesses], next_y[S::kAccesses],
      next_x[S::kAccesses], next_g[S::kAccesses];
  float next_stats[4] = {0.f, 0.f, 0.f, 0.f};
  auto fetch_row = [&](long row) {
    auto of = [&](const void* p, long stride) {
      return p == nullptr ? nullptr
                          : static_cast<const void*>(static_cast<const T*>(p) +
                                                     row * stride);
    };
    S::fetch(of(r.t.x, r.x_stride), channels, next_x);
    if (pre) {
      S::fetch(of(d.g.grad_normed, channels), channels, next_u);
      S::fetch(of(r.t.sum, channels), channels, next_y);
    }
    S::fetch(of(d.g.grad_sum, channels), channels, next_d);
    if (r.gate != SNN_HIP_GATE_NONE)
      S::fetch(static_cast<const T*>(r.t.gate) +
                   static_cast<int>(row) / r.gate_rows * r.gate_stride,
               channels, next_g);
    if (r.t.stats != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i) next_stats[i] = r.t.stats[4 * row + i];
    }
  };

  for (int run = blockIdx.x; run < d.runs; run += d.groups) {
    const int gate_row = run / d.per_gate;
    const long first = static_cast<long>(gate_row) * d.gate_span +
                       static_cast<long>(run - gate_row * d.per_gate) * d.run_rows;
    const long last = min(min(first + d.run_rows,
                              (gate_row + 1l) * d.gate_span),
                          static_cast<long>(r.rows));
    if constexpr (SHARED) {
#pragma unroll
      for (int i = 0; i < PT; ++i) gate_sum[i] = 0.f;
    }
    if (!kLean && first + team < last) fetch_row(first + team);
    for (long row = first + team; row < last; row += kTeams) {
      const long at = row * channels;
      if constexpr (kLean) {
        fetch_row(row);
        fetch_pre();
      }
      float dy[PT], xh[PT], u[PT], yh[PT], gate[PT];
      S::expand(next_d, channels, dy);
      S::expand(next_x, channels, xh);
      if (pre) {
        S::expand(next_u, channels, u);
        S::expand(next_y, channels, yh);
      }
      if (r.gate != SNN_HIP_GATE_NONE) S::expand(next_g, channels, gate);
      const float mean0 = next_stats[0], rstd0 = next_stats[1],
                  mean1 = next_stats[2], rstd1 = next_stats[3];
      if (!kLean && row + kTeams < last) fetch_row(row + kTeams);

      float w[PT];
      if (pre) {
        S::expand(pre_weight, channels, w);
        float m[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < PT; ++i) {
          yh[i] = S::inside(i, channels) ? (yh[i] - mean1) * rstd1 : 0.f;
          add(kPreWeight, i, u[i] * yh[i]);
          if constexpr (BIASES) add(kPreBias, i, u[i]);
          u[i] *= w[i];
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
      if constexpr (kLean) fetch_post();

      // n, of which the gate and the scale have their gradients
      float n[PT], s[PT];
      if (r.post != SNN_HIP_NORM_NONE) {
#pragma unroll
        for (int i = 0; i < PT; ++i)
          xh[i] = S::inside(i, channels) ? (xh[i] - mean0) * rstd0 : 0.f;
      }
      S::expand(post_weight, channels, w);
      S::expand(post_bias, channels, n);
      S::expand(scale, channels, s);
#pragma unroll
      for (int i = 0; i < PT; ++i) n[i] += xh[i] * w[i];
      if (r.gate != SNN_HIP_GATE_NONE) {
        float dg[PT];
#pragma unroll
        for (int i = 0; i < PT; ++i) dg[i] = dy[i] * s[i] * n[i];
        if (r.gate != SNN_HIP_GATE_VALUE) {
          const bool silu = r.gate == SNN_HIP_GATE_SILU;
#pragma unroll
          for (int i = 0; i < PT; ++i) {
            float sg, rest;
            seq::sigmoid<T>(gate[i], &sg, &rest);
            const float weight = silu ? gate[i] : 1.f;
            dg[i] *= sg * ((silu ? 1.f : 0.f) + weight * rest);
            gate[i] = weight * sg;
          }
        }
#pragma unroll
        for (int i = 0; i < PT; ++i) dy[i] *= gate[i];
        if constexpr (SHARED) {
#pragma unroll
          for (int i = 0; i < PT; ++i) gate_sum[i] += dg[i];
        } else if (d.g.grad_gate != nullptr) {
          S::store(static_cast<T*>(d.g.grad_gate) + at, channels, dg);
        }
      }
      // dy is dy * gate from here on
      float m[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < PT; ++i) {
        add(kScale, i, dy[i] * n[i]);
        dy[i] *= s[i];
        add(kPostWeight, i, dy[i] * xh[i]);
        if constexpr (BIASES) add(kPostBias, i, dy[i]);
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
    if constexpr (SHARED) {
      if (d.g.grad_gate != nullptr) {
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
  }
  if (d.sums == nullptr) return;
  float* const to =
      d.sums + static_cast<long>(blockIdx.x) * kOwn * channels;
#pragma unroll
  for (int s = 0; s < kOwn; ++s) {
    if (s < kInLds) {
#pragma unroll
      for (int i = 0; i < PT; ++i) sums[s][i] = place(s, i);
    }
    gather(sums[s]);
    if (team == 0) store_floats(to + static_cast<long>(s) * channels, sums[s]);
  }
}

// Work-groups that walk the rows, and the runs they take: eight waves a CU, which
// leaves each the registers for its sums, the weights and the row on its way
// (16384 x 2048 bfloat16: 120 us; twelve waves without a row on its way 130,
// sixteen, whose registers do not fit, 383).
constexpr int kMostWaves = 8 * 256;
// Rows of a run at least, so that its sums cost little beside them; fewer where
// there are few rows, which then wait for one another less (64 x 1024 fp32).
inline int least_rows(int rows) { return std::min(8, std::max(1, rows / 256)); }

void plan_runs(const snn_hip_residual_norm_params& p, Grad* d) {
  const bool shared = p.gate != SNN_HIP_GATE_NONE && p.gate_rows > 1;
  const int span = shared ? std::min(p.gate_rows, p.rows) : p.rows;
  const int gates = ceil_div(p.rows, span);
  const int waves = p.channels <= 512 ? 4 : ceil_div(p.channels, 512);
  const int groups = std::max(256, kMostWaves / waves);
  const int teams = p.channels <= 512 ? 4 : 1;
  const int target =
      std::max(least_rows(p.rows) * teams, ceil_div(p.rows, groups));
  d->gate_span = span;
  d->per_gate = ceil_div(span, target);
  d->run_rows = ceil_div(span, d->per_gate);
  d->runs = gates * d->per_gate;
  d->groups = std::min(d->runs, groups);
}

size_t sum_floats(const snn_hip_residual_norm_params& p, const Grad& d) {
  return static_cast<size_t>(d.groups) * kSums * p.channels;
}
size_t gate_floats(const snn_hip_residual_norm_params& p, const Grad& d) {
  return p.gate != SNN_HIP_GATE_NONE && p.gate_rows > 1 && d.per_gate > 1
             ? static_cast<size_t>(d.runs) * p.channels
             : 0;
}

template <typename T, int VEC, int PT, int WAVES, bool WHOLE>
int launch_as(const Rows& r, const Grad& d, hipStream_t stream) {
  const bool biases =
      d.g.grad_post_bias != nullptr || d.g.grad_pre_bias != nullptr;
  const bool shared = r.gate != SNN_HIP_GATE_NONE && r.gate_rows > 1;
  const auto kernel =
      biases
          ? (shared
                 ? residual_norm_grad_kernel<T, VEC, PT, WAVES, WHOLE, true, true>
                 : residual_norm_grad_kernel<T, VEC, PT, WAVES, WHOLE, true,
                                             false>)
          : (shared
                 ? residual_norm_grad_kernel<T, VEC, PT, WAVES, WHOLE, false, true>
                 : residual_norm_grad_kernel<T, VEC, PT, WAVES, WHOLE, false,
                                             false>);
  KernelTimer timer(stream);
  hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(d.groups)),
                     dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, stream, r, d);
  SNN_HIP_CHECK_LAUNCH();
  if (d.sums != nullptr) {
    const seq::SumOutputs outputs = {{d.g.grad_scale, d.g.grad_post_weight,
                                      d.g.grad_pre_weight, d.g.grad_post_bias,
                                      d.g.grad_pre_bias}};
    const int own = biases ? static_cast<int>(kSums) : kWeightSums;
    hipLaunchKernelGGL(seq::add_rows_kernel<T>,
                       seq::columns_grid(r.channels, own), dim3(1024), 0,
                       stream, d.sums, outputs, static_cast<T*>(nullptr),
                       r.channels, d.groups,
                       static_cast<long>(own) * r.channels,
                       static_cast<long>(r.channels));
    SNN_HIP_CHECK_LAUNCH();
  }
  if (d.gate_sums != nullptr) {
    hipLaunchKernelGGL(
        seq::add_rows_kernel<T>,
        seq::columns_grid(r.channels, d.runs / d.per_gate), dim3(1024), 0,
        stream, d.gate_sums, seq::SumOutputs{}, static_cast<T*>(d.g.grad_gate),
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
  if (r.channels < VEC)
    return launch_as<T, 1, 8, 1, true>(r, d, as_stream(stream));
  return norm::by_channels<VEC>(
      r.channels, [&](auto waves, auto values, auto whole) {
        // (the long rows' kernels have no registers for accesses that begin in
        // front of what is theirs: 256 x 7195 fp32 75 us, value by value 50, and
        // 36 since LDS holds sums)
        constexpr bool kSingly = decltype(waves)::value == 16 &&
                                 !decltype(whole)::value;
        return launch_as<T, kSingly ? 1 : VEC, decltype(values)::value,
                         decltype(waves)::value,
                         kSingly || decltype(whole)::value>(
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
