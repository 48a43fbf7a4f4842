// The entry points of the gated product and its gradients (the products:
// gated_matmul.h).
//
//   g = lhs op(G) + b,  u = lhs op(U) + c,  output = act(g) u
//   dg = grad u act'(g)                     du = grad act(g)
//   grad lhs = dg op(G)^T + du op(U)^T      grad op(G) = lhs^T dg, grad op(U) = lhs^T du
//
// dg and du are one pass over grad_output, g and u in front of the products, which
// sums the biases' gradients on the way and keeps both in the workspace, rounded to the
// data type: see matmul_bias_act.hip.
#include <algorithm>

#include "gated_matmul.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using gated::Pair;
using seq::Pack;

// dg and du of a block of 32 VEC columns and `rows` rows: 8 rows at a time, and their
// sums at the end.  Rows of the two are `stride` values apart.  Bound by memory:
// bfloat16, 4096 x 8192, 72 us, 336 MB, 4.7 TB/s.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    gated_grad_kernel(const T* __restrict__ grad, long grad_stride,
                      const T* __restrict__ gate, const T* __restrict__ up,
                      T* __restrict__ dg, T* __restrict__ du, long stride,
                      float* __restrict__ sums, int m, int n, int rows,
                      int activation) {
  typedef typename Pack<T, VEC>::type V;
  __shared__ float part[2][8][32 * VEC];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int first = (blockIdx.x * 32 + lane) * VEC;
  const int begin = blockIdx.y * rows, end = min(m, begin + rows);
  const seq::Group<VEC> at(first, n);
  float sum[2][VEC] = {};
  if (first < n) {
    for (int row = begin + line; row < end; row += 8) {
      const long place = static_cast<long>(row) * n + at.c;
      float d[VEC], g[VEC], u[VEC], value[VEC];
      seq::unpack<T, VEC>(
          *reinterpret_cast<const V*>(grad + row * grad_stride + at.c), d);
      seq::unpack<T, VEC>(*reinterpret_cast<const V*>(gate + place), g);
      seq::unpack<T, VEC>(*reinterpret_cast<const V*>(up + place), u);
#pragma unroll
      for (int i = 0; i < VEC; ++i) value[i] = g[i];
      epi::activate(value, activation);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        g[i] = d[i] * u[i] * epi::activation_slope(g[i], activation);
        u[i] = d[i] * value[i];
        sum[0][i] += g[i];
        sum[1][i] += u[i];
      }
      if (dg != nullptr) {
        // (two lanes write the same values where they overlap)
        const long to = row * stride + at.c;
        *reinterpret_cast<V*>(dg + to) = seq::pack<T, VEC>(g);
        *reinterpret_cast<V*>(du + to) = seq::pack<T, VEC>(u);
      }
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (first < n && i >= at.skip) {
      const int c = at.c + i - blockIdx.x * 32 * VEC;
      part[0][line][c] = sum[0][i];
      part[1][line][c] = sum[1][i];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 32 * VEC; i += 256) {
    const int which = i / (32 * VEC), c = i % (32 * VEC);
    const int col = blockIdx.x * 32 * VEC + c;
    if (col >= n) continue;
    float s = 0.f;
#pragma unroll
    for (int l = 0; l < 8; ++l) s += part[which][l][c];
    sums[(static_cast<long>(which) * gridDim.y + blockIdx.y) * n + col] = s;
  }
}

// Rows that a work-group of that pass takes: enough work-groups for the GPU, and few
// enough that their sums are little beside the rows.
int rows_per_group(int m, int n) {
  const int columns = ceil_div(n, 256);
  const int groups = std::max(1, 2048 / columns);
  return std::max(32, ceil_div(ceil_div(m, groups), 8) * 8);
}

int elem_size(int dtype) { return dtype == SNN_HIP_DTYPE_F32 ? 4 : 2; }
long or_else(int stride, int row) { return stride == 0 ? row : stride; }
size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

int check(const snn_hip_gated_matmul_params* p, int size, const void* workspace) {
  if (p == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(p->m > 0 && p->k > 0 && p->n > 0);
  SNN_REQUIRE(p->activation >= SNN_HIP_ACTIVATION_NONE &&
              p->activation <= SNN_HIP_ACTIVATION_SILU);
  auto stride_ok = [](int stride, int row) {
    return stride == 0 || stride >= row;
  };
  SNN_REQUIRE(stride_ok(p->lhs_stride, p->k));
  SNN_REQUIRE(stride_ok(p->rhs_stride, p->transpose_rhs ? p->k : p->n));
  SNN_REQUIRE(stride_ok(p->output_stride, p->n));
  SNN_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
  // (columns and reductions are counted in 31 bits of bytes, two operands' in turn)
  const int most = (1 << 29) / size;
  if (p->m >= most || p->k >= most || p->n >= most) return SNN_HIP_INDEX_EXCEEDED;
  return SNN_HIP_OK;
}

template <typename T>
int run(Pair& g, void* workspace, size_t bytes, hipStream_t stream) {
  if (std::is_same<T, float>::value)
    return gated::run_f32(g, workspace, bytes, stream);
  if (std::is_same<T, _Float16>::value)
    return gated::run_f16(g, workspace, bytes, stream);
  return gated::run_bf16(g, workspace, bytes, stream);
}
template <typename T>
int run(epi::Product& g, void* workspace, size_t bytes, hipStream_t stream) {
  if (std::is_same<T, float>::value)
    return epi::run_f32(g, workspace, bytes, stream);
  if (std::is_same<T, _Float16>::value)
    return epi::run_f16(g, workspace, bytes, stream);
  return epi::run_bf16(g, workspace, bytes, stream);
}

// The products, but for the addresses.
Pair forward_pair(const snn_hip_gated_matmul_params& p) {
  Pair g = {};
  g.p_stride = or_else(p.lhs_stride, p.k);
  g.q_stride = or_else(p.rhs_stride, p.transpose_rhs ? p.k : p.n);
  g.q_k_inner = p.transpose_rhs != 0;
  g.m = p.m;
  g.n = p.n;
  g.k = p.k;
  g.gated = true;
  g.out_stride = or_else(p.output_stride, p.n);
  g.activation = p.activation;
  return g;
}
// Values from row to row of dg and du: rows that start at multiples of 16 bytes.
long factor_stride(const snn_hip_gated_matmul_params& p, int size) {
  return epi::copied_stride(p.n, size);
}
Pair lhs_pair(const snn_hip_gated_matmul_params& p, int size) {
  Pair g = {};
  g.p_stride = factor_stride(p, size);
  g.q_stride = or_else(p.rhs_stride, p.transpose_rhs ? p.k : p.n);
  g.q_k_inner = p.transpose_rhs == 0;
  g.m = p.m;
  g.n = p.k;
  g.k = p.n;
  g.gated = false;
  g.out_stride = p.k;
  return g;
}
// lhs^T d, or its transpose: stored as the weight is.
epi::Product weight_product(const snn_hip_gated_matmul_params& p, int size,
                            const void* lhs, const void* d) {
  epi::Product g = {};
  g.k = p.m;
  const long of_lhs = or_else(p.lhs_stride, p.k), of_d = factor_stride(p, size);
  const bool swap = p.transpose_rhs != 0;
  g.p = swap ? d : lhs;
  g.p_stride = swap ? of_d : of_lhs;
  g.m = swap ? p.n : p.k;
  g.q = swap ? lhs : d;
  g.q_stride = swap ? of_lhs : of_d;
  g.n = swap ? p.k : p.n;
  g.out_stride = g.n;
  return g;
}

// Where the gradients' workspace has what: dg and du, the biases' partial sums, and
// what the products take in turn.
struct GradSpace {
  size_t factor, sums, products;
};
GradSpace grad_space(const snn_hip_gated_matmul_params& p, int size) {
  GradSpace s = {};
  s.factor = round16(static_cast<size_t>(p.m) * factor_stride(p, size) * size);
  s.sums = round16(2 * static_cast<size_t>(ceil_div(p.m, rows_per_group(p.m, p.n))) *
                   p.n * sizeof(float));
  s.products = std::max(gated::workspace_bytes(lhs_pair(p, size), size),
                        epi::workspace_bytes(
                            weight_product(p, size, nullptr, nullptr), size));
  return s;
}

template <typename T>
int forward(const void* lhs, const void* gate_weight, const void* up_weight,
            const void* gate_bias, const void* up_bias, void* output, void* gate,
            void* up, const snn_hip_gated_matmul_params* params, void* workspace,
            size_t elems, void* stream) {
  const int v = check(params, sizeof(T), workspace);
  if (v != SNN_HIP_OK) return v;
  SNN_REQUIRE(lhs != nullptr && gate_weight != nullptr && up_weight != nullptr &&
              output != nullptr);
  SNN_REQUIRE((gate != nullptr) == (up != nullptr));
  Pair g = forward_pair(*params);
  g.p[0] = lhs;
  g.q[0] = gate_weight;
  g.q[1] = up_weight;
  g.bias[0] = gate_bias;
  g.bias[1] = up_bias;
  g.out = output;
  g.pre[0] = gate;
  g.pre[1] = up;
  KernelTimer timer(as_stream(stream));
  return run<T>(g, workspace, workspace == nullptr ? 0 : elems * sizeof(T),
                as_stream(stream));
}

template <typename T, int VEC>
int launch_factors(const snn_hip_gated_matmul_params& p, const void* grad,
                   const void* gate, const void* up, void* dg, void* du,
                   float* sums, hipStream_t stream) {
  const int rows = rows_per_group(p.m, p.n);
  const unsigned groups = static_cast<unsigned>(ceil_div(p.m, rows));
  if (groups > 65535) return SNN_HIP_INDEX_EXCEEDED;
  hipLaunchKernelGGL(
      (gated_grad_kernel<T, VEC>),
      dim3(static_cast<unsigned>(ceil_div(p.n, 32 * VEC)), groups), dim3(256), 0,
      stream, static_cast<const T*>(grad), or_else(p.output_stride, p.n),
      static_cast<const T*>(gate), static_cast<const T*>(up), static_cast<T*>(dg),
      static_cast<T*>(du), factor_stride(p, sizeof(T)), sums, p.m, p.n, rows,
      p.activation);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T>
int backward(const void* grad, const void* lhs, const void* gate_weight,
             const void* up_weight, const void* gate, const void* up,
             void* grad_lhs, void* grad_gate_weight, void* grad_up_weight,
             void* grad_gate_bias, void* grad_up_bias,
             const snn_hip_gated_matmul_params* params, void* workspace,
             size_t elems, void* stream_arg) {
  const int v = check(params, sizeof(T), workspace);
  if (v != SNN_HIP_OK) return v;
  const snn_hip_gated_matmul_params& p = *params;
  SNN_REQUIRE(grad != nullptr && gate != nullptr && up != nullptr);
  SNN_REQUIRE(grad_lhs == nullptr ||
              (gate_weight != nullptr && up_weight != nullptr));
  const bool weights = grad_gate_weight != nullptr || grad_up_weight != nullptr;
  const bool biases = grad_gate_bias != nullptr || grad_up_bias != nullptr;
  SNN_REQUIRE(!weights || lhs != nullptr);
  SNN_REQUIRE(grad_lhs != nullptr || weights || biases);
  const hipStream_t stream = as_stream(stream_arg);
  GradSpace space = grad_space(p, sizeof(T));
  if (grad_lhs == nullptr && !weights) space.factor = 0;
  if (!biases) space.sums = 0;
  const size_t bytes = workspace == nullptr ? 0 : elems * sizeof(T);
  const size_t fixed = 2 * space.factor + space.sums;
  if (bytes < fixed) return SNN_HIP_INSUFFICIENT_WORKSPACE;
  char* const at = static_cast<char*>(workspace);
  T* const dg = space.factor > 0 ? reinterpret_cast<T*>(at) : nullptr;
  T* const du =
      space.factor > 0 ? reinterpret_cast<T*>(at + space.factor) : nullptr;
  float* const sums =
      biases ? reinterpret_cast<float*>(at + 2 * space.factor) : nullptr;
  void* const rest = at + fixed;
  const size_t rest_bytes = bytes - fixed;

  KernelTimer timer(stream);
  constexpr int VEC = 16 / sizeof(T);
  int s = p.n >= VEC ? launch_factors<T, VEC>(p, grad, gate, up, dg, du, sums, stream)
                     : launch_factors<T, 1>(p, grad, gate, up, dg, du, sums, stream);
  if (s != SNN_HIP_OK) return s;
  if (biases) {
    const int count = ceil_div(p.m, rows_per_group(p.m, p.n));
    const seq::SumOutputs outputs = {{grad_gate_bias, grad_up_bias}};
    hipLaunchKernelGGL(seq::add_rows_kernel<T>, seq::columns_grid(p.n, 2),
                       dim3(1024), 0, stream, sums, outputs,
                       static_cast<T*>(nullptr), p.n, count,
                       static_cast<long>(p.n), static_cast<long>(count) * p.n);
    SNN_HIP_CHECK_LAUNCH();
  }
  if (grad_lhs != nullptr) {
    Pair g = lhs_pair(p, sizeof(T));
    g.p[0] = dg;
    g.p[1] = du;
    g.q[0] = gate_weight;
    g.q[1] = up_weight;
    g.out = grad_lhs;
    s = run<T>(g, rest, rest_bytes, stream);
    if (s != SNN_HIP_OK) return s;
  }
  for (int which = 0; which < 2; ++which) {
    void* const out = which == 0 ? grad_gate_weight : grad_up_weight;
    if (out == nullptr) continue;
    epi::Product g = weight_product(p, sizeof(T), lhs, which == 0 ? dg : du);
    g.out = out;
    s = run<T>(g, rest, rest_bytes, stream);
    if (s != SNN_HIP_OK) return s;
  }
  return SNN_HIP_OK;
}

}  // namespace

namespace gated {

size_t workspace_bytes(const Pair& g, int elem_size) {
  // (with aligned addresses and without: other tiles, other shares)
  size_t most = 0;
  for (const bool aligned : {false, true}) {
    const Plan p = make_plan(g, elem_size, ~size_t{0}, aligned, aligned);
    const size_t shares = p.splits > 1 ? static_cast<size_t>(g.m) * g.n *
                                             (g.gated ? 2 : 1) * p.splits *
                                             sizeof(float)
                                       : 0;
    // (copies only for what the sizes and strides ask for)
    const size_t copies = (g.gated ? 1 : 2) * p.p_bytes + 2 * p.q_bytes;
    most = std::max(most, shares + (aligned ? copies : 0));
  }
  return (most + 15) / 16 * 16;
}

}  // namespace gated
}  // namespace snn

#define SNN_GATED_MATMUL(suffix, T)                                            \
  int snn_hip_gated_matmul_##suffix(                                           \
      const void* lhs, const void* gate_weight, const void* up_weight,         \
      const void* gate_bias, const void* up_bias, void* output, void* gate,    \
      void* up, const snn_hip_gated_matmul_params* params, void* workspace,    \
      size_t workspace_elems, void* stream) {                                  \
    return snn::forward<T>(lhs, gate_weight, up_weight, gate_bias, up_bias,    \
                           output, gate, up, params, workspace,                \
                           workspace_elems, stream);                           \
  }                                                                            \
  int snn_hip_gated_matmul_grad_##suffix(                                      \
      const void* grad_output, const void* lhs, const void* gate_weight,       \
      const void* up_weight, const void* gate, const void* up, void* grad_lhs, \
      void* grad_gate_weight, void* grad_up_weight, void* grad_gate_bias,      \
      void* grad_up_bias, const snn_hip_gated_matmul_params* params,           \
      void* workspace, size_t workspace_elems, void* stream) {                 \
    return snn::backward<T>(grad_output, lhs, gate_weight, up_weight, gate,    \
                            up, grad_lhs, grad_gate_weight, grad_up_weight,    \
                            grad_gate_bias, grad_up_bias, params, workspace,   \
                            workspace_elems, stream);                          \
  }

extern "C" {

SNN_GATED_MATMUL(f32, float)
SNN_GATED_MATMUL(f16, _Float16)
SNN_GATED_MATMUL(bf16, __bf16)

int snn_hip_gated_matmul_workspace_size(
    const snn_hip_gated_matmul_params* params, int grad, int dtype,
    size_t* required_elems, size_t* recommended_elems) {
  if (dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16 ||
      required_elems == nullptr || recommended_elems == nullptr)
    return SNN_HIP_INVALID_PARAMETER;
  const int size = snn::elem_size(dtype);
  const int v = snn::check(params, size, nullptr);
  if (v != SNN_HIP_OK) return v;
  if (grad != 0) {
    const snn::GradSpace s = snn::grad_space(*params, size);
    *required_elems = (2 * s.factor + s.sums) / size;
    *recommended_elems = (2 * s.factor + s.sums + s.products) / size;
  } else {
    *required_elems = 0;
    *recommended_elems =
        snn::gated::workspace_bytes(snn::forward_pair(*params), size) / size;
  }
  return SNN_HIP_OK;
}

int snn_hip_gated_matmul_planned(
    const snn_hip_gated_matmul_params* params, int product, int dtype,
    int aligned, size_t workspace_elems, snn_hip_matmul_bias_act_plan* plan) {
  if (dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16 || product < 0 ||
      product > 2 || plan == nullptr)
    return SNN_HIP_INVALID_PARAMETER;
  const int size = snn::elem_size(dtype);
  const int v = snn::check(params, size, nullptr);
  if (v != SNN_HIP_OK) return v;
  const bool at16 = aligned != 0;
  size_t bytes = workspace_elems * size;
  if (product > 0) {
    const snn::GradSpace s = snn::grad_space(*params, size);
    if (bytes < 2 * s.factor + s.sums) return SNN_HIP_INSUFFICIENT_WORKSPACE;
    bytes -= 2 * s.factor + s.sums;
  }
  if (product == 2) {
    const snn::epi::Product g =
        snn::weight_product(*params, size, nullptr, nullptr);
    // (the factor's gradient is in the workspace)
    const bool first = params->transpose_rhs != 0;
    const snn::epi::Plan p =
        snn::epi::make_plan(g, size, bytes, first || at16, !first || at16);
    if (p.splits == 0) return SNN_HIP_INDEX_EXCEEDED;
    const snn::epi::Shape& shape = snn::epi::shape_of(size, p.kernel);
    *plan = {shape.bm,
             shape.bn,
             shape.chunks > 1,
             p.kernel >= snn::epi::kAny16x16,
             p.kernel == snn::epi::kTile128Pair,
             g.p_k_inner,
             g.q_k_inner,
             p.copy_p,
             p.copy_q,
             p.splits};
    return SNN_HIP_OK;
  }
  const snn::gated::Pair g = product == 0 ? snn::forward_pair(*params)
                                          : snn::lhs_pair(*params, size);
  const snn::gated::Plan p =
      snn::gated::make_plan(g, size, bytes, product == 1 || at16, at16);
  if (p.splits == 0) return SNN_HIP_INDEX_EXCEEDED;
  const snn::epi::Shape shape = snn::gated::shape_of(size, p.kernel);
  *plan = {shape.bm,
           shape.bn,
           shape.chunks > 1,
           p.kernel >= snn::gated::kDirectKernels,
           p.kernel == snn::gated::kTile128Pair,
           1,
           g.q_k_inner,
           p.copy_p,
           p.copy_q,
           p.splits};
  return SNN_HIP_OK;
}

}  // extern "C"
