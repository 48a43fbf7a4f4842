// The entry points of the matrix product with bias, activation and residual,
// and its gradients (the product itself: gemm_epilogue.h).
//
//   z = op(lhs) op(rhs) + bias,  output = act(z) + residual
//   dz = grad_output act'(z)     grad_bias = sum over rows of dz
//   grad op(lhs) = dz op(rhs)^T  grad op(rhs) = op(lhs)^T dz
//
// dz is one pass over grad_output and z in front of the two products, which sums
// the bias's gradient on the way and keeps dz in the workspace, rounded to the
// data type: the products take 16-bit operands, and a rounding of every factor
// is as large an error in a sum as the rounding of that sum itself (8192 x 2048 x
// 8192 bfloat16: 2.3e-3 of the gradients' norm against 64 bits, 1.7e-3 without it;
// dz held in two values would take the products twice, 430 us more).
#include <algorithm>

#include "gemm_epilogue.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using epi::Product;
using seq::Pack;

// dz of a block of 32 VEC columns and `rows` rows: 8 rows at a time, and their
// sums at the end.  Bound by memory: 8192 x 8192 bfloat16 through gelu's slope, 403
// MB, in 73-79 us, 5.1-5.5 TB/s.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
    activation_grad_kernel(const T* __restrict__ grad, long grad_stride,
                           const T* __restrict__ z, T* __restrict__ dz,
                           float* __restrict__ sums, int m, int n, int rows,
                           int activation) {
  typedef typename Pack<T, VEC>::type V;
  __shared__ float part[8][32 * VEC];
  const int lane = threadIdx.x & 31, line = threadIdx.x >> 5;
  const int first = (blockIdx.x * 32 + lane) * VEC;
  const int begin = blockIdx.y * rows, end = min(m, begin + rows);
  const seq::Group<VEC> at(first, n);
  float sum[VEC] = {};
  if (first < n) {
    for (int row = begin + line; row < end; row += 8) {
      float g[VEC];
      seq::unpack<T, VEC>(
          *reinterpret_cast<const V*>(grad + row * grad_stride + at.c), g);
      if (activation != SNN_HIP_ACTIVATION_NONE) {
        const long place = static_cast<long>(row) * n + at.c;
        float v[VEC];
        seq::unpack<T, VEC>(*reinterpret_cast<const V*>(z + place), v);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
          g[i] *= epi::activation_slope(v[i], activation);
        // (two lanes write the same values where they overlap)
        if (dz != nullptr)
          *reinterpret_cast<V*>(dz + place) = seq::pack<T, VEC>(g);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) sum[i] += g[i];
    }
  }
  if (sums == nullptr) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (first < n && i >= at.skip) part[line][at.c + i - blockIdx.x * 32 * VEC] = sum[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * VEC; i += 256) {
    const int col = blockIdx.x * 32 * VEC + i;
    if (col >= n) continue;
    float s = 0.f;
#pragma unroll
    for (int l = 0; l < 8; ++l) s += part[l][i];
    sums[static_cast<long>(blockIdx.y) * n + col] = s;
  }
}

// Rows that a work-group of that pass takes: enough work-groups for the GPU,
// and few enough that their sums are little beside the rows.
int rows_per_group(int m, int n) {
  const int columns = ceil_div(n, 256);
  const int groups = std::max(1, 2048 / columns);
  return std::max(32, ceil_div(ceil_div(m, groups), 8) * 8);
}

int run(int dtype, Product& g, void* workspace, size_t bytes,
        hipStream_t stream) {
  switch (dtype) {
    case SNN_HIP_DTYPE_F32:
      return epi::run_f32(g, workspace, bytes, stream);
    case SNN_HIP_DTYPE_F16:
      return epi::run_f16(g, workspace, bytes, stream);
    default:
      return epi::run_bf16(g, workspace, bytes, stream);
  }
}

int elem_size(int dtype) { return dtype == SNN_HIP_DTYPE_F32 ? 4 : 2; }

int check(const snn_hip_matmul_bias_act_params* p, int size,
          const void* workspace) {
  if (p == nullptr) return SNN_HIP_INVALID_PARAMETER;
  SNN_REQUIRE(p->m > 0 && p->k > 0 && p->n > 0);
  SNN_REQUIRE(p->activation >= SNN_HIP_ACTIVATION_NONE &&
              p->activation <= SNN_HIP_ACTIVATION_SILU);
  auto stride_ok = [](int stride, int row) {
    return stride == 0 || stride >= row;
  };
  SNN_REQUIRE(stride_ok(p->lhs_stride, p->transpose_lhs ? p->m : p->k));
  SNN_REQUIRE(stride_ok(p->rhs_stride, p->transpose_rhs ? p->k : p->n));
  SNN_REQUIRE(stride_ok(p->residual_stride, p->n));
  SNN_REQUIRE(stride_ok(p->output_stride, p->n));
  SNN_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15u) == 0);
  // (columns and reductions are counted in 31 bits of bytes)
  const int most = (1 << 30) / size;
  if (p->m >= most || p->k >= most || p->n >= most)
    return SNN_HIP_INDEX_EXCEEDED;
  return SNN_HIP_OK;
}

long or_else(int stride, int row) { return stride == 0 ? row : stride; }

size_t round16(size_t bytes) { return (bytes + 15) / 16 * 16; }

// The forward product and those of the gradients, but for the addresses.
Product forward_product(const snn_hip_matmul_bias_act_params& p) {
  Product g = {};
  g.p_stride = or_else(p.lhs_stride, p.transpose_lhs ? p.m : p.k);
  g.p_k_inner = !p.transpose_lhs;
  g.q_stride = or_else(p.rhs_stride, p.transpose_rhs ? p.k : p.n);
  g.q_k_inner = p.transpose_rhs != 0;
  g.m = p.m;
  g.n = p.n;
  g.k = p.k;
  g.residual_stride = or_else(p.residual_stride, p.n);
  g.out_stride = or_else(p.output_stride, p.n);
  g.pre_stride = p.n;
  g.activation = p.activation;
  return g;
}

// An operand of the gradients' products: the address, its values with the
// result's dimension first, and whether the reduction is contiguous.
struct Side {
  const void* at;
  long stride;
  bool k_inner;
  int rows;
};
Product grad_product(const Side& a, const Side& b, int k) {
  Product g = {};
  g.p = a.at;
  g.p_stride = a.stride;
  g.p_k_inner = a.k_inner;
  g.m = a.rows;
  g.q = b.at;
  g.q_stride = b.stride;
  g.q_k_inner = b.k_inner;
  g.n = b.rows;
  g.k = k;
  g.out_stride = b.rows;
  return g;
}
// over n: dz (m x n) and op(rhs) (k x n)
Product lhs_product(const snn_hip_matmul_bias_act_params& p, const void* d,
                    long d_stride, const void* rhs) {
  const Side of_d = {d, d_stride, true, p.m};
  const Side of_r = {rhs, or_else(p.rhs_stride, p.transpose_rhs ? p.k : p.n),
                     !p.transpose_rhs, p.k};
  return p.transpose_lhs ? grad_product(of_r, of_d, p.n)
                         : grad_product(of_d, of_r, p.n);
}
// over m: op(lhs)^T (k x m) and dz^T (n x m)
Product rhs_product(const snn_hip_matmul_bias_act_params& p, const void* d,
                    long d_stride, const void* lhs) {
  const Side of_l = {lhs, or_else(p.lhs_stride, p.transpose_lhs ? p.m : p.k),
                     p.transpose_lhs != 0, p.k};
  const Side of_d = {d, d_stride, false, p.n};
  return p.transpose_rhs ? grad_product(of_d, of_l, p.m)
                         : grad_product(of_l, of_d, p.m);
}

// Where the gradients' workspace has what: dz, the bias's partial sums, and
// what the two products take in turn.
struct GradSpace {
  size_t dz, sums, products;
};
GradSpace grad_space(const snn_hip_matmul_bias_act_params& p, int size) {
  GradSpace s = {};
  const bool act = p.activation != SNN_HIP_ACTIVATION_NONE;
  if (act) s.dz = round16(static_cast<size_t>(p.m) * p.n * size);
  s.sums = round16(static_cast<size_t>(ceil_div(p.m, rows_per_group(p.m, p.n))) *
                   p.n * sizeof(float));
  const long stride = act ? p.n : or_else(p.output_stride, p.n);
  s.products =
      std::max(epi::workspace_bytes(lhs_product(p, nullptr, stride, nullptr),
                                    size),
               epi::workspace_bytes(rhs_product(p, nullptr, stride, nullptr),
                                    size));
  return s;
}

template <typename T>
int forward(int dtype, const void* lhs, const void* rhs, const void* bias,
            const void* residual, void* output, void* pre,
            const snn_hip_matmul_bias_act_params* params, void* workspace,
            size_t elems, void* stream) {
  const int v = check(params, sizeof(T), workspace);
  if (v != SNN_HIP_OK) return v;
  SNN_REQUIRE(lhs != nullptr && rhs != nullptr && output != nullptr);
  Product g = forward_product(*params);
  g.p = lhs;
  g.q = rhs;
  g.bias = bias;
  g.residual = residual;
  g.out = output;
  g.pre = pre;
  KernelTimer timer(as_stream(stream));
  return run(dtype, g, workspace, workspace == nullptr ? 0 : elems * sizeof(T),
             as_stream(stream));
}

template <typename T, int VEC>
int launch_activation_grad(const snn_hip_matmul_bias_act_params& p,
                           const void* grad, const void* z, void* dz,
                           float* sums, hipStream_t stream) {
  const int rows = rows_per_group(p.m, p.n);
  const unsigned groups = static_cast<unsigned>(ceil_div(p.m, rows));
  if (groups > 65535) return SNN_HIP_INDEX_EXCEEDED;
  hipLaunchKernelGGL(
      (activation_grad_kernel<T, VEC>),
      dim3(static_cast<unsigned>(ceil_div(p.n, 32 * VEC)), groups), dim3(256),
      0, stream, static_cast<const T*>(grad), or_else(p.output_stride, p.n),
      static_cast<const T*>(z), static_cast<T*>(dz), sums, p.m, p.n, rows,
      p.activation);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T>
int backward(int dtype, const void* grad, const void* lhs, const void* rhs,
             const void* z, void* grad_lhs, void* grad_rhs, void* grad_bias,
             const snn_hip_matmul_bias_act_params* params, void* workspace,
             size_t elems, void* stream_arg) {
  const int v = check(params, sizeof(T), workspace);
  if (v != SNN_HIP_OK) return v;
  const snn_hip_matmul_bias_act_params& p = *params;
  const bool act = p.activation != SNN_HIP_ACTIVATION_NONE;
  SNN_REQUIRE(grad != nullptr && (!act || z != nullptr));
  SNN_REQUIRE(grad_lhs == nullptr || rhs != nullptr);
  SNN_REQUIRE(grad_rhs == nullptr || lhs != nullptr);
  SNN_REQUIRE(grad_lhs != nullptr || grad_rhs != nullptr ||
              grad_bias != nullptr);
  const hipStream_t stream = as_stream(stream_arg);
  const bool products = grad_lhs != nullptr || grad_rhs != nullptr;
  GradSpace space = grad_space(p, sizeof(T));
  if (!products) space.dz = 0;
  if (grad_bias == nullptr) space.sums = 0;
  const size_t bytes = workspace == nullptr ? 0 : elems * sizeof(T);
  if (bytes < space.dz + space.sums) return SNN_HIP_INSUFFICIENT_WORKSPACE;
  char* const at = static_cast<char*>(workspace);
  T* const dz = space.dz > 0 ? reinterpret_cast<T*>(at) : nullptr;
  float* const sums =
      space.sums > 0 ? reinterpret_cast<float*>(at + space.dz) : nullptr;
  void* const rest = bytes > 0 ? at + space.dz + space.sums : nullptr;
  const size_t rest_bytes = bytes - space.dz - space.sums;

  KernelTimer timer(stream);
  const long grad_stride = or_else(p.output_stride, p.n);
  if (dz != nullptr || sums != nullptr) {
    constexpr int VEC = 16 / sizeof(T);
    const int s =
        p.n >= VEC
            ? launch_activation_grad<T, VEC>(p, grad, z, dz, sums, stream)
            : launch_activation_grad<T, 1>(p, grad, z, dz, sums, stream);
    if (s != SNN_HIP_OK) return s;
  }
  if (sums != nullptr) {
    hipLaunchKernelGGL(
        seq::add_rows_kernel<T>,
        seq::columns_grid(p.n, 1), dim3(1024), 0, stream, sums, seq::SumOutputs{}, static_cast<T*>(grad_bias), p.n,
        ceil_div(p.m, rows_per_group(p.m, p.n)), static_cast<long>(p.n), 0l);
    SNN_HIP_CHECK_LAUNCH();
  }

  const void* const d = dz != nullptr ? static_cast<const void*>(dz) : grad;
  const long d_stride = dz != nullptr ? p.n : grad_stride;
  if (grad_lhs != nullptr) {
    Product g = lhs_product(p, d, d_stride, rhs);
    g.out = grad_lhs;
    const int s = run(dtype, g, rest, rest_bytes, stream);
    if (s != SNN_HIP_OK) return s;
  }
  if (grad_rhs != nullptr) {
    Product g = rhs_product(p, d, d_stride, lhs);
    g.out = grad_rhs;
    const int s = run(dtype, g, rest, rest_bytes, stream);
    if (s != SNN_HIP_OK) return s;
  }
  return SNN_HIP_OK;
}

}  // namespace

namespace epi {

size_t workspace_bytes(const Product& g, int elem_size) {
  // (with aligned addresses and without: other tiles, other shares)
  size_t most = 0;
  for (const bool aligned : {false, true}) {
    const Plan p = make_plan(g, elem_size, ~size_t{0}, aligned, aligned);
    const size_t shares = p.splits > 1 ? static_cast<size_t>(g.m) * g.n *
                                             p.splits * sizeof(float)
                                       : 0;
    // (copies only for what the sizes and strides ask for)
    most = std::max(most, shares + (aligned ? p.p_bytes + p.q_bytes : 0));
  }
  return round16(most);
}

}  // namespace epi
}  // namespace snn

#define SNN_MATMUL_BIAS_ACT(suffix, T, dtype)                                 \
  int snn_hip_matmul_bias_act_##suffix(                                       \
      const void* lhs, const void* rhs, const void* bias,                     \
      const void* residual, void* output, void* pre_activation,               \
      const snn_hip_matmul_bias_act_params* params, void* workspace,          \
      size_t workspace_elems, void* stream) {                                 \
    return snn::forward<T>(dtype, lhs, rhs, bias, residual, output,           \
                           pre_activation, params, workspace,                 \
                           workspace_elems, stream);                          \
  }                                                                           \
  int snn_hip_matmul_bias_act_grad_##suffix(                                  \
      const void* grad_output, const void* lhs, const void* rhs,              \
      const void* pre_activation, void* grad_lhs, void* grad_rhs,             \
      void* grad_bias, const snn_hip_matmul_bias_act_params* params,          \
      void* workspace, size_t workspace_elems, void* stream) {                \
    return snn::backward<T>(dtype, grad_output, lhs, rhs, pre_activation,     \
                            grad_lhs, grad_rhs, grad_bias, params, workspace, \
                            workspace_elems, stream);                         \
  }

extern "C" {

SNN_MATMUL_BIAS_ACT(f32, float, SNN_HIP_DTYPE_F32)
SNN_MATMUL_BIAS_ACT(f16, _Float16, SNN_HIP_DTYPE_F16)
SNN_MATMUL_BIAS_ACT(bf16, __bf16, SNN_HIP_DTYPE_BF16)

int snn_hip_matmul_bias_act_workspace_size(
    const snn_hip_matmul_bias_act_params* params, int grad, int dtype,
    size_t* required_elems, size_t* recommended_elems) {
  if (dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16 ||
      required_elems == nullptr || recommended_elems == nullptr)
    return SNN_HIP_INVALID_PARAMETER;
  const int size = snn::elem_size(dtype);
  const int v = snn::check(params, size, nullptr);
  if (v != SNN_HIP_OK) return v;
  if (grad != 0) {
    const snn::GradSpace s = snn::grad_space(*params, size);
    *required_elems = (s.dz + s.sums) / size;
    *recommended_elems = (s.dz + s.sums + s.products) / size;
  } else {
    *required_elems = 0;
    *recommended_elems =
        snn::epi::workspace_bytes(snn::forward_product(*params), size) / size;
  }
  return SNN_HIP_OK;
}

int snn_hip_matmul_bias_act_planned(
    const snn_hip_matmul_bias_act_params* params, int product, int dtype,
    int aligned, size_t workspace_elems, snn_hip_matmul_bias_act_plan* plan) {
  if (dtype < SNN_HIP_DTYPE_F32 || dtype > SNN_HIP_DTYPE_BF16 || product < 0 ||
      product > 2 || plan == nullptr)
    return SNN_HIP_INVALID_PARAMETER;
  const int size = snn::elem_size(dtype);
  const int v = snn::check(params, size, nullptr);
  if (v != SNN_HIP_OK) return v;
  const bool at16 = aligned != 0;
  size_t bytes = workspace_elems * size;
  snn::epi::Product g;
  bool p_at16 = at16, q_at16 = at16;
  if (product == 0) {
    g = snn::forward_product(*params);
  } else {
    const snn::GradSpace s = snn::grad_space(*params, size);
    if (bytes < s.dz + s.sums) return SNN_HIP_INSUFFICIENT_WORKSPACE;
    bytes -= s.dz + s.sums;
    const long stride =
        s.dz > 0 ? params->n : snn::or_else(params->output_stride, params->n);
    g = product == 1 ? snn::lhs_product(*params, nullptr, stride, nullptr)
                     : snn::rhs_product(*params, nullptr, stride, nullptr);
    // (the gradient in front of the activation is in the workspace)
    const bool first = product == 1 ? params->transpose_lhs == 0
                                    : params->transpose_rhs != 0;
    if (s.dz > 0) (first ? p_at16 : q_at16) = true;
  }
  const snn::epi::Plan p = snn::epi::make_plan(g, size, bytes, p_at16, q_at16);
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

}  // extern "C"
