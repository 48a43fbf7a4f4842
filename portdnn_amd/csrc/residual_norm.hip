// The norms before and after a block with its gate and residual scale, forward
// (gfx950):
//
//   n = post_norm(x) * post_weight + post_bias
//   sum = residual + scale * gate * n
//   normed = pre_norm(sum) * pre_weight + pre_bias
//
// Bound by memory: a row is read once (x, residual and the gate), stays in the
// registers of the waves that share it and is written once (sum, normed), so
// that the row sums of both norms cost no pass of their own.  Up to 512 channels
// a wave holds a row and no barrier is needed; longer rows are shared by the
// waves of a work-group.  Mean and squares are summed in fp32, the squares from
// the centred values, and the second norm takes the sum as it is in front of its
// rounding.  32768 x 4096 bfloat16 with both norms and 8 gates: 218 us,
// 1074 MB at 4.9 TB/s (a stream that only reads and writes 5.95); 8 x 4096 fp32: 4.6
// us, a launch's latency and that of two row sums.
#include "residual_norm.h"
#include "snn_kernels.h"

namespace snn {
namespace {

using norm::Rows;

// Subtracts the mean (LAYER) and returns it and the reciprocal deviation; v
// becomes the normalised values.
template <typename S, int PT, int WAVES>
__device__ __forceinline__ void normalise(float (&v)[PT], int kind,
                                          int channels, float epsilon,
                                          float* lds, int* turn, float* mean,
                                          float* rstd) {
  const float per = 1.f / static_cast<float>(channels);
  *mean = 0.f;
  if (kind == SNN_HIP_NORM_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < PT; ++i) s[0] += v[i];
    norm::row_sums<WAVES>(s, lds, turn);
    *mean = s[0] * per;
#pragma unroll
    for (int i = 0; i < PT; ++i)
      v[i] = S::inside(i, channels) ? v[i] - *mean : 0.f;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int i = 0; i < PT; ++i) q[0] += v[i] * v[i];
  norm::row_sums<WAVES>(q, lds, turn);
  *rstd = 1.f / sqrtf(q[0] * per + epsilon);
#pragma unroll
  for (int i = 0; i < PT; ++i) v[i] *= *rstd;
}

template <int PT>
__device__ __forceinline__ void scaled(float (&v)[PT], const float (&w)[PT]) {
#pragma unroll
  for (int i = 0; i < PT; ++i) v[i] *= w[i];
}
template <int PT>
__device__ __forceinline__ void shifted(float (&v)[PT], const float (&b)[PT]) {
#pragma unroll
  for (int i = 0; i < PT; ++i) v[i] += b[i];
}

template <typename T, int VEC, int PT, int WAVES, bool WHOLE>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES)
    residual_norm_kernel(Rows r) {
  typedef norm::Slice<T, VEC, PT, WAVES, WHOLE> S;
  __shared__ float lds[WAVES == 1 ? 1 : 4 * WAVES];
  int turn = 0;
  const long row = WAVES == 1
                       ? seq::group_of_grid() * 4l + (threadIdx.x >> 6)
                       : static_cast<long>(seq::group_of_grid());
  if (row >= r.rows) return;
  const int channels = r.channels;
  const long at = row * channels;
  auto tensor = [&](const void* p, long offset) {
    return static_cast<const void*>(static_cast<const T*>(p) + offset);
  };
  float v[PT], other[PT];
  S::load(tensor(r.t.x, row * r.x_stride), channels, v);
  float gate[PT];
  if (r.gate != SNN_HIP_GATE_NONE) {
    S::load(tensor(r.t.gate, row / r.gate_rows * r.gate_stride), channels, gate);
    if (r.gate != SNN_HIP_GATE_VALUE) {
      const bool silu = r.gate == SNN_HIP_GATE_SILU;
#pragma unroll
      for (int i = 0; i < PT; ++i)
        gate[i] = (silu ? gate[i] : 1.f) * seq::sigmoid_alone<T>(gate[i]);
    }
  }
  float residual[PT];
  if (r.t.residual != nullptr)
    S::load(tensor(r.t.residual, at), channels, residual);
  float mean0 = 0.f, rstd0 = 0.f, mean1 = 0.f, rstd1 = 0.f;
  if (r.post != SNN_HIP_NORM_NONE) {
    normalise<S, PT, WAVES>(v, r.post, channels, r.epsilon, lds, &turn, &mean0,
                            &rstd0);
    if (r.t.post_weight != nullptr) {
      S::load(r.t.post_weight, channels, other);
      scaled(v, other);
    }
    if (r.t.post_bias != nullptr) {
      S::load(r.t.post_bias, channels, other);
      shifted(v, other);
    }
  }
  if (r.gate != SNN_HIP_GATE_NONE) scaled(v, gate);
  if (r.t.scale != nullptr) {
    S::load(r.t.scale, channels, other);
    scaled(v, other);
  }
  if (r.t.residual != nullptr) shifted(v, residual);
  if (r.t.sum != nullptr)
    S::store(static_cast<T*>(r.t.sum) + at, channels, v);
  if (r.pre != SNN_HIP_NORM_NONE) {
    normalise<S, PT, WAVES>(v, r.pre, channels, r.epsilon, lds, &turn, &mean1,
                            &rstd1);
    if (r.t.pre_weight != nullptr) {
      S::load(r.t.pre_weight, channels, other);
      scaled(v, other);
    }
    if (r.t.pre_bias != nullptr) {
      S::load(r.t.pre_bias, channels, other);
      shifted(v, other);
    }
    if (r.t.normed != nullptr)
      S::store(static_cast<T*>(r.t.normed) + at, channels, v);
  }
  if (r.t.stats != nullptr && S::lane() == 0) {
    float* const s = r.t.stats + 4 * row;
    s[0] = mean0;
    s[1] = rstd0;
    s[2] = mean1;
    s[3] = rstd1;
  }
}

template <typename T, int VEC, int PT, int WAVES, bool WHOLE>
int launch_as(const Rows& r, hipStream_t stream) {
  const size_t rows = r.rows, groups = WAVES == 1 ? ceil_div(rows, size_t{4}) : rows;
  KernelTimer timer(stream);
  hipLaunchKernelGGL((residual_norm_kernel<T, VEC, PT, WAVES, WHOLE>),
                     seq::grid_of(groups), dim3(WAVES == 1 ? 256 : 64 * WAVES), 0, stream, r);
  SNN_HIP_CHECK_LAUNCH();
  return SNN_HIP_OK;
}

template <typename T>
int residual_norm(const snn_hip_residual_norm_tensors* tensors,
                  const snn_hip_residual_norm_params* params, void* stream) {
  int v = norm::check_params(params);
  if (v == SNN_HIP_OK) v = norm::check_operands(tensors, *params);
  if (v != SNN_HIP_OK) return v;
  const snn_hip_residual_norm_tensors& t = *tensors;
  SNN_REQUIRE(t.sum != nullptr || t.normed != nullptr);
  SNN_REQUIRE(t.normed == nullptr || params->pre_norm != SNN_HIP_NORM_NONE);
  const Rows r = norm::rows_of(t, *params);
  constexpr int VEC = 16 / sizeof(T);
  if (r.channels < VEC)
    return launch_as<T, 1, 8, 1, true>(r, as_stream(stream));
  return norm::by_channels<VEC>(
      r.channels, [&](auto waves, auto values, auto whole) {
        return launch_as<T, VEC, decltype(values)::value,
                         decltype(waves)::value, decltype(whole)::value>(
            r, as_stream(stream));
      });
}

}  // namespace
}  // namespace snn

extern "C" {

int snn_hip_residual_norm_f32(const snn_hip_residual_norm_tensors* tensors,
                              const snn_hip_residual_norm_params* params,
                              void* stream) {
  return snn::residual_norm<float>(tensors, params, stream);
}
int snn_hip_residual_norm_f16(const snn_hip_residual_norm_tensors* tensors,
                              const snn_hip_residual_norm_params* params,
                              void* stream) {
  return snn::residual_norm<_Float16>(tensors, params, stream);
}
int snn_hip_residual_norm_bf16(const snn_hip_residual_norm_tensors* tensors,
                               const snn_hip_residual_norm_params* params,
                               void* stream) {
  return snn::residual_norm<__bf16>(tensors, params, stream);
}

}  // extern "C"
