// Not in portDNN: the operators of a residual block over sequences on the HIP
// backend, in the form of its launches.  What they compute, their shapes and
// what may be null stand with their entry points in snn_hip.h.
#ifndef PORTDNN_HIP_RESIDUAL_BLOCK_H_
#define PORTDNN_HIP_RESIDUAL_BLOCK_H_

#include <cstdint>
#include <type_traits>
#include <vector>

#include "portdnn/hip/core.h"
#include "snn_hip.h"

namespace sycldnn {

// The storage of a bfloat16 value.  Launches take it as their element type;
// any other type of two bytes is binary16.
struct bfloat16 {
  std::uint16_t bits;
};

namespace hip {
namespace detail {

template <typename T>
constexpr int data_type() {
  static_assert(std::is_same<T, float>::value || sizeof(T) == 2,
                "supported data types: float, half and bfloat16");
  return std::is_same<T, float>::value      ? SNN_HIP_DTYPE_F32
         : std::is_same<T, bfloat16>::value ? SNN_HIP_DTYPE_BF16
                                            : SNN_HIP_DTYPE_F16;
}

// The entry point of element type T.
template <typename T, typename F>
constexpr F* entry(F* f32, F* f16, F* bf16) {
  return data_type<T>() == SNN_HIP_DTYPE_F32   ? f32
         : data_type<T>() == SNN_HIP_DTYPE_F16 ? f16
                                               : bf16;
}

// Waits for `events`, calls the entry point, records what ends it.
template <typename Backend, typename F, typename... Args>
SNNStatus call(Backend& backend, const std::vector<Event>& events, F* f,
               Args... args) {
  hipStream_t stream = backend.get_stream();
  wait_for(stream, events);
  return finish(f(args..., stream), stream);
}

}  // namespace detail
}  // namespace hip

namespace matmul_bias_act {

using Params = snn_hip_matmul_bias_act_params;

struct WorkspaceSize {
  size_t required_size;     // elements of T
  size_t recommended_size;  // elements of T
};

// Of launch, or of launch_grad.
template <typename T>
WorkspaceSize query_workspace_size(Params const& params, bool grad = false) {
  WorkspaceSize ws{0, 0};
  (void)snn_hip_matmul_bias_act_workspace_size(
      &params, grad, hip::detail::data_type<T>(), &ws.required_size,
      &ws.recommended_size);
  return ws;
}

// output = act(op(lhs) op(rhs) + bias) + residual.
template <typename T, typename Backend>
SNNStatus launch(typename Backend::template pointer_type<T const> lhs,
                 typename Backend::template pointer_type<T const> rhs,
                 typename Backend::template pointer_type<T const> bias,
                 typename Backend::template pointer_type<T const> residual,
                 typename Backend::template pointer_type<T> output,
                 typename Backend::template pointer_type<T> pre_activation,
                 Params const& params, Backend& backend,
                 typename Backend::template pointer_type<T> workspace,
                 size_t workspace_size,
                 const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_matmul_bias_act_f32,
                            snn_hip_matmul_bias_act_f16,
                            snn_hip_matmul_bias_act_bf16),
      lhs, rhs, bias, residual, output, pre_activation, &params, workspace,
      workspace_size);
}

// The gradients of lhs, rhs and bias; those that are null are left out.
template <typename T, typename Backend>
SNNStatus launch_grad(
    typename Backend::template pointer_type<T const> grad_output,
    typename Backend::template pointer_type<T const> lhs,
    typename Backend::template pointer_type<T const> rhs,
    typename Backend::template pointer_type<T const> pre_activation,
    typename Backend::template pointer_type<T> grad_lhs,
    typename Backend::template pointer_type<T> grad_rhs,
    typename Backend::template pointer_type<T> grad_bias, Params const& params,
    Backend& backend, typename Backend::template pointer_type<T> workspace,
    size_t workspace_size, const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_matmul_bias_act_grad_f32,
                            snn_hip_matmul_bias_act_grad_f16,
                            snn_hip_matmul_bias_act_grad_bf16),
      grad_output, lhs, rhs, pre_activation, grad_lhs, grad_rhs, grad_bias,
      &params, workspace, workspace_size);
}

}  // namespace matmul_bias_act

namespace residual_norm {

using Params = snn_hip_residual_norm_params;
using Tensors = snn_hip_residual_norm_tensors;  // of elements T
using Gradients = snn_hip_residual_norm_gradients;

struct WorkspaceSize {
  size_t required_size;     // elements of T
  size_t recommended_size;  // elements of T
};

// Of launch_grad; launch takes none.
template <typename T>
WorkspaceSize query_grad_workspace_size(Params const& params) {
  WorkspaceSize ws{0, 0};
  (void)snn_hip_residual_norm_grad_workspace_size(
      &params, hip::detail::data_type<T>(), &ws.required_size,
      &ws.recommended_size);
  return ws;
}

// sum = residual + scale * gate * post_norm(x), normed = pre_norm(sum).
template <typename T, typename Backend>
SNNStatus launch(Tensors const& tensors, Params const& params, Backend& backend,
                 const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_residual_norm_f32,
                            snn_hip_residual_norm_f16,
                            snn_hip_residual_norm_bf16),
      &tensors, &params);
}

template <typename T, typename Backend>
SNNStatus launch_grad(Tensors const& tensors, Gradients const& gradients,
                      Params const& params, Backend& backend,
                      typename Backend::template pointer_type<T> workspace,
                      size_t workspace_size,
                      const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_residual_norm_grad_f32,
                            snn_hip_residual_norm_grad_f16,
                            snn_hip_residual_norm_grad_bf16),
      &tensors, &gradients, &params, workspace, workspace_size);
}

}  // namespace residual_norm

namespace linear_recurrence {

using Params = snn_hip_linear_recurrence_params;

struct WorkspaceSize {
  size_t required_size;     // elements of T
  size_t recommended_size;  // elements of T
};

// Of launch and launch_grad alike.
template <typename T>
WorkspaceSize query_workspace_size(Params const& params) {
  WorkspaceSize ws{0, 0};
  (void)snn_hip_linear_recurrence_workspace_size(
      &params, hip::detail::data_type<T>(), &ws.required_size,
      &ws.recommended_size);
  return ws;
}

// h_t = sigmoid(forget_t) h_{t-1} + w_t x_t.
template <typename T, typename Backend>
SNNStatus launch(
    typename Backend::template pointer_type<T const> x,
    typename Backend::template pointer_type<T const> forget,
    typename Backend::template pointer_type<T const> input_gate,
    typename Backend::template pointer_type<unsigned char const> resets,
    typename Backend::template pointer_type<int const> lengths,
    typename Backend::template pointer_type<float const> initial_state,
    typename Backend::template pointer_type<T> h,
    typename Backend::template pointer_type<float> final_state,
    Params const& params, Backend& backend,
    typename Backend::template pointer_type<T> workspace,
    size_t workspace_size, const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_linear_recurrence_f32,
                            snn_hip_linear_recurrence_f16,
                            snn_hip_linear_recurrence_bf16),
      x, forget, input_gate, resets, lengths, initial_state, h, final_state,
      &params, workspace, workspace_size);
}

template <typename T, typename Backend>
SNNStatus launch_grad(
    typename Backend::template pointer_type<T const> grad_h,
    typename Backend::template pointer_type<float const> grad_final_state,
    typename Backend::template pointer_type<T const> x,
    typename Backend::template pointer_type<T const> forget,
    typename Backend::template pointer_type<T const> input_gate,
    typename Backend::template pointer_type<unsigned char const> resets,
    typename Backend::template pointer_type<int const> lengths,
    typename Backend::template pointer_type<float const> initial_state,
    typename Backend::template pointer_type<T const> h,
    typename Backend::template pointer_type<T> grad_x,
    typename Backend::template pointer_type<T> grad_forget,
    typename Backend::template pointer_type<T> grad_input_gate,
    typename Backend::template pointer_type<float> grad_initial_state,
    Params const& params, Backend& backend,
    typename Backend::template pointer_type<T> workspace,
    size_t workspace_size, const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_linear_recurrence_grad_f32,
                            snn_hip_linear_recurrence_grad_f16,
                            snn_hip_linear_recurrence_grad_bf16),
      grad_h, grad_final_state, x, forget, input_gate, resets, lengths,
      initial_state, h, grad_x, grad_forget, grad_input_gate,
      grad_initial_state, &params, workspace, workspace_size);
}

}  // namespace linear_recurrence
}  // namespace sycldnn

#endif  // PORTDNN_HIP_RESIDUAL_BLOCK_H_
