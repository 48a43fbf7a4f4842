// Not in portDNN: the operators of a linear-attention block on the HIP backend, in
// the form of its launches.  What they compute, their shapes and what may be null
// stand with their entry points in snn_hip.h.
#ifndef PORTDNN_HIP_LINEAR_ATTENTION_BLOCK_H_
#define PORTDNN_HIP_LINEAR_ATTENTION_BLOCK_H_

#include <vector>

#include "portdnn/hip/residual_block.h"

namespace sycldnn {
namespace gated_matmul {

using Params = snn_hip_gated_matmul_params;

struct WorkspaceSize {
  size_t required_size;     // elements of T
  size_t recommended_size;  // elements of T
};

// Of launch, or of launch_grad.
template <typename T>
WorkspaceSize query_workspace_size(Params const& params, bool grad = false) {
  WorkspaceSize ws{0, 0};
  (void)snn_hip_gated_matmul_workspace_size(
      &params, grad, hip::detail::data_type<T>(), &ws.required_size,
      &ws.recommended_size);
  return ws;
}

// output = act(lhs gate_weight + gate_bias) * (lhs up_weight + up_bias).
template <typename T, typename Backend>
SNNStatus launch(typename Backend::template pointer_type<T const> lhs,
                 typename Backend::template pointer_type<T const> gate_weight,
                 typename Backend::template pointer_type<T const> up_weight,
                 typename Backend::template pointer_type<T const> gate_bias,
                 typename Backend::template pointer_type<T const> up_bias,
                 typename Backend::template pointer_type<T> output,
                 typename Backend::template pointer_type<T> gate,
                 typename Backend::template pointer_type<T> up,
                 Params const& params, Backend& backend,
                 typename Backend::template pointer_type<T> workspace,
                 size_t workspace_size,
                 const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_gated_matmul_f32, snn_hip_gated_matmul_f16,
                            snn_hip_gated_matmul_bf16),
      lhs, gate_weight, up_weight, gate_bias, up_bias, output, gate, up, &params,
      workspace, workspace_size);
}

// The gradients of the five operands; those that are null are left out.
template <typename T, typename Backend>
SNNStatus launch_grad(
    typename Backend::template pointer_type<T const> grad_output,
    typename Backend::template pointer_type<T const> lhs,
    typename Backend::template pointer_type<T const> gate_weight,
    typename Backend::template pointer_type<T const> up_weight,
    typename Backend::template pointer_type<T const> gate,
    typename Backend::template pointer_type<T const> up,
    typename Backend::template pointer_type<T> grad_lhs,
    typename Backend::template pointer_type<T> grad_gate_weight,
    typename Backend::template pointer_type<T> grad_up_weight,
    typename Backend::template pointer_type<T> grad_gate_bias,
    typename Backend::template pointer_type<T> grad_up_bias,
    Params const& params, Backend& backend,
    typename Backend::template pointer_type<T> workspace, size_t workspace_size,
    const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_gated_matmul_grad_f32,
                            snn_hip_gated_matmul_grad_f16,
                            snn_hip_gated_matmul_grad_bf16),
      grad_output, lhs, gate_weight, up_weight, gate, up, grad_lhs,
      grad_gate_weight, grad_up_weight, grad_gate_bias, grad_up_bias, &params,
      workspace, workspace_size);
}

}  // namespace gated_matmul

namespace rotary {

using Params = snn_hip_rotary_params;

// Positions by rotation; the gradient is the launch with params.inverse.
template <typename T, typename Backend>
SNNStatus launch(
    typename Backend::template pointer_type<T const> input,
    typename Backend::template pointer_type<double const> frequencies,
    typename Backend::template pointer_type<int const> positions,
    typename Backend::template pointer_type<T> output, Params const& params,
    Backend& backend, const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_rotary_f32, snn_hip_rotary_f16,
                            snn_hip_rotary_bf16),
      input, frequencies, positions, output, &params);
}

// The table of launch, in host memory.
inline StatusCode frequencies(int turned, double base, double* table,
                              snn_hip_rotary_scaling scaling =
                                  SNN_HIP_ROTARY_SCALING_NONE,
                              double factor = 1.0, double context = 0.0,
                              double low = 1.0, double high = 32.0) {
  return static_cast<StatusCode>(snn_hip_rotary_frequencies(
      turned, base, scaling, factor, context, low, high, table));
}

}  // namespace rotary

namespace linear_attention {

using Params = snn_hip_linear_attention_params;

struct WorkspaceSize {
  size_t required_size;     // elements of T
  size_t recommended_size;  // elements of T
};

// Of launch, or of launch_grad.
template <typename T>
WorkspaceSize query_workspace_size(Params const& params, bool grad = false) {
  WorkspaceSize ws{0, 0};
  (void)snn_hip_linear_attention_workspace_size(
      &params, grad, hip::detail::data_type<T>(), &ws.required_size,
      &ws.recommended_size);
  return ws;
}

// S_t = exp(decay) S_{t-1} + k_t^T v_t, o_t = scale q_t S_t.
template <typename T, typename Backend>
SNNStatus launch(
    typename Backend::template pointer_type<T const> q,
    typename Backend::template pointer_type<T const> k,
    typename Backend::template pointer_type<T const> v,
    typename Backend::template pointer_type<float const> decay,
    typename Backend::template pointer_type<unsigned char const> resets,
    typename Backend::template pointer_type<int const> lengths,
    typename Backend::template pointer_type<float const> initial_state,
    typename Backend::template pointer_type<T> output,
    typename Backend::template pointer_type<float> final_state,
    Params const& params, Backend& backend,
    typename Backend::template pointer_type<T> workspace, size_t workspace_size,
    const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_linear_attention_f32,
                            snn_hip_linear_attention_f16,
                            snn_hip_linear_attention_bf16),
      q, k, v, decay, resets, lengths, initial_state, output, final_state,
      &params, workspace, workspace_size);
}

template <typename T, typename Backend>
SNNStatus launch_grad(
    typename Backend::template pointer_type<T const> grad_output,
    typename Backend::template pointer_type<float const> grad_final_state,
    typename Backend::template pointer_type<T const> q,
    typename Backend::template pointer_type<T const> k,
    typename Backend::template pointer_type<T const> v,
    typename Backend::template pointer_type<float const> decay,
    typename Backend::template pointer_type<unsigned char const> resets,
    typename Backend::template pointer_type<int const> lengths,
    typename Backend::template pointer_type<float const> initial_state,
    typename Backend::template pointer_type<T> grad_q,
    typename Backend::template pointer_type<T> grad_k,
    typename Backend::template pointer_type<T> grad_v,
    typename Backend::template pointer_type<float> grad_initial_state,
    Params const& params, Backend& backend,
    typename Backend::template pointer_type<T> workspace, size_t workspace_size,
    const std::vector<hip::Event>& events = {}) {
  return hip::detail::call(
      backend, events,
      hip::detail::entry<T>(snn_hip_linear_attention_grad_f32,
                            snn_hip_linear_attention_grad_f16,
                            snn_hip_linear_attention_grad_bf16),
      grad_output, grad_final_state, q, k, v, decay, resets, lengths,
      initial_state, grad_q, grad_k, grad_v, grad_initial_state, &params,
      workspace, workspace_size);
}

}  // namespace linear_attention
}  // namespace sycldnn

#endif  // PORTDNN_HIP_LINEAR_ATTENTION_BLOCK_H_
