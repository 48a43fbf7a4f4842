// gated_matmul.h for __bf16.
#include "gated_matmul_run.h"

namespace snn {
namespace gated {

int run_bf16(Pair& g, void* workspace, size_t bytes, hipStream_t stream) {
  return run<__bf16>(g, workspace, bytes, stream);
}

}  // namespace gated
}  // namespace snn
