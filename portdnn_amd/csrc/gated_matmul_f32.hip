// gated_matmul.h for float.
#include "gated_matmul_run.h"

namespace snn {
namespace gated {

int run_f32(Pair& g, void* workspace, size_t bytes, hipStream_t stream) {
  return run<float>(g, workspace, bytes, stream);
}

}  // namespace gated
}  // namespace snn
