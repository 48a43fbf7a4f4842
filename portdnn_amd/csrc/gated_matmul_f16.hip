// gated_matmul.h for _Float16.
#include "gated_matmul_run.h"

namespace snn {
namespace gated {

int run_f16(Pair& g, void* workspace, size_t bytes, hipStream_t stream) {
  return run<_Float16>(g, workspace, bytes, stream);
}

}  // namespace gated
}  // namespace snn
