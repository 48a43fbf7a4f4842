// gemm_epilogue.h for float.
#include "gemm_epilogue_run.h"

namespace snn {
namespace epi {

int run_f32(Product& g, void* workspace, size_t bytes, hipStream_t stream) {
  return run<float>(g, workspace, bytes, stream);
}

}  // namespace epi
}  // namespace snn
