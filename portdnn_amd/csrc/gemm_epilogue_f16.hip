// gemm_epilogue.h for _Float16.
#include "gemm_epilogue_run.h"

namespace snn {
namespace epi {

int run_f16(Product& g, void* workspace, size_t bytes, hipStream_t stream) {
  return run<_Float16>(g, workspace, bytes, stream);
}

}  // namespace epi
}  // namespace snn
