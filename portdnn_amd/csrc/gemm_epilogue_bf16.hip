// gemm_epilogue.h for __bf16.
#include "gemm_epilogue_run.h"

namespace snn {
namespace epi {

int run_bf16(Product& g, void* workspace, size_t bytes, hipStream_t stream) {
  return run<__bf16>(g, workspace, bytes, stream);
}

}  // namespace epi
}  // namespace snn
