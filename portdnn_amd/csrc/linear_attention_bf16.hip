// The kernels of linear_attention.h for bfloat16.
#include "linear_attention.h"

namespace snn {
namespace att {

int run_walks_bf16(const Problem& p, int keys_class, int waves, bool outputs,
                  hipStream_t stream) {
  return run_walks<__bf16>(p, keys_class, waves, outputs, stream);
}

}  // namespace att
}  // namespace snn
