// The kernels of linear_attention.h for fp32.
#include "linear_attention.h"

namespace snn {
namespace att {

int run_walks_f32(const Problem& p, int keys_class, int waves, bool outputs,
                 hipStream_t stream) {
  return run_walks<float>(p, keys_class, waves, outputs, stream);
}

}  // namespace att
}  // namespace snn
