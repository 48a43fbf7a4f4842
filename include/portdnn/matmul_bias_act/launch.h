// Not a portDNN include path: in the form of those of its operators.
#ifndef SNN_FWD_MATMUL_BIAS_ACT_LAUNCH_H
#define SNN_FWD_MATMUL_BIAS_ACT_LAUNCH_H
#include "portdnn/hip/residual_block.h"
#endif
