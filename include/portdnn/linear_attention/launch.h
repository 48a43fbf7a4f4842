// Not a portDNN include path: in the form of those of its operators.
#ifndef SNN_FWD_LINEAR_ATTENTION_LAUNCH_H
#define SNN_FWD_LINEAR_ATTENTION_LAUNCH_H
#include "portdnn/hip/linear_attention_block.h"
#endif
