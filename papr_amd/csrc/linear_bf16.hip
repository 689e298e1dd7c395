#include "linear_kernels.h"

PAPR_LINEAR_INSTANCES(bf16)
