// float16 rows, float16 weights.
#include "linear_kernel.h"

template struct chx::LinearKernels<chx::kHalfHalf>;
