// float16 rows, int8 weights.
#include "linear_kernel.h"

template struct chx::LinearKernels<chx::kHalfInt8>;
