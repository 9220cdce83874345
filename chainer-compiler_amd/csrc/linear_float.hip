// float32 rows and weights.
#include "linear_kernel.h"

template struct chx::LinearKernels<chx::kFloatFloat>;
