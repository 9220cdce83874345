// float32
#include "attention_kernel.h"

template struct chx::AttentionKernels<false>;
