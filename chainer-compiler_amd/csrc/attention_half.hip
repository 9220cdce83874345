// float16
#include "attention_kernel.h"

template struct chx::AttentionKernels<true>;
