#ifndef INFINICORE_AMD_PAGED_ATTENTION_FP4_AMD_H
#define INFINICORE_AMD_PAGED_ATTENTION_FP4_AMD_H

#include "../paged_attention_fp4.h"

DESCRIPTOR(amd)

#endif
