#ifndef INFINICORE_AMD_PAGED_CACHING_FP4_AMD_H
#define INFINICORE_AMD_PAGED_CACHING_FP4_AMD_H

#include "../paged_caching_fp4.h"

DESCRIPTOR(amd)

#endif
