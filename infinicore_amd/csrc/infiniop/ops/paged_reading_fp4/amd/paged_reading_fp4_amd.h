#ifndef INFINICORE_AMD_PAGED_READING_FP4_AMD_H
#define INFINICORE_AMD_PAGED_READING_FP4_AMD_H

#include "../paged_reading_fp4.h"

DESCRIPTOR(amd)

#endif
