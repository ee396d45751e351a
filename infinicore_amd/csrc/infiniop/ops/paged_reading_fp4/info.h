// Create-time validation of the paged_reading_fp4 operands: the same tensors in the same relation as paged_caching_fp4's, with
// k and v as the outputs, which may not overlap themselves.
#ifndef INFINICORE_AMD_PAGED_READING_FP4_INFO_H
#define INFINICORE_AMD_PAGED_READING_FP4_INFO_H

#include "../paged_caching_fp4/info.h"

namespace op::paged_reading_fp4 {

struct PagedReadingFp4Info : paged_caching_fp4::PagedCachingFp4Info {
    static utils::Result<PagedReadingFp4Info> create(infiniopTensorDescriptor_t k_desc, infiniopTensorDescriptor_t v_desc,
                                                     infiniopTensorDescriptor_t k_codes_desc,
                                                     infiniopTensorDescriptor_t v_codes_desc,
                                                     infiniopTensorDescriptor_t k_scales_desc,
                                                     infiniopTensorDescriptor_t v_scales_desc,
                                                     infiniopTensorDescriptor_t slot_mapping_desc) {
        auto base = PagedCachingFp4Info::create(k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc, k_desc, v_desc,
                                                slot_mapping_desc);
        CHECK_RESULT(base);
        for (auto *d : {k_desc, v_desc}) { // broadcast rows: every token's or head's values would land on one another
            CHECK_OR_RETURN((d->dim(0) <= 1 || d->stride(0) != 0) && (d->dim(1) <= 1 || d->stride(1) != 0),
                            INFINI_STATUS_BAD_TENSOR_STRIDES);
        }
        return PagedReadingFp4Info{base.take()};
    }
};

} // namespace op::paged_reading_fp4

#endif
