// Create-time validation of the paged_attention_prefill_fp4 operands: paged_attention_fp4's, with rows of several tokens per
// sequence and their prefix sums, checked as paged_attention_prefill checks them.
#ifndef INFINICORE_AMD_PAGED_ATTENTION_PREFILL_FP4_INFO_H
#define INFINICORE_AMD_PAGED_ATTENTION_PREFILL_FP4_INFO_H

#include "../paged_attention_fp4/info.h"

namespace op::paged_attention_prefill_fp4 {

struct PagedAttentionPrefillFp4Info : paged_attention_fp4::AttentionFp4Info {
    static utils::Result<PagedAttentionPrefillFp4Info> create(infiniopTensorDescriptor_t out_desc,
                                                              infiniopTensorDescriptor_t q_desc,
                                                              infiniopTensorDescriptor_t k_codes_desc,
                                                              infiniopTensorDescriptor_t v_codes_desc,
                                                              infiniopTensorDescriptor_t k_scales_desc,
                                                              infiniopTensorDescriptor_t v_scales_desc,
                                                              infiniopTensorDescriptor_t block_tables_desc,
                                                              infiniopTensorDescriptor_t seq_lens_desc,
                                                              infiniopTensorDescriptor_t cum_seq_lens_q_desc,
                                                              infiniopTensorDescriptor_t alibi_slopes_desc, float scale) {
        if (!cum_seq_lens_q_desc) {
            return INFINI_STATUS_NULL_POINTER;
        }
        auto base = AttentionFp4Info::create(out_desc, q_desc, k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc,
                                             block_tables_desc, seq_lens_desc, alibi_slopes_desc, scale);
        CHECK_RESULT(base);
        PagedAttentionPrefillFp4Info info{base.take()};
        if (cum_seq_lens_q_desc->dtype() != info.index_dtype) {
            return INFINI_STATUS_BAD_TENSOR_DTYPE;
        }
        if (cum_seq_lens_q_desc->ndim() != 1) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        if (cum_seq_lens_q_desc->dim(0) != info.num_seqs + 1) {
            return INFINI_STATUS_BAD_PARAM;
        }
        CHECK_OR_RETURN(cum_seq_lens_q_desc->stride(0) == 1 || info.num_seqs == 0, INFINI_STATUS_BAD_TENSOR_STRIDES);
        // rows of the grid and of a sequence are counted in 32 bits
        if (info.num_rows * info.num_heads > 0x3fffffff) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        return info;
    }
};

} // namespace op::paged_attention_prefill_fp4

#endif
