// Create-time validation of the paged_caching_fp4 operands and capture of every size and stride the kernel needs. The order
// of the checks is that of paged_caching: null descriptors, types, ranks and sizes, strides.
#ifndef INFINICORE_AMD_PAGED_CACHING_FP4_INFO_H
#define INFINICORE_AMD_PAGED_CACHING_FP4_INFO_H

#include "../fp4_pool.h"

namespace op::paged_caching_fp4 {

struct PagedCachingFp4Info {
    infiniDtype_t dtype; // F16, BF16 or F32: k and v
    fp4::PoolInfo pool;
    size_t num_tokens;
    // element strides
    ptrdiff_t k_token_stride, k_head_stride;
    ptrdiff_t v_token_stride, v_head_stride;

    static utils::Result<PagedCachingFp4Info> create(infiniopTensorDescriptor_t k_codes_desc,
                                                     infiniopTensorDescriptor_t v_codes_desc,
                                                     infiniopTensorDescriptor_t k_scales_desc,
                                                     infiniopTensorDescriptor_t v_scales_desc,
                                                     infiniopTensorDescriptor_t k_desc, infiniopTensorDescriptor_t v_desc,
                                                     infiniopTensorDescriptor_t slot_mapping_desc) {
        if (!k_desc || !v_desc || !slot_mapping_desc) {
            return INFINI_STATUS_NULL_POINTER;
        }
        auto pool = fp4::PoolInfo::create(k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc);
        CHECK_RESULT(pool);
        PagedCachingFp4Info info{};
        info.pool = pool.take();
        info.dtype = k_desc->dtype();
        CHECK_DTYPE(info.dtype, INFINI_DTYPE_F16, INFINI_DTYPE_BF16, INFINI_DTYPE_F32);
        if (v_desc->dtype() != info.dtype || slot_mapping_desc->dtype() != INFINI_DTYPE_I64) {
            return INFINI_STATUS_BAD_TENSOR_DTYPE;
        }
        if (k_desc->ndim() != 3 || v_desc->ndim() != 3 || slot_mapping_desc->ndim() != 1) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        info.num_tokens = slot_mapping_desc->dim(0);
        if (k_desc->dim(0) != info.num_tokens || v_desc->dim(0) != info.num_tokens
            || k_desc->dim(1) != info.pool.num_kv_heads || v_desc->dim(1) != info.pool.num_kv_heads
            || k_desc->dim(2) != info.pool.k_size || v_desc->dim(2) != info.pool.v_size) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        // counted in 32 bits, 65 535 workgroups of 256 lanes of eight elements to a token
        if (info.num_tokens > 0x3fffffff || info.pool.num_kv_heads > 0x7fff800 || info.pool.k_size + info.pool.v_size > 0x7fff800
            || info.pool.num_kv_heads * (info.pool.k_size + info.pool.v_size) > 0x7fff800) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        CHECK_OR_RETURN(k_desc->stride(2) == 1 || k_desc->dim(2) == 0, INFINI_STATUS_BAD_TENSOR_STRIDES);
        CHECK_OR_RETURN(v_desc->stride(2) == 1 || v_desc->dim(2) == 0, INFINI_STATUS_BAD_TENSOR_STRIDES);
        CHECK_OR_RETURN(slot_mapping_desc->stride(0) == 1 || info.num_tokens <= 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        info.k_token_stride = k_desc->stride(0);
        info.k_head_stride = k_desc->stride(1);
        info.v_token_stride = v_desc->stride(0);
        info.v_head_stride = v_desc->stride(1);
        return info;
    }
};

} // namespace op::paged_caching_fp4

#endif
