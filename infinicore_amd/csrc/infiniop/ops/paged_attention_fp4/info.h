// Create-time validation of the paged_attention_fp4 operands and capture of every size and stride the decode needs. Checks,
// their order and statuses follow paged_attention's; the pool's tensors are checked by fp4_pool.h.
#ifndef INFINICORE_AMD_PAGED_ATTENTION_FP4_INFO_H
#define INFINICORE_AMD_PAGED_ATTENTION_FP4_INFO_H

#include "../fp4_pool.h"

namespace op::paged_attention_fp4 {

// What decode and prefill over the pool have in common.
struct AttentionFp4Info {
    infiniDtype_t dtype;       // F16 or BF16: q and out
    infiniDtype_t index_dtype; // I64, I32 or U32: block_tables and lengths
    float scale;
    bool has_alibi;
    fp4::PoolInfo pool;
    size_t num_seqs;
    size_t num_rows; // of q and out
    size_t num_heads;
    size_t head_size;
    size_t max_num_blocks_per_seq;
    // element strides
    ptrdiff_t q_stride, q_head_stride;
    ptrdiff_t o_stride, o_head_stride;
    ptrdiff_t block_table_batch_stride;

    static bool isIndexDtype(infiniDtype_t dt) {
        return dt == INFINI_DTYPE_I64 || dt == INFINI_DTYPE_I32 || dt == INFINI_DTYPE_U32;
    }

    // `lens_desc`: tokens of the sequences
    static utils::Result<AttentionFp4Info> create(infiniopTensorDescriptor_t out_desc, infiniopTensorDescriptor_t q_desc,
                                                  infiniopTensorDescriptor_t k_codes_desc,
                                                  infiniopTensorDescriptor_t v_codes_desc,
                                                  infiniopTensorDescriptor_t k_scales_desc,
                                                  infiniopTensorDescriptor_t v_scales_desc,
                                                  infiniopTensorDescriptor_t block_tables_desc,
                                                  infiniopTensorDescriptor_t lens_desc,
                                                  infiniopTensorDescriptor_t alibi_slopes_desc, // may be null
                                                  float scale) {
        if (!out_desc || !q_desc || !block_tables_desc || !lens_desc) {
            return INFINI_STATUS_NULL_POINTER;
        }
        const infiniDtype_t dtype = q_desc->dtype();
        CHECK_DTYPE(dtype, INFINI_DTYPE_F16, INFINI_DTYPE_BF16);
        if (out_desc->dtype() != dtype) {
            return INFINI_STATUS_BAD_TENSOR_DTYPE;
        }
        if (q_desc->ndim() != 3 || out_desc->ndim() != 3 || block_tables_desc->ndim() != 2 || lens_desc->ndim() != 1) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        CHECK_OR_RETURN(q_desc->stride(2) == 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        CHECK_OR_RETURN(out_desc->stride(2) == 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        auto pool = fp4::PoolInfo::create(k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc);
        CHECK_RESULT(pool);
        if (!isIndexDtype(block_tables_desc->dtype()) || lens_desc->dtype() != block_tables_desc->dtype()) {
            return INFINI_STATUS_BAD_TENSOR_DTYPE;
        }
        CHECK_OR_RETURN(block_tables_desc->stride(1) == 1 || block_tables_desc->dim(1) <= 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        CHECK_OR_RETURN(lens_desc->stride(0) == 1 || lens_desc->dim(0) <= 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        if (alibi_slopes_desc != nullptr) {
            if (alibi_slopes_desc->dtype() != INFINI_DTYPE_F32) {
                return INFINI_STATUS_BAD_TENSOR_DTYPE;
            }
            if (alibi_slopes_desc->ndim() != 1) {
                return INFINI_STATUS_BAD_TENSOR_SHAPE;
            }
            CHECK_OR_RETURN(alibi_slopes_desc->stride(0) == 1 || alibi_slopes_desc->dim(0) <= 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        }

        AttentionFp4Info info{};
        info.dtype = dtype;
        info.index_dtype = block_tables_desc->dtype();
        info.scale = scale;
        info.has_alibi = alibi_slopes_desc != nullptr;
        info.pool = pool.take();
        info.num_seqs = lens_desc->dim(0);
        info.num_rows = q_desc->dim(0);
        info.num_heads = q_desc->dim(1);
        info.head_size = q_desc->dim(2);
        info.max_num_blocks_per_seq = block_tables_desc->dim(1);
        const size_t hs = info.head_size;
        if (hs != 64 && hs != 128 && hs != 192 && hs != 256) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        if (info.pool.k_size != hs || info.pool.v_size != hs) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        if (info.pool.num_kv_heads == 0 || info.num_heads % info.pool.num_kv_heads != 0 || info.pool.block_size == 0) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        for (size_t i = 0; i < 3; ++i) {
            if (out_desc->dim(i) != q_desc->dim(i)) {
                return INFINI_STATUS_BAD_TENSOR_SHAPE;
            }
        }
        if (block_tables_desc->dim(0) < info.num_seqs
            || (alibi_slopes_desc != nullptr && alibi_slopes_desc->dim(0) < info.num_heads)) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        // the kernels load 16 bytes of codes and up to four scales at a time, and their offsets inside a page are of 32 bits
        CHECK_OR_RETURN(info.pool.codeRowsAligned(16), INFINI_STATUS_BAD_TENSOR_STRIDES);
        CHECK_OR_RETURN(info.pool.scaleRowsAligned(info.scaleBytes()), INFINI_STATUS_BAD_TENSOR_STRIDES);
        const fp4::PoolInfo &p = info.pool;
        for (ptrdiff_t row : {p.k_codes.row, p.v_codes.row, p.k_scales.row, p.v_scales.row}) {
            CHECK_OR_RETURN(row >= 0 && row <= 0xffffff, INFINI_STATUS_BAD_TENSOR_STRIDES);
            CHECK_OR_RETURN(p.block_size <= 0x7fffffff / static_cast<size_t>(row > 0 ? row : 1), INFINI_STATUS_BAD_TENSOR_STRIDES);
        }
        // outputs of two rows or heads at one place would be written by different wavefronts
        CHECK_OR_RETURN((out_desc->dim(0) <= 1 || out_desc->stride(0) != 0) && (out_desc->dim(1) <= 1 || out_desc->stride(1) != 0),
                        INFINI_STATUS_BAD_TENSOR_STRIDES);
        // counted in 32 bits
        if (info.num_seqs > 0xffff || info.num_heads > 0xffff || info.num_rows > 0x3fffffff || p.block_size > 0xffffff
            || info.max_num_blocks_per_seq > 0x3fffffff) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        info.q_stride = q_desc->stride(0);
        info.q_head_stride = q_desc->stride(1);
        info.o_stride = out_desc->stride(0);
        info.o_head_stride = out_desc->stride(1);
        info.block_table_batch_stride = block_tables_desc->stride(0);
        return info;
    }

    // Scales that are loaded at a time: a row's, where it has two or four, else a part of them.
    size_t scaleBytes() const { return head_size % 128 == 0 ? 4 : 2; }

    // Tokens that a row of the block table can hold, at most 2^30.
    int capacity() const {
        const size_t tokens = max_num_blocks_per_seq * pool.block_size;
        return static_cast<int>(tokens < (size_t{1} << 30) ? tokens : (size_t{1} << 30));
    }
};

struct PagedAttentionFp4Info : AttentionFp4Info {
    static utils::Result<PagedAttentionFp4Info> create(infiniopTensorDescriptor_t out_desc, infiniopTensorDescriptor_t q_desc,
                                                       infiniopTensorDescriptor_t k_codes_desc,
                                                       infiniopTensorDescriptor_t v_codes_desc,
                                                       infiniopTensorDescriptor_t k_scales_desc,
                                                       infiniopTensorDescriptor_t v_scales_desc,
                                                       infiniopTensorDescriptor_t block_tables_desc,
                                                       infiniopTensorDescriptor_t seq_lens_desc,
                                                       infiniopTensorDescriptor_t alibi_slopes_desc, float scale) {
        auto base = AttentionFp4Info::create(out_desc, q_desc, k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc,
                                             block_tables_desc, seq_lens_desc, alibi_slopes_desc, scale);
        CHECK_RESULT(base);
        PagedAttentionFp4Info info{base.take()};
        if (info.num_seqs != info.num_rows) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        return info;
    }
};

} // namespace op::paged_attention_fp4

#endif
