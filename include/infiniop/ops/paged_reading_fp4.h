/*
 * Tokens of a paged pool held in 4 bits, read back as the values they stand for: the inverse of
 * infiniopPagedCachingFp4, whose header describes the pool.
 *
 * Tensors (strides in elements; the innermost dimension packed everywhere):
 *   k             [num_tokens, num_kv_heads, head_size]   out, F16 | BF16 | F32, any token and head strides but 0
 *   v             [num_tokens, num_kv_heads, value_size]  out, same dtype
 *   k_codes       [num_blocks, num_kv_heads, block_size, head_size / 2]    U8, any strides on dims 0-2
 *   v_codes       [num_blocks, num_kv_heads, block_size, value_size / 2]   U8
 *   k_scales      [num_blocks, num_kv_heads, block_size, head_size / 32]   U8
 *   v_scales      [num_blocks, num_kv_heads, block_size, value_size / 32]  U8
 *   slot_mapping  [num_tokens] I64, contiguous; the same slot may be read any number of times
 *
 * Row i of k and v becomes the values e2m1(code) * 2^(s - 127) of slot slot_mapping[i], rounded once to the outputs'
 * type (exact for every pool that infiniopPagedCachingFp4 wrote); NaN where s = 255. A slot that is negative (padding) or
 * past the pool reads as zeros.
 */
#ifndef INFINICORE_AMD_INFINIOP_PAGED_READING_FP4_H
#define INFINICORE_AMD_INFINIOP_PAGED_READING_FP4_H

#include "../operator_descriptor.h"

typedef struct InfiniopDescriptor *infiniopPagedReadingFp4Descriptor_t;

__INFINI_C __export infiniStatus_t infiniopCreatePagedReadingFp4Descriptor(
    infiniopHandle_t handle,
    infiniopPagedReadingFp4Descriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc,
    infiniopTensorDescriptor_t k_codes_desc,
    infiniopTensorDescriptor_t v_codes_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t slot_mapping_desc);

/* Always reports 0. */
__INFINI_C __export infiniStatus_t infiniopGetPagedReadingFp4WorkspaceSize(
    infiniopPagedReadingFp4Descriptor_t desc,
    size_t *size);

/* Enqueues on `stream`; BAD_PARAM where the calling thread's current device is not the descriptor's. */
__INFINI_C __export infiniStatus_t infiniopPagedReadingFp4(
    infiniopPagedReadingFp4Descriptor_t desc,
    void *workspace,
    size_t workspace_size,
    void *k,
    void *v,
    const void *k_codes,
    const void *v_codes,
    const void *k_scales,
    const void *v_scales,
    const void *slot_mapping,
    void *stream);

__INFINI_C __export infiniStatus_t infiniopDestroyPagedReadingFp4Descriptor(
    infiniopPagedReadingFp4Descriptor_t desc);

#endif /* INFINICORE_AMD_INFINIOP_PAGED_READING_FP4_H */
