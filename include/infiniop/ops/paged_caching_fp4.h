/*
 * Paged caching into a pool held in 4 bits: quantise freshly computed K/V vectors of a chunk of tokens
 * and scatter them into their slots.
 *
 * Tensors (strides in elements; the innermost dimension packed everywhere):
 *   k_codes       [num_blocks, num_kv_heads, block_size, head_size / 2]    U8, any strides on dims 0-2
 *   v_codes       [num_blocks, num_kv_heads, block_size, value_size / 2]   U8
 *   k_scales      [num_blocks, num_kv_heads, block_size, head_size / 32]   U8
 *   v_scales      [num_blocks, num_kv_heads, block_size, value_size / 32]  U8
 *   k             [num_tokens, num_kv_heads, head_size]   F16 | BF16 | F32, any token and head strides
 *   v             [num_tokens, num_kv_heads, value_size]  same dtype
 *   slot_mapping  [num_tokens] I64, contiguous
 * Sizes are multiples of 32.
 *
 * The format is the 4-bit one of the OCP microscaling (MX) specification: a byte of codes holds two e2m1
 * floats, the even element in its low half (bit 3 sign; magnitudes of codes 0..7: 0, 0.5, 1, 1.5, 2, 3, 4, 6), and
 * 32 neighbouring elements share one scale byte s, which stands for 2^(s - 127). A group is written with
 *   s = 127 + clamp(floor(log2(largest magnitude)) - 2, -23, 13),
 * its elements rounded to the nearest (ties to the even code, magnitudes over 6 held at 6, the sign kept). With
 * exponents in that range every stored value is exact in F16 as in BF16: magnitudes over 49152 are held there, groups
 * below 2^-21 lose elements below 2^-25 (half of the smallest F16). A group with an infinity or a NaN is written as scale
 * 255 with codes 0, and reads as NaN.
 *
 * Token i goes to page slot_mapping[i] / block_size, row slot_mapping[i] % block_size, for every KV
 * head; a negative slot marks padding and is skipped, one past the pool is dropped. Bytes of the pool that no slot
 * names are not touched. Two tokens of a call that name the same slot race: what that slot then holds may be of both.
 */
#ifndef INFINICORE_AMD_INFINIOP_PAGED_CACHING_FP4_H
#define INFINICORE_AMD_INFINIOP_PAGED_CACHING_FP4_H

#include "../operator_descriptor.h"

typedef struct InfiniopDescriptor *infiniopPagedCachingFp4Descriptor_t;

__INFINI_C __export infiniStatus_t infiniopCreatePagedCachingFp4Descriptor(
    infiniopHandle_t handle,
    infiniopPagedCachingFp4Descriptor_t *desc_ptr,
    infiniopTensorDescriptor_t k_codes_desc,
    infiniopTensorDescriptor_t v_codes_desc,
    infiniopTensorDescriptor_t k_scales_desc,
    infiniopTensorDescriptor_t v_scales_desc,
    infiniopTensorDescriptor_t k_desc,
    infiniopTensorDescriptor_t v_desc,
    infiniopTensorDescriptor_t slot_mapping_desc);

/* Always reports 0. */
__INFINI_C __export infiniStatus_t infiniopGetPagedCachingFp4WorkspaceSize(
    infiniopPagedCachingFp4Descriptor_t desc,
    size_t *size);

/* Enqueues on `stream`; BAD_PARAM where the calling thread's current device is not the descriptor's. */
__INFINI_C __export infiniStatus_t infiniopPagedCachingFp4(
    infiniopPagedCachingFp4Descriptor_t desc,
    void *workspace,
    size_t workspace_size,
    void *k_codes,
    void *v_codes,
    void *k_scales,
    void *v_scales,
    const void *k,
    const void *v,
    const void *slot_mapping,
    void *stream);

__INFINI_C __export infiniStatus_t infiniopDestroyPagedCachingFp4Descriptor(
    infiniopPagedCachingFp4Descriptor_t desc);

#endif /* INFINICORE_AMD_INFINIOP_PAGED_CACHING_FP4_H */
