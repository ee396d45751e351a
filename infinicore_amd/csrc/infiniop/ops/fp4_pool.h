// The four tensors of a paged KV pool held in 4 bits, as every operator on it checks and captures them.
//   codes  [num_blocks, num_kv_heads, block_size, size / 2]   U8: two e2m1 codes per byte, the even element in the low half
//   scales [num_blocks, num_kv_heads, block_size, size / 32]  U8: one exponent (bias 127) for each 32 elements, 255 = NaN
// for keys and for values. A value is e2m1(code) * 2^(scale - 127): the 4-bit format of the OCP microscaling (MX)
// specification.
#ifndef INFINICORE_AMD_FP4_POOL_H
#define INFINICORE_AMD_FP4_POOL_H

#include "../../utils/check.h"
#include "../../utils/result.h"
#include "../tensor.h"

namespace op::fp4 {

constexpr size_t kGroup = 32; // elements under one scale

// Byte strides of one of the two tensors of keys or of values.
struct PoolStrides {
    ptrdiff_t block, head, row;
};

struct PoolInfo {
    size_t num_blocks, num_kv_heads, block_size;
    size_t k_size, v_size; // elements of a key / value vector
    PoolStrides k_codes, v_codes, k_scales, v_scales;

    static utils::Result<PoolInfo> create(infiniopTensorDescriptor_t k_codes_desc, infiniopTensorDescriptor_t v_codes_desc,
                                          infiniopTensorDescriptor_t k_scales_desc,
                                          infiniopTensorDescriptor_t v_scales_desc) {
        if (!k_codes_desc || !v_codes_desc || !k_scales_desc || !v_scales_desc) {
            return INFINI_STATUS_NULL_POINTER;
        }
        PoolInfo info{};
        for (auto *d : {k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc}) {
            CHECK_DTYPE(d->dtype(), INFINI_DTYPE_U8);
        }
        for (auto *d : {k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc}) {
            if (d->ndim() != 4) {
                return INFINI_STATUS_BAD_TENSOR_SHAPE;
            }
            for (size_t i = 0; i < 3; ++i) {
                if (d->dim(i) != k_codes_desc->dim(i)) {
                    return INFINI_STATUS_BAD_TENSOR_SHAPE;
                }
            }
        }
        info.num_blocks = k_codes_desc->dim(0);
        info.num_kv_heads = k_codes_desc->dim(1);
        info.block_size = k_codes_desc->dim(2);
        info.k_size = 2 * k_codes_desc->dim(3);
        info.v_size = 2 * v_codes_desc->dim(3);
        if (info.k_size % kGroup != 0 || info.v_size % kGroup != 0 || k_scales_desc->dim(3) != info.k_size / kGroup
            || v_scales_desc->dim(3) != info.v_size / kGroup) {
            return INFINI_STATUS_BAD_TENSOR_SHAPE;
        }
        for (auto *d : {k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc}) {
            CHECK_OR_RETURN(d->stride(3) == 1 || d->dim(3) <= 1, INFINI_STATUS_BAD_TENSOR_STRIDES);
        }
        auto strides = [](infiniopTensorDescriptor_t d) { return PoolStrides{d->stride(0), d->stride(1), d->stride(2)}; };
        info.k_codes = strides(k_codes_desc);
        info.v_codes = strides(v_codes_desc);
        info.k_scales = strides(k_scales_desc);
        info.v_scales = strides(v_scales_desc);
        return info;
    }

    // Whether every row of the codes (scales) begins at a multiple of `bytes` from the base.
    bool codeRowsAligned(size_t bytes) const { return rowsAligned(k_codes, bytes) && rowsAligned(v_codes, bytes); }
    bool scaleRowsAligned(size_t bytes) const { return rowsAligned(k_scales, bytes) && rowsAligned(v_scales, bytes); }

    bool rowsAligned(const PoolStrides &s, size_t bytes) const {
        const size_t extent[3] = {num_blocks, num_kv_heads, block_size};
        const ptrdiff_t stride[3] = {s.block, s.head, s.row};
        for (int i = 0; i < 3; ++i) {
            if (extent[i] > 1 && static_cast<size_t>(stride[i]) % bytes != 0) {
                return false;
            }
        }
        return true;
    }
};

} // namespace op::fp4

#endif
