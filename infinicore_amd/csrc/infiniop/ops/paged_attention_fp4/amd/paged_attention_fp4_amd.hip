// paged_attention_fp4 on AMD Instinct (gfx950): descriptor, workspace and launches of the decode kernels in decode_fp4.h.
#include "paged_attention_fp4_amd.h"
#include "../../../devices/amd/amd_device.h"
#include "../../../handle.h"
#include "decode_fp4_launch.h"

namespace op::paged_attention_fp4::amd {

namespace {

template <typename T, int HEAD>
void launchHead(const DecodeFp4Args &a, const DecodePlan &plan, hipStream_t stream) {
    if (a.block_size % 16 == 0) {
        launchDecode<T, HEAD, 16, false>(a, plan, stream);
    } else if (a.block_size % 8 == 0) {
        launchDecode<T, HEAD, 8, false>(a, plan, stream);
    } else {
        launchDecode<T, HEAD, 1, false>(a, plan, stream);
    }
}

template <typename T>
void launchType(const DecodeFp4Args &a, size_t head, const DecodePlan &plan, hipStream_t stream) {
    switch (head) {
    case 64: launchHead<T, 64>(a, plan, stream); break;
    case 128: launchHead<T, 128>(a, plan, stream); break;
    case 192: launchHead<T, 192>(a, plan, stream); break;
    default: launchHead<T, 256>(a, plan, stream); break;
    }
}

} // namespace

struct Descriptor::Opaque {
    DecodePlan plan;
};

Descriptor::~Descriptor() { delete _opaque; }

infiniStatus_t Descriptor::create(infiniopHandle_t handle, Descriptor **desc_ptr, infiniopTensorDescriptor_t out_desc,
                                  infiniopTensorDescriptor_t q_desc, infiniopTensorDescriptor_t k_codes_desc,
                                  infiniopTensorDescriptor_t v_codes_desc, infiniopTensorDescriptor_t k_scales_desc,
                                  infiniopTensorDescriptor_t v_scales_desc, infiniopTensorDescriptor_t block_tables_desc,
                                  infiniopTensorDescriptor_t seq_lens_desc, infiniopTensorDescriptor_t alibi_slopes_desc,
                                  float scale) {
    auto info = PagedAttentionFp4Info::create(out_desc, q_desc, k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc,
                                              block_tables_desc, seq_lens_desc, alibi_slopes_desc, scale);
    CHECK_RESULT(info);
    const PagedAttentionFp4Info in = info.take();
    const DecodePlan plan = planDecode(in, false, device::amd::deviceInfo(handle->device_id).compute_units);
    if (!plan.possible) {
        return INFINI_STATUS_BAD_TENSOR_SHAPE; // more steps than are counted in 32 bits
    }
    *desc_ptr = new Descriptor(new Opaque{plan}, in, plan.workspaceBytes(), handle->device, handle->device_id);
    return INFINI_STATUS_SUCCESS;
}

infiniStatus_t Descriptor::calculate(void *workspace, size_t workspace_size, void *out, const void *q, const void *k_codes,
                                     const void *v_codes, const void *k_scales, const void *v_scales,
                                     const void *block_tables, const void *seq_lens, const void *alibi_slopes,
                                     void *stream_) const {
    const PagedAttentionFp4Info &in = _info;
    const DecodePlan &plan = _opaque->plan;
    if (workspace_size < _workspace_size || (_workspace_size > 0 && workspace == nullptr)) {
        return INFINI_STATUS_INSUFFICIENT_WORKSPACE;
    }
    if (in.num_seqs == 0 || in.num_heads == 0) {
        return INFINI_STATUS_SUCCESS;
    }
    if (out == nullptr || q == nullptr || k_codes == nullptr || v_codes == nullptr || k_scales == nullptr
        || v_scales == nullptr || block_tables == nullptr || seq_lens == nullptr || (in.has_alibi && alibi_slopes == nullptr)) {
        return INFINI_STATUS_NULL_POINTER;
    }
    if (in.capacity() == 0 || in.pool.num_blocks == 0) {
        return INFINI_STATUS_SUCCESS; // no sequence can hold a token
    }
    int current_device = -1;
    if (hipGetDevice(&current_device) != hipSuccess || current_device != device_id) {
        return INFINI_STATUS_BAD_PARAM;
    }
    auto address = [](const void *p) { return reinterpret_cast<uintptr_t>(p); };
    const size_t index_bytes = infiniSizeOf(in.index_dtype);
    if ((address(k_codes) | address(v_codes)) % 16 != 0 || (address(k_scales) | address(v_scales)) % in.scaleBytes() != 0
        || (address(q) | address(out)) % 2 != 0
        || (address(block_tables) | address(seq_lens)) % index_bytes != 0 || address(alibi_slopes) % 4 != 0) {
        return INFINI_STATUS_BAD_PARAM;
    }

    const DecodeFp4Args a = decodeArgs(in, plan, workspace, out, q, k_codes, v_codes, k_scales, v_scales, block_tables, seq_lens,
                                       nullptr, alibi_slopes);
    auto stream = static_cast<hipStream_t>(stream_);
    if (in.dtype == INFINI_DTYPE_F16) {
        launchType<TileF16>(a, in.head_size, plan, stream);
    } else {
        launchType<TileBF16>(a, in.head_size, plan, stream);
    }
    return hipGetLastError() == hipSuccess ? INFINI_STATUS_SUCCESS : INFINI_STATUS_INTERNAL_ERROR;
}

} // namespace op::paged_attention_fp4::amd
