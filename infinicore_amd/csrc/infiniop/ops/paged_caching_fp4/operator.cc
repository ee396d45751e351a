// C entry points of paged_caching_fp4: pick the backend from the handle's / descriptor's device type; the only backend in
// this build is amd, every other device type answers DEVICE_TYPE_NOT_SUPPORTED.
#include "infiniop/ops/paged_caching_fp4.h"
#include "../../handle.h"
#include "../../operator.h"
#include "amd/paged_caching_fp4_amd.h"

using AmdDescriptor = op::paged_caching_fp4::amd::Descriptor;

__INFINI_C infiniStatus_t infiniopCreatePagedCachingFp4Descriptor(infiniopHandle_t handle,
                                                                  infiniopPagedCachingFp4Descriptor_t *desc_ptr,
                                                                  infiniopTensorDescriptor_t k_codes_desc,
                                                                  infiniopTensorDescriptor_t v_codes_desc,
                                                                  infiniopTensorDescriptor_t k_scales_desc,
                                                                  infiniopTensorDescriptor_t v_scales_desc,
                                                                  infiniopTensorDescriptor_t k_desc,
                                                                  infiniopTensorDescriptor_t v_desc,
                                                                  infiniopTensorDescriptor_t slot_mapping_desc) {
    if (handle == nullptr || desc_ptr == nullptr) {
        return INFINI_STATUS_NULL_POINTER;
    }
    switch (handle->device) {
    case INFINI_DEVICE_AMD:
        return AmdDescriptor::create(handle, reinterpret_cast<AmdDescriptor **>(desc_ptr), k_codes_desc, v_codes_desc,
                                     k_scales_desc, v_scales_desc, k_desc, v_desc, slot_mapping_desc);
    default:
        return INFINI_STATUS_DEVICE_TYPE_NOT_SUPPORTED;
    }
}

__INFINI_C infiniStatus_t infiniopGetPagedCachingFp4WorkspaceSize(infiniopPagedCachingFp4Descriptor_t desc, size_t *size) {
    if (desc == nullptr || size == nullptr) {
        return INFINI_STATUS_NULL_POINTER;
    }
    switch (desc->device_type) {
    case INFINI_DEVICE_AMD:
        *size = reinterpret_cast<AmdDescriptor *>(desc)->workspaceSize();
        return INFINI_STATUS_SUCCESS;
    default:
        return INFINI_STATUS_DEVICE_TYPE_NOT_SUPPORTED;
    }
}

__INFINI_C infiniStatus_t infiniopPagedCachingFp4(infiniopPagedCachingFp4Descriptor_t desc, void *workspace,
                                                  size_t workspace_size, void *k_codes, void *v_codes, void *k_scales,
                                                  void *v_scales, const void *k, const void *v, const void *slot_mapping,
                                                  void *stream) {
    if (desc == nullptr) {
        return INFINI_STATUS_NULL_POINTER;
    }
    switch (desc->device_type) {
    case INFINI_DEVICE_AMD:
        return reinterpret_cast<AmdDescriptor *>(desc)->calculate(workspace, workspace_size, k_codes, v_codes, k_scales,
                                                                  v_scales, k, v, slot_mapping, stream);
    default:
        return INFINI_STATUS_DEVICE_TYPE_NOT_SUPPORTED;
    }
}

__INFINI_C infiniStatus_t infiniopDestroyPagedCachingFp4Descriptor(infiniopPagedCachingFp4Descriptor_t desc) {
    if (desc == nullptr) {
        return INFINI_STATUS_NULL_POINTER;
    }
    switch (desc->device_type) {
    case INFINI_DEVICE_AMD:
        delete reinterpret_cast<AmdDescriptor *>(desc);
        return INFINI_STATUS_SUCCESS;
    default:
        return INFINI_STATUS_DEVICE_TYPE_NOT_SUPPORTED;
    }
}
