// Shape of a backend descriptor class for paged_caching_fp4. A backend instantiates it in its own namespace with
// DESCRIPTOR(ns) and defines create/calculate/~Descriptor.
#ifndef INFINICORE_AMD_PAGED_CACHING_FP4_H
#define INFINICORE_AMD_PAGED_CACHING_FP4_H

#include "../../operator.h"
#include "info.h"

#define DESCRIPTOR(NAMESPACE)                                                                                    \
    namespace op::paged_caching_fp4::NAMESPACE {                                                                 \
    class Descriptor final : public InfiniopDescriptor {                                                         \
        struct Opaque;                                                                                           \
        Opaque *_opaque;                                                                                         \
        PagedCachingFp4Info _info;                                                                               \
        size_t _workspace_size;                                                                                  \
                                                                                                                 \
        Descriptor(Opaque *opaque, const PagedCachingFp4Info &info, size_t workspace_size,                       \
                   infiniDevice_t device_type, int device_id)                                                    \
            : InfiniopDescriptor{device_type, device_id}, _opaque(opaque), _info(info),                          \
              _workspace_size(workspace_size) {}                                                                 \
                                                                                                                 \
    public:                                                                                                      \
        ~Descriptor();                                                                                           \
        size_t workspaceSize() const { return _workspace_size; }                                                 \
        static infiniStatus_t create(infiniopHandle_t handle, Descriptor **desc_ptr,                             \
                                     infiniopTensorDescriptor_t k_codes_desc,                                    \
                                     infiniopTensorDescriptor_t v_codes_desc,                                    \
                                     infiniopTensorDescriptor_t k_scales_desc,                                   \
                                     infiniopTensorDescriptor_t v_scales_desc, infiniopTensorDescriptor_t k_desc, \
                                     infiniopTensorDescriptor_t v_desc,                                          \
                                     infiniopTensorDescriptor_t slot_mapping_desc);                              \
        infiniStatus_t calculate(void *workspace, size_t workspace_size, void *k_codes, void *v_codes,           \
                                 void *k_scales, void *v_scales, const void *k, const void *v,                   \
                                 const void *slot_mapping, void *stream) const;                                  \
    };                                                                                                           \
    }

#endif
