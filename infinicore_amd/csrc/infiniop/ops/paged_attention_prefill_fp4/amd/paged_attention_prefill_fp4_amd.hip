// paged_attention_prefill_fp4 on AMD Instinct (gfx950): descriptor and launches of the kernel in prefill_fp4.h.
#include "paged_attention_prefill_fp4_amd.h"
#include "../../../devices/amd/amd_device.h"
#include "../../../handle.h"
#include "prefill_fp4.h"
#include <algorithm>

namespace op::paged_attention_prefill_fp4::amd {

namespace {

template <typename T, int HEAD, int R>
void launchRows(const PrefillFp4Args &a, hipStream_t stream) {
    constexpr int BM = 64 * R;
    // every sequence has at most one row block that is not full
    const int64_t blocks = static_cast<int64_t>(a.total_q_tokens) * a.group / BM + a.num_seqs;
    const dim3 grid(static_cast<unsigned>(blocks * a.num_kv_heads));
    if (a.block_size % kTile == 0) {
        prefillFp4Kernel<T, HEAD, R, true><<<grid, kPrefillThreads, 0, stream>>>(a);
    } else {
        prefillFp4Kernel<T, HEAD, R, false><<<grid, kPrefillThreads, 0, stream>>>(a);
    }
}

template <typename T>
void launchType(const PrefillFp4Args &a, size_t head, bool wide, hipStream_t stream) {
    switch (head) {
    case 64: wide ? launchRows<T, 64, 2>(a, stream) : launchRows<T, 64, 1>(a, stream); break;
    case 128: wide ? launchRows<T, 128, 2>(a, stream) : launchRows<T, 128, 1>(a, stream); break;
    case 192: launchRows<T, 192, 1>(a, stream); break;
    default: launchRows<T, 256, 1>(a, stream); break;
    }
}

PoolSide sideOf(const void *base, const fp4::PoolStrides &s) {
    return PoolSide{static_cast<const char *>(base), s.block, s.head, static_cast<int32_t>(s.row)};
}

} // namespace

struct Descriptor::Opaque {
    bool wide; // 128 rows per workgroup
};

Descriptor::~Descriptor() { delete _opaque; }

infiniStatus_t Descriptor::create(infiniopHandle_t handle, Descriptor **desc_ptr, infiniopTensorDescriptor_t out_desc,
                                  infiniopTensorDescriptor_t q_desc, infiniopTensorDescriptor_t k_codes_desc,
                                  infiniopTensorDescriptor_t v_codes_desc, infiniopTensorDescriptor_t k_scales_desc,
                                  infiniopTensorDescriptor_t v_scales_desc, infiniopTensorDescriptor_t block_tables_desc,
                                  infiniopTensorDescriptor_t seq_lens_desc, infiniopTensorDescriptor_t cum_seq_lens_q_desc,
                                  infiniopTensorDescriptor_t alibi_slopes_desc, float scale) {
    auto info = PagedAttentionPrefillFp4Info::create(out_desc, q_desc, k_codes_desc, v_codes_desc, k_scales_desc,
                                                     v_scales_desc, block_tables_desc, seq_lens_desc,
                                                     cum_seq_lens_q_desc, alibi_slopes_desc, scale);
    CHECK_RESULT(info);
    const PagedAttentionPrefillFp4Info in = info.take();
    const int64_t rows = static_cast<int64_t>(in.num_rows * in.num_heads); // of all KV heads
    const int64_t units = device::amd::deviceInfo(handle->device_id).compute_units;
    *desc_ptr = new Descriptor(new Opaque{rows / 128 >= 2 * units}, in, 0, handle->device, handle->device_id);
    return INFINI_STATUS_SUCCESS;
}

infiniStatus_t Descriptor::calculate(void *workspace, size_t workspace_size, void *out, const void *q, const void *k_codes,
                                     const void *v_codes, const void *k_scales, const void *v_scales,
                                     const void *block_tables, const void *seq_lens, const void *cum_seq_lens_q,
                                     const void *alibi_slopes, void *stream_) const {
    (void)workspace;
    (void)workspace_size;
    const PagedAttentionPrefillFp4Info &in = _info;
    if (in.num_seqs == 0 || in.num_rows == 0 || in.num_heads == 0) {
        return INFINI_STATUS_SUCCESS;
    }
    if (out == nullptr || q == nullptr || k_codes == nullptr || v_codes == nullptr || k_scales == nullptr
        || v_scales == nullptr || block_tables == nullptr || seq_lens == nullptr || cum_seq_lens_q == nullptr
        || (in.has_alibi && alibi_slopes == nullptr)) {
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
        || (address(block_tables) | address(seq_lens) | address(cum_seq_lens_q)) % index_bytes != 0
        || address(alibi_slopes) % 4 != 0) {
        return INFINI_STATUS_BAD_PARAM;
    }

    PrefillFp4Args a{};
    a.out = out;
    a.q = q;
    a.k_codes = sideOf(k_codes, in.pool.k_codes);
    a.v_codes = sideOf(v_codes, in.pool.v_codes);
    a.k_scales = sideOf(k_scales, in.pool.k_scales);
    a.v_scales = sideOf(v_scales, in.pool.v_scales);
    a.block_tables = block_tables;
    a.kv_lens = seq_lens;
    a.cu_seqlens_q = cum_seq_lens_q;
    a.alibi_slopes = in.has_alibi ? static_cast<const float *>(alibi_slopes) : nullptr;
    a.index_type = in.index_dtype == INFINI_DTYPE_I64 ? IndexType::i64 : in.index_dtype == INFINI_DTYPE_I32 ? IndexType::i32 : IndexType::u32;
    a.scale_log2 = in.scale * kLog2e;
    a.num_seqs = static_cast<int32_t>(in.num_seqs);
    a.total_q_tokens = static_cast<int32_t>(in.num_rows);
    a.num_heads = static_cast<int32_t>(in.num_heads);
    a.num_kv_heads = static_cast<int32_t>(in.pool.num_kv_heads);
    a.group = static_cast<int32_t>(in.num_heads / in.pool.num_kv_heads);
    a.block_size = static_cast<int32_t>(in.pool.block_size);
    a.num_blocks = static_cast<int32_t>(std::min<size_t>(in.pool.num_blocks, 0x7fffffff));
    a.capacity = in.capacity();
    auto aligned = [&](const void *p, ptrdiff_t row, ptrdiff_t head) { return (address(p) | static_cast<uintptr_t>((row | head) * 2)) % 16 == 0; };
    a.q_aligned = aligned(q, in.q_stride, in.q_head_stride);
    a.out_aligned = aligned(out, in.o_stride, in.o_head_stride);
    a.q_stride = in.q_stride;
    a.q_head_stride = in.q_head_stride;
    a.o_stride = in.o_stride;
    a.o_head_stride = in.o_head_stride;
    a.block_table_stride = in.block_table_batch_stride;

    auto stream = static_cast<hipStream_t>(stream_);
    if (in.dtype == INFINI_DTYPE_F16) {
        launchType<TileF16>(a, in.head_size, _opaque->wide, stream);
    } else {
        launchType<TileBF16>(a, in.head_size, _opaque->wide, stream);
    }
    return hipGetLastError() == hipSuccess ? INFINI_STATUS_SUCCESS : INFINI_STATUS_INTERNAL_ERROR;
}

} // namespace op::paged_attention_prefill_fp4::amd
