// paged_attention_prefill_fp4 on AMD Instinct (gfx950): descriptor and launches of the kernel in prefill_fp4.h, and for a few
// new tokens per sequence of the decode kernels that take rows of several tokens (decode_fp4.h).
#include "paged_attention_prefill_fp4_amd.h"
#include "../../../devices/amd/amd_device.h"
#include "../../../handle.h"
#include "../../paged_attention_fp4/amd/decode_fp4_launch.h"
#include "prefill_fp4.h"
#include <algorithm>
#include <cmath>

namespace op::paged_attention_prefill_fp4::amd {

namespace {

using op::paged_attention_fp4::amd::decodeArgs;
using op::paged_attention_fp4::amd::DecodeFp4Args;
using op::paged_attention_fp4::amd::DecodePlan;
using op::paged_attention_fp4::amd::indexType;
using op::paged_attention_fp4::amd::launchDecode;
using op::paged_attention_fp4::amd::planDecode;
using op::paged_attention_fp4::amd::rowsAligned;
using op::paged_attention_fp4::amd::sideOf;

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

template <typename T, int HEAD>
void launchFew(const DecodeFp4Args &a, const DecodePlan &plan, hipStream_t stream) {
    if (a.block_size % 16 == 0) {
        launchDecode<T, HEAD, 16, true>(a, plan, stream);
    } else if (a.block_size % 8 == 0) {
        launchDecode<T, HEAD, 8, true>(a, plan, stream);
    } else {
        launchDecode<T, HEAD, 1, true>(a, plan, stream);
    }
}
template <typename T>
void launchFewType(const DecodeFp4Args &a, size_t head, const DecodePlan &plan, hipStream_t stream) {
    switch (head) {
    case 64: launchFew<T, 64>(a, plan, stream); break;
    case 128: launchFew<T, 128>(a, plan, stream); break;
    case 192: launchFew<T, 192>(a, plan, stream); break;
    default: launchFew<T, 256>(a, plan, stream); break;
    }
}

// Whether rows of 16, whose tokens the wavefronts of the whole chip divide among themselves (decode_fp4.h), beat row blocks
// of 64 that each walk all of theirs. A row block takes 1.2 us per 64 tokens on its own and 0.66 us of a compute unit's time;
// 16 rows take 0.36 us of it, and dividing and joining 12 us. (Head 128; how much a table holds stands for the lengths.)
// Measured, row blocks / rows of 16, in us: 32 sequences of 6000 tokens, 8 KV heads: 8 rows each 121 / 54, 32 rows 121 / 91,
// 64 rows 121 / 141; of 1000 tokens: 8 rows 26 / 22, 32 rows 27 / 32; 1 sequence of 20000: 128 rows 380 / 46.
bool fewRows(const PagedAttentionPrefillFp4Info &in, int units) {
    const double steps = std::max(1.0, static_cast<double>(in.capacity()) / 64);
    const double seqs = static_cast<double>(in.num_seqs), rows = static_cast<double>(in.num_rows * in.num_heads / in.pool.num_kv_heads);
    const double heads_per_unit = static_cast<double>(in.pool.num_kv_heads) / units;
    const double blocks = seqs * std::ceil(rows / seqs / 64) * heads_per_unit, chunks = seqs * std::ceil(rows / seqs / 16) * heads_per_unit;
    return 12 + 0.36 * steps * chunks < steps * std::max(1.2, 0.66 * blocks);
}

} // namespace

struct Descriptor::Opaque {
    bool few;        // the decode kernels, by `plan`
    DecodePlan plan;
    bool wide;       // 128 rows per workgroup
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
    const int units = device::amd::deviceInfo(handle->device_id).compute_units;
    Opaque o{};
    const int64_t rows = static_cast<int64_t>(in.num_rows * in.num_heads); // of all KV heads
    o.wide = rows / 128 >= 2 * units;
    if (fewRows(in, units)) {
        o.plan = planDecode(in, true, units);
        o.few = o.plan.possible && static_cast<int64_t>(o.plan.max_segments) * o.plan.part_rows <= 0x7fffffff; // (the merge's grid)
    }
    *desc_ptr = new Descriptor(new Opaque{o}, in, o.few ? o.plan.workspaceBytes() : 0, handle->device, handle->device_id);
    return INFINI_STATUS_SUCCESS;
}

infiniStatus_t Descriptor::calculate(void *workspace, size_t workspace_size, void *out, const void *q, const void *k_codes,
                                     const void *v_codes, const void *k_scales, const void *v_scales,
                                     const void *block_tables, const void *seq_lens, const void *cum_seq_lens_q,
                                     const void *alibi_slopes, void *stream_) const {
    const PagedAttentionPrefillFp4Info &in = _info;
    if (workspace_size < _workspace_size || (_workspace_size > 0 && workspace == nullptr)) {
        return INFINI_STATUS_INSUFFICIENT_WORKSPACE;
    }
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

    auto stream = static_cast<hipStream_t>(stream_);
    if (_opaque->few) {
        const DecodeFp4Args a = decodeArgs(in, _opaque->plan, workspace, out, q, k_codes, v_codes, k_scales, v_scales, block_tables,
                                           seq_lens, cum_seq_lens_q, alibi_slopes);
        if (in.dtype == INFINI_DTYPE_F16) {
            launchFewType<TileF16>(a, in.head_size, _opaque->plan, stream);
        } else {
            launchFewType<TileBF16>(a, in.head_size, _opaque->plan, stream);
        }
        return hipGetLastError() == hipSuccess ? INFINI_STATUS_SUCCESS : INFINI_STATUS_INTERNAL_ERROR;
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
    a.index_type = indexType(in.index_dtype);
    a.scale_log2 = in.scale * kLog2e;
    a.num_seqs = static_cast<int32_t>(in.num_seqs);
    a.total_q_tokens = static_cast<int32_t>(in.num_rows);
    a.num_heads = static_cast<int32_t>(in.num_heads);
    a.num_kv_heads = static_cast<int32_t>(in.pool.num_kv_heads);
    a.group = static_cast<int32_t>(in.num_heads / in.pool.num_kv_heads);
    a.block_size = static_cast<int32_t>(in.pool.block_size);
    a.num_blocks = static_cast<int32_t>(std::min<size_t>(in.pool.num_blocks, 0x7fffffff));
    a.capacity = in.capacity();
    a.q_aligned = rowsAligned(q, in.q_stride, in.q_head_stride);
    a.out_aligned = rowsAligned(out, in.o_stride, in.o_head_stride);
    a.q_stride = in.q_stride;
    a.q_head_stride = in.q_head_stride;
    a.o_stride = in.o_stride;
    a.o_head_stride = in.o_head_stride;
    a.block_table_stride = in.block_table_batch_stride;

    if (in.dtype == INFINI_DTYPE_F16) {
        launchType<TileF16>(a, in.head_size, _opaque->wide, stream);
    } else {
        launchType<TileBF16>(a, in.head_size, _opaque->wide, stream);
    }
    return hipGetLastError() == hipSuccess ? INFINI_STATUS_SUCCESS : INFINI_STATUS_INTERNAL_ERROR;
}

} // namespace op::paged_attention_prefill_fp4::amd
