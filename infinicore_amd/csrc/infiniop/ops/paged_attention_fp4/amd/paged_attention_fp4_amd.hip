// paged_attention_fp4 on AMD Instinct (gfx950): descriptor, workspace and launches of the decode kernels in decode_fp4.h.
#include "paged_attention_fp4_amd.h"
#include "../../../devices/amd/amd_device.h"
#include "../../../handle.h"
#include "decode_fp4.h"
#include <algorithm>

namespace op::paged_attention_fp4::amd {

namespace {

// How a call is cut: runs of steps per stream (a KV head and up to 16 of its query heads), and where partial results lie.
struct Plan {
    int head_chunks;
    int runs; // per stream
    int part_rows;
    size_t acc_bytes, ml_bytes;

    size_t workspaceBytes() const { return runs > 1 ? acc_bytes + ml_bytes + 256 : 0; } // (256: to align it here)
};

// Two workgroups of four wavefronts fit a compute unit: that many runs fill the device once.
constexpr int kWavesPerUnit = 8;

Plan makePlan(const PagedAttentionFp4Info &in, const device::amd::DeviceInfo &dev) {
    Plan plan{};
    const int64_t group = static_cast<int64_t>(in.num_heads / in.pool.num_kv_heads);
    plan.head_chunks = static_cast<int>((group + kHeadsPerWave - 1) / kHeadsPerWave);
    plan.part_rows = static_cast<int>(std::min<int64_t>(group, kHeadsPerWave));
    const int64_t streams = static_cast<int64_t>(in.pool.num_kv_heads) * plan.head_chunks;
    const int64_t steps = static_cast<int64_t>(in.num_seqs) * ((in.capacity() + kStepTokens - 1) / kStepTokens);
    const int64_t fill = (static_cast<int64_t>(dev.compute_units) * kWavesPerUnit + streams - 1) / std::max<int64_t>(streams, 1);
    plan.runs = static_cast<int>(std::max<int64_t>(1, std::min(fill, (steps + kLeastSteps - 1) / kLeastSteps)));
    const size_t rows = static_cast<size_t>(streams) * plan.runs * 2 * plan.part_rows;
    plan.acc_bytes = (rows * in.head_size * sizeof(float) + 255) / 256 * 256;
    plan.ml_bytes = rows * sizeof(float2);
    return plan;
}

template <typename T, int HEAD>
void launchHead(const DecodeFp4Args &a, int runs, hipStream_t stream) {
    constexpr int kWaves = kDecodeThreads / 64;
    const unsigned streams = static_cast<unsigned>(a.num_kv_heads) * a.head_chunks;
    const dim3 grid(streams * ((runs + kWaves - 1) / kWaves));
    if (a.block_size % 16 == 0) {
        decodeFp4Kernel<T, HEAD, 16><<<grid, kDecodeThreads, 0, stream>>>(a);
    } else if (a.block_size % 8 == 0) {
        decodeFp4Kernel<T, HEAD, 8><<<grid, kDecodeThreads, 0, stream>>>(a);
    } else {
        decodeFp4Kernel<T, HEAD, 1><<<grid, kDecodeThreads, 0, stream>>>(a);
    }
    if (runs > 1) {
        mergeFp4Kernel<T, HEAD><<<static_cast<unsigned>(a.num_seqs) * a.num_heads, 64, 0, stream>>>(a);
    }
}

template <typename T>
void launchType(const DecodeFp4Args &a, size_t head, int runs, hipStream_t stream) {
    switch (head) {
    case 64: launchHead<T, 64>(a, runs, stream); break;
    case 128: launchHead<T, 128>(a, runs, stream); break;
    case 192: launchHead<T, 192>(a, runs, stream); break;
    default: launchHead<T, 256>(a, runs, stream); break;
    }
}

PoolSide sideOf(const void *base, const fp4::PoolStrides &s) {
    return PoolSide{static_cast<const char *>(base), s.block, s.head, static_cast<int32_t>(s.row)};
}

} // namespace

struct Descriptor::Opaque {
    Plan plan;
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
    const Plan plan = makePlan(in, device::amd::deviceInfo(handle->device_id));
    *desc_ptr = new Descriptor(new Opaque{plan}, in, plan.workspaceBytes(), handle->device, handle->device_id);
    return INFINI_STATUS_SUCCESS;
}

infiniStatus_t Descriptor::calculate(void *workspace, size_t workspace_size, void *out, const void *q, const void *k_codes,
                                     const void *v_codes, const void *k_scales, const void *v_scales,
                                     const void *block_tables, const void *seq_lens, const void *alibi_slopes,
                                     void *stream_) const {
    const PagedAttentionFp4Info &in = _info;
    const Plan &plan = _opaque->plan;
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
    if ((address(k_codes) | address(v_codes)) % 16 != 0 || (address(q) | address(out)) % 2 != 0
        || (address(block_tables) | address(seq_lens)) % index_bytes != 0 || address(alibi_slopes) % 4 != 0) {
        return INFINI_STATUS_BAD_PARAM;
    }

    DecodeFp4Args a{};
    a.out = out;
    a.q = q;
    a.k_codes = sideOf(k_codes, in.pool.k_codes);
    a.v_codes = sideOf(v_codes, in.pool.v_codes);
    a.k_scales = sideOf(k_scales, in.pool.k_scales);
    a.v_scales = sideOf(v_scales, in.pool.v_scales);
    a.block_tables = block_tables;
    a.seq_lens = seq_lens;
    a.alibi_slopes = in.has_alibi ? static_cast<const float *>(alibi_slopes) : nullptr;
    a.index_type = in.index_dtype == INFINI_DTYPE_I64 ? IndexType::i64 : in.index_dtype == INFINI_DTYPE_I32 ? IndexType::i32 : IndexType::u32;
    if (plan.runs > 1) {
        char *ws = reinterpret_cast<char *>((address(workspace) + 255) & ~static_cast<uintptr_t>(255));
        a.part_acc = reinterpret_cast<float *>(ws);
        a.part_ml = reinterpret_cast<float2 *>(ws + plan.acc_bytes);
    }
    a.part_rows = plan.part_rows;
    a.scale_log2 = in.scale * kLog2e;
    a.num_seqs = static_cast<int32_t>(in.num_seqs);
    a.num_heads = static_cast<int32_t>(in.num_heads);
    a.num_kv_heads = static_cast<int32_t>(in.pool.num_kv_heads);
    a.group = static_cast<int32_t>(in.num_heads / in.pool.num_kv_heads);
    a.head_chunks = plan.head_chunks;
    a.runs = plan.runs;
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
        launchType<TileF16>(a, in.head_size, plan.runs, stream);
    } else {
        launchType<TileBF16>(a, in.head_size, plan.runs, stream);
    }
    return hipGetLastError() == hipSuccess ? INFINI_STATUS_SUCCESS : INFINI_STATUS_INTERNAL_ERROR;
}

} // namespace op::paged_attention_fp4::amd
