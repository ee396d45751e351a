// Host side of the kernels in decode_fp4.h: how a call is cut, its workspace, arguments and launches; used by decode and, for
// runs of a few tokens per sequence, by prefill.
#ifndef INFINICORE_AMD_PA_DECODE_FP4_LAUNCH_H
#define INFINICORE_AMD_PA_DECODE_FP4_LAUNCH_H

#include "../info.h"
#include "decode_fp4.h"
#include <algorithm>

namespace op::paged_attention_fp4::amd {

// Runs of steps per stream (a KV head and up to 16 of its query heads), and where partial results lie.
struct DecodePlan {
    bool possible;
    int head_chunks;
    int runs;           // per stream
    int part_rows;
    int max_segments;   // per stream
    int merge_waves;
    size_t acc_bytes, ml_bytes, segment_bytes;

    size_t workspaceBytes() const { return runs > 1 ? acc_bytes + ml_bytes + segment_bytes + 256 + 256 : 0; } // (256: to align it here; a count)
};

// Wavefronts that a compute unit holds at a time: that many runs fill the device once.
inline int wavesPerUnit(size_t head) {
    const int groups = head == 64 ? Layout<64>::kPerUnit : head == 128 ? Layout<128>::kPerUnit : head == 192 ? Layout<192>::kPerUnit : Layout<256>::kPerUnit;
    return groups * (kDecodeThreads / 64);
}

// `by_rows`: several query tokens per sequence (RUNS).
inline DecodePlan planDecode(const AttentionFp4Info &in, bool by_rows, int compute_units) {
    DecodePlan plan{};
    const int64_t group = static_cast<int64_t>(in.num_heads / in.pool.num_kv_heads);
    plan.head_chunks = by_rows ? 1 : static_cast<int>((group + kHeadsPerWave - 1) / kHeadsPerWave);
    plan.part_rows = by_rows ? kHeadsPerWave : static_cast<int>(std::min<int64_t>(group, kHeadsPerWave));
    const int64_t streams = std::max<int64_t>(static_cast<int64_t>(in.pool.num_kv_heads) * plan.head_chunks, 1);
    const int64_t segments = static_cast<int64_t>(in.num_seqs) + (by_rows ? static_cast<int64_t>(in.num_rows) * group / kHeadsPerWave : 0);
    const int64_t per_segment = (static_cast<int64_t>(in.capacity()) + kStepTokens - 1) / kStepTokens;
    plan.possible = segments <= 0x3fffffff && segments * per_segment <= 0x7fffffff;
    if (!plan.possible) {
        return plan;
    }
    plan.max_segments = static_cast<int>(segments);
    const int64_t steps = segments * per_segment;
    const int64_t fill = (static_cast<int64_t>(compute_units) * wavesPerUnit(in.head_size) + streams - 1) / streams;
    plan.runs = static_cast<int>(std::max<int64_t>(1, std::min(fill, (steps + kLeastSteps - 1) / kLeastSteps)));
    // wavefronts that join the parts of a row, by how many parts there are if the segments are alike
    const int64_t parts = plan.runs / std::max<int64_t>(segments, 1) + 2;
    plan.merge_waves = parts <= 8 ? 1 : (parts <= 48 ? 4 : 16);
    const size_t rows = static_cast<size_t>(streams) * plan.runs * 2 * plan.part_rows;
    auto padded = [](size_t bytes) { return (bytes + 255) / 256 * 256; };
    plan.acc_bytes = padded(rows * in.head_size * sizeof(float));
    plan.ml_bytes = padded(rows * sizeof(float2));
    plan.segment_bytes = padded(static_cast<size_t>(plan.max_segments) * sizeof(int4));
    return plan;
}

inline PoolSide sideOf(const void *base, const fp4::PoolStrides &s) {
    return PoolSide{static_cast<const char *>(base), s.block, s.head, static_cast<int32_t>(s.row)};
}
inline IndexType indexType(infiniDtype_t dtype) {
    return dtype == INFINI_DTYPE_I64 ? IndexType::i64 : dtype == INFINI_DTYPE_I32 ? IndexType::i32 : IndexType::u32;
}
// Whether every row of [rows, heads, head] begins at a multiple of 16 bytes.
inline bool rowsAligned(const void *p, ptrdiff_t row, ptrdiff_t head) {
    return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>((row | head) * 2)) % 16 == 0;
}

// `cu`: nullptr but for RUNS.
inline DecodeFp4Args decodeArgs(const AttentionFp4Info &in, const DecodePlan &plan, void *workspace, void *out, const void *q,
                                const void *k_codes, const void *v_codes, const void *k_scales, const void *v_scales,
                                const void *block_tables, const void *seq_lens, const void *cu, const void *alibi_slopes) {
    DecodeFp4Args a{};
    a.out = out;
    a.q = q;
    a.k_codes = sideOf(k_codes, in.pool.k_codes);
    a.v_codes = sideOf(v_codes, in.pool.v_codes);
    a.k_scales = sideOf(k_scales, in.pool.k_scales);
    a.v_scales = sideOf(v_scales, in.pool.v_scales);
    a.block_tables = block_tables;
    a.seq_lens = seq_lens;
    a.cu_seqlens_q = cu;
    a.alibi_slopes = in.has_alibi ? static_cast<const float *>(alibi_slopes) : nullptr;
    a.index_type = indexType(in.index_dtype);
    if (plan.runs > 1) {
        char *ws = reinterpret_cast<char *>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~static_cast<uintptr_t>(255));
        a.part_acc = reinterpret_cast<float *>(ws);
        a.part_ml = reinterpret_cast<float2 *>(ws + plan.acc_bytes);
        a.segments = reinterpret_cast<int4 *>(ws + plan.acc_bytes + plan.ml_bytes);
        a.num_segments = reinterpret_cast<int32_t *>(ws + plan.acc_bytes + plan.ml_bytes + plan.segment_bytes);
    }
    a.part_rows = plan.part_rows;
    a.scale_log2 = in.scale * kLog2e;
    a.num_seqs = static_cast<int32_t>(in.num_seqs);
    a.num_heads = static_cast<int32_t>(in.num_heads);
    a.num_kv_heads = static_cast<int32_t>(in.pool.num_kv_heads);
    a.total_q_tokens = static_cast<int32_t>(in.num_rows);
    a.group = static_cast<int32_t>(in.num_heads / in.pool.num_kv_heads);
    a.head_chunks = plan.head_chunks;
    a.runs = plan.runs;
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
    return a;
}

template <typename T, int HEAD, int GRAIN, bool RUNS>
void launchDecode(const DecodeFp4Args &a, const DecodePlan &plan, hipStream_t stream) {
    constexpr int kWaves = kDecodeThreads / 64;
    unsigned groups = static_cast<unsigned>((plan.runs + kWaves - 1) / kWaves);
    groups += a.num_kv_heads % 2 == 0 && groups > 1 && groups % 2 != 0 ? 1 : 0; // (pairs of KV heads: see the kernel)
#define EARLY a.seq_lens, a.cu_seqlens_q, static_cast<int32_t>(a.index_type), a.num_seqs, a.capacity, a.runs
    decodeFp4Kernel<T, HEAD, GRAIN, RUNS><<<dim3(a.num_kv_heads, groups, plan.head_chunks), kDecodeThreads, 0, stream>>>(EARLY, a);
    if (plan.runs > 1) {
        const dim3 grid(static_cast<unsigned>(plan.max_segments) * plan.part_rows, a.num_kv_heads, plan.head_chunks);
        switch (plan.merge_waves) {
        case 1: mergeFp4Kernel<T, HEAD, RUNS, 1><<<grid, 64, 0, stream>>>(EARLY, a); break;
        case 4: mergeFp4Kernel<T, HEAD, RUNS, 4><<<grid, 256, 0, stream>>>(EARLY, a); break;
        default: mergeFp4Kernel<T, HEAD, RUNS, 16><<<grid, 1024, 0, stream>>>(EARLY, a); break;
        }
    }
#undef EARLY
}

} // namespace op::paged_attention_fp4::amd

#endif
