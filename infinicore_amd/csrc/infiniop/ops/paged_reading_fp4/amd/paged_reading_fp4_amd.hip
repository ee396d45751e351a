// paged_reading_fp4 on AMD Instinct (gfx950): tokens of a pool held in 4 bits, gathered and written out as 16- or 32-bit
// values. The mirror of paged_caching_fp4: a lane has eight elements (a dword of codes, the byte of their scale), four
// conversion instructions make them the values they stand for, and one or two 16-byte stores write them. HBM-bound: 0.53
// bytes are read and two (four) written per element.
#include "paged_reading_fp4_amd.h"
#include "../../../devices/amd/amd_fp4.h"
#include "../../../devices/amd/amd_streaming.h"
#include "../../../handle.h"
#include "../../../../utils/check.h"

namespace op::paged_reading_fp4::amd {

namespace {

using namespace device::amd;

constexpr int kThreads = 256;
constexpr int kPerLane = 8; // elements

struct Side { // keys or values
    const uint8_t *codes, *scales;
    void *to;
    int64_t code_block, code_head, code_row;    // bytes
    int64_t scale_block, scale_head, scale_row; // bytes
    int64_t token_stride, head_stride;          // elements
    uint32_t lanes_per_row;                     // size / 8
};

struct ReadArgs {
    Side k, v;
    const int64_t *slot_mapping;
    int64_t num_slots;
    uint32_t num_tokens;
    uint32_t k_lanes;     // of a token: heads x k.lanes_per_row
    uint32_t token_lanes; // of its keys and values
    uint32_t block_tokens; // tokens of a workgroup
    uint32_t block_size;
    int32_t block_shift;  // log2(block_size) when it is a power of two, else -1
};

// Eight values as they are stored.
struct EightBF16 {
    using Element = uint16_t;
    uint4 w;
    __device__ __forceinline__ void of(uint32_t codes, float s) { w = mx::toBF16x8(codes, s); }
    __device__ __forceinline__ void store(Element *p) const { storeStreamed(p, w); }
    __device__ __forceinline__ void storeEach(Element *p) const {
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = static_cast<uint16_t>(words[i / 2] >> (16 * (i & 1)));
        }
    }
};
struct EightF16 : EightBF16 {
    __device__ __forceinline__ void of(uint32_t codes, float s) { w = mx::toF16x8(codes, s); }
};
struct EightF32 {
    using Element = float;
    mx::f32x2 w[4];
    __device__ __forceinline__ void of(uint32_t codes, float s) {
        w[0] = mx::toF32<0>(codes, s);
        w[1] = mx::toF32<1>(codes, s);
        w[2] = mx::toF32<2>(codes, s);
        w[3] = mx::toF32<3>(codes, s);
    }
    __device__ __forceinline__ void store(Element *p) const {
        storeStreamed(p, make_float4(w[0][0], w[0][1], w[1][0], w[1][1]));
        storeStreamed(p + 4, make_float4(w[2][0], w[2][1], w[3][0], w[3][1]));
    }
    __device__ __forceinline__ void storeEach(Element *p) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[i] = w[i / 2][i & 1];
        }
    }
};

// ALIGNED: outputs at multiples of 16 bytes, rows of codes at multiples of 4; otherwise element by element, byte by byte.
template <typename Eight, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) pagedReadingFp4Kernel(ReadArgs a) {
    const uint32_t first = blockIdx.x * a.block_tokens;
    const uint32_t lanes = min(a.block_tokens, a.num_tokens - first) * a.token_lanes;
    for (uint32_t at = threadIdx.x; at < lanes; at += kThreads) {
        const uint32_t t = at / a.token_lanes;
        uint32_t u = at - t * a.token_lanes;
        const bool value = u >= a.k_lanes;
        u -= value ? a.k_lanes : 0;
        const Side &side = value ? a.v : a.k;
        const uint32_t head = u / side.lanes_per_row, chunk = u - head * side.lanes_per_row;
        const uint32_t token = first + t;
        const int64_t slot = a.slot_mapping[token];
        uint32_t codes = 0, scale = 0;
        if (slot >= 0 && slot < a.num_slots) {
            const int64_t page = a.block_shift >= 0 ? slot >> a.block_shift : slot / a.block_size;
            const int64_t row = slot - page * a.block_size;
            const uint8_t *from = side.codes + page * side.code_block + head * side.code_head + row * side.code_row + chunk * 4;
            if constexpr (ALIGNED) {
                codes = loadStreamed<uint32_t>(from);
            } else {
                codes = from[0] | from[1] << 8 | from[2] << 16 | static_cast<uint32_t>(from[3]) << 24;
            }
            scale = side.scales[page * side.scale_block + head * side.scale_head + row * side.scale_row + (chunk >> 2)];
        }
        Eight eight;
        eight.of(codes, mx::scaleOf(scale));
        auto *to = static_cast<typename Eight::Element *>(side.to) + token * side.token_stride + head * side.head_stride
                 + chunk * kPerLane;
        if constexpr (ALIGNED) {
            eight.store(to);
        } else {
            eight.storeEach(to);
        }
    }
}

Side sideOf(const void *codes, const void *scales, void *to, const fp4::PoolStrides &c, const fp4::PoolStrides &s,
            ptrdiff_t token_stride, ptrdiff_t head_stride, size_t size) {
    return Side{static_cast<const uint8_t *>(codes), static_cast<const uint8_t *>(scales), to, c.block, c.head, c.row,
                s.block, s.head, s.row, token_stride, head_stride, static_cast<uint32_t>(size / kPerLane)};
}

} // namespace

struct Descriptor::Opaque {};

Descriptor::~Descriptor() { delete _opaque; }

infiniStatus_t Descriptor::create(infiniopHandle_t handle, Descriptor **desc_ptr, infiniopTensorDescriptor_t k_desc,
                                  infiniopTensorDescriptor_t v_desc, infiniopTensorDescriptor_t k_codes_desc,
                                  infiniopTensorDescriptor_t v_codes_desc, infiniopTensorDescriptor_t k_scales_desc,
                                  infiniopTensorDescriptor_t v_scales_desc, infiniopTensorDescriptor_t slot_mapping_desc) {
    auto info = PagedReadingFp4Info::create(k_desc, v_desc, k_codes_desc, v_codes_desc, k_scales_desc, v_scales_desc,
                                            slot_mapping_desc);
    CHECK_RESULT(info);
    const PagedReadingFp4Info in = info.take();
    // the kernel counts tokens, rows of a page and the lanes of a workgroup in 32 bits
    if (in.num_tokens > 0x7fffffff || in.pool.block_size > 0x7fffffff || in.pool.num_kv_heads > 0xffff
        || in.pool.k_size > 0xffff || in.pool.v_size > 0xffff) {
        return INFINI_STATUS_BAD_TENSOR_SHAPE;
    }
    *desc_ptr = new Descriptor(new Opaque{}, in, 0, handle->device, handle->device_id);
    return INFINI_STATUS_SUCCESS;
}

infiniStatus_t Descriptor::calculate(void *workspace, size_t workspace_size, void *k, void *v, const void *k_codes,
                                     const void *v_codes, const void *k_scales, const void *v_scales,
                                     const void *slot_mapping, void *stream_) const {
    (void)workspace;
    (void)workspace_size;
    const PagedReadingFp4Info &in = _info;
    const fp4::PoolInfo &pool = in.pool;
    if (in.num_tokens == 0 || pool.num_kv_heads == 0 || pool.k_size + pool.v_size == 0) {
        return INFINI_STATUS_SUCCESS;
    }
    const bool keys = pool.k_size > 0, values = pool.v_size > 0;
    const bool empty = pool.num_blocks == 0 || pool.block_size == 0; // every slot is past the pool
    if (slot_mapping == nullptr || (keys && k == nullptr) || (values && v == nullptr)
        || (!empty && keys && (k_codes == nullptr || k_scales == nullptr))
        || (!empty && values && (v_codes == nullptr || v_scales == nullptr))) {
        return INFINI_STATUS_NULL_POINTER;
    }
    int current_device = -1;
    if (hipGetDevice(&current_device) != hipSuccess || current_device != device_id) {
        return INFINI_STATUS_BAD_PARAM;
    }
    const uint64_t es = infiniSizeOf(in.dtype);
    auto address = [](const void *p) { return reinterpret_cast<uint64_t>(p); };
    if ((address(k) | address(v)) % es != 0 || address(slot_mapping) % 8 != 0) {
        return INFINI_STATUS_BAD_PARAM; // a base address that is not aligned to the element size
    }

    ReadArgs a{};
    a.k = sideOf(k_codes, k_scales, k, pool.k_codes, pool.k_scales, in.k_token_stride, in.k_head_stride, pool.k_size);
    a.v = sideOf(v_codes, v_scales, v, pool.v_codes, pool.v_scales, in.v_token_stride, in.v_head_stride, pool.v_size);
    a.slot_mapping = static_cast<const int64_t *>(slot_mapping);
    a.num_slots = static_cast<int64_t>(pool.num_blocks) * static_cast<int64_t>(pool.block_size);
    a.num_tokens = static_cast<uint32_t>(in.num_tokens);
    a.k_lanes = static_cast<uint32_t>(pool.num_kv_heads) * a.k.lanes_per_row;
    a.token_lanes = a.k_lanes + static_cast<uint32_t>(pool.num_kv_heads) * a.v.lanes_per_row;
    a.block_tokens = a.token_lanes >= kThreads ? 1 : kThreads / a.token_lanes;
    a.block_size = static_cast<uint32_t>(pool.block_size);
    a.block_shift = a.block_size > 0 && (a.block_size & (a.block_size - 1)) == 0 ? __builtin_ctz(a.block_size) : -1;

    const uint64_t targets = address(k) | address(v)
                           | (static_cast<uint64_t>(in.k_token_stride | in.k_head_stride | in.v_token_stride | in.v_head_stride) * es);
    const bool aligned = targets % 16 == 0 && (address(k_codes) | address(v_codes)) % 4 == 0 && pool.codeRowsAligned(4);
    const uint32_t grid = (a.num_tokens + a.block_tokens - 1) / a.block_tokens;
    auto stream = static_cast<hipStream_t>(stream_);
    auto launch = [&](auto eight) {
        using Eight = decltype(eight);
        if (aligned) {
            pagedReadingFp4Kernel<Eight, true><<<grid, kThreads, 0, stream>>>(a);
        } else {
            pagedReadingFp4Kernel<Eight, false><<<grid, kThreads, 0, stream>>>(a);
        }
    };
    switch (in.dtype) {
    case INFINI_DTYPE_BF16: launch(EightBF16{}); break;
    case INFINI_DTYPE_F16: launch(EightF16{}); break;
    default: launch(EightF32{}); break;
    }
    return hipGetLastError() == hipSuccess ? INFINI_STATUS_SUCCESS : INFINI_STATUS_INTERNAL_ERROR;
}

} // namespace op::paged_reading_fp4::amd
