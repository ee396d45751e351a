// Conversions between 4-bit floats (e2m1) under a shared power-of-two scale and 16- / 32-bit floats, by the gfx950
// instructions that take the scale along (v_cvt_scalef32_pk_*). Each costs as much as one fused multiply-add and covers two
// elements; encoding from 32 bits takes twice that. Held against the definition on the device for every code under every
// scale, and every bf16 / fp16 value under every scale that is written: equal in all, subnormals and NaN (scale 255) among
// them; magnitudes over 6 are held at 6, ties go to the even code.
#ifndef INFINICORE_AMD_FP4_H
#define INFINICORE_AMD_FP4_H

#include <cstdint>
#include <hip/hip_runtime.h>

namespace device::amd::mx {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// A scale byte as the conversions take it: a float of which only the exponent counts (0 stands for 2^-127, 255 for NaN).
__device__ __forceinline__ float scaleOf(uint32_t byte) { return __uint_as_float(byte << 23); }

// The exponents that are written. Every stored value is then exact in fp16 as in bf16 (0.5 * 2^-23 = 2^-24 is the smallest
// fp16, 6 * 2^13 = 49152 fits), so that a kernel may take whichever of the two its products want.
constexpr int kLeastScale = 127 - 23, kMostScale = 127 + 13;

// The scale of a group whose largest magnitude is `top` (not NaN-quieted: an integer maximum of the bits keeps a NaN on top):
// its exponent less that of e2m1's largest magnitude, 6 = 1.5 * 2^2.
__device__ __forceinline__ uint32_t scaleFor(float top) {
    const int e = static_cast<int>((__float_as_uint(top) >> 23) & 0xff);
    const int s = e - 2 < kLeastScale ? kLeastScale : (e - 2 > kMostScale ? kMostScale : e - 2);
    return static_cast<uint32_t>(e == 0xff ? 0xff : s);
}

// Elements 2 B, 2 B + 1 of the eight in `codes`.
template <int B>
__device__ __forceinline__ uint32_t toBF16(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, B));
}
template <int B>
__device__ __forceinline__ uint32_t toF16(uint32_t codes, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, scale, B));
}
template <int B>
__device__ __forceinline__ f32x2 toF32(uint32_t codes, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes, scale, B);
}
__device__ __forceinline__ uint4 toBF16x8(uint32_t codes, float scale) {
    return make_uint4(toBF16<0>(codes, scale), toBF16<1>(codes, scale), toBF16<2>(codes, scale), toBF16<3>(codes, scale));
}
__device__ __forceinline__ uint4 toF16x8(uint32_t codes, float scale) {
    return make_uint4(toF16<0>(codes, scale), toF16<1>(codes, scale), toF16<2>(codes, scale), toF16<3>(codes, scale));
}

// Two elements (packed as in memory) into byte B of `codes`.
template <int B>
__device__ __forceinline__ uint32_t fromBF16(uint32_t codes, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(codes, __builtin_bit_cast(bf16x2, pair), scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t fromF16(uint32_t codes, uint32_t pair, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(codes, __builtin_bit_cast(f16x2, pair), scale, B);
}
template <int B>
__device__ __forceinline__ uint32_t fromF32(uint32_t codes, float lo, float hi, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, lo, hi, scale, B);
}

} // namespace device::amd::mx

#endif
