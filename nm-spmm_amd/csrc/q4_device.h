// Device code that the products with 4-bit operands share (q4_linear.hip, q4_gemm.hip).
#ifndef NMSPMM_Q4_DEVICE_H
#define NMSPMM_Q4_DEVICE_H

#include "internal.h"

namespace nmspmm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <ElementType T>
__device__ inline f32x4 product(u32x4 a, u32x4 b, f32x4 c)
{
    if (T == kF16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 16.0 twice, kept in a vector register: an instruction takes one scalar, and mask-and-or needs this and the mask (with both
// as constants the compiler makes a mask and an or of it: half as many instructions again).
template <ElementType T>
__device__ inline uint32_t sixteens()
{
    uint32_t one = T == kF16 ? 0x4c004c00u : 0x41804180u;
    asm("" : "+v"(one));
    return one;
}

// Eight codes -> eight operand elements 16 + code (a word's bits are rotated so that the first pair is in place for bf16: q4.hip).
template <ElementType T>
__device__ inline u32x4 widened(uint32_t w, uint32_t one)
{
    const uint32_t mask = T == kF16 ? 0x03c003c0u : 0x00780078u;
    if (T == kF16)
        return u32x4{((w << 3) & mask) | one, ((w >> 1) & mask) | one, ((w >> 5) & mask) | one,
                     (__builtin_amdgcn_alignbit(w, w, 9) & mask) | one};
    return u32x4{(w & mask) | one, ((w >> 4) & mask) | one, ((w >> 8) & mask) | one, (__builtin_amdgcn_alignbit(w, w, 12) & mask) | one};
}

// Eight 8-bit floats that stand for code - zero times 2^-9 -> eight operand elements code - zero (exact).
template <ElementType T>
__device__ inline u32x4 from_bytes(uint32_t low, uint32_t high)
{
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const float unit = 512.0f;
    if (T == kF16)
        return u32x4{__builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, unit, false)),
                     __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(low, unit, true)),
                     __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, unit, false)),
                     __builtin_bit_cast(uint32_t, (f16x2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(high, unit, true))};
    return u32x4{__builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, unit, false)),
                 __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(low, unit, true)),
                 __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, unit, false)),
                 __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(high, unit, true))};
}

// Eight codes -> eight bf16 elements code - zero (exact): 16 + code in fp16, `offset` (twice - (16 + zero) in fp16) added, and to bf16 by way
// of 8-bit floats, which hold these numbers: two instructions for two of them, where fp32 would take three.
__device__ inline u32x4 differences(uint32_t w, uint32_t sixteen, uint32_t offset)
{
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    typedef short i16x2 __attribute__((ext_vector_type(2)));
    const u32x4 u = widened<kF16>(w, sixteen);
    u32x4 d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2 two = __builtin_bit_cast(f16x2, (uint32_t)u[i]) + __builtin_bit_cast(f16x2, offset);
        const i16x2 bytes = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(i16x2{0, 0}, two, 1.0f, false);
        d[i] = __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(__builtin_bit_cast(uint32_t, bytes), 1.0f, false));
    }
    return d;
}

template <ElementType T>
__device__ inline void store_result(void* y, size_t at, float v)
{
    if (T == kF32)
        static_cast<float*>(y)[at] = v;
    else if (T == kBF16)
        static_cast<uint16_t*>(y)[at] = __builtin_bit_cast(uint16_t, (__bf16)v);
    else
        static_cast<uint16_t*>(y)[at] = __builtin_bit_cast(uint16_t, (_Float16)v);
}

// The same through a descriptor, at a byte offset from its base; beyond its bounds nothing is stored.
template <ElementType T>
__device__ inline void store_bounded(__amdgpu_buffer_rsrc_t r, uint32_t offset, float v)
{
    if (T == kF32)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), r, (int)offset, 0, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(T == kBF16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v),
                                              r, (int)offset, 0, 0);
}

} // namespace nmspmm
#endif
