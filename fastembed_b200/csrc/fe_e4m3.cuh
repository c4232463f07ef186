// fe_e4m3.cuh — device helpers of the 8-bit (OCP e4m3: 4 exponent bits, 3 mantissa bits,
// largest value 448, no infinities) kernels: conversions and the scale rules.
#pragma once

#include <cuda_fp16.h>

#include "fe_common.cuh"

namespace fe {

constexpr float kE4m3Max = 448.0f;
// The smallest row maximum that sets a row scale: keeps the scale and its reciprocal normal
// fp32 numbers, so that a row of zeros needs no special case.
constexpr float kTinyAmax = 7.70371977754894341e-34f;  // 2^-110

// Two fp32 values to two e4m3 codes (lo in bits 0-7), round to nearest even, saturating;
// NaN gives the NaN code.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi)
{
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

__device__ __forceinline__ uint32_t pack_e4m3x4(float a, float b, float c, float d)
{
    return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
}

// Two e4m3 codes (the low 16 bits) to two f16 values: exact, subnormals included, NaN kept.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t codes)
{
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(codes)));
    return r;
}

__device__ __forceinline__ float2 e4m3x2_to_f32x2(uint32_t codes)
{
    const uint32_t h = e4m3x2_to_f16x2(codes);
    return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// |v| where v is finite, 0 where it is infinite or NaN (the row and block maxima leave those out)
__device__ __forceinline__ float finite_abs(float v)
{
    const float a = fabsf(v);
    return a <= 3.402823466e38f ? a : 0.f;
}

// v, or NaN where v is not finite (the saturating conversion would make an infinity 448)
__device__ __forceinline__ float finite_or_nan(float v)
{
    return fabsf(v) <= 3.402823466e38f ? v : __int_as_float(0x7fffffff);
}

// v / scale, with inv = 1 / scale: a product, then the quotient's remainder by one fma and what it adds by another
// (Markstein's division).  The product alone puts quotients on a border between two codes, of which rows
// of bf16 numbers have some (3 codes of 10,000), on either side of it.  Equal to the fp32 quotient but for
// those within 2^-46 of halfway between two fp32 numbers, and all of a bf16 v and a bf16 maximum / 448 are equal.
// The signs are such that -0 stays -0.  The compiler's division in its place: 26,508 x 1,024 with the norm
// 54.6 us, so 50.
__device__ __forceinline__ float div_by(float v, float scale, float inv)
{
    const float p = -v * -inv;
    return fmaf(fmaf(p, scale, -v), -inv, p);
}

__device__ __forceinline__ void div_by2(float &a, float &b, float scale, float inv)
{
    const float na = -a, nb = -b;
    float p = na, q = nb, r, s;
    mul_f32x2(p, q, -inv, -inv);
    fma_f32x2v(r, s, p, q, scale, scale, na, nb);
    fma_f32x2v(a, b, r, s, -inv, -inv, p, q);
}

}  // namespace fe
