// fp32 values as sums of two fp16 values, for products on the fp16 matrix instructions.
//
// x s = h + l + r with h and l fp16 and s a power of two: each rounds to nearest, so |r| <= 2^-22 |x s| where neither is subnormal.
// x y is then h h' + h l' + l h', the dropped l l' and the two r again 2^-22 each of the product at most: 22 bits where fp32 has 24,
// and rounded three times instead of once, for three products at fp16's rate.  (Three bf16 values hold fp32 exactly and take six.)
// s brings the largest value of a set (a query, a tile of keys or of values) to 2^14 .. 2^15; fp16 keeps full precision down to
// 2^-14, l down to 2^-24, so values are held to 22 bits down to 2^-17 of the largest and to 2^-40 of the largest below.
#pragma once
#include "common.hpp"

namespace fdx {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// the power of two that brings `largest` to 2^14 .. 2^15 (as near as fp32 has powers of two), and its reciprocal
struct Pow2 {
    float up, down;
};
__device__ __forceinline__ Pow2 pow2_for(float largest)
{
    int field = 268 - (int)(__builtin_bit_cast(uint32_t, largest) >> 23 & 255u);
    field = field > 253 ? 253 : field;
    return { __builtin_bit_cast(float, (uint32_t)field << 23), __builtin_bit_cast(float, (uint32_t)(254 - field) << 23) };
}

// Two instructions a value: the mixed-precision multiply-add rounds x s to h, and x s - h to l, without a register for either in fp32
// (the compiler takes three, a product among them).
__device__ __forceinline__ void split2x8(const float (&x)[8], float s, f16x8& h, f16x8& l)
{
    typedef uint32_t u32x4_ __attribute__((ext_vector_type(4)));
    u32x4_ hw, lw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t a, b;
        asm("v_fma_mixlo_f16 %0, %1, %2, 0" : "=v"(a) : "v"(x[2 * i]), "v"(s));
        asm("v_fma_mixhi_f16 %0, %1, %2, 0" : "+v"(a) : "v"(x[2 * i + 1]), "v"(s));
        asm("v_fma_mixlo_f16 %0, %1, %2, -%3 op_sel_hi:[0,0,1]" : "=v"(b) : "v"(x[2 * i]), "v"(s), "v"(a));
        asm("v_fma_mixhi_f16 %0, %1, %2, -%3 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(b) : "v"(x[2 * i + 1]), "v"(s), "v"(a));
        hw[i] = a;
        lw[i] = b;
    }
    h = __builtin_bit_cast(f16x8, hw);
    l = __builtin_bit_cast(f16x8, lw);
}
// the same for values that need no power
__device__ __forceinline__ void split2x8(const float (&x)[8], f16x8& h, f16x8& l)
{
    typedef uint32_t u32x4_ __attribute__((ext_vector_type(4)));
    u32x4_ hw, lw;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __builtin_bit_cast(uint32_t, f16x2 { (_Float16)x[2 * i], (_Float16)x[2 * i + 1] });
        uint32_t b;
        asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(b) : "v"(x[2 * i]), "v"(a));
        asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(b) : "v"(x[2 * i + 1]), "v"(a));
        hw[i] = a;
        lw[i] = b;
    }
    h = __builtin_bit_cast(f16x8, hw);
    l = __builtin_bit_cast(f16x8, lw);
}
// max(a, b, c) and max(a, |b|, |c|) as one instruction each: the compiler's maximum of values that it has not computed itself takes another
// one a value, for NaNs
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max3_abs(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, abs(%2), abs(%3)" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

} // namespace fdx
