// fp32 values as sums of two fp16 values, for products on the fp16 matrix instructions.
//
// x s = h + l + r with h and l fp16 and s a power of two: each rounds to nearest, so |r| <= 2^-22 |x s| where neither is subnormal.
// x y is then h h' + h l' + l h', the dropped l l' and the two r again 2^-22 each of the product at most: 22 bits where fp32 has 24,
// and rounded three times instead of once, for three products at fp16's rate.  (Three bf16 values hold fp32 exactly and take six.)
// s brings the largest value of a set (a query, a tile of keys or of values) to 2^14 .. 2^15; fp16 keeps full precision down to
// 2^-14 and has a last bit of 2^-24, so values are held to 22 bits down to 2^-17 of the largest and to 2^-40 of the largest below.
#pragma once
#include "common.hpp"

namespace fdx {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// A power of two that brings values of up to 2^(e - 127 + 1) to at most 2^15 (as near as fp32 has powers of two), and its reciprocal.  STEP:
// its exponent is a multiple of STEP, for powers that should not change with every set; the largest value then ends up STEP - 1 powers lower
// at worst.
struct Pow2 {
    float up, down;
};
template <int STEP>
__device__ __forceinline__ Pow2 pow2_for(int e)
{
    int field = (268 - e) / STEP * STEP;
    field = field > 253 ? 253 / STEP * STEP : field; // 12 or more: e is at most 255
    return { __builtin_bit_cast(float, (uint32_t)field << 23), __builtin_bit_cast(float, (uint32_t)(254 - field) << 23) };
}
__device__ __forceinline__ int exponent(float x) { return (int)(__builtin_bit_cast(uint32_t, x) >> 23 & 255u); }

// Sets of rows that share a power: keys and values of a tile.  A row keeps 22 bits of its own largest value as long as that is not below
// 2^-17 of the set's (2^-14 with a power in steps of four: fp16's last bit is 2^-24, and half of that has to be 2^-22 of the row's); sets that
// reach further are not for these products.  Two rows' largest values,
// one in each half, as what the set's spread is found from: `top` has their exponents, `low` 255 less each, 0 for a row of zeros.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
struct Spread {
    u16x2 top, low;
};
__device__ __forceinline__ Spread row_spread(float a, float b)
{
    const int ea = exponent(a), eb = exponent(b);
    return { u16x2 { (unsigned short)ea, (unsigned short)eb },
        u16x2 { (unsigned short)(a == 0.f ? 0 : 255 - ea), (unsigned short)(b == 0.f ? 0 : 255 - eb) } };
}
__device__ __forceinline__ u16x2 most(u16x2 a, u16x2 b) { return __builtin_elementwise_max(a, b); }
template <int CTRL>
__device__ __forceinline__ u16x2 most_dpp(u16x2 v)
{
    return most(v, __builtin_bit_cast(u16x2, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true)));
}
// over a wave whose groups of N neighbouring lanes (4 or 8) agree
template <int N>
__device__ __forceinline__ u16x2 most_of_wave(u16x2 v)
{
    if (N == 4)
        v = most_dpp<0x141>(v); // row_half_mirror
    v = most_dpp<0x140>(v);     // row_mirror
    uint32_t x = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    v = most(__builtin_bit_cast(u16x2, (uint32_t)r[0]), __builtin_bit_cast(u16x2, (uint32_t)r[1]));
    x = __builtin_bit_cast(uint32_t, v);
    const auto q = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return most(__builtin_bit_cast(u16x2, (uint32_t)q[0]), __builtin_bit_cast(u16x2, (uint32_t)q[1]));
}
// whether keys (first half) and values (second half, in steps of four) can share their powers
__device__ __forceinline__ bool spread_fits(u16x2 top, u16x2 low) { return top[0] + low[0] <= 255 + 17 && top[1] + low[1] <= 255 + 14; }

// Both roundings are of mixed-precision multiply-adds, x s and x s - h, which take and give either type.
__device__ __forceinline__ void split2x8(const float (&x)[8], float s, f16x8& h, f16x8& l)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = (_Float16)__builtin_fmaf(x[i], s, 0.f);
        l[i] = (_Float16)__builtin_fmaf(x[i], s, -(float)h[i]);
    }
}
// the same for values that need no power; the factor of one, which the compiler does not know, keeps x - h the multiply-add that takes h
// as it is (a subtraction takes two conversions more)
__device__ __forceinline__ void split2x8(const float (&x)[8], f16x8& h, f16x8& l)
{
    float one = 1.f;
    asm("" : "+s"(one));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = (_Float16)x[i];
        l[i] = (_Float16)__builtin_fmaf(x[i], one, -(float)h[i]);
    }
}
// the largest of three, NaN if one is: one instruction (fmaxf takes another one for every value that the compiler did not compute itself)
__device__ __forceinline__ float max3(float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); }

// the larger of a lane's value and that of the lane 32 away, on the vector unit (a shuffle is a trip through LDS)
__device__ __forceinline__ float max_halves(float v)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

} // namespace fdx
