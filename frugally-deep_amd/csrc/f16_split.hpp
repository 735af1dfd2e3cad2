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

__device__ __forceinline__ void split2x8(const float (&x)[8], float s, f16x8& h, f16x8& l)
{
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        h[i] = (_Float16)(x[i] * s);
        l[i] = (_Float16)__builtin_fmaf(x[i], s, -(float)h[i]);
    }
}

} // namespace fdx
