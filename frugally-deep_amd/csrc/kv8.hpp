// Elements of a cache in 8 bits: a code times the fp32 scale of its block (fdx_kv_pages8).
#pragma once
#include "ragged_attn.hpp"

namespace fdx {

enum { kI8 = 0, kE4M3 = 1 };
constexpr float kMostI8 = 127.f, kMostE4M3 = 448.f;
constexpr float kLeastScale = 0x1p-126f; // of a block of zeros too: its reciprocal is finite

template <int KIND>
__device__ __forceinline__ constexpr float most_code() { return KIND == kI8 ? kMostI8 : kMostE4M3; }

// four values, in units of codes, as four codes
template <int KIND>
__device__ __forceinline__ uint32_t to_codes(const float (&x)[4])
{
    if constexpr (KIND == kI8) {
        // beside 1.5 * 2^23 the last bit is one: the sum is rounded to a whole number, ties to even, and its last byte is the code
        uint32_t r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            r[e] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_fmed3f(x[e], -kMostI8, kMostI8) + 12582912.f);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(r[3], r[2], 0x0c0c0400u), __builtin_amdgcn_perm(r[1], r[0], 0x0c0c0400u), 0x05040100u);
    } else {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[e] = __builtin_amdgcn_fmed3f(x[e], -kMostE4M3, kMostE4M3);
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
    }
}
// and back
template <int KIND>
__device__ __forceinline__ void from_codes(uint32_t c, float (&x)[4])
{
    if constexpr (KIND == kI8) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            x[e] = (float)(int8_t)(c >> (8 * e));
    } else {
        x[0] = __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
        x[1] = __builtin_amdgcn_cvt_f32_fp8((int)c, 1);
        x[2] = __builtin_amdgcn_cvt_f32_fp8((int)c, 2);
        x[3] = __builtin_amdgcn_cvt_f32_fp8((int)c, 3);
    }
}

// Four codes as four fp16 values, exactly: two pairs
template <int KIND>
__device__ __forceinline__ void f16_of_codes(uint32_t c, uint32_t& lo, uint32_t& hi)
{
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    if constexpr (KIND == kI8) {
        // 1024 + n has n as its last bits for n = code + 128
        const uint32_t n = c ^ 0x80808080u;
        const f16x2 off = { (_Float16)1152.f, (_Float16)1152.f };
        lo = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(n, 0x64646464u, 0x00050004u)) - off);
        hi = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(n, 0x64646464u, 0x00070006u)) - off);
    } else {
        lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, false));
        hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(c, 1.f, true));
    }
}
// four rows of four codes, transposed
__device__ __forceinline__ void transpose_codes(const uint32_t (&r)[4], uint32_t (&t)[4])
{
    const uint32_t a = __builtin_amdgcn_perm(r[1], r[0], 0x05010400u), b = __builtin_amdgcn_perm(r[3], r[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(r[1], r[0], 0x07030602u), d = __builtin_amdgcn_perm(r[3], r[2], 0x07030602u);
    t[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    t[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    t[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    t[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}

// sum over the lanes up to this one
__device__ __forceinline__ int wave_prefix(int v)
{
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true); // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true); // the last lane of a row to the row behind it
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true); // lane 31 to lanes 32 ..
    return v;
}
// the largest of sixteen lanes' numbers, in all of them
template <int CTRL>
__device__ __forceinline__ uint32_t most_dpp(uint32_t v)
{
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, true);
    return o > v ? o : v;
}
__device__ __forceinline__ uint32_t row16_most(uint32_t v) { return most_dpp<0x140>(most_dpp<0x141>(most_dpp<0x4E>(most_dpp<0xB1>(v)))); }

// where the scales of a cache are
struct Scales8 {
    const float *k, *v;
    Divisor block;
};

} // namespace fdx
