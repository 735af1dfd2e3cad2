// New keys and values into the pages of a cache in 8 bits.
#include <cfloat>

#include "kv8.hpp"

namespace fdx {

struct Append8Params {
    const float *k, *v;
    int64_t ldk, ldv;
    const int32_t* starts;
    int tokens;
    fdx_kv_pages c;
    float *k_scale, *v_scale;
    int block, wide;
    Divisor page_size, by_block;
    int* error_flag;
};

// Blocks that the new tokens of sequence i touch have numbers from starts[i] / block + 2 i on: n tokens touch at most floor(n / block) + 2 of them,
// and floor((a + n) / block) - floor(a / block) + 2 is not less.  The numbers that are left over are no block.
__device__ __forceinline__ int64_t first_block(int start, int i, const Divisor& block) { return (int64_t)quotient(start, block) + 2 * i; }

// W codes of a row from depth d on, as fp32 values or codes; W is 4 or 1
template <int KIND, int W>
__device__ __forceinline__ void store_codes(uint8_t* to, const float (&x)[4])
{
    const uint32_t c = to_codes<KIND>(x);
    if constexpr (W == 4)
        *reinterpret_cast<uint32_t*>(to) = c;
    else
        *to = (uint8_t)c;
}

// A wave takes a head's keys, or values, in one block of one sequence.
template <int KIND, int W>
__global__ __launch_bounds__(256) void kv8_append_kernel(Append8Params p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    if (p.error_flag && blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.c.n_seqs; i += 256)
            if (!packed_start_ok(p.starts, i, p.tokens))
                *p.error_flag = 1;
    const int64_t number = item / (2 * p.c.kv_heads);
    const int which = (int)(item - number * (2 * p.c.kv_heads)), head = which >> 1;
    const int s = not_above(SearchWave(), p.c.n_seqs, [&](int i) {
        const int a = p.starts[i];
        return first_block(a < 0 ? 0 : (a > p.tokens ? p.tokens : a), i, p.by_block) <= number;
    }) - 1;
    if (s < 0)
        return;
    const Span span = packed_span(p.starts, s, p.tokens);
    if (span.count == 0)
        return;
    // positions first .. end - 1 are new, those out of the cache aside
    const int64_t pos0 = (int64_t)p.c.lens[s] - span.count, end0 = pos0 + span.count;
    const int64_t first = pos0 < 0 ? 0 : pos0, end = end0 > p.c.max_len ? p.c.max_len : end0;
    if (p.error_flag && lane == 0 && (first != pos0 || end != end0))
        *p.error_flag = 1;
    if (first >= end)
        return;
    const int64_t blk = first / p.block + (number - first_block(span.first, s, p.by_block));
    const int64_t begin = blk * p.block > first ? blk * p.block : first, stop = (blk + 1) * p.block < end ? (blk + 1) * p.block : end;
    if (begin >= stop)
        return;
    const int row0 = page_row(p.c.table + (int64_t)s * p.c.table_width, p.c.table_width, p.c.n_pages, p.page_size, (int)(blk * p.block));
    if (row0 < 0) {
        if (p.error_flag && lane == 0)
            *p.error_flag = 1;
        return;
    }
    const bool is_v = which & 1;
    const int depth = is_v ? p.c.dv : p.c.dk, a_row = p.c.kv_heads * depth;
    const int64_t ld = is_v ? p.ldv : p.ldk;
    const float* from = (is_v ? p.v : p.k) + (span.first + (begin - pos0)) * ld + (int64_t)head * depth;
    uint8_t* to = static_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + ((int64_t)row0 + (begin - blk * p.block)) * a_row + (int64_t)head * depth;
    float* scale = (is_v ? p.v_scale : p.k_scale) + (int64_t)quotient(row0, p.by_block) * p.c.kv_heads + head;
    const int old = (int)(begin - blk * p.block), rows = (int)(stop - begin), chunks = (depth + W - 1) / W;
    const float before = old > 0 ? *scale : 0.f;
    uint32_t top = 0; // of |x| as a whole number: infinities and NaN are the largest
    for (int r = 0; r < rows; ++r)
        for (int d = lane; d < chunks; d += 64)
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const uint32_t b = __builtin_bit_cast(uint32_t, from[r * ld + d * W + e]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
    for (int w = 32; w > 0; w >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, w, 64);
        top = o > top ? o : top;
    }
    const float most = __builtin_bit_cast(float, top);
    const bool odd = !(most < INFINITY) || !(before < INFINITY);
    float now = fmaxf(most / most_code<KIND>(), kLeastScale);
    now = odd ? NAN : fmaxf(now, before);
    const float up = odd ? 0.f : 1.f / now;
    if (old > 0 && now != before) { // NaN too
        const float by = odd ? 0.f : before / now;
        for (int r = 0; r < old; ++r)
            for (int d = lane; d < chunks; d += 64) {
                uint8_t* at = to + (int64_t)(r - old) * a_row + d * W;
                float x[4] = { 0.f, 0.f, 0.f, 0.f };
                if (!odd) {
                    from_codes<KIND>(W == 4 ? *reinterpret_cast<uint32_t*>(at) : *at, x);
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        x[e] *= by;
                }
                store_codes<KIND, W>(at, x);
            }
    }
    for (int r = 0; r < rows; ++r)
        for (int d = lane; d < chunks; d += 64) {
            float x[4] = { 0.f, 0.f, 0.f, 0.f };
            if (!odd)
#pragma unroll
                for (int e = 0; e < W; ++e)
                    x[e] = from[r * ld + d * W + e] * up;
            store_codes<KIND, W>(to + (int64_t)r * a_row + d * W, x);
        }
    if (lane == 0)
        *scale = now;
}

template <int KIND>
static void append8_launch(const Append8Params& p, dim3 grid)
{
    if (p.wide)
        hipLaunchKernelGGL((kv8_append_kernel<KIND, 4>), grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL((kv8_append_kernel<KIND, 1>), grid, dim3(256), 0, stream(), p);
}

} // namespace fdx

using namespace fdx;

extern "C" fdx_status fdx_kv8_append_f32(const float* k, int64_t ldk, const float* v, int64_t ldv, const int32_t* starts, int tokens,
    const fdx_kv_pages8* cache, int* error_flag_dev)
{
    const fdx_status st = check_kv_pages8("kv8_append", cache);
    if (st != FDX_OK)
        return st;
    const fdx_kv_pages& c = cache->pages;
    FDX_REQUIRE(k && v && starts, "kv8_append: null pointer");
    FDX_REQUIRE(tokens > 0 && tokens <= (1 << 24), "kv8_append: 1 to 2^24 tokens");
    const int64_t nk = (int64_t)c.kv_heads * c.dk, nv = (int64_t)c.kv_heads * c.dv;
    FDX_REQUIRE(ldk >= nk && ldv >= nv, "kv8_append: rows overlap");
    const int64_t items = ((int64_t)tokens / cache->block + 2 * (int64_t)c.n_seqs + 1) * 2 * c.kv_heads;
    FDX_REQUIRE(items < ((int64_t)1 << 32), "kv8_append: blocks * key heads too many for one launch");
    // vectors of four wherever every row and head starts on one
    const uintptr_t rows = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)
        | 4 * (reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v));
    const int wide = (rows & 15) == 0 && ((ldk | ldv | c.dk | c.dv) & 3) == 0;
    const Append8Params p { k, v, ldk, ldv, starts, tokens, c, cache->k_scale, cache->v_scale, cache->block, wide, make_divisor(c.page_size),
        make_divisor(cache->block), error_flag_dev };
    const dim3 grid((unsigned)((items + 3) / 4));
    profile_begin();
    if (c.type == FDX_KV_I8)
        append8_launch<kI8>(p, grid);
    else
        append8_launch<kE4M3>(p, grid);
    profile_end("kv8_append_f32", 0.0, (double)tokens * (double)(nk + nv) * 5.0);
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
