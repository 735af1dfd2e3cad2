// New keys and values into the pages of a cache in 8 bits.
//
//   s = max(max |x| / Q, 2^-126, s of earlier tokens), code = round(x (1 / s)); earlier codes c -> round(c (s0 / s)) where s grows from s0
// Reads 4 bytes an element and writes 1, bound by memory for prompts and by the launch for a decode step.  A wave takes the keys, or the values, of one
// head over a strip of whole blocks, some 1024 vectors, which it holds in registers between the maximum and the codes: all of its loads are on
// their way together, and the search and the page look-ups (a lane a block) are paid once a strip.  Twenty prompts of 300
// to 4000 tokens, 8 heads of 128 (277 MB): 67 us, 4.1 TB/s, with blocks of 1 to 32 tokens; a token each for 64 sequences 6 us of kernel, less than a
// call takes the host.
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
    int block, strip, wide; // positions of a block, of a strip (whole blocks, 64 at most)
    Divisor page_size, by_block, by_strip, k_chunks, v_chunks, by_items;
    int* error_flag;
};

// Strips that the new tokens of sequence i touch have numbers from starts[i] / strip + 2 i on: n tokens touch at most floor(n / strip) + 2 of them,
// and floor((a + n) / strip) - floor(a / strip) + 2 is not less.  The numbers that are left over are no strip.
__device__ __forceinline__ int first_strip(int start, int i, const Divisor& strip) { return quotient(start, strip) + 2 * i; }

// W codes; W is 4 or 1
template <int KIND, int W>
__device__ __forceinline__ void store_codes(uint8_t* to, const float (&x)[4])
{
    const uint32_t c = to_codes<KIND>(x);
    if constexpr (W == 4)
        *reinterpret_cast<uint32_t*>(to) = c;
    else
        *to = (uint8_t)c;
}

template <int KIND, int W, int IT> // vectors of W, IT of a lane
__global__ __launch_bounds__(256) void kv8_append_kernel(Append8Params p)
{
    typedef float fv __attribute__((ext_vector_type(W)));
    // of a wave's blocks: their first rows among all pages (-1: no page), the largest |x|, 1 / scale
    __shared__ int row_of[4][64];
    __shared__ uint32_t most_of[4][64];
    __shared__ float up_of[4][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t item = blockIdx.x * 4 + wave;
    if (p.error_flag && blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.c.n_seqs; i += 256)
            if (!packed_start_ok(p.starts, i, p.tokens))
                *p.error_flag = 1;
    const int number = (int)(item / (uint32_t)p.by_items.by), which = (int)(item - (uint32_t)number * p.by_items.by), head = which < p.c.kv_heads ? which : which - p.c.kv_heads;
    const int s = __builtin_amdgcn_readfirstlane(not_above(SearchWave(), p.c.n_seqs, [&](int i) {
        const int a = p.starts[i];
        return first_strip(a < 0 ? 0 : (a > p.tokens ? p.tokens : a), i, p.by_strip) <= number;
    })) - 1;
    if (s < 0)
        return;
    const Span span = packed_span(p.starts, s, p.tokens);
    if (span.count == 0)
        return;
    // positions first .. end - 1 are new, those out of the cache aside
    const int64_t pos0 = (int64_t)p.c.lens[s] - span.count, end0 = pos0 + span.count;
    const int first = pos0 < 0 ? 0 : (pos0 > p.c.max_len ? p.c.max_len : (int)pos0), end = end0 > p.c.max_len ? p.c.max_len : (int)end0;
    if (p.error_flag && lane == 0 && (first != pos0 || end != end0))
        *p.error_flag = 1;
    if (first >= end)
        return;
    const int64_t strip_at = (int64_t)(quotient(first, p.by_strip) + (number - first_strip(span.first, s, p.by_strip))) * p.strip;
    if (strip_at >= end)
        return;
    const int begin = strip_at > first ? (int)strip_at : first, stop = end - strip_at < p.strip ? end : (int)strip_at + p.strip;
    if (begin >= stop)
        return;
    const int block0 = quotient(begin, p.by_block), blocks = quotient(stop - 1, p.by_block) - block0 + 1, old = begin - block0 * p.block; // blocks: up to 64
    const bool is_v = which >= p.c.kv_heads; // the waves of a workgroup have heads next to each other
    const int depth = is_v ? p.c.dv : p.c.dk;
    const int64_t a_row = (int64_t)p.c.kv_heads * depth, ld = is_v ? p.ldv : p.ldk;
    const float* from = (is_v ? p.v : p.k) + (span.first + (begin - pos0)) * ld + (int64_t)head * depth;
    uint8_t* to = static_cast<uint8_t*>(is_v ? p.c.v : p.c.k) + (int64_t)head * depth;
    float* scales = (is_v ? p.v_scale : p.k_scale) + head;
    int row0 = -1; // of block0 + lane
    if (lane < blocks)
        row0 = page_row(p.c.table + (int64_t)s * p.c.table_width, p.c.table_width, p.c.n_pages, p.page_size, (block0 + lane) * p.block);
    const Divisor by_chunks = is_v ? p.v_chunks : p.k_chunks;
    const int chunks = (int)by_chunks.by, total = (stop - begin) * chunks;
    const bool rows_of_16 = (chunks & 15) == 0; // sixteen lanes have one row
    fv x[IT];
    // a lane's vectors are 64 apart: their rows and depths follow from one another without quotients; lanes behind the last one have that
    struct Item {
        int row, chunk;
    };
    const int step_rows = quotient(64, by_chunks), step_chunks = 64 - step_rows * chunks, last_row = stop - begin - 1;
    auto item_at = [&](int base) {
        const int e = base + lane, r = quotient(e, by_chunks);
        return Item { r, e - r * chunks };
    };
    auto next = [&](Item& i) {
        i.row += step_rows;
        i.chunk += step_chunks;
        const bool over = i.chunk >= chunks;
        i.row += over;
        i.chunk -= over ? chunks : 0;
    };
    auto load = [&](int base) {
        Item i = item_at(base);
#pragma unroll
        for (int it = 0; it < IT; ++it)
            if (base + it * 64 < total) {
                const int r = i.row < last_row ? i.row : last_row;
                x[it] = *reinterpret_cast<const fv*>(from + r * ld + i.chunk * W);
                next(i);
            }
    };
    load(0); // on its way beside the look-ups
    if (lane < blocks) {
        row_of[wave][lane] = row0;
        most_of[wave][lane] = 0;
        if (row0 < 0 && p.error_flag)
            *p.error_flag = 1;
    }
    float* scale = scales + (int64_t)quotient(row0 < 0 ? 0 : row0, p.by_block) * p.c.kv_heads;
    const float before = lane == 0 && old > 0 && row0 >= 0 ? *scale : 0.f;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int base = 0; base < total; base += 64 * IT) {
        if (base > 0)
            load(base);
        Item item = item_at(base);
#pragma unroll
        for (int it = 0; it < IT; ++it)
            if (base + it * 64 < total) {
                uint32_t top = 0; // of |x| as a whole number: infinities and NaN are the largest
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const float one = x[it][i]; // the cast of a vector's element takes its first one
                    const uint32_t b = __builtin_bit_cast(uint32_t, one) & 0x7fffffffu;
                    top = b > top ? b : top;
                }
                const int at = quotient(old + (item.row < last_row ? item.row : last_row), p.by_block);
                next(item);
                if (rows_of_16) {
                    top = row16_most(top);
                    if ((lane & 15) == 0)
                        atomicMax(&most_of[wave][at], top);
                } else {
                    atomicMax(&most_of[wave][at], top);
                }
            }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    float by = 1.f; // of the first block's earlier codes; below zero where they become 0
    if (lane < blocks && row0 >= 0) {
        const float most = __builtin_bit_cast(float, most_of[wave][lane]);
        const bool odd = !(most < INFINITY) || !(before < INFINITY);
        const float now = odd ? NAN : fmaxf(fmaxf(most / most_code<KIND>(), kLeastScale), before);
        up_of[wave][lane] = odd ? 0.f : 1.f / now;
        by = odd ? -1.f : before / now;
        *scale = now;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    for (int base = 0; base < total; base += 64 * IT) {
        if (total > 64 * IT)
            load(base);
        Item item = item_at(base);
#pragma unroll
        for (int it = 0; it < IT; ++it)
            if (base + it * 64 < total) {
                const int r = item.row < last_row ? item.row : last_row, at = quotient(old + r, p.by_block), row = row_of[wave][at];
                const float up = up_of[wave][at];
                float y[4] = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
                for (int i = 0; i < W; ++i)
                    y[i] = up != 0.f ? x[it][i] * up : 0.f; // an infinity's codes are 0
                if (row >= 0 && item.row <= last_row)
                    store_codes<KIND, W>(to + (row + (old + r - at * p.block)) * a_row + item.chunk * W, y);
                next(item);
            }
    }
    // earlier tokens of the first block, whose scale has grown (or become NaN)
    const int first_row = __builtin_amdgcn_readfirstlane(row0);
    by = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, by)));
    if (old > 0 && first_row >= 0 && by != 1.f)
        for (int e = lane; e < old * chunks; e += 64) {
            const int r = quotient(e, by_chunks);
            uint8_t* at = to + (first_row + r) * a_row + (e - r * chunks) * W;
            float y[4] = { 0.f, 0.f, 0.f, 0.f };
            if (by >= 0.f) { // where a scale has grown 2^150-fold this is zero, and codes are zeros of their own sign
                from_codes<KIND>(W == 4 ? *reinterpret_cast<uint32_t*>(at) : *at, y);
#pragma unroll
                for (int i = 0; i < W; ++i)
                    y[i] *= by;
            }
            store_codes<KIND, W>(at, y);
        }
}

// Blocks of more than 1024 vectors a head would be read twice, for the maximum and for the codes; up to 2048 they fit into twice the registers
// (blocks of 64 tokens, 8 heads of 128, 20 prompts of 300 to 4000: 95 -> 78 us; blocks that fit into half of them keep more waves, 67 us).
template <int KIND>
static void append8_launch(const Append8Params& p, dim3 grid)
{
    const int chunks = (int)(p.k_chunks.by > p.v_chunks.by ? p.k_chunks.by : p.v_chunks.by);
    if (!p.wide)
        hipLaunchKernelGGL((kv8_append_kernel<KIND, 1, 16>), grid, dim3(256), 0, stream(), p);
    else if ((int64_t)p.strip * chunks <= 1024 || (int64_t)p.strip * chunks > 2048)
        hipLaunchKernelGGL((kv8_append_kernel<KIND, 4, 16>), grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL((kv8_append_kernel<KIND, 4, 32>), grid, dim3(256), 0, stream(), p);
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
    // vectors of four wherever every row and head starts on one
    const uintptr_t rows = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)
        | 4 * (reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v));
    const int wide = (rows & 15) == 0 && ((ldk | ldv | c.dk | c.dv) & 3) == 0;
    const int k_chunks = wide ? c.dk / 4 : c.dk, v_chunks = wide ? c.dv / 4 : c.dv;
    int64_t blocks = 1024 / (int64_t)(k_chunks > v_chunks ? k_chunks : v_chunks) / cache->block;
    blocks = blocks < 1 ? 1 : (blocks > 64 ? 64 : blocks);
    const int strip = (int)blocks * cache->block;
    FDX_REQUIRE((int64_t)cache->block * (k_chunks > v_chunks ? k_chunks : v_chunks) < ((int64_t)1 << 30), "kv8_append: blocks of more than 2^30 elements of a head");
    const int64_t items = ((int64_t)tokens / strip + 2 * (int64_t)c.n_seqs + 1) * 2 * c.kv_heads;
    FDX_REQUIRE(items < ((int64_t)1 << 25), "kv8_append: strips * key heads too many for one launch");
    const Append8Params p { k, v, ldk, ldv, starts, tokens, c, cache->k_scale, cache->v_scale, cache->block, strip, wide, make_divisor(c.page_size),
        make_divisor(cache->block), make_divisor(strip), make_divisor(k_chunks), make_divisor(v_chunks), make_divisor(2 * c.kv_heads), error_flag_dev };
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
