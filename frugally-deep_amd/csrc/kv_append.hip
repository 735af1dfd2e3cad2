// New keys and values into the pages of a cache.
//
// A copy with computed places: reads 4 bytes and writes 4 (2 in bf16 pages) an element, bound by memory for prompts and by the
// launch for a decode step.  Twenty prompts of 300 to 4000 tokens, 8 heads of 128, fp32 pages (444 MB): 84 us, 5.3 TB/s; a token each for 64
// sequences 3.7 us of kernel, less than a call takes the host.
#include <cstdint>

#include "ragged_attn.hpp"

namespace fdx {

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));

struct AppendParams {
    const float *k, *v;
    int64_t ldk, ldv;
    const int32_t* starts;
    int tokens;
    fdx_kv_pages c;
    Divisor page_size;
    int* error_flag;
};

template <typename T, int W>
__device__ __forceinline__ void append_row(const float* __restrict__ from, T* __restrict__ to, int count, int lane)
{
    typedef float fv __attribute__((ext_vector_type(W)));
    typedef T tv __attribute__((ext_vector_type(W)));
    for (int i = lane * W; i < count; i += 64 * W)
        *reinterpret_cast<tv*>(to + i) = __builtin_convertvector(*reinterpret_cast<const fv*>(from + i), tv);
}

// A wave takes a token's keys or its values.
template <typename T, int W>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    if (p.error_flag && blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.c.n_seqs; i += 256)
            if (!packed_start_ok(p.starts, i, p.tokens))
                *p.error_flag = 1;
    const int row = (int)(item >> 1);
    if (row >= p.tokens)
        return;
    const int s = find_row(SearchWave(), p.starts, p.c.n_seqs, p.tokens, row);
    if (s < 0)
        return;
    const Span span = packed_span(p.starts, s, p.tokens);
    const int64_t pos = (int64_t)p.c.lens[s] - span.count + (row - span.first);
    const int at = pos < 0 || pos >= p.c.max_len
        ? -1
        : page_row(p.c.table + (int64_t)s * p.c.table_width, p.c.table_width, p.c.n_pages, p.page_size, (int)pos);
    if (at < 0) {
        if (p.error_flag && lane == 0)
            *p.error_flag = 1;
        return;
    }
    const int nk = p.c.kv_heads * p.c.dk, nv = p.c.kv_heads * p.c.dv;
    if (item & 1)
        append_row<T, W>(p.v + (int64_t)row * p.ldv, static_cast<T*>(p.c.v) + (int64_t)at * nv, nv, lane);
    else
        append_row<T, W>(p.k + (int64_t)row * p.ldk, static_cast<T*>(p.c.k) + (int64_t)at * nk, nk, lane);
}

// what every call asks of a cache whose elements have `size` bytes
static fdx_status check_kv_shape(const char* who, const fdx_kv_pages* c, bool type_ok, uintptr_t size)
{
    FDX_REQUIRE(c && c->k && c->v && c->table && c->lens, "%s: null pointer", who);
    FDX_REQUIRE(type_ok, "%s: unknown element type %d of the cache", who, c->type);
    FDX_REQUIRE(c->n_pages > 0 && c->page_size > 0 && c->kv_heads > 0 && c->dk > 0 && c->dv > 0 && c->n_seqs > 0 && c->table_width > 0
            && c->max_len > 0,
        "%s: bad shape of the cache", who);
    FDX_REQUIRE((int64_t)c->n_pages * c->page_size < ((int64_t)1 << 31), "%s: more than 2^31 positions in the cache", who);
    FDX_REQUIRE((int64_t)c->kv_heads * c->dk < ((int64_t)1 << 31) && (int64_t)c->kv_heads * c->dv < ((int64_t)1 << 31),
        "%s: rows of the cache too long", who);
    FDX_REQUIRE(c->max_len <= (1 << 30), "%s: sequences of more than 2^30 positions", who);
    FDX_REQUIRE((int64_t)c->table_width * c->page_size >= c->max_len, "%s: the table does not reach max_len", who);
    FDX_REQUIRE(((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & (size - 1)) == 0,
        "%s: pages that are not aligned to their elements", who);
    return FDX_OK;
}
fdx_status check_kv_pages(const char* who, const fdx_kv_pages* c)
{
    return check_kv_shape(who, c, c && (c->type == FDX_KV_F32 || c->type == FDX_KV_BF16), c && c->type == FDX_KV_BF16 ? 2 : 4);
}
fdx_status check_kv_pages8(const char* who, const fdx_kv_pages8* c)
{
    const fdx_kv_pages* pages = c ? &c->pages : nullptr;
    const fdx_status st = check_kv_shape(who, pages, pages && (pages->type == FDX_KV_I8 || pages->type == FDX_KV_E4M3), 1);
    if (st != FDX_OK)
        return st;
    FDX_REQUIRE(c->k_scale && c->v_scale, "%s: null pointer", who);
    FDX_REQUIRE(((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) == 0, "%s: scales that are not aligned", who);
    FDX_REQUIRE(c->block > 0 && pages->page_size % c->block == 0, "%s: blocks of %d positions do not divide pages of %d", who, c->block, pages->page_size);
    return FDX_OK;
}

} // namespace fdx

using namespace fdx;

extern "C" fdx_status fdx_kv_append_f32(const float* k, int64_t ldk, const float* v, int64_t ldv, const int32_t* starts, int tokens,
    const fdx_kv_pages* cache, int* error_flag_dev)
{
    fdx_status st = check_kv_pages("kv_append", cache);
    if (st != FDX_OK)
        return st;
    FDX_REQUIRE(k && v && starts, "kv_append: null pointer");
    FDX_REQUIRE(tokens > 0 && tokens <= (1 << 24), "kv_append: 1 to 2^24 tokens");
    const int64_t nk = (int64_t)cache->kv_heads * cache->dk, nv = (int64_t)cache->kv_heads * cache->dv;
    FDX_REQUIRE(ldk >= nk && ldv >= nv, "kv_append: rows overlap");
    const AppendParams p { k, v, ldk, ldv, starts, tokens, *cache, make_divisor(cache->page_size), error_flag_dev };
    const dim3 grid((unsigned)((2 * (int64_t)tokens + 3) / 4));
    // vectors of four wherever every row of the four tensors starts on one
    const uintptr_t rows = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)
        | (cache->type == FDX_KV_BF16 ? 2 : 1) * (reinterpret_cast<uintptr_t>(cache->k) | reinterpret_cast<uintptr_t>(cache->v));
    const bool wide = (rows & 15) == 0 && ((ldk | ldv | nk | nv) & 3) == 0;
    hipStream_t s = stream();
    profile_begin();
    if (cache->type == FDX_KV_F32) {
        if (wide)
            hipLaunchKernelGGL((kv_append_kernel<float, 4>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((kv_append_kernel<float, 1>), grid, dim3(256), 0, s, p);
    } else {
        if (wide)
            hipLaunchKernelGGL((kv_append_kernel<__bf16, 4>), grid, dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((kv_append_kernel<__bf16, 1>), grid, dim3(256), 0, s, p);
    }
    profile_end("kv_append_f32", 0.0, (double)tokens * (double)(nk + nv) * (cache->type == FDX_KV_BF16 ? 6.0 : 8.0));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
