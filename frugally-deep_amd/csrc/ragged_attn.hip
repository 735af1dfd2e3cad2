// Attention over packed prompts and over paged caches (gfx950), query heads in groups that share a key / value head.
#include "ragged_attn.hpp"

namespace fdx {

fdx_status check_kv_pages(const char* who, const fdx_kv_pages* c); // kv_append.hip

// ---- one wave, one query row: the formula as it stands ----
template <int KIND>
__global__ __launch_bounds__(256) void ragged_plain_kernel(RaggedParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (p.error_flag && blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens));
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int row = (int)(item / p.heads), head = (int)(item % p.heads);
    if (row >= p.tokens)
        return;
    const int index = find_row(p.starts, p.n_seqs, p.tokens, row);
    if (index < 0)
        return;
    const Sequence s = sequence_of<KIND>(p, index, packed_span(p.starts, index, p.tokens));
    raise_flag(p, s.cut);
    if (row - s.span.first >= s.span.count)
        return;
    const int visible = visible_keys(p, s, row - s.span.first);
    float m, l, o[2];
    bool missing = false;
    plain_row<KIND>(p, s, p.q + (int64_t)row * p.ldq + (int64_t)head * p.dk, head / p.group, 0, visible, m, l, o, missing);
    raise_flag(p, missing);
    const bool sees = __any(m != -INFINITY) || visible > 0;
    float* to = p.out + (int64_t)row * p.ldo + (int64_t)head * p.dv;
    if (lane < p.dv)
        to[lane] = finish(o[0], l, sees);
    if (64 + lane < p.dv)
        to[64 + lane] = finish(o[1], l, sees);
}

template <int KIND>
static void ragged_launch(const RaggedParams& p, void* scratch)
{
    (void)scratch;
    hipLaunchKernelGGL(ragged_plain_kernel<KIND>, dim3((unsigned)(((int64_t)p.tokens * p.heads + 3) / 4)), dim3(256), 0, stream(), p);
}

static fdx_status check_ragged(const char* who, const RaggedParams& p, const void* scratch, size_t need)
{
    FDX_REQUIRE(p.q && p.k && p.v && p.starts && p.out, "%s: null pointer", who);
    FDX_REQUIRE(p.n_seqs > 0 && p.tokens > 0 && p.heads > 0 && p.kv_heads > 0 && p.dk > 0 && p.dv > 0, "%s: bad shape", who);
    FDX_REQUIRE(p.heads % p.kv_heads == 0, "%s: %d query heads cannot share %d key heads", who, p.heads, p.kv_heads);
    FDX_REQUIRE((int64_t)p.tokens * p.heads <= ((int64_t)1 << 26) && p.n_seqs <= (1 << 22) && p.heads <= 65535,
        "%s: tokens * heads or sequences too many for one launch", who);
    FDX_REQUIRE(p.ldq >= (int64_t)p.heads * p.dk && p.ldo >= (int64_t)p.heads * p.dv && p.ldk >= (int64_t)p.kv_heads * p.dk
            && p.ldv >= (int64_t)p.kv_heads * p.dv,
        "%s: rows overlap", who);
    FDX_REQUIRE(need == 0 || (scratch && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0), "%s: scratch missing or not 16-byte aligned", who);
    if (p.dk > 128 || p.dv > 128) {
        set_error("%s: depths up to 128, not %d and %d", who, p.dk, p.dv);
        return FDX_ERR_UNSUPPORTED;
    }
    return FDX_OK;
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_mha_packed_scratch_bytes(int tokens, int n_seqs, int heads, int kv_heads, int dk, int dv)
{
    (void)tokens; (void)n_seqs; (void)heads; (void)kv_heads; (void)dk; (void)dv;
    return 0;
}

extern "C" fdx_status fdx_mha_packed_f32(const float* q, int64_t ldq, const float* k, int64_t ldk, const float* v, int64_t ldv,
    const int32_t* starts, int n_seqs, int tokens, int heads, int kv_heads, int dk, int dv, int causal, float* out, int64_t ldo,
    void* scratch_dev, int* error_flag_dev)
{
    RaggedParams p {};
    p.q = q; p.ldq = ldq; p.k = k; p.ldk = ldk; p.v = v; p.ldv = ldv; p.out = out; p.ldo = ldo;
    p.starts = starts; p.n_seqs = n_seqs; p.tokens = tokens;
    p.heads = heads; p.kv_heads = kv_heads; p.group = kv_heads > 0 ? heads / kv_heads : 0;
    p.dk = dk; p.dv = dv; p.causal = causal != 0;
    p.error_flag = error_flag_dev;
    const fdx_status st = check_ragged("mha_packed", p, scratch_dev, fdx_mha_packed_scratch_bytes(tokens, n_seqs, heads, kv_heads, dk, dv));
    if (st != FDX_OK)
        return st;
    p.scale = (float)(1.0 / std::sqrt((double)dk));
    profile_begin();
    ragged_launch<kPackedF32>(p, scratch_dev);
    profile_end("mha_packed_f32", 0.0, 4.0 * tokens * ((double)heads + kv_heads) * (dk + dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}

extern "C" size_t fdx_mha_paged_scratch_bytes(int tokens, int max_new, int heads, const fdx_kv_pages* cache)
{
    (void)tokens; (void)max_new; (void)heads; (void)cache;
    return 0;
}

extern "C" fdx_status fdx_mha_paged_f32(const float* q, int64_t ldq, const int32_t* starts, int tokens, int max_new, int heads,
    const fdx_kv_pages* cache, float* out, int64_t ldo, void* scratch_dev, int* error_flag_dev)
{
    fdx_status st = check_kv_pages("mha_paged", cache);
    if (st != FDX_OK)
        return st;
    FDX_REQUIRE(max_new > 0, "mha_paged: bad shape");
    RaggedParams p {};
    p.q = q; p.ldq = ldq; p.out = out; p.ldo = ldo;
    p.k = cache->k; p.ldk = (int64_t)cache->kv_heads * cache->dk; p.v = cache->v; p.ldv = (int64_t)cache->kv_heads * cache->dv;
    p.starts = starts; p.n_seqs = cache->n_seqs; p.tokens = tokens;
    p.heads = heads; p.kv_heads = cache->kv_heads; p.group = heads / cache->kv_heads;
    p.dk = cache->dk; p.dv = cache->dv; p.causal = 1;
    p.table = cache->table; p.lens = cache->lens; p.table_width = cache->table_width; p.n_pages = cache->n_pages;
    p.page_size = cache->page_size; p.max_len = cache->max_len; p.max_new = max_new < tokens ? max_new : tokens;
    p.error_flag = error_flag_dev;
    st = check_ragged("mha_paged", p, scratch_dev, fdx_mha_paged_scratch_bytes(tokens, max_new, heads, cache));
    if (st != FDX_OK)
        return st;
    p.scale = (float)(1.0 / std::sqrt((double)p.dk));
    profile_begin();
    if (cache->type == FDX_KV_F32)
        ragged_launch<kPagedF32>(p, scratch_dev);
    else
        ragged_launch<kPagedBf16>(p, scratch_dev);
    profile_end("mha_paged_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
