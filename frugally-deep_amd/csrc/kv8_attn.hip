// Attention over paged caches in 8 bits, query heads in groups that share a key / value head.
#include <cfloat>

#include "kv8.hpp"

namespace fdx {

// A wave takes a row: a lane has a key's score, then depths lane and 64 + lane of the output.
template <int KIND>
__global__ __launch_bounds__(256) void paged8_kernel(RaggedParams p, const float* k_scale, const float* v_scale, Divisor block)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens) || p.lens[i] < 0 || p.lens[i] > p.max_len);
    const int row = (int)(item / p.heads), head = (int)(item - (int64_t)row * p.heads);
    if (row >= p.tokens)
        return;
    const int index = find_row(SearchWave(), p.starts, p.n_seqs, p.tokens, row);
    if (index < 0)
        return;
    const Sequence s = sequence_of<kPagedF32>(p, index, packed_span(p.starts, index, p.tokens));
    raise_flag(p, s.cut);
    const int token = row - s.span.first;
    if (token >= s.span.count)
        return;
    const int kv_head = quotient(head, p.by_group), last = visible_keys(p, s, token);
    const float* q = p.q + (int64_t)row * p.ldq + (int64_t)head * p.dk;
    const uint8_t* kb = static_cast<const uint8_t*>(p.k) + (int64_t)kv_head * p.dk;
    const uint8_t* vb = static_cast<const uint8_t*>(p.v) + (int64_t)kv_head * p.dv;
    float m = -INFINITY, l = 0.f, o[2] = { 0.f, 0.f };
    bool seen = false;
    for (int j0 = 0; j0 < last; j0 += 64) {
        const int at = j0 + lane < last ? key_row<kPagedF32>(p, s, j0 + lane) : -1;
        seen = seen || __any(at >= 0);
        raise_flag(p, j0 + lane < last && at < 0);
        float sc = -INFINITY, vs = 0.f;
        if (at >= 0) {
            const int64_t scale = (int64_t)quotient(at, block) * p.kv_heads + kv_head;
            float dot = 0.f;
            for (int d = 0; d < p.dk; ++d) {
                float x[4];
                from_codes<KIND>(kb[(int64_t)at * p.ldk + d], x);
                dot = fmaf(q[d], x[0], dot);
            }
            sc = dot * (p.scale * kLog2e) * k_scale[scale];
            vs = v_scale[scale];
        }
        const bool nan = __any(sc != sc);
        const float m_new = nan ? NAN : fmaxf(m, wave_all<true>(sc)), m_use = m_new == -INFINITY ? 0.f : m_new;
        const float corr = __builtin_amdgcn_exp2f(m - m_use), pr = at >= 0 ? __builtin_amdgcn_exp2f(sc - m_use) : 0.f;
        l = l * corr + wave_all<false>(pr);
        m = m_new;
        float part[2] = { 0.f, 0.f }; // of these keys: one chain over all of them would round a thousand times
        const float w = at >= 0 ? pr * vs : 0.f;
        for (int j = 0; j < 64; ++j) {
            const int r = __shfl(at, j, 64);
            const float wj = __shfl(w, j, 64);
            if (r < 0)
                continue;
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (64 * i + lane < p.dv) {
                    float x[4];
                    from_codes<KIND>(vb[(int64_t)r * p.ldv + 64 * i + lane], x);
                    part[i] = fmaf(wj, x[0], part[i]);
                }
        }
        o[0] = fmaf(o[0], corr, part[0]);
        o[1] = fmaf(o[1], corr, part[1]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (64 * i + lane < p.dv)
            p.out[(int64_t)row * p.ldo + (int64_t)head * p.dv + 64 * i + lane] = finish(o[i], l, seen);
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_mha_paged8_scratch_bytes(int tokens, int max_new, int heads, const fdx_kv_pages8* cache)
{
    return cache ? fdx_mha_paged_scratch_bytes(tokens, max_new, heads, &cache->pages) : 0;
}

extern "C" fdx_status fdx_mha_paged8_f32(const float* q, int64_t ldq, const int32_t* starts, int tokens, int max_new, int heads,
    const fdx_kv_pages8* cache, float* out, int64_t ldo, void* scratch_dev, int* error_flag_dev)
{
    fdx_status st = check_kv_pages8("mha_paged8", cache);
    if (st != FDX_OK)
        return st;
    RaggedParams p {};
    RaggedPlan plan;
    st = paged_params("mha_paged8", q, ldq, starts, tokens, max_new, heads, &cache->pages, out, ldo, scratch_dev, error_flag_dev, p, plan);
    if (st != FDX_OK)
        return st;
    const Divisor block = make_divisor(cache->block);
    const dim3 grid((unsigned)(((int64_t)tokens * heads + 3) / 4));
    profile_begin();
    if (cache->pages.type == FDX_KV_I8)
        hipLaunchKernelGGL(paged8_kernel<kI8>, grid, dim3(256), 0, stream(), p, cache->k_scale, cache->v_scale, block);
    else
        hipLaunchKernelGGL(paged8_kernel<kE4M3>, grid, dim3(256), 0, stream(), p, cache->k_scale, cache->v_scale, block);
    profile_end("mha_paged8_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
