// Attention over paged caches in 8 bits, query heads in groups that share a key / value head.
#include <cfloat>

#include "bf16_split.hpp"
#include "kv8.hpp"

namespace fdx {

// ---- few query rows: keys and values pass once, straight from memory to the matrix instructions ----
//
// A workgroup takes the rows that a sequence brings to one key head, over one range of its keys; its waves take 32 keys a turn.  Up to sixteen
// rows: every fourth turn is a wave's; up to thirty-two: two waves for either half of the rows take every second one.
//  * S^T = K Q^T: lane (c, g) of 16 x 4 loads 16 codes of keys c and 16 + c at depths 64 i + 16 g, and has the scores of keys 4 g .. 4 g + 3 and
//    16 + 4 g .. of row c.
//  * O^T = V^T P^T over the turn's 32 keys: lane (c, g) loads D / 16 codes of those eight keys at depth D / 16 c, so the probabilities it has are
//    the operand, and gets depths D / 16 (4 g + i) + e of row c.
//  * Codes are bf16 values exactly; queries, and probabilities times their values' scales, are the exact sums of three bf16 values.  A key's scale
//    meets its score, so neither takes a step of its own: lane (c, g) has looked up one scale, and a lane's number in its row of sixteen names it.
template <int D, bool WIDE>
struct Block8 {
    static constexpr int NK = D / 64, DL = D / 16;
    uint32_t k[2][NK][4]; // of keys c and 16 + c
    uint32_t v[8][DL / 4];
    float scale;          // of keys 4 g + (c & 3) + 4 (c & 4): of its keys for c < 8, of its values behind
    int row;              // place of key lane % 32
};

// 4 N codes of a row from depth d on, zeros behind `depth`
template <int N, bool WIDE>
__device__ __forceinline__ void load_codes(const uint8_t* row, int d, int depth, uint32_t* c)
{
    typedef uint32_t cv __attribute__((ext_vector_type(N)));
    if constexpr (WIDE) {
        cv x;
#pragma unroll
        for (int e = 0; e < N; ++e)
            x[e] = 0;
        if (d < depth)
            x = *reinterpret_cast<const cv*>(row + d);
#pragma unroll
        for (int e = 0; e < N; ++e)
            c[e] = x[e];
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            c[e] = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (d + 4 * e + i < depth)
                    c[e] |= (uint32_t)row[d + 4 * e + i] << (8 * i);
        }
    }
}
template <>
__device__ __forceinline__ void load_codes<1, true>(const uint8_t* row, int d, int depth, uint32_t* c)
{
    c[0] = d < depth ? *reinterpret_cast<const uint32_t*>(row + d) : 0;
}

template <int D, int KIND, bool WIDE>
__global__ __launch_bounds__(256, WIDE ? 2 : 1) void paged8_few_kernel(RaggedParams p, Scales8 scales)
{
    typedef Block8<D, WIDE> Block;
    constexpr int NK = Block::NK, DL = Block::DL;
    __shared__ float meet[4 * 16 * (D + 4)], meet_m[4][16], meet_l[4][16];
    auto meet_o = [&](int w, int row) { return meet + (w * 16 + row) * (D + 4); };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int seq = blockIdx.x / p.kv_heads, kv_head = blockIdx.x % p.kv_heads;
    if (p.error_flag && blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = tid; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens));
    const Sequence s = sequence_of<kPagedF32>(p, seq, packed_span(p.starts, seq, p.tokens));
    if (tid == 0)
        raise_flag(p, s.cut);
    const int count = s.span.count * p.group;
    if (count == 0 || !s.few)
        return;
    const bool halves = count > 16;
    const int step = halves ? 2 : 4, slot = halves ? wave & 1 : wave, r_first = halves ? (wave >> 1) * 16 : 0; // of this wave
    int k_end = visible_keys(p, s, s.span.count - 1);
    const int64_t k_from = (int64_t)blockIdx.y * s.range;
    if (blockIdx.y > 0 && k_from >= k_end)
        return;
    const int k_first = (int)k_from;
    if (k_end - k_first > s.range)
        k_end = k_first + s.range;
    const int blocks = k_end > k_first ? (k_end - k_first + 31) / 32 : 0;

    const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + (int64_t)kv_head * p.dk;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + (int64_t)kv_head * p.dv;
    const float* scale_base = (c < 8 ? scales.k : scales.v) + kv_head;
    const int scale_key = 4 * g + (c & 3) + 4 * (c & 4);
    auto look_up = [&](int blk) { // the place of key lane % 32 of a block; positions behind the range repeat its last one
        const int at = k_first + blk * 32 + (lane & 31);
        return key_row<kPagedF32>(p, s, at < k_end ? at : k_end - 1);
    };
    auto fetch = [&](Block& b, int row) {
        b.row = row;
        row = row < 0 ? 0 : row;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const uint8_t* kr = kbase + (int64_t)__shfl(row, 16 * z + c, 64) * p.ldk;
#pragma unroll
            for (int i = 0; i < NK; ++i)
                load_codes<4, WIDE>(kr, 64 * i + 16 * g, p.dk, b.k[z][i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            load_codes<DL / 4, WIDE>(vbase + (int64_t)__shfl(row, 16 * (i >> 2) + 4 * g + (i & 3), 64) * p.ldv, DL * c, p.dv, b.v[i]);
        b.scale = scale_base[(int64_t)quotient(__shfl(row, scale_key, 64), scales.block) * p.kv_heads];
    };
    Block a, b;
    int row_b = 0;
    if (slot < blocks) {
        const int row_a = look_up(slot);
        row_b = look_up(slot + step);
        fetch(a, row_a);
    }

    // the query: step (i, h) has depths 64 i + 16 g + 8 h ..
    bf16x8 q[2 * NK][3];
    const bool q_ok = r_first + c < count;
    const int q_token = quotient(q_ok ? r_first + c : 0, p.by_group);
    const int visible = q_ok ? visible_keys(p, s, q_token) : 0;
    {
        const float* from = p.q + (int64_t)(s.span.first + q_token) * p.ldq
            + (int64_t)(kv_head * p.group + (q_ok ? r_first + c : 0) - q_token * p.group) * p.dk;
#pragma unroll
        for (int u = 0; u < 2 * NK; ++u) {
            const int d = 64 * (u >> 1) + 16 * g + 8 * (u & 1);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                f32x4 y = { 0.f, 0.f, 0.f, 0.f };
                if (WIDE) {
                    if (d + e < p.dk)
                        y = *reinterpret_cast<const f32x4*>(from + d + e);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (d + e + i < p.dk)
                            y[i] = from[d + e + i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    x[e + i] = y[i] * (p.scale * kLog2e);
            }
            uint32_t w[3][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                split3(x[2 * i], x[2 * i + 1], w[0][i], w[1][i], w[2][i]);
#pragma unroll
            for (int z = 0; z < 3; ++z)
                q[u][z] = __builtin_bit_cast(bf16x8, (u32x4 { w[z][0], w[z][1], w[z][2], w[z][3] }));
        }
    }
    float m_run = -INFINITY, l_run = 0.f;
    f32x4 oacc[DL];
#pragma unroll
    for (int e = 0; e < DL; ++e)
        oacc[e] = f32x4 { 0.f, 0.f, 0.f, 0.f };
    // keys that the first row sees are seen by all
    const int first_sees = visible_keys(p, s, quotient(r_first, p.by_group)), all_see = first_sees < k_end ? first_sees : k_end;
    bool missing = false, seen = false;
    auto mfma = [](bf16x8 x, bf16x8 y, const f32x4& acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, y, acc, 0, 0, 0); };
    auto work = [&](Block& x, int blk) {
        f32x4 acc[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            acc[z] = f32x4 { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int u = 0; u < 2 * NK; ++u) {
                u32x4 w;
                uint32_t lo, hi;
                bf16_of_codes<KIND>(x.k[z][u >> 1][2 * (u & 1)], lo, hi);
                w[0] = lo;
                w[1] = hi;
                bf16_of_codes<KIND>(x.k[z][u >> 1][2 * (u & 1) + 1], lo, hi);
                w[2] = lo;
                w[3] = hi;
#pragma unroll
                for (int n = 2; n >= 0; --n) // small ones first
                    acc[z] = mfma(__builtin_bit_cast(bf16x8, w), q[u][n], acc[z]);
            }
        }
        float sc[8], vs[8]; // keys 4 g + i, then 16 + 4 g + i
        sc[0] = acc[0][0] * dpp_move<0x150>(x.scale); // row_newbcast: lane n of a row of sixteen, for all of them
        sc[1] = acc[0][1] * dpp_move<0x151>(x.scale);
        sc[2] = acc[0][2] * dpp_move<0x152>(x.scale);
        sc[3] = acc[0][3] * dpp_move<0x153>(x.scale);
        sc[4] = acc[1][0] * dpp_move<0x154>(x.scale);
        sc[5] = acc[1][1] * dpp_move<0x155>(x.scale);
        sc[6] = acc[1][2] * dpp_move<0x156>(x.scale);
        sc[7] = acc[1][3] * dpp_move<0x157>(x.scale);
        vs[0] = dpp_move<0x158>(x.scale);
        vs[1] = dpp_move<0x159>(x.scale);
        vs[2] = dpp_move<0x15A>(x.scale);
        vs[3] = dpp_move<0x15B>(x.scale);
        vs[4] = dpp_move<0x15C>(x.scale);
        vs[5] = dpp_move<0x15D>(x.scale);
        vs[6] = dpp_move<0x15E>(x.scale);
        vs[7] = dpp_move<0x15F>(x.scale);
        const int at = k_first + blk * 32;
        const bool absent = __any(x.row < 0);
        if (at + 32 > all_see || absent) {
            missing = missing || absent;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = 16 * (i >> 2) + 4 * g + (i & 3);
                const bool there = __shfl(x.row, key, 64) >= 0;
                const bool sees = there && at + key < (visible < k_end ? visible : k_end);
                sc[i] = sees ? sc[i] : -INFINITY;
                vs[i] = sees ? vs[i] : 0.f; // a scale of NaN is for the rows that see it
                seen = seen || sees;
#pragma unroll
                for (int e = 0; e < DL / 4; ++e)
                    x.v[i][e] = there ? x.v[i][e] : 0;
            }
        } else {
            seen = true;
        }
        float mx = fmaxf(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])), fmaxf(fmaxf(sc[4], sc[5]), fmaxf(sc[6], sc[7])));
        if (__any(mx > m_run + 8.f)) { // the maximum moves when a score passes it by 2^8
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float m_new = fmaxf(m_run, mx);
            const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= corr;
#pragma unroll
            for (int e = 0; e < DL; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    oacc[e][i] *= corr;
        }
        const float base = m_run == -INFINITY ? 0.f : m_run;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sc[i] = __builtin_amdgcn_exp2f(sc[i] - base);
            sum += sc[i];
            sc[i] *= vs[i];
        }
        l_run += sum;
        uint32_t w[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            split3(sc[2 * i], sc[2 * i + 1], w[0][i], w[1][i], w[2][i]);
        bf16x8 pr[3];
#pragma unroll
        for (int z = 0; z < 3; ++z)
            pr[z] = __builtin_bit_cast(bf16x8, (u32x4 { w[z][0], w[z][1], w[z][2], w[z][3] }));
#pragma unroll
        for (int e = 0; e < DL; e += 4) {
            uint32_t t[2][4];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const uint32_t r[4] = { x.v[4 * z][e / 4], x.v[4 * z + 1][e / 4], x.v[4 * z + 2][e / 4], x.v[4 * z + 3][e / 4] };
                transpose_codes(r, t[z]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u32x4 v;
                uint32_t lo, hi;
                bf16_of_codes<KIND>(t[0][i], lo, hi);
                v[0] = lo;
                v[1] = hi;
                bf16_of_codes<KIND>(t[1][i], lo, hi);
                v[2] = lo;
                v[3] = hi;
#pragma unroll
                for (int z = 2; z >= 0; --z)
                    oacc[e + i] = mfma(__builtin_bit_cast(bf16x8, v), pr[z], oacc[e + i]);
            }
        }
    };
    for (int blk = slot; blk < blocks; blk += 2 * step) {
        const bool more = blk + step < blocks;
        int row_a = 0;
        if (more) {
            fetch(b, row_b);
            row_a = look_up(blk + 2 * step);
        }
        work(a, blk);
        if (!more)
            break;
        if (blk + 2 * step < blocks) {
            fetch(a, row_a);
            row_b = look_up(blk + 3 * step);
        }
        work(b, blk + step);
    }
    raise_flag(p, missing);

    // the waves' sums meet: 16 threads a row, DL depths each
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);
    const uint64_t seen_by = __ballot(seen); // by lanes c, 16 + c, 32 + c or 48 + c
    const bool some = ((seen_by | seen_by >> 16 | seen_by >> 32 | seen_by >> 48) >> c & 1) != 0;
    if (g == 0) {
        meet_m[wave][c] = some && m_run == -INFINITY ? -FLT_MAX : m_run;
        meet_l[wave][c] = l_run;
    }
#pragma unroll
    for (int e = 0; e < DL; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            meet_o(wave, c)[DL * (4 * g + i) + e] = oacc[e][i];
    __syncthreads();
    const int row_at = tid >> 4, d0 = (tid & 15) * DL;
    for (int half = 0; half <= (halves ? 1 : 0); ++half) {
        const int w_first = 2 * half, w_last = halves ? w_first + 1 : 3; // the waves that have these rows
        float top = -INFINITY;
        for (int w = w_first; w <= w_last; ++w)
            top = fmaxf(top, meet_m[w][row_at]);
        const float m = top == -INFINITY ? 0.f : top;
        float l = 0.f, o[DL];
#pragma unroll
        for (int e = 0; e < DL; ++e)
            o[e] = 0.f;
        for (int w = w_first; w <= w_last; ++w) {
            const float f = __builtin_amdgcn_exp2f(meet_m[w][row_at] - m);
            l += f * meet_l[w][row_at];
#pragma unroll
            for (int e = 0; e < DL; ++e)
                o[e] += f * meet_o(w, row_at)[d0 + e];
        }
        const int r = 16 * half + row_at;
        if (r >= count)
            continue;
        const int token = quotient(r, p.by_group), head = kv_head * p.group + r - token * p.group;
        const int sees = visible_keys(p, s, token);
        const bool in_parts = sees > s.range;
        if (in_parts ? k_first >= sees : blockIdx.y > 0)
            continue;
        float* to = p.out + (int64_t)(s.span.first + token) * p.ldo + (int64_t)head * p.dv;
        if (in_parts) {
            const int64_t id = part_row(p, s, token, head);
            to = p.few.out(blockIdx.y, id, p.dv);
            float* size_at = p.few.size(blockIdx.y, id, p.dv);
            if ((tid & 15) == 0) {
                size_at[0] = top;
                size_at[1] = l;
            }
        }
#pragma unroll
        for (int e = 0; e < DL; ++e)
            o[e] = finish(o[e], l, top != -INFINITY && !in_parts);
#pragma unroll
        for (int e = 0; e < DL; e += 4) {
            if (WIDE) {
                if (d0 + e < p.dv)
                    *reinterpret_cast<f32x4*>(to + d0 + e) = f32x4 { o[e], o[e + 1], o[e + 2], o[e + 3] };
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (d0 + e + i < p.dv)
                        to[d0 + e + i] = o[e + i];
            }
        }
    }
}

// A wave takes a row: a lane has a key's score, then depths lane and 64 + lane of the output.
template <int KIND>
__global__ __launch_bounds__(256) void paged8_kernel(RaggedParams p, Scales8 scales)
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
    if (token >= s.span.count || s.few)
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
            const int64_t scale = (int64_t)quotient(at, scales.block) * p.kv_heads + kv_head;
            float dot = 0.f;
            for (int d = 0; d < p.dk; ++d) {
                float x[4];
                from_codes<KIND>(kb[(int64_t)at * p.ldk + d], x);
                dot = fmaf(q[d], x[0], dot);
            }
            sc = dot * (p.scale * kLog2e) * scales.k[scale];
            vs = scales.v[scale];
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

template <int D, int KIND>
static void paged8_launch(const RaggedParams& p, const RaggedPlan& plan, const Scales8& scales)
{
    // rows of codes are whole 16-byte vectors (values: of a lane's codes), those of q and out whole float4
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.k)
        | reinterpret_cast<uintptr_t>(p.v);
    const bool wide = (all & 15) == 0 && ((p.ldq | p.ldo) & 3) == 0 && p.dk % 16 == 0 && p.dv % (D / 16) == 0;
    const dim3 few((unsigned)(p.n_seqs * p.kv_heads), (unsigned)plan.few_ranges);
    if (plan.few_ranges > 0) {
        if (wide)
            hipLaunchKernelGGL((paged8_few_kernel<D, KIND, true>), few, dim3(256), 0, stream(), p, scales);
        else
            hipLaunchKernelGGL((paged8_few_kernel<D, KIND, false>), few, dim3(256), 0, stream(), p, scales);
    }
    if (plan.tiles > 0)
        hipLaunchKernelGGL(paged8_kernel<KIND>, dim3((unsigned)(((int64_t)p.tokens * p.heads + 3) / 4)), dim3(256), 0, stream(), p, scales);
    if (plan.few_ranges > 1 || plan.tile_ranges > 1)
        ragged_join_launch(p);
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
    p.tile.keys = 0x7fffffff;
    plan.tile_ranges = 1;
    const Scales8 scales { cache->k_scale, cache->v_scale, make_divisor(cache->block) };
    const bool small = p.dk <= 64 && p.dv <= 64;
    profile_begin();
    if (cache->pages.type == FDX_KV_I8)
        small ? paged8_launch<64, kI8>(p, plan, scales) : paged8_launch<128, kI8>(p, plan, scales);
    else
        small ? paged8_launch<64, kE4M3>(p, plan, scales) : paged8_launch<128, kE4M3>(p, plan, scales);
    profile_end("mha_paged8_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
