// Attention over packed prompts and over paged caches (gfx950), query heads in groups that share a key / value head.
#include <cfloat>
#include <climits>

#include "f16_split.hpp"
#include "ragged_attn.hpp"

namespace fdx {

fdx_status check_kv_pages(const char* who, const fdx_kv_pages* c); // kv_append.hip

// a row by plain sums, into its place
template <int KIND>
__device__ __forceinline__ void store_plain_row(const RaggedParams& p, const Sequence& s, int token, int head, int kv_head, int range, int lane)
{
    const int visible = visible_keys(p, s, token);
    const bool in_parts = visible > p.split_keys;
    const int first = range * p.split_keys;
    if (in_parts ? first >= visible : range > 0)
        return;
    const int last = in_parts && visible - first > p.split_keys ? first + p.split_keys : visible;
    const int64_t row = s.span.first + token, id = row * p.heads + head;
    float m, l, o[2];
    bool seen, missing;
    plain_row<KIND>(p, s, p.q + row * p.ldq + (int64_t)head * p.dk, kv_head, first, last, m, l, o, seen, missing);
    raise_flag(p, missing);
    float* to = in_parts ? part_out(p, range, id) : p.out + row * p.ldo + (int64_t)head * p.dv;
    if (in_parts && lane == 0) {
        part_size(p, range, id)[0] = seen && m == -INFINITY ? -FLT_MAX : m;
        part_size(p, range, id)[1] = l;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (64 * i + lane < p.dv)
            to[64 * i + lane] = in_parts ? finish(o[i], l, false) : finish(o[i], l, seen);
}

// ---- many query rows: tiles on the fp16 matrix instructions ----
//
// A workgroup takes 128 rows of one key head of one sequence, rows counting through the query heads of the group first (row = token *
// group + head), so that short sequences fill a tile and a key is read once for all heads that share it; a wave takes 32 of them.
// Keys and values pass through LDS in tiles of 64, split in two fp16 planes on the way (f16_split.hpp).  Products are taken
// transposed, S^T = K Q^T: a query is a lane's column and keys are the accumulator's registers, so the softmax's running maximum and sum
// are one register a lane, and the probabilities lie as the second product O^T = V^T P^T takes them.
//  * LDS holds blocks of eight contraction indices: keys [plane][depth block][key][16 bytes], values [plane][key block][depth][16 bytes].
//    Depth block 4 g + l holds depths 32 g + 4 l .. + 3 and 32 g + 16 + 4 l .. + 3, the two 16-byte chunks that lane l of four fetches
//    of a key row; a key block the eight keys whose probabilities one lane half has in eight consecutive accumulator registers.
//  * A query row, a tile's keys and the values so far are each brought to fp16's range by a power of two; a tile whose values are larger than
//    any before lowers the sums' power (a test a tile, rare).
//  * The maximum that a row's exponentials refer to moves only when a score passes it by 2^4, so sums are rescaled a few times a row
//    instead of every tile; exponentials carry 2^10 to stay clear of fp16's small end, at most 2^14.
//  * Rows whose sums are not finite (infinite or NaN operands, whether the row sees them or not) are taken again by plain_row.
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <typename T, int W>
__device__ __forceinline__ void load_depths(const T* row, int d, int depth, bool wide, float (&x)[W])
{
    typedef T tv __attribute__((ext_vector_type(W)));
    if (wide) {
        if (d < depth) {
            const tv v = *reinterpret_cast<const tv*>(row + d);
#pragma unroll
            for (int e = 0; e < W; ++e)
                x[e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < W; ++e)
                x[e] = 0.f;
        }
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
            x[e] = d + e < depth ? (float)row[d + e] : 0.f;
    }
}

constexpr float kShift = 10.f; // exponentials are 2^kShift times the probability's numerator

template <int D, int KIND, bool WIDE>
__global__ __launch_bounds__(256, 2) void ragged_tile_kernel(RaggedParams p)
{
    typedef typename KvElement<KIND>::type T;
    constexpr int KB = D / 8, STEPS = D / 16, KL = D / 32, VD = D / 32, DB = D / 32;
    constexpr int KBLK = 64 * 16 + 32, VBLK = D * 16 + 32; // bytes of a block, offset against each other
    constexpr bool kPaged = KIND != kPackedF32;
    __shared__ __attribute__((aligned(16))) unsigned char ks[2 * KB * KBLK];
    __shared__ __attribute__((aligned(16))) unsigned char vs[2 * 8 * VBLK];
    __shared__ float largest[2][4];
    __shared__ int rows_of[2][64];
    __shared__ uint64_t absent[2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, half = lane >> 5;
    if (p.error_flag && blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = tid; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens));
    // key heads next to each other: consecutive workgroups go to the eight XCDs in turn, so that an XCD's cache holds few heads'
    // keys; later tiles of a sequence, which see more keys, first
    const int kv_head = blockIdx.x % p.kv_heads;
    const Tile tile = find_tile(p.starts, p.n_seqs, p.tokens, p.group, 128, gridDim.x / p.kv_heads - 1 - blockIdx.x / p.kv_heads);
    if (tile.seq < 0)
        return;
    const Sequence s = sequence_of<KIND>(p, tile.seq, tile.span);
    if (tid == 0)
        raise_flag(p, s.cut);
    const int count = s.span.count * p.group; // rows
    const int r_first = tile.index * 128;
    if (r_first >= count || s.span.count * p.group < p.tile_from)
        return;
    const int r = r_first + wave * 32 + c;
    const bool q_ok = r < count;
    const int token = (q_ok ? r : count - 1) / p.group, head = kv_head * p.group + (q_ok ? r : count - 1) - token * p.group;
    const int64_t q_row = s.span.first + token;
    const int visible = visible_keys(p, s, token);

    const int r_last = r_first + 128 < count ? r_first + 127 : count - 1;
    const int k_first = blockIdx.y * p.split_keys;
    int k_end = visible_keys(p, s, r_last / p.group); // of the workgroup's last row
    if (blockIdx.y > 0 && k_first >= k_end)
        return;
    if (k_end > k_first + p.split_keys)
        k_end = k_first + p.split_keys;
    const int tiles = k_end > k_first ? (k_end - k_first + 63) / 64 : 0;
    // what the wave's rows see: all of them the first `wave_all_see`, some the first `wave_any`
    const int w_first = r_first + wave * 32, w_last = w_first + 31 < count ? w_first + 31 : count - 1;
    const int wave_all_see = visible_keys(p, s, (w_first < count ? w_first : count - 1) / p.group), wave_any = visible_keys(p, s, w_last / p.group);

    // the query: depth block 2 u + half
    f16x8 qh[STEPS], ql[STEPS];
    float q_down;
    {
        float x[STEPS][8], top = 0.f;
        const float* from = p.q + q_row * p.ldq + (int64_t)head * p.dk;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int blk = 2 * u + half, d0 = 32 * (blk >> 2) + 4 * (blk & 3);
            float lo[4], hi[4];
            load_depths<float, 4>(from, d0, p.dk, WIDE, lo);
            load_depths<float, 4>(from, d0 + 16, p.dk, WIDE, hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[u][e] = lo[e];
                x[u][4 + e] = hi[e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                top = fmaxf(top, fabsf(x[u][e]));
        }
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const Pow2 sq = pow2_for(top);
        q_down = sq.down * (p.scale * kLog2e);
#pragma unroll
        for (int u = 0; u < STEPS; ++u)
            split2x8(x[u], sq.up, qh[u], ql[u]);
    }

    const T* kbase = static_cast<const T*>(p.k) + (int64_t)kv_head * p.dk;
    const T* vbase = static_cast<const T*>(p.v) + (int64_t)kv_head * p.dv;
    const int krow = tid >> 2, kl = tid & 3, vblk = tid >> 5, vd = (tid & 31) * VD;
    float kst[KL][8], vst[8][VD];
    // positions behind the range repeat its last one: masked, and as finite as it is
    auto place = [&](int j0, int key, int buf) -> int64_t {
        if constexpr (kPaged)
            return rows_of[buf][key];
        else
            return s.span.first + (j0 + key < k_end ? j0 + key : k_end - 1);
    };
    auto look_up = [&](int j0) { // lane of wave 0: the place of key j0 + lane
        return key_row<KIND>(p, s, j0 + lane < k_end ? j0 + lane : k_end - 1);
    };
    auto keep_place = [&](int row, int buf) {
        rows_of[buf][lane] = row < 0 ? 0 : row;
        const uint64_t none = __ballot(row < 0);
        if (lane == 0) {
            absent[buf] = none;
            raise_flag(p, none != 0);
        }
    };
    auto fetch = [&](int j0, int buf) {
        const T* kr = kbase + place(j0, krow, buf) * p.ldk;
#pragma unroll
        for (int g = 0; g < KL; ++g) {
            float lo[4], hi[4];
            load_depths<T, 4>(kr, 32 * g + 4 * kl, p.dk, WIDE, lo);
            load_depths<T, 4>(kr, 32 * g + 16 + 4 * kl, p.dk, WIDE, hi);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                kst[g][e] = lo[e];
                kst[g][4 + e] = hi[e];
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            load_depths<T, VD>(vbase + place(j0, 16 * (vblk >> 1) + 4 * (vblk & 1) + 8 * (j >> 2) + (j & 3), buf) * p.ldv, vd, p.dv, WIDE, vst[j]);
    };
    auto measure = [&] { // the largest finite key and value of the fetched tile
        float km = 0.f, vm = 0.f;
#pragma unroll
        for (int g = 0; g < KL; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                km = fmaxf(km, fabsf(kst[g][e]));
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int d = 0; d < VD; ++d)
                vm = fmaxf(vm, fabsf(vst[j][d]));
        km = wave_all<true>(km);
        vm = wave_all<true>(vm);
        if (__builtin_expect(km == INFINITY || vm == INFINITY, 0)) { // rows that do not see the infinity keep their sums
            km = vm = 0.f;
#pragma unroll
            for (int g = 0; g < KL; ++g)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    km = fmaxf(km, fabsf(kst[g][e]) < INFINITY ? fabsf(kst[g][e]) : 0.f);
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int d = 0; d < VD; ++d)
                    vm = fmaxf(vm, fabsf(vst[j][d]) < INFINITY ? fabsf(vst[j][d]) : 0.f);
            km = wave_all<true>(km);
            vm = wave_all<true>(vm);
        }
        if (lane == 0) {
            largest[0][wave] = km;
            largest[1][wave] = vm;
        }
    };
    auto mfma = [](f16x8 a, f16x8 b, const f32x16& acc) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0); };
    constexpr f32x16 kZero = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };

    f32x16 oacc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
        oacc[d] = kZero;
    float m_run = -INFINITY, l_run = 0.f, v_top = 0.f;
    Pow2 sv = pow2_for(0.f);
    int next_row = 0;

    if (tiles > 0) {
        if constexpr (kPaged) {
            if (wave == 0) {
                keep_place(look_up(k_first), 0);
                next_row = look_up(k_first + 64);
            }
            __syncthreads();
        }
        fetch(k_first, 0);
        measure();
    }
    for (int t = 0; t < tiles; ++t) {
        const int j0 = k_first + t * 64;
        __syncthreads(); // every wave is done with the previous tile
        const Pow2 sk = pow2_for(fmaxf(fmaxf(largest[0][0], largest[0][1]), fmaxf(largest[0][2], largest[0][3])));
        const float vm = fmaxf(fmaxf(largest[1][0], largest[1][1]), fmaxf(largest[1][2], largest[1][3]));
        if (vm > v_top) { // the same for the whole workgroup
            v_top = vm;
            const Pow2 now = pow2_for(vm);
            const float f = now.up * sv.down;
            sv = now;
            if (f != 1.f) {
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        oacc[d][e] *= f;
            }
        }
#pragma unroll
        for (int g = 0; g < KL; ++g) {
            f16x8 h, l;
            split2x8(kst[g], sk.up, h, l);
            *reinterpret_cast<f16x8*>(&ks[(4 * g + kl) * KBLK + krow * 16]) = h;
            *reinterpret_cast<f16x8*>(&ks[(KB + 4 * g + kl) * KBLK + krow * 16]) = l;
        }
#pragma unroll
        for (int d = 0; d < VD; ++d) {
            const float x[8] = { vst[0][d], vst[1][d], vst[2][d], vst[3][d], vst[4][d], vst[5][d], vst[6][d], vst[7][d] };
            f16x8 h, l;
            split2x8(x, sv.up, h, l);
            *reinterpret_cast<f16x8*>(&vs[vblk * VBLK + (vd + d) * 16]) = h;
            *reinterpret_cast<f16x8*>(&vs[(8 + vblk) * VBLK + (vd + d) * 16]) = l;
        }
        if constexpr (kPaged)
            if (wave == 0 && t + 1 < tiles)
                keep_place(next_row, (t + 1) & 1);
        __syncthreads();
        if (t + 1 < tiles) {
            fetch(j0 + 64, (t + 1) & 1); // in flight while this tile is worked on
            if (kPaged && wave == 0 && t + 2 < tiles)
                next_row = look_up(j0 + 128);
        }
        if (j0 < wave_any) { // some row of this wave sees some key of the tile
            // S^T: 64 keys x 32 rows
            f32x16 sacc[2];
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                sacc[kb] = kZero;
#pragma unroll
                for (int u = 0; u < STEPS; ++u) {
                    const f16x8 kh = *reinterpret_cast<const f16x8*>(&ks[(2 * u + half) * KBLK + (kb * 32 + c) * 16]);
                    const f16x8 kw = *reinterpret_cast<const f16x8*>(&ks[(KB + 2 * u + half) * KBLK + (kb * 32 + c) * 16]);
                    sacc[kb] = mfma(kw, qh[u], sacc[kb]);
                    sacc[kb] = mfma(kh, ql[u], sacc[kb]);
                    sacc[kb] = mfma(kh, qh[u], sacc[kb]);
                }
            }
            const int limit = (visible < k_end ? visible : k_end) - j0; // keys of the tile that this lane's row sees
            if (j0 + 64 > wave_all_see || j0 + 64 > k_end) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3) >= limit)
                            sacc[kb][e] = -INFINITY;
            }
            if constexpr (kPaged) {
                const uint64_t none = absent[t & 1];
                if (none != 0) {
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (none >> (kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3)) & 1)
                                sacc[kb][e] = -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    mx = fmaxf(mx, sacc[kb][e]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float to_log2 = fmaxf(q_down * sk.down, 1.17549435e-38f); // above zero: -infinity stays what it is
            mx *= to_log2;
            if (__any(mx > m_run + 4.f)) {
                const float m_new = fmaxf(m_run, mx);
                const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= corr;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        oacc[d][e] *= corr;
            }
            const float base = kShift - (m_run == -INFINITY ? 0.f : m_run); // a row that has seen no key yet adds zeros
            float rs = 0.f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sacc[kb][e] = __builtin_amdgcn_exp2f(fmaf(sacc[kb][e], to_log2, base));
                    rs += sacc[kb][e];
                }
            l_run += rs; // the other half of the tile's keys lies in lane + 32: they meet at the end
            // O^T += V^T P^T
#pragma unroll
            for (int u = 0; u < 4; ++u) { // keys of block 2 u + half: registers 8 (u % 2) .. + 7 of half tile u / 2
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = sacc[u >> 1][8 * (u & 1) + j];
                f16x8 ph, pl;
                split2x8(x, 1.f, ph, pl);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const f16x8 vh = *reinterpret_cast<const f16x8*>(&vs[(2 * u + half) * VBLK + (d * 32 + c) * 16]);
                    const f16x8 vl = *reinterpret_cast<const f16x8*>(&vs[(8 + 2 * u + half) * VBLK + (d * 32 + c) * 16]);
                    oacc[d] = mfma(vl, ph, oacc[d]);
                    oacc[d] = mfma(vh, pl, oacc[d]);
                    oacc[d] = mfma(vh, ph, oacc[d]);
                }
            }
        }
        if (t + 1 < tiles)
            measure();
    }

    l_run += __shfl_xor(l_run, 32, 64);
    float size = l_run;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            size += fabsf(oacc[d][e]);
    // a row's two lanes hold half of its depths each
    const uint64_t odd_lanes = __ballot(q_ok && !(size < INFINITY));
    uint32_t odd = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    const bool in_parts = visible > p.split_keys;
    const int64_t id = q_row * p.heads + head;
    if (q_ok && !(odd >> c & 1) && (in_parts ? k_first < visible : blockIdx.y == 0)) {
        const float f = l_run > 0.f ? sv.down / l_run : 0.f; // no key: zeros
        float* to = in_parts ? part_out(p, blockIdx.y, id) : p.out + q_row * p.ldo + (int64_t)head * p.dv;
        if (in_parts && half == 0) {
            float* at = part_size(p, blockIdx.y, id);
            at[0] = m_run - kShift;
            at[1] = l_run;
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int depth = 32 * d + 8 * g + 4 * half;
                const f32x4 o = { oacc[d][4 * g] * f, oacc[d][4 * g + 1] * f, oacc[d][4 * g + 2] * f, oacc[d][4 * g + 3] * f };
                if (WIDE) {
                    if (depth < p.dv)
                        *reinterpret_cast<f32x4*>(to + depth) = o;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (depth + e < p.dv)
                            to[depth + e] = o[e];
                }
            }
    }
    if (__builtin_expect(odd == 0, 1))
        return;
#pragma clang loop unroll(disable)
    while (odd) {
        const int r1 = r_first + wave * 32 + __builtin_ctz(odd);
        odd &= odd - 1;
        const int t1 = r1 / p.group, h1 = kv_head * p.group + r1 - t1 * p.group;
        store_plain_row<KIND>(p, s, t1, h1, kv_head, blockIdx.y, lane);
    }
}

// Rows that more than one range of keys was summed for: sum of 2^(m - M) l o over the ranges, divided by that of 2^(m - M) l.
template <int KIND>
__global__ __launch_bounds__(256) void ragged_join_kernel(RaggedParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t id = (int64_t)blockIdx.x * 4 + wave;
    const int row = (int)(id / p.heads), head = (int)(id % p.heads);
    if (row >= p.tokens)
        return;
    const int index = find_row(p.starts, p.n_seqs, p.tokens, row);
    if (index < 0)
        return;
    const Sequence s = sequence_of<KIND>(p, index, packed_span(p.starts, index, p.tokens));
    if (row - s.span.first >= s.span.count)
        return;
    const int visible = visible_keys(p, s, row - s.span.first);
    if (visible <= p.split_keys)
        return;
    const int parts = (visible + p.split_keys - 1) / p.split_keys;
    float top = -INFINITY;
    for (int i = 0; i < parts; ++i)
        top = fmaxf(top, part_size(p, i, id)[0]);
    const float m = top == -INFINITY ? 0.f : top;
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int i = 0; i < parts; ++i) {
        const float* at = part_size(p, i, id);
        const float w = at[1] * __builtin_amdgcn_exp2f(at[0] - m);
        const float* from = part_out(p, i, id);
        l += w;
        if (lane < p.dv)
            o0 = fmaf(w, from[lane], o0);
        if (64 + lane < p.dv)
            o1 = fmaf(w, from[64 + lane], o1);
    }
    float* to = p.out + (int64_t)row * p.ldo + (int64_t)head * p.dv;
    if (lane < p.dv)
        to[lane] = finish(o0, l, top != -INFINITY);
    if (64 + lane < p.dv)
        to[64 + lane] = finish(o1, l, top != -INFINITY);
}

template <int D, int KIND>
static void tile_launch(const RaggedParams& p, bool wide)
{
    const int64_t tiles = KIND == kPackedF32
        ? tile_numbers(p.tokens, p.n_seqs, p.group, 128)
        : tile_numbers(p.tokens, p.n_seqs, p.group, 128);
    const dim3 grid((unsigned)(tiles * p.kv_heads), (unsigned)p.splits);
    if (wide)
        hipLaunchKernelGGL((ragged_tile_kernel<D, KIND, true>), grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL((ragged_tile_kernel<D, KIND, false>), grid, dim3(256), 0, stream(), p);
}

// rows of every tensor start on vectors of four elements
static bool wide_rows(const RaggedParams& p, int size)
{
    const uintptr_t f = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out);
    const uintptr_t kv = reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v);
    return (f & 15) == 0 && (kv & (4 * size - 1)) == 0 && ((p.ldq | p.ldo | p.ldk | p.ldv | p.dk | p.dv) & 3) == 0;
}

template <int KIND>
static void ragged_launch(const RaggedParams& p)
{
    const bool wide = wide_rows(p, KIND == kPagedBf16 ? 2 : 4);
    if (p.dk <= 64 && p.dv <= 64)
        tile_launch<64, KIND>(p, wide);
    else
        tile_launch<128, KIND>(p, wide);
    if (p.splits > 1)
        hipLaunchKernelGGL(ragged_join_kernel<KIND>, dim3((unsigned)(((int64_t)p.tokens * p.heads + 3) / 4)), dim3(256), 0, stream(), p);
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
    p.splits = 1;
    p.split_keys = INT_MAX;
    ragged_launch<kPackedF32>(p);
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
    p.splits = 1;
    p.split_keys = INT_MAX;
    if (cache->type == FDX_KV_F32)
        ragged_launch<kPagedF32>(p);
    else
        ragged_launch<kPagedBf16>(p);
    profile_end("mha_paged_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
