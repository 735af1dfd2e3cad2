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
// Keys and values pass through LDS in tiles of 4096 / D keys, split in two fp16 planes on the way (f16_split.hpp).  Products are taken
// transposed, S^T = K Q^T: a query is a lane's column and keys are the accumulator's registers, so the softmax's running maximum and sum
// are one register a lane, and the probabilities lie as the second product O^T = V^T P^T takes them.
//  * LDS holds two tiles: while one is multiplied the next one is split and written beside the first product's matrix instructions and the
//    one behind it is on its way to registers, one barrier a tile.  (One tile in LDS and two barriers: the vector units' and the matrix units' times
//    added up instead of passing side by side.)
//  * LDS holds blocks of eight contraction indices: keys [plane][depth block][key][16 bytes], values [plane][key block][depth][16 bytes].
//    N = D / 16 threads fetch a key: depth block N g + l holds the 16-byte chunks 2 N g + l and 2 N g + N + l of the row, which lane l of the N
//    has; a key block the eight keys whose probabilities one lane half has in eight consecutive accumulator registers.
//  * A query row, a tile's keys and the values so far are each brought to fp16's range by a power of two; a tile whose values are larger than
//    any before lowers the sums' power (a test a tile, rare).
//  * The maximum that a row's exponentials refer to moves only when a score passes it by 2^4, so sums are rescaled a few times a row
//    instead of every tile; exponentials carry 2^10 to stay clear of fp16's small end, at most 2^14.
//  * Rows whose sums are not finite (infinite or NaN operands, whether the row sees them or not) are taken again by plain_row.
typedef float f32x16 __attribute__((ext_vector_type(16)));

// W elements of a row from depth d on, zeros behind `depth`; EXACT: all are there and lie on vectors
template <typename T, int W, bool EXACT>
__device__ __forceinline__ void load_depths(const T* row, int d, int depth, int wide, float* x)
{
    typedef T tv __attribute__((ext_vector_type(W)));
    if (EXACT || (wide && d < depth)) {
        const tv v = *reinterpret_cast<const tv*>(row + d);
#pragma unroll
        for (int e = 0; e < W; ++e)
            x[e] = (float)v[e];
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
            x[e] = d + e < depth ? (float)row[d + e] : 0.f;
    }
}

constexpr float kShift = 10.f; // exponentials are 2^kShift times the probability's numerator

template <int D, int KIND, bool EXACT>
__global__ __launch_bounds__(256, 2) void ragged_tile_kernel(RaggedParams p)
{
    typedef typename KvElement<KIND>::type T;
    constexpr int KT = 4096 / D, HALVES = KT / 32, N = D / 16; // keys of a tile, in accumulators of 32; threads that fetch a key
    constexpr int KB = D / 8, VB = KT / 8, STEPS = D / 16, DB = D / 32;
    constexpr int KBLK = KT * 16 + 32, VBLK = D * 16 + 32; // bytes of a block, offset against each other
    constexpr bool kPaged = KIND != kPackedF32;
    __shared__ __attribute__((aligned(16))) unsigned char ks0[2 * KB * KBLK], ks1[2 * KB * KBLK];
    __shared__ __attribute__((aligned(16))) unsigned char vs0[2 * VB * VBLK], vs1[2 * VB * VBLK];
    __shared__ float largest[2][2][4];
    __shared__ int rows_of[4][KT];
    __shared__ uint64_t absent[4];
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
    if (r_first >= count || count <= p.few_rows)
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
    if (k_end - k_first > p.split_keys)
        k_end = k_first + p.split_keys;
    const int tiles = k_end > k_first ? (k_end - k_first + KT - 1) / KT : 0;
    // what the wave's rows see: all of them the first `wave_all_see`, some the first `wave_any`
    const int w_first = r_first + wave * 32, w_last = w_first + 31 < count ? w_first + 31 : count - 1;
    const int wave_all_see = visible_keys(p, s, (w_first < count ? w_first : count - 1) / p.group);
    const int wave_any = visible_keys(p, s, w_last / p.group);

    // the query: depth block 2 u + half
    f16x8 qh[STEPS], ql[STEPS];
    float q_down;
    {
        float x[STEPS][8], top = 0.f;
        const float* from = p.q + q_row * p.ldq + (int64_t)head * p.dk;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int blk = 2 * u + half, d0 = 8 * N * (blk / N) + 4 * (blk % N);
            load_depths<float, 4, EXACT>(from, d0, p.dk, p.wide, x[u]);
            load_depths<float, 4, EXACT>(from, d0 + 4 * N, p.dk, p.wide, x[u] + 4);
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
    const int krow = tid / N, kl = tid % N, vblk = tid / (D / 2), vd = tid % (D / 2) * 2;
    float kst[2][8], vst[8][2];
    // positions behind the range repeat its last one: masked, and as finite as it is
    auto place = [&](int t, int key) -> int64_t {
        if constexpr (kPaged) {
            return rows_of[t & 3][key];
        } else {
            const int at = k_first + t * KT + key;
            return s.span.first + (at < k_end ? at : k_end - 1);
        }
    };
    auto look_up = [&](int t) { // lane of wave 0: the place of a key of tile t
        const int at = k_first + t * KT + (lane & (KT - 1));
        return key_row<KIND>(p, s, at < k_end ? at : k_end - 1);
    };
    auto keep_place = [&](int row, int t) {
        if (lane < KT)
            rows_of[t & 3][lane] = row < 0 ? 0 : row;
        const uint64_t none = __ballot(row < 0);
        if (lane == 0) {
            absent[t & 3] = none;
            raise_flag(p, none != 0);
        }
    };
    const uint32_t ld_k = (uint32_t)p.ldk, ld_v = (uint32_t)p.ldv;
    const int vkey = 16 * (vblk >> 1) + 4 * (vblk & 1); // the first of the eight keys, the others 1, 2, 3, 8, 9, 10, 11 behind it
    auto fetch = [&](int t) {
        if (EXACT && !kPaged && k_first + (t + 1) * KT <= k_end) { // a whole tile: one base, offsets that stay
            const int64_t row = s.span.first + k_first + t * KT;
            const T *kr = kbase + row * p.ldk, *vr = vbase + row * p.ldv;
            const uint32_t ko = krow * ld_k + 4 * kl, vo = vkey * ld_v + vd;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                load_depths<T, 4, EXACT>(kr + (ko + 8 * N * g), 0, 0, 1, kst[g]);
                load_depths<T, 4, EXACT>(kr + (ko + 8 * N * g + 4 * N), 0, 0, 1, kst[g] + 4);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
                load_depths<T, 2, EXACT>(vr + (vo + (8 * (j >> 2) + (j & 3)) * ld_v), 0, 0, 1, vst[j]);
            return;
        }
        const T* kr = kbase + place(t, krow) * p.ldk;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            load_depths<T, 4, EXACT>(kr, 8 * N * g + 4 * kl, p.dk, p.wide, kst[g]);
            load_depths<T, 4, EXACT>(kr, 8 * N * g + 4 * N + 4 * kl, p.dk, p.wide, kst[g] + 4);
        }
        if (EXACT && kPaged && p.page_size % 16 == 0) { // the eight keys lie in one page
            const T* vr = vbase + place(t, vkey) * p.ldv + vd;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                load_depths<T, 2, EXACT>(vr + (8 * (j >> 2) + (j & 3)) * ld_v, 0, 0, 1, vst[j]);
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
            load_depths<T, 2, EXACT>(vbase + place(t, vkey + 8 * (j >> 2) + (j & 3)) * p.ldv, vd, p.dv, p.wide, vst[j]);
    };
    auto measure = [&](int t) { // the largest finite key and value of the fetched tile
        float km = 0.f, vm = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            km = max3_abs(km, kst[0][e], kst[1][e]);
            vm = max3_abs(vm, vst[e][0], vst[e][1]);
        }
        km = wave_all<true>(km);
        vm = wave_all<true>(vm);
        if (__builtin_expect(km == INFINITY || vm == INFINITY, 0)) { // rows that do not see the infinity keep their sums
            km = vm = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    km = fmaxf(km, fabsf(kst[g][e]) < INFINITY ? fabsf(kst[g][e]) : 0.f);
                    vm = fmaxf(vm, fabsf(vst[e][g]) < INFINITY ? fabsf(vst[e][g]) : 0.f);
                }
            km = wave_all<true>(km);
            vm = wave_all<true>(vm);
        }
        if (lane == 0) {
            largest[t & 1][0][wave] = km;
            largest[t & 1][1][wave] = vm;
        }
    };
    auto four = [](const float* v) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); };
    auto mfma = [](f16x8 a, f16x8 b, const f32x16& acc) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0); };
    constexpr f32x16 kZero = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };

    f32x16 oacc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
        oacc[d] = kZero;
    float m_run = -INFINITY, l_run = 0.f, v_top = 0.f;
    Pow2 sk = pow2_for(0.f), sv = sk, sk_next = sk, sv_next = sk; // of the tile at work (sv: of the sums) and of the one behind it
    int next_row = 0;
    auto scale_next = [&](int t) {
        sk_next = pow2_for(four(largest[t & 1][0]));
        v_top = fmaxf(v_top, four(largest[t & 1][1]));
        sv_next = pow2_for(v_top);
    };
    auto stage = [&](unsigned char* ks, unsigned char* vs) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            f16x8 h, l;
            split2x8(kst[g], sk_next.up, h, l);
            *reinterpret_cast<f16x8*>(&ks[(N * g + kl) * KBLK + krow * 16]) = h;
            *reinterpret_cast<f16x8*>(&ks[(KB + N * g + kl) * KBLK + krow * 16]) = l;
        }
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const float x[8] = { vst[0][d], vst[1][d], vst[2][d], vst[3][d], vst[4][d], vst[5][d], vst[6][d], vst[7][d] };
            f16x8 h, l;
            split2x8(x, sv_next.up, h, l);
            *reinterpret_cast<f16x8*>(&vs[vblk * VBLK + (vd + d) * 16]) = h;
            *reinterpret_cast<f16x8*>(&vs[(VB + vblk) * VBLK + (vd + d) * 16]) = l;
        }
    };
    auto turn = [&](int t, const unsigned char* ks, const unsigned char* vs, unsigned char* ks_next, unsigned char* vs_next) {
        const int j0 = k_first + t * KT;
        const bool work = j0 < wave_any; // some row of this wave sees some key of the tile
        const float f = sv_next.up * sv.down;
        sk = sk_next;
        if (work)
            sv = sv_next; // a wave that is through keeps its sums as they are
        if (t + 1 < tiles)
            scale_next(t + 1);
        // S^T: KT keys x 32 rows, for a wave that sees none of them too; beside it tile t + 1 goes to LDS (the last time what the
        // registers still hold, for nobody)
        f32x16 sacc[HALVES];
#pragma unroll
        for (int kb = 0; kb < HALVES; ++kb) {
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
        stage(ks_next, vs_next);
        if constexpr (kPaged)
            if (wave == 0 && t + 3 < tiles)
                keep_place(next_row, t + 3);
        if (t + 2 < tiles) {
            fetch(t + 2);
            if (kPaged && wave == 0 && t + 4 < tiles)
                next_row = look_up(t + 4);
        }
        if (work) {
            const int limit = (visible < k_end ? visible : k_end) - j0; // keys of the tile that this lane's row sees
            if (j0 + KT > wave_all_see || j0 + KT > k_end) {
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3) >= limit)
                            sacc[kb][e] = -INFINITY;
            }
            if constexpr (kPaged) {
                const uint64_t none = absent[t & 3];
                if (none != 0) {
#pragma unroll
                    for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            if (none >> (kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3)) & 1)
                                sacc[kb][e] = -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                for (int e = 0; e < 16; e += 2)
                    mx = max3(mx, sacc[kb][e], sacc[kb][e + 1]);
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float to_log2 = fmaxf(q_down * sk.down, 1.17549435e-38f); // above zero: -infinity stays what it is
            mx *= to_log2;
            if (__any(mx > m_run + 4.f) || f != 1.f) {
                const float m_new = mx > m_run + 4.f ? mx : m_run;
                const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= corr;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        oacc[d][e] *= corr * f;
            }
            const float base = kShift - (m_run == -INFINITY ? 0.f : m_run); // a row that has seen no key yet adds zeros
            float rs = 0.f;
#pragma unroll
            for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sacc[kb][e] = __builtin_amdgcn_exp2f(fmaf(sacc[kb][e], to_log2, base));
                    rs += sacc[kb][e];
                }
            l_run += rs; // the other half of the tile's keys lies in lane + 32: they meet at the end
            // O^T += V^T P^T
#pragma unroll
            for (int u = 0; u < KT / 16; ++u) { // keys of block 2 u + half: registers 8 (u % 2) .. + 7 of accumulator u / 2
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = sacc[u >> 1][8 * (u & 1) + j];
                f16x8 ph, pl;
                split2x8(x, ph, pl);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const f16x8 vh = *reinterpret_cast<const f16x8*>(&vs[(2 * u + half) * VBLK + (d * 32 + c) * 16]);
                    const f16x8 vl = *reinterpret_cast<const f16x8*>(&vs[(VB + 2 * u + half) * VBLK + (d * 32 + c) * 16]);
                    oacc[d] = mfma(vl, ph, oacc[d]);
                    oacc[d] = mfma(vh, pl, oacc[d]);
                    oacc[d] = mfma(vh, ph, oacc[d]);
                }
            }
        }
        if (t + 2 < tiles)
            measure(t + 2);
        __syncthreads();
    };

    if (tiles > 0) {
        if constexpr (kPaged) {
            if (wave == 0) {
                const int row0 = look_up(0), row1 = look_up(1), row2 = look_up(2);
                next_row = look_up(3);
                keep_place(row0, 0);
                keep_place(row1, 1);
                keep_place(row2, 2);
            }
            __syncthreads();
        }
        fetch(0);
        measure(0);
        __syncthreads();
        scale_next(0);
        stage(ks0, vs0);
        if (tiles > 1) {
            fetch(1);
            measure(1);
        }
        __syncthreads();
        sv = sv_next;
    }
    for (int t = 0; t < tiles; t += 2) {
        turn(t, ks0, vs0, ks1, vs1);
        if (t + 1 < tiles)
            turn(t + 1, ks1, vs1, ks0, vs0);
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
                if (EXACT || (p.wide && depth < p.dv)) {
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

// ---- few query rows: keys and values pass once, straight from memory to the fp32 matrix instructions ----
//
// A workgroup takes all rows (up to 16 R) that a sequence brings to one key head, over one range of its keys; its four waves take every
// fourth block of 16 keys, each with sums of its own, and meet at the end.  Bound by memory: a lane's loads are the operands of
// the 16x16x4 fp32 products, nothing is staged, and a block's loads are on their way while the block before is worked on.
//  * S^T = K Q^T: lane (c, g) of 16 x 4 loads chunks of key c, chunk i at depth 4 W i + W g (W elements are 16 bytes), and has scores of keys
//    4 g .. 4 g + 3 of row c.
//  * O^T = V^T P^T: lane (c, g) loads depths V c .. V c + V - 1 of keys 4 g .. + 3, so the probabilities it has are the operand, and gets
//    depths V (4 g + i) + e of row c.  The products are exact in fp32; what they cost, 32 cycles per 16 keys, 16 rows and 4 depths, is less
//    than the memory's share of a CU needs for the keys.
template <typename T, int W, bool WIDE>
__device__ __forceinline__ auto load_chunk(const T* row, int d, int depth)
{
    typedef T tv __attribute__((ext_vector_type(W)));
    tv v;
#pragma unroll
    for (int e = 0; e < W; ++e)
        v[e] = (T)0.f;
    if (WIDE) {
        if (d < depth)
            v = *reinterpret_cast<const tv*>(row + d);
    } else {
#pragma unroll
        for (int e = 0; e < W; ++e)
            if (d + e < depth)
                v[e] = row[d + e];
    }
    return v;
}

template <int D, int KIND, int R, bool WIDE>
__global__ __launch_bounds__(256) void ragged_few_kernel(RaggedParams p)
{
    typedef typename KvElement<KIND>::type T;
    constexpr int W = 16 / (int)sizeof(T), NK = D / (4 * W); // elements of a key chunk, chunks of a lane
    constexpr int DL = D / 16, VW = DL < W ? DL : W, NV = DL / VW; // depths of a lane, in NV loads of VW
    typedef T kvec __attribute__((ext_vector_type(W)));
    typedef T vvec __attribute__((ext_vector_type(VW)));
    struct Block {
        kvec k[NK];
        vvec v[4][NV];
        int row;
    };
    __shared__ float meet_o[4][16][D + 4];
    __shared__ float meet_m[4][16 * R], meet_l[4][16 * R];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int seq = blockIdx.x / p.kv_heads, kv_head = blockIdx.x % p.kv_heads;
    if (p.error_flag && blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = tid; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens));
    const Sequence s = sequence_of<KIND>(p, seq, packed_span(p.starts, seq, p.tokens));
    if (tid == 0)
        raise_flag(p, s.cut);
    const int count = s.span.count * p.group;
    if (count == 0 || count > p.few_rows)
        return;
    const int k_first = blockIdx.y * p.split_keys;
    int k_end = visible_keys(p, s, s.span.count - 1);
    if (blockIdx.y > 0 && k_first >= k_end)
        return;
    if (k_end - k_first > p.split_keys)
        k_end = k_first + p.split_keys;
    const int blocks = k_end > k_first ? (k_end - k_first + 15) / 16 : 0;

    const T* kbase = static_cast<const T*>(p.k) + (int64_t)kv_head * p.dk;
    const T* vbase = static_cast<const T*>(p.v) + (int64_t)kv_head * p.dv;
    auto look_up = [&](int blk) { // the place of key c of a block; positions behind the range repeat its last one
        const int at = k_first + blk * 16 + c;
        return key_row<KIND>(p, s, at < k_end ? at : k_end - 1);
    };
    auto fetch = [&](Block& b, int row) {
        b.row = row;
        const T* kr = kbase + (int64_t)(row < 0 ? 0 : row) * p.ldk;
#pragma unroll
        for (int i = 0; i < NK; ++i)
            b.k[i] = load_chunk<T, W, WIDE>(kr, 4 * W * i + W * g, p.dk);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int vrow = __shfl(row, 4 * g + i, 64);
            const T* vr = vbase + (int64_t)(vrow < 0 ? 0 : vrow) * p.ldv;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                b.v[i][j] = load_chunk<T, VW, WIDE>(vr, 16 * VW * j + VW * c, p.dv);
        }
    };
    Block a, b;
    int row_b = 0;
    if (wave < blocks) {
        const int row_a = look_up(wave);
        row_b = look_up(wave + 4);
        fetch(a, row_a);
    }

    float q[R][NK][W];
    int visible[R];
    float m_run[R], l_run[R];
    f32x4 oacc[R][DL];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const bool ok = 16 * r + c < count;
        const int at = ok ? 16 * r + c : 0, token = at / p.group;
        visible[r] = ok ? visible_keys(p, s, token) : 0;
        const float* from = p.q + (int64_t)(s.span.first + token) * p.ldq + (int64_t)(kv_head * p.group + at - token * p.group) * p.dk;
#pragma unroll
        for (int i = 0; i < NK; ++i)
#pragma unroll
            for (int h = 0; h < W; h += 4) {
                const f32x4 x = load_chunk<float, 4, WIDE>(from, 4 * W * i + W * g + h, p.dk);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    q[r][i][h + e] = x[e] * (p.scale * kLog2e);
            }
        m_run[r] = -INFINITY;
        l_run[r] = 0.f;
#pragma unroll
        for (int e = 0; e < DL; ++e)
            oacc[r][e] = f32x4 { 0.f, 0.f, 0.f, 0.f };
    }
    // keys that the first row sees are seen by all
    const int first_sees = visible_keys(p, s, 0), all_see = first_sees < k_end ? first_sees : k_end;
    bool missing = false;
    auto work = [&](const Block& x, int blk) {
        f32x4 sc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            sc[r] = f32x4 { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int i = 0; i < NK; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e)
                    sc[r] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)x.k[i][e], q[r][i][e], sc[r], 0, 0, 0);
        }
        const int at = k_first + blk * 16;
        if (at + 16 > all_see) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + 4 * g + i >= (visible[r] < k_end ? visible[r] : k_end))
                        sc[r][i] = -INFINITY;
        }
        if (__any(x.row < 0)) {
            missing = true;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool none = __shfl(x.row, 4 * g + i, 64) < 0;
#pragma unroll
                for (int r = 0; r < R; ++r)
                    sc[r][i] = none ? -INFINITY : sc[r][i];
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float mx = fmaxf(fmaxf(sc[r][0], sc[r][1]), fmaxf(sc[r][2], sc[r][3]));
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (__any(mx > m_run[r] + 8.f)) { // the maximum moves when a score passes it by 2^8
                const float m_new = fmaxf(m_run[r], mx);
                const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[r] - m_new);
                m_run[r] = m_new;
                l_run[r] *= corr;
#pragma unroll
                for (int e = 0; e < DL; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        oacc[r][e][i] *= corr;
            }
            const float base = m_run[r] == -INFINITY ? 0.f : m_run[r];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[r][i] = __builtin_amdgcn_exp2f(sc[r][i] - base);
                l_run[r] += sc[r][i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < VW; ++e)
                        oacc[r][j * VW + e] = __builtin_amdgcn_mfma_f32_16x16x4f32((float)x.v[i][j][e], sc[r][i], oacc[r][j * VW + e], 0, 0, 0);
        }
    };
    for (int blk = wave; blk < blocks; blk += 8) {
        const bool more = blk + 4 < blocks;
        int row_a = 0;
        if (more) {
            fetch(b, row_b);
            row_a = look_up(blk + 8);
        }
        work(a, blk);
        if (!more)
            break;
        if (blk + 8 < blocks) {
            fetch(a, row_a);
            row_b = look_up(blk + 12);
        }
        work(b, blk + 4);
    }
    raise_flag(p, missing);

    // the waves' sums meet, 16 rows at a time: 16 threads a row, DL depths each
    uint32_t odd = 0; // of this wave's rows those whose sums are not finite, or empty though there are keys
#pragma unroll
    for (int r = 0; r < R; ++r) {
        l_run[r] += __shfl_xor(l_run[r], 16, 64);
        l_run[r] += __shfl_xor(l_run[r], 32, 64);
        if (r > 0)
            __syncthreads();
        if (g == 0) {
            meet_m[wave][16 * r + c] = m_run[r];
            meet_l[wave][16 * r + c] = l_run[r];
        }
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < VW; ++e)
                    meet_o[wave][c][16 * VW * j + VW * (4 * g + i) + e] = oacc[r][j * VW + e][i];
        __syncthreads();
        const int at = 16 * r + (tid >> 4), d0 = (tid & 15) * DL;
        const float top = fmaxf(fmaxf(meet_m[0][at], meet_m[1][at]), fmaxf(meet_m[2][at], meet_m[3][at]));
        const float m = top == -INFINITY ? 0.f : top;
        float l = 0.f, o[DL], size;
#pragma unroll
        for (int e = 0; e < DL; ++e)
            o[e] = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(meet_m[w][at] - m);
            l += f * meet_l[w][at];
#pragma unroll
            for (int e = 0; e < DL; ++e)
                o[e] += f * meet_o[w][tid >> 4][d0 + e];
        }
        size = l;
#pragma unroll
        for (int e = 0; e < DL; ++e)
            size += fabsf(o[e]);
        const int token = (at < count ? at : 0) / p.group, head = kv_head * p.group + (at < count ? at : 0) - token * p.group;
        const int sees = visible_keys(p, s, token);
        const bool in_parts = sees > p.split_keys, mine = at < count && (in_parts ? k_first < sees : blockIdx.y == 0);
        const uint64_t bad = __ballot(mine && (!(size < INFINITY) || (l == 0.f && k_first < sees)));
        if (mine && (bad >> (lane & 48) & 0xffff) == 0) {
            const int64_t q_row = s.span.first + token, id = q_row * p.heads + head;
            const float f = l > 0.f ? 1.f / l : 0.f; // no key: zeros
            float* to = in_parts ? part_out(p, blockIdx.y, id) : p.out + q_row * p.ldo + (int64_t)head * p.dv;
            if (in_parts && (tid & 15) == 0) {
                float* size_at = part_size(p, blockIdx.y, id);
                size_at[0] = top;
                size_at[1] = l;
            }
#pragma unroll
            for (int e = 0; e < DL; e += 4) {
                if (WIDE) {
                    if (d0 + e < p.dv)
                        *reinterpret_cast<f32x4*>(to + d0 + e) = f32x4 { o[e] * f, o[e + 1] * f, o[e + 2] * f, o[e + 3] * f };
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (d0 + e + i < p.dv)
                            to[d0 + e + i] = o[e + i] * f;
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) // rows 4 wave .. 4 wave + 3 of the sixteen
            if (bad >> (16 * k) & 0xffff)
                odd |= 1u << (16 * r + 4 * wave + k);
    }
    if (__builtin_expect(odd == 0, 1))
        return;
#pragma clang loop unroll(disable)
    while (odd) {
        const int r1 = __builtin_ctz(odd);
        odd &= odd - 1;
        const int token = r1 / p.group;
        store_plain_row<KIND>(p, s, token, kv_head * p.group + r1 - token * p.group, kv_head, blockIdx.y, lane);
    }
}

// Rows that more than one range of keys was summed for: sum of 2^(m - M) l o over the ranges, divided by that of 2^(m - M) l.
template <int KIND>
__global__ __launch_bounds__(256) void ragged_join_kernel(RaggedParams p, int few_keys, int tile_keys)
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
    const int keys = s.span.count * p.group <= p.few_rows ? few_keys : tile_keys;
    if (visible <= keys)
        return;
    const int parts = (visible + keys - 1) / keys;
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

// How a call is cut: sequences of few rows (up to `few_rows`) go to ragged_few_kernel in ranges of few_keys keys, the others to
// ragged_tile_kernel in ranges of tile_keys.
struct RaggedPlan {
    int few_rows, few_ranges, few_keys; // few_ranges 0: no such launch
    int tile_ranges, tile_keys;
    int64_t tiles;
    int ranges() const { return few_ranges > tile_ranges ? few_ranges : tile_ranges; }
    size_t scratch(int tokens, int heads, int dv) const
    {
        return ranges() > 1 ? sizeof(float) * (size_t)ranges() * tokens * heads * (2 + (size_t)dv) : 0;
    }
};

static int ranges_of(int64_t keys, int64_t want, int least, int* range_keys)
{
    int64_t per = (keys + want - 1) / want;
    per = (per < least ? least : per) + 63 & ~(int64_t)63;
    *range_keys = per > INT_MAX - 64 ? INT_MAX - 64 : (int)per;
    return (int)((keys + *range_keys - 1) / *range_keys);
}

static RaggedPlan paged_plan(int tokens, int max_new, int heads, const fdx_kv_pages* c)
{
    RaggedPlan r {};
    const int group = heads / c->kv_heads;
    const int64_t most = (int64_t)(max_new < tokens ? max_new : tokens) * group; // rows of a sequence
    r.few_rows = most <= 16 ? 16 : 32;
    if (group <= r.few_rows) {
        const int64_t items = (int64_t)c->n_seqs * c->kv_heads;
        r.few_ranges = ranges_of(c->max_len, (4096 + items - 1) / items, 256, &r.few_keys);
    }
    if (most > r.few_rows || r.few_ranges == 0) {
        r.tiles = tile_numbers(tokens, c->n_seqs, group, 128) * c->kv_heads;
        const int64_t full = ((int64_t)tokens * group + 127) / 128 * c->kv_heads;
        r.tile_ranges = ranges_of(c->max_len, full >= 256 ? 1 : (512 + full - 1) / full, 512, &r.tile_keys);
    }
    if (r.few_ranges == 0)
        r.few_rows = 0;
    return r;
}

static RaggedPlan packed_plan(int tokens, int n_seqs, int heads, int kv_heads)
{
    RaggedPlan r {};
    r.tiles = tile_numbers(tokens, n_seqs, heads / kv_heads, 128) * kv_heads;
    r.tile_ranges = 1;
    r.tile_keys = INT_MAX - 64;
    return r;
}

// rows of every tensor start on vectors of four elements (eight in bf16 pages)
template <int KIND>
static bool wide_rows(const RaggedParams& p)
{
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.k)
        | reinterpret_cast<uintptr_t>(p.v);
    const int64_t unit = KIND == kPagedBf16 ? 7 : 3;
    return (all & 15) == 0 && ((p.ldq | p.ldo | p.ldk | p.ldv | p.dk | p.dv) & unit) == 0;
}

template <int D, int KIND, bool WIDE>
static void ragged_launch(RaggedParams p, const RaggedPlan& plan)
{
    p.few_rows = plan.few_rows;
    p.wide = WIDE;
    p.ranges = plan.ranges();
    if constexpr (KIND != kPackedF32) {
        if (plan.few_ranges > 0) {
            p.split_keys = plan.few_keys;
            const dim3 grid((unsigned)(p.n_seqs * p.kv_heads), (unsigned)plan.few_ranges);
            if (plan.few_rows <= 16)
                hipLaunchKernelGGL((ragged_few_kernel<D, KIND, 1, WIDE>), grid, dim3(256), 0, stream(), p);
            else
                hipLaunchKernelGGL((ragged_few_kernel<D, KIND, 2, WIDE>), grid, dim3(256), 0, stream(), p);
        }
    }
    if (plan.tiles > 0) {
        p.split_keys = plan.tile_keys;
        const dim3 grid((unsigned)plan.tiles, (unsigned)plan.tile_ranges);
        if (WIDE && p.dk == D && p.dv == D && p.ldk < (1 << 24) && p.ldv < (1 << 24)) // offsets inside a tile in 32 bits
            hipLaunchKernelGGL((ragged_tile_kernel<D, KIND, true>), grid, dim3(256), 0, stream(), p);
        else
            hipLaunchKernelGGL((ragged_tile_kernel<D, KIND, false>), grid, dim3(256), 0, stream(), p);
    }
    if (plan.ranges() > 1)
        hipLaunchKernelGGL(ragged_join_kernel<KIND>, dim3((unsigned)(((int64_t)p.tokens * p.heads + 3) / 4)), dim3(256), 0, stream(), p, plan.few_keys,
            plan.tile_keys);
}

template <int KIND>
static void ragged_dispatch(const RaggedParams& p, const RaggedPlan& plan)
{
    const bool small = p.dk <= 64 && p.dv <= 64;
    if (wide_rows<KIND>(p)) {
        if (small)
            ragged_launch<64, KIND, true>(p, plan);
        else
            ragged_launch<128, KIND, true>(p, plan);
    } else {
        if (small)
            ragged_launch<64, KIND, false>(p, plan);
        else
            ragged_launch<128, KIND, false>(p, plan);
    }
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
    (void)dk;
    if (tokens <= 0 || n_seqs <= 0 || heads <= 0 || kv_heads <= 0 || dv <= 0)
        return 0;
    return packed_plan(tokens, n_seqs, heads, kv_heads).scratch(tokens, heads, dv);
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
    p.error_flag = error_flag_dev; p.part = static_cast<float*>(scratch_dev);
    const fdx_status st = check_ragged("mha_packed", p, scratch_dev, fdx_mha_packed_scratch_bytes(tokens, n_seqs, heads, kv_heads, dk, dv));
    if (st != FDX_OK)
        return st;
    p.scale = (float)(1.0 / std::sqrt((double)dk));
    profile_begin();
    ragged_dispatch<kPackedF32>(p, packed_plan(tokens, n_seqs, heads, kv_heads));
    profile_end("mha_packed_f32", 0.0, 4.0 * tokens * ((double)heads + kv_heads) * (dk + dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}

extern "C" size_t fdx_mha_paged_scratch_bytes(int tokens, int max_new, int heads, const fdx_kv_pages* c)
{
    if (!c || tokens <= 0 || max_new <= 0 || heads <= 0 || c->kv_heads <= 0 || heads % c->kv_heads != 0 || c->dk <= 0 || c->dv <= 0 || c->n_seqs <= 0
        || c->max_len <= 0)
        return 0;
    return paged_plan(tokens, max_new, heads, c).scratch(tokens, heads, c->dv);
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
    p.error_flag = error_flag_dev; p.part = static_cast<float*>(scratch_dev);
    st = check_ragged("mha_paged", p, scratch_dev, fdx_mha_paged_scratch_bytes(tokens, max_new, heads, cache));
    if (st != FDX_OK)
        return st;
    FDX_REQUIRE((int64_t)p.n_seqs * p.kv_heads <= (1 << 22), "mha_paged: sequences * key heads too many for one launch");
    p.scale = (float)(1.0 / std::sqrt((double)p.dk));
    const RaggedPlan plan = paged_plan(tokens, max_new, heads, cache);
    profile_begin();
    if (cache->type == FDX_KV_F32)
        ragged_dispatch<kPagedF32>(p, plan);
    else
        ragged_dispatch<kPagedBf16>(p, plan);
    profile_end("mha_paged_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
