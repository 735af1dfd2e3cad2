// Attention over paged caches in 8 bits, query heads in groups that share a key / value head.
#include <cfloat>
#include <climits>

#include "bf16_split.hpp"
#include "f16_split.hpp"
#include "kv8.hpp"

namespace fdx {

// ---- few query rows: keys and values pass once, straight from memory to the matrix instructions ----
//
// A key head's blocks of 32 keys, those of all sequences one behind the other, are dealt to its workgroups in equal shares, from the lengths that
// are there: none waits for a longer one, there are as many as the GPU takes at once, and those of all heads walk through the same rows of the
// cache side by side.  Where a share ends inside a sequence, its rows' sums are kept for paged8_join_kernel.  A workgroup takes the rows that a
// sequence brings to its key head over the blocks that are its, 32 keys a turn of a wave.  Up to sixteen rows: every fourth block is a wave's;
// up to thirty-two: two waves for either half of the rows take every second one.
//  * S^T = K Q^T: lane (c, g) of 16 x 4 loads 16 codes of keys c and 16 + c at depths 64 i + 16 g, and has the scores of keys 4 g .. 4 g + 3 and
//    16 + 4 g .. of row c.
//  * O^T = V^T P^T over the turn's 32 keys: lane (c, g) loads D / 16 codes of those eight keys at depth D / 16 c, so the probabilities it has are
//    the operand, and gets depths D / 16 (4 g + i) + e of row c.
//  * Codes are fp16 values exactly; a query is held as two fp16 values (f16_split.hpp), and so are its probabilities times their values' scales, by a
//    power that keeps the largest of them so far in fp16's range: a row has sums of its own power, and none depends on keys that it does not see.
//  * A key's scale meets its score; lane (c, g) has looked up one scale, and a lane's number in its row of sixteen names it for all of them.
// Bound by memory: a wave has its next block on its way beside the one it works on.  64 sequences of 4000 keys, 32 / 8 heads of 128 (528 MB), 106 us,
// 4.9 TB/s; 64 of 300 to 7900 (315 MB) 84, 3.8 TB/s: beginnings and ends of segments, two or three a workgroup, take a sixth; one token over 100 003 keys (205
// MB) 49, 4.2.  A third block on its way 91 -> 94 us; three workgroups a CU would spill 37 registers.
template <int D, bool WIDE>
struct Block8 {
    static constexpr int NK = D / 64, DL = D / 16;
    uint32_t k[2][NK][4]; // of keys c and 16 + c
    uint32_t v[8][DL / 4];
    float scale;          // of keys 4 g + (c & 3) + 4 (c & 4): of its keys for c < 8, of its values behind
    int row;              // place of key lane % 32
};

// 4 N codes of a row from depth d on; WIDE: from its first on where d is behind `depth`, any codes: queries are zeros there, and nobody stores that depth
template <int N, bool WIDE>
__device__ __forceinline__ void load_codes(const uint8_t* row, int d, int depth, uint32_t (&c)[N])
{
    if constexpr (WIDE) {
        const uint8_t* from = row + (d < depth ? d : 0);
        if constexpr (N == 4) {
            const u32x4 x = *reinterpret_cast<const u32x4*>(from);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                c[e] = x[e];
        } else if constexpr (N == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(from);
            c[0] = x.x;
            c[1] = x.y;
        } else {
            c[0] = *reinterpret_cast<const uint32_t*>(from);
        }
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

// LDS where the waves' sums meet: a wave's 16 (D + 4) floats each, and 2 * 4 * 16 of m and l; and of 64 sequences their ends among the blocks, first
// rows, new tokens, keys, positions of their first new tokens
struct Meet8 {
    float *of_0, *of_1, *of_2, *of_3, *ml;
    int (*seqs)[64];
    unsigned char* q; // queries of either half of the rows, as the products read them: [half][step][plane][lane][16 bytes]
};

// the shares of sequences with few rows
struct Few8 {
    float* parts;    // [share][key head][2][row][dv] of o / l, then as much of [m, l]: of its first sequence (0) if that began before, of its last (1)
    int shares;      // of a key head
    int rows;        // of a sequence and key head at most
    int unit;        // blocks that shares are counted in: one, or so many that there are fewer than 2^31
    int kv_heads;
    int2* split;     // [sequence] the share that it begins in, how many it has

    __device__ __forceinline__ int64_t row_of(int share, int head, int slot, int row) const
    {
        return ((int64_t)(share * kv_heads + head) * 2 + slot) * rows + row;
    }
    __device__ __forceinline__ float* out(int64_t row, int dv) const { return parts + row * dv; }
    __device__ __forceinline__ float* size(int64_t row, int dv) const { return parts + (int64_t)shares * kv_heads * 2 * rows * dv + row * 2; }
};
// Blocks of a share at least, a turn of each wave; up to kWhole are not shared, which saves the join's launch.  us with 8 and 8 / with 4 and 12, one token:
// 12 heads of 64, 300 keys 13.0 / 9.7, 1000 13.2 / 11.8; 32 / 8 heads of 128, 300 keys 15.0 / 11.8, 380 and eight tokens 19.7 / 18.5, 2000 15.3 / 13.3, 8000
// 16.8 / 17.4; 64 sequences of 50 to 400 32.5 / 27.7.  With up to 16 whole, 400 keys and eight tokens take 19.9 instead of 16.0.
constexpr int kLeastShare = 4, kWhole = 12;

// one of the sequences with few rows: its new rows, its keys, its units of blocks.  One that sees no key has a unit all the same: its rows get zeros.
struct FewSequence {
    int first, count, keys, ahead, units;
};
__device__ __forceinline__ FewSequence few_sequence(const RaggedParams& p, const Few8& few, int i)
{
    if (i >= p.n_seqs)
        return { 0, 0, 0, 0, 0 };
    const Sequence s = sequence_of<kPagedF32>(p, i, packed_span(p.starts, i, p.tokens));
    if (s.span.count == 0 || !s.few)
        return { 0, 0, 0, 0, 0 };
    const int blocks = (s.keys + 31) / 32;
    return { s.span.first, s.span.count, s.keys, s.ahead, blocks > 0 ? (blocks - 1) / few.unit + 1 : 1 };
}
__device__ __forceinline__ int share_of(const Few8& few, int all)
{
    const int share = (all + few.shares - 1) / few.shares, least = (kLeastShare + few.unit - 1) / few.unit;
    return share < least ? least : share;
}

template <int D, int KIND, bool WIDE>
__device__ __forceinline__ void few8_segment(const RaggedParams& p, const Scales8& scales, const Few8& few, const Meet8& meet, const Sequence& s,
    int kv_head, int first_block, int last_block, int share, int part)
{
    typedef Block8<D, WIDE> Block;
    constexpr int NK = Block::NK, DL = Block::DL;
    float (*meet_m)[16] = reinterpret_cast<float (*)[16]>(meet.ml), (*meet_l)[16] = meet_m + 4;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid)); // what follows from it is found out for each segment, no register keeps it
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int count = s.span.count * p.group;
    const bool halves = count > 16;
    const int step = halves ? 2 : 4, slot = halves ? wave & 1 : wave, r_first = halves ? (wave >> 1) * 16 : 0; // of this wave
    const int k_first = first_block * 32, k_end = last_block * 32 < s.keys ? last_block * 32 : s.keys;
    const int blocks = (k_end - k_first + 31) / 32;

    const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + (int64_t)kv_head * p.dk;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + (int64_t)kv_head * p.dv;
    const float* scale_base = (c < 8 ? scales.k : scales.v) + kv_head;
    const int scale_key = 4 * g + (c & 3) + 4 * (c & 4);
    auto look_up = [&](int blk) { // the place of key lane % 32 of a block; positions behind the range repeat its last one
        const int at = k_first + blk * 32 + (lane & 31);
        return key_row<kPagedF32>(p, s, at < k_end ? at : k_end - 1);
    };
    // where rows start is 32 bits in units of 16 bytes (see `wide` of paged8_launch), which saves the products of 64 bits
    const uint32_t k_units = (uint32_t)(p.ldk >> 4), v_units = (uint32_t)(p.ldv >> 4);
    const int lane_c = 4 * c, lane_g = 16 * g, lane_scale = 4 * scale_key; // bytes, as the lane that a number comes from is told
    auto of_lane = [](int v, int lane, int more) { return __builtin_amdgcn_ds_bpermute(lane + 4 * more, v); };
    auto fetch = [&](Block& b, int row) {
        b.row = row;
        row = row < 0 ? 0 : row;
        const uint32_t k_at = (uint32_t)row * k_units, v_at = (uint32_t)row * v_units;
#pragma unroll
        for (int z = 0; z < 2; ++z) {
            const uint8_t* kr = WIDE ? kbase + ((uint64_t)(uint32_t)of_lane((int)k_at, lane_c, 16 * z) << 4) : kbase + (int64_t)of_lane(row, lane_c, 16 * z) * p.ldk;
#pragma unroll
            for (int i = 0; i < NK; ++i)
                load_codes<4, WIDE>(kr, 64 * i + 16 * g, p.dk, b.k[z][i]);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = 16 * (i >> 2) + (i & 3);
            const uint8_t* vr = WIDE ? vbase + ((uint64_t)(uint32_t)of_lane((int)v_at, lane_g, key) << 4) : vbase + (int64_t)of_lane(row, lane_g, key) * p.ldv;
            load_codes<DL / 4, WIDE>(vr, DL * c, p.dv, b.v[i]);
        }
        b.scale = scale_base[(int64_t)quotient(of_lane(row, lane_scale, 0), scales.block) * p.kv_heads];
    };
    Block a, b;
    int row_b = 0;
    if (slot < blocks) {
        const int row_a = look_up(slot);
        row_b = look_up(slot + step);
        fetch(a, row_a);
    }

    // the query: step (i, h) has depths 64 i + 16 g + 8 h ..
    // In LDS, which leaves registers to the blocks on their way; waves that share rows write the same.
    f16x8* q_at = reinterpret_cast<f16x8*>(meet.q) + (r_first > 0 ? 4 * NK * 64 : 0) + lane;
    // Scores over codes are up to 2^15 * 448 * 128 < 2^31 times to_log2, which may pass fp32's range before a small scale brings them back: factors above 2^90
    // leave 2^30 for behind the scale.
    float to_log2, behind;
    bool some_behind;
    const bool q_ok = r_first + c < count;
    const int q_token = quotient(q_ok ? r_first + c : 0, p.by_group);
    const int visible = q_ok ? visible_keys(p, s, q_token) : 0;
    {
        const float* from = p.q + (int64_t)(s.span.first + q_token) * p.ldq
            + (int64_t)(kv_head * p.group + (q_ok ? r_first + c : 0) - q_token * p.group) * p.dk;
        float x[2 * NK][8], top = 0.f;
#pragma unroll
        for (int u = 0; u < 2 * NK; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const int d = 64 * (u >> 1) + 16 * g + 8 * (u & 1) + e;
                f32x4 y = { 0.f, 0.f, 0.f, 0.f };
                if (WIDE) {
                    if (d < p.dk)
                        y = *reinterpret_cast<const f32x4*>(from + d);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (d + i < p.dk)
                            y[i] = from[d + i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[u][e + i] = y[i];
                    top = fmaxf(top, fabsf(y[i]));
                }
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        const Pow2 sq = pow2_for<1>(exponent(max_halves(top)));
        to_log2 = sq.down * (p.scale * kLog2e);
        behind = to_log2 > 0x1p90f ? 0x1p30f : 1.f;
        to_log2 = to_log2 > 0x1p90f ? to_log2 * 0x1p-30f : to_log2;
        some_behind = __any(behind != 1.f);
#pragma unroll
        for (int u = 0; u < 2 * NK; ++u)
        {
            f16x8 h, l;
            split2x8(x[u], sq.up, h, l);
            q_at[(2 * u) * 64] = l;
            q_at[(2 * u + 1) * 64] = h;
        }
    }
    float m_run = -INFINITY, l_run = 0.f;
    float w_most = 0.f; // the largest probability times scale so far, to within 2^4
    Pow2 power = pow2_for<1>(0); // of the sums
    f32x4 oacc[DL];
#pragma unroll
    for (int e = 0; e < DL; ++e)
        oacc[e] = f32x4 { 0.f, 0.f, 0.f, 0.f };
    // keys that the first row sees are seen by all
    const int first_sees = visible_keys(p, s, quotient(r_first, p.by_group)), all_see = first_sees < k_end ? first_sees : k_end;
    bool missing = false, seen = false;
    auto mfma = [](f16x8 x, f16x8 y, const f32x4& acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(x, y, acc, 0, 0, 0); };
    auto most_of_row = [](float x) { return max_halves(fmaxf(x, __shfl_xor(x, 16, 64))); }; // lanes c, 16 + c, 32 + c and 48 + c
    auto work = [&](Block& x, int blk) {
        auto operand = [](uint32_t a, uint32_t b) {
            u32x4 w;
            uint32_t lo, hi;
            f16_of_codes<KIND>(a, lo, hi);
            w[0] = lo;
            w[1] = hi;
            f16_of_codes<KIND>(b, lo, hi);
            w[2] = lo;
            w[3] = hi;
            return __builtin_bit_cast(f16x8, w);
        };
        f32x4 acc[2] = { { 0.f, 0.f, 0.f, 0.f }, { 0.f, 0.f, 0.f, 0.f } };
#pragma unroll
        for (int u = 0; u < 2 * NK; ++u) {
            const f16x8 ql = q_at[(2 * u) * 64], qh = q_at[(2 * u + 1) * 64];
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const f16x8 k = operand(x.k[z][u >> 1][2 * (u & 1)], x.k[z][u >> 1][2 * (u & 1) + 1]);
                acc[z] = mfma(k, ql, acc[z]);
                acc[z] = mfma(k, qh, acc[z]);
            }
        }
        float sc[8], vs[8]; // keys 4 g + i, then 16 + 4 g + i
#pragma unroll
        for (int i = 0; i < 8; ++i)
            sc[i] = acc[i >> 2][i & 3] * to_log2;
        sc[0] *= dpp_move<0x150>(x.scale); // row_newbcast: lane n of a row of sixteen, for all of them
        sc[1] *= dpp_move<0x151>(x.scale);
        sc[2] *= dpp_move<0x152>(x.scale);
        sc[3] *= dpp_move<0x153>(x.scale);
        sc[4] *= dpp_move<0x154>(x.scale);
        sc[5] *= dpp_move<0x155>(x.scale);
        sc[6] *= dpp_move<0x156>(x.scale);
        sc[7] *= dpp_move<0x157>(x.scale);
        if (__builtin_expect(some_behind, 0)) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                sc[i] *= behind;
        }
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
        if (__builtin_expect(at + 32 > all_see || absent, 0)) {
            missing = missing || absent;
            int g4 = 4 * g;
            asm volatile("" : "+v"(g4)); // no register keeps the keys' numbers for the next time
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int key = 16 * (i >> 2) + g4 + (i & 3);
                const bool there = of_lane(x.row, lane_g, 16 * (i >> 2) + (i & 3)) >= 0;
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
        float corr = 1.f;
        // The maximum moves when a score passes it by 4: what is added is below 2^4, and 2^4 times a value's scale, up to 2^128 / 127, is in fp32's range
        if (__any(mx > m_run + 4.f)) {
            const float m_new = fmaxf(m_run, most_of_row(mx));
            corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
            m_run = m_new;
            l_run *= corr;
            w_most *= corr;
        }
        const float base = m_run == -INFINITY ? 0.f : m_run;
        float sum = 0.f, most = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sc[i] = __builtin_amdgcn_exp2f(sc[i] - base);
            sum += sc[i];
            sc[i] *= vs[i];
            most = fmaxf(most, sc[i]);
        }
        l_run += sum;
        if (__any(most > w_most * 16.f || corr != 1.f)) {
            w_most = fmaxf(w_most, most_of_row(most));
            const Pow2 now = pow2_for<1>(exponent(w_most) + 5); // at most 2^10
            const float by = corr * now.up * power.down; // from the left: the powers' product alone may pass fp32's range
            power = now;
#pragma unroll
            for (int e = 0; e < DL; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    oacc[e][i] *= by;
        }
        f16x8 ph, pl;
        split2x8(sc, power.up, ph, pl);
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
                const f16x8 v = operand(t[0][i], t[1][i]);
                oacc[e + i] = mfma(v, pl, oacc[e + i]);
                oacc[e + i] = mfma(v, ph, oacc[e + i]);
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
    const float part_of = l_run > 0.f ? 1.f / l_run : 0.f; // sums meet as means, which stay in fp32's range where the values are; NaN stays NaN below
    auto leave = [&](float* of) {
#pragma unroll
        for (int e = 0; e < DL; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                of[c * (D + 4) + DL * (4 * g + i) + e] = oacc[e][i] * part_of * power.down;
    };
    if (wave == 0) // no pointer is chosen by a number: that would be a table in scratch memory
        leave(meet.of_0);
    else if (wave == 1)
        leave(meet.of_1);
    else if (wave == 2)
        leave(meet.of_2);
    else
        leave(meet.of_3);
    __syncthreads();
    const int row_at = tid >> 4, d0 = (tid & 15) * DL;
    for (int half = 0; half <= (halves ? 1 : 0); ++half) {
        const int w_first = 2 * half, w_last = halves ? w_first + 1 : 3; // the waves that have these rows
        float top = -INFINITY;
        for (int w = w_first; w <= w_last; ++w)
            top = fmaxf(top, meet_m[w][row_at]);
        const float m = top == -INFINITY ? 0.f : top;
        float l = 0.f, o[DL];
        for (int w = w_first; w <= w_last; ++w)
            l += __builtin_amdgcn_exp2f(meet_m[w][row_at] - m) * meet_l[w][row_at];
#pragma unroll
        for (int e = 0; e < DL; ++e)
            o[e] = 0.f;
        const float none = top != -INFINITY && part < 0 ? NAN : 0.f; // as finish() has it
        auto add = [&](int w, const float* of) {
            const float f = __builtin_amdgcn_exp2f(meet_m[w][row_at] - m) * meet_l[w][row_at] / l;
#pragma unroll
            for (int e = 0; e < DL; ++e)
                o[e] = fmaf(f, of[row_at * (D + 4) + d0 + e], o[e]);
        };
        if (l != 0.f) {
            if (w_first == 0) {
                add(0, meet.of_0);
                add(1, meet.of_1);
            }
            if (w_last == 3) {
                add(2, meet.of_2);
                add(3, meet.of_3);
            }
        } else {
#pragma unroll
            for (int e = 0; e < DL; ++e)
                o[e] = none;
        }
        const int r = 16 * half + row_at;
        if (r >= count)
            continue;
        const int token = quotient(r, p.by_group), head = kv_head * p.group + r - token * p.group;
        float* to = p.out + (int64_t)(s.span.first + token) * p.ldo + (int64_t)head * p.dv;
        if (part >= 0) {
            const int64_t id = few.row_of(share, kv_head, part, r);
            to = few.out(id, p.dv);
            float* size_at = few.size(id, p.dv);
            if ((tid & 15) == 0) {
                size_at[0] = top;
                size_at[1] = l;
            }
        }
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

template <int D, int KIND, bool WIDE>
__device__ __forceinline__ void few8_body(const RaggedParams& p, const Scales8& scales, const Few8& few, int wg, const Meet8& meet)
{
    const int kv_head = wg % p.kv_heads, mine = wg / p.kv_heads;
    if (p.error_flag && wg == 0)
        for (int i = threadIdx.x; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens) || sequence_of<kPagedF32>(p, i, packed_span(p.starts, i, p.tokens)).cut);
    int at = 0, end = 0, share = 1, from = 0, front = 0; // units; those in front of sequences i0 ..
    auto deal = [&](int all) {
        share = share_of(few, all);
        if ((int64_t)mine * share >= all)
            return false;
        at = mine * share;
        end = all - at < share ? all : at + share;
        return true;
    };
    if (p.n_seqs > 64) { // 64 runs of sequences, sixteen a wave: where the share begins among them
        const int lane = threadIdx.x & 63, length = (p.n_seqs / 64 + 64) & ~63;
        for (int j = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); j < 64; j += 4) {
            int sum = 0;
            for (int64_t i = (int64_t)j * length; i < (int64_t)(j + 1) * length && i < p.n_seqs; i += 64)
                sum += few_sequence(p, few, (int)i + lane).units;
            sum = wave_prefix(sum);
            if (lane == 63)
                meet.seqs[0][j] = sum;
        }
        __syncthreads();
        const int up_to = wave_prefix(meet.seqs[0][lane]);
        __syncthreads();
        if (!deal(__builtin_amdgcn_readlane(up_to, 63)))
            return;
        const int run = __builtin_popcountll(__ballot(up_to <= at));
        front = run > 0 ? __builtin_amdgcn_readlane(up_to, run - 1) : 0;
        from = run * length;
    }
    for (int i0 = from; i0 < p.n_seqs; i0 += 64) {
        int tid = threadIdx.x;
        asm volatile("" : "+v"(tid));
        const int lane = tid & 63;
        const FewSequence of_lane = few_sequence(p, few, i0 + lane);
        const int up_to = front + wave_prefix(of_lane.units), before = front;
        front = __builtin_amdgcn_readlane(up_to, 63);
        if (p.n_seqs <= 64 && !deal(front))
            return;
        if (at >= front)
            continue;
        if (tid < 64) { // no register keeps it through the segments
            meet.seqs[0][lane] = up_to;
            meet.seqs[1][lane] = of_lane.first;
            meet.seqs[2][lane] = of_lane.count;
            meet.seqs[3][lane] = of_lane.keys;
            meet.seqs[4][lane] = of_lane.ahead;
        }
        __syncthreads();
        while (at < end && at < front) {
            int me = threadIdx.x;
            asm volatile("" : "+v"(me));
            const int of = __builtin_popcountll(__ballot(meet.seqs[0][me & 63] <= at));
            auto number = [&](int which, int i) { return __builtin_amdgcn_readfirstlane(meet.seqs[which][i]); };
            const int first = of > 0 ? number(0, of - 1) : before, last = number(0, of);
            const Sequence s { { number(1, of), number(2, of) }, number(3, of), number(4, of), i0 + of, true, INT_MAX, false };
            const int stop = end < last ? end : last;
            if (few.split && kv_head == 0 && at == first && me == 0)
                few.split[i0 + of] = int2 { mine, (last - 1) / share - mine + 1 };
            few8_segment<D, KIND, WIDE>(p, scales, few, meet, s, kv_head, (at - first) * few.unit, (stop - first) * few.unit, mine,
                at == first && stop == last ? -1 : (at > first ? 0 : 1));
            at = stop;
            __syncthreads(); // the waves' sums have been read
        }
        if (at >= end)
            return;
        __syncthreads();
    }
}

template <int D, int KIND, bool WIDE>
__global__ __launch_bounds__(256, WIDE ? 2 : 1) void paged8_few_kernel(RaggedParams p, Scales8 scales, Few8 few)
{
    __shared__ float meet[4][16 * (D + 4)], ml[2 * 4 * 16];
    __shared__ int seqs[5][64];
    __shared__ __attribute__((aligned(16))) unsigned char q[2 * D / 32 * 2 * 1024];
    few8_body<D, KIND, WIDE>(p, scales, few, blockIdx.x, Meet8 { meet[0], meet[1], meet[2], meet[3], ml, seqs, q });
}

// ---- many query rows: tiles on the fp16 matrix instructions ----
//
// A workgroup takes 128 rows of one key head of one sequence, rows counting through the query heads of the group first (row = token *
// group + head), a wave 32 of them; keys and values pass through LDS in tiles of 4096 / D keys, codes as the fp16 values that they are.  Products
// are taken transposed, S^T = K Q^T and O^T = V^T P^T: a query is a lane's column and keys are the accumulator's registers.
//  * A query row is brought to fp16's range by a power of two and held as two fp16 values (f16_split.hpp).  So are its probabilities times
//    the values' scales, by a power that keeps the largest of them so far between 2^6 and 2^15: a row has sums of its own power, and none
//    depends on keys that it does not see.  A key's scale meets its score.
// Vector instructions (60 % of the time) and matrix instructions (44 %) mostly add up: four sequences that bring 1000 tokens to 3000 keys, 32 / 8
// heads of 128 (164 GFLOP), 371 us, 442 TFLOP/s, where two products for one leave 620.
//  * LDS holds two tiles.  While the probabilities of tile t meet its values, the scores of tile t + 1 are multiplied; tile t + 2's keys and tile
//    t + 1's values go to LDS, what comes behind them to registers; one barrier a tile.
template <int D>
struct Tile8 {
    static constexpr int KT = 4096 / D, N = 256 / KT; // keys of a tile; threads that fetch a key, 16 codes each
    static constexpr int KBLK = KT * 16 + 128 / N, VROW = D * 2 + 32; // bytes of a block of 8 depths, of a row of values, offset against each other
    static constexpr int kKeys = D / 8 * KBLK, kValues = KT * VROW; // bytes of a tile
    static constexpr int kAhead = 512; // places of two halves of as many positions are looked up ahead, all threads at once
};
struct TileLds8 {
    unsigned char *ks0, *ks1, *vs0, *vs1;
    float *scale0, *scale1; // of a tile's keys, then of its values
    int *rows_of, *some_absent;
};
#define FDX_TILE8_LDS(D, lds)                                                                                               \
    __shared__ __attribute__((aligned(16))) unsigned char lds##_ks0[Tile8<D>::kKeys], lds##_ks1[Tile8<D>::kKeys];           \
    __shared__ __attribute__((aligned(16))) unsigned char lds##_vs0[Tile8<D>::kValues], lds##_vs1[Tile8<D>::kValues];       \
    __shared__ __attribute__((aligned(16))) float lds##_scale0[2 * Tile8<D>::KT], lds##_scale1[2 * Tile8<D>::KT];           \
    __shared__ int lds##_rows_of[2 * Tile8<D>::kAhead];                                                                     \
    __shared__ int lds##_absent;                                                                                            \
    const TileLds8 lds { lds##_ks0, lds##_ks1, lds##_vs0, lds##_vs1, lds##_scale0, lds##_scale1, lds##_rows_of, &lds##_absent }

template <int D, int KIND, bool WIDE, bool SIXTEENS>
__device__ __forceinline__ void tile8_body(const RaggedParams& p, const Scales8& scales, const Place& place_in, const TileLds8& lds)
{
    typedef Tile8<D> S;
    typedef float f32x16 __attribute__((ext_vector_type(16)));
    constexpr int KT = S::KT, HALVES = KT / 32, N = S::N, STEPS = D / 16, DB = D / 32, KBLK = S::KBLK, VROW = S::VROW, kAhead = S::kAhead;
    int* rows_of = lds.rows_of;
    int& some_absent = *lds.some_absent;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, half = lane >> 5;
    if (p.error_flag && place_in.x == 0 && place_in.y == 0)
        for (int i = tid; i < p.n_seqs; i += 256) // lengths too: a sequence without new tokens has no tile
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens) || p.lens[i] < 0 || p.lens[i] > p.max_len);
    // key heads next to each other, later tiles of a sequence, which see more keys, first
    const int kv_head = place_in.x % p.kv_heads;
    const int64_t number = place_in.x / p.kv_heads;
    const Tile tile = p.n_seqs <= 64 ? late_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, p.group, 128, number)
                                     : find_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, p.group, 128, place_in.nx / p.kv_heads - 1 - number);
    if (tile.seq < 0)
        return;
    const Sequence s = sequence_of<kPagedF32>(p, tile.seq, tile.span);
    if (tid == 0)
        raise_flag(p, s.cut);
    const int count = s.span.count * p.group; // rows
    const int r_first = tile.index * 128;
    if (r_first >= count || s.few)
        return;
    const int mine = r_first + wave * 32 + c;
    const bool q_ok = mine < count;
    const int token = quotient(q_ok ? mine : count - 1, p.by_group), head = kv_head * p.group + (q_ok ? mine : count - 1) - token * p.group;
    const int64_t q_row = s.span.first + token;
    const int visible = visible_keys(p, s, token);
    const int r_last = r_first + 128 < count ? r_first + 127 : count - 1;
    int k_end = visible_keys(p, s, quotient(r_last, p.by_group)); // of the workgroup's last row
    const int64_t k_from = (int64_t)place_in.y * s.range;
    if (place_in.y > 0 && k_from >= k_end)
        return;
    const int k_first = (int)k_from;
    if (k_end - k_first > s.range)
        k_end = k_first + s.range;
    const int tiles = k_end > k_first ? (k_end - k_first + KT - 1) / KT : 0;
    // what the wave's rows see: all of them the first `wave_all_see`, some the first `wave_any`
    const int w_first = r_first + wave * 32, w_last = w_first + 31 < count ? w_first + 31 : count - 1;
    const int wave_all_see = visible_keys(p, s, quotient(w_first < count ? w_first : count - 1, p.by_group));
    const int wave_any = visible_keys(p, s, quotient(w_last, p.by_group));

    const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + (int64_t)kv_head * p.dk;
    const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + (int64_t)kv_head * p.dv;
    const int krow = tid / N, kl = tid % N;
    // 2 KT threads, whole waves or halves of one, fetch a scale each: of a key, or of its values
    const bool scaled = tid < 2 * KT;
    const float* scale_base = (tid < KT ? scales.k : scales.v) + kv_head;
    uint32_t kst[4], vst[4];
    float sst = 0.f;
    auto place = [&](int t, int key) { return rows_of[(t * KT + key) & (2 * kAhead - 1)]; };
    auto look_up = [&](int first) { // places of positions first .. first + kAhead - 1 of the range; those behind it repeat its last one
#pragma unroll
        for (int i = 0; i < kAhead; i += 256) {
            const int at = k_first + first + i + tid;
            const int row = key_row<kPagedF32>(p, s, at < k_end ? at : k_end - 1);
            rows_of[(first + i + tid) & (2 * kAhead - 1)] = row;
            if (row < 0) {
                some_absent = 1;
                raise_flag(p, true);
            }
        }
    };
    auto zero_codes = [](uint32_t (&x)[4]) { x[0] = x[1] = x[2] = x[3] = 0; };
    auto fetch_keys = [&](int t) {
        const int row = place(t, krow);
        load_codes<4, WIDE>(kbase + (int64_t)(row < 0 ? 0 : row) * p.ldk, 16 * kl, p.dk, kst);
        if (row < 0)
            zero_codes(kst);
    };
    auto fetch_values = [&](int t) {
        const int row = place(t, krow);
        load_codes<4, WIDE>(vbase + (int64_t)(row < 0 ? 0 : row) * p.ldv, 16 * kl, p.dv, vst);
        if (row < 0)
            zero_codes(vst);
        if (scaled) {
            const int at = place(t, tid & (KT - 1));
            sst = at < 0 ? 0.f : scale_base[(int64_t)quotient(at, scales.block) * p.kv_heads];
        }
    };
    auto stage_keys = [&](unsigned char* ks) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 w;
            uint32_t lo, hi;
            f16_of_codes<KIND>(kst[2 * h], lo, hi);
            w[0] = lo;
            w[1] = hi;
            f16_of_codes<KIND>(kst[2 * h + 1], lo, hi);
            w[2] = lo;
            w[3] = hi;
            *reinterpret_cast<u32x4*>(&ks[(2 * kl + h) * KBLK + krow * 16]) = w;
        }
    };
    auto stage_values = [&](unsigned char* vs, float* scale) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 w;
            uint32_t lo, hi;
            f16_of_codes<KIND>(vst[2 * h], lo, hi);
            w[0] = lo;
            w[1] = hi;
            f16_of_codes<KIND>(vst[2 * h + 1], lo, hi);
            w[2] = lo;
            w[3] = hi;
            *reinterpret_cast<u32x4*>(&vs[krow * VROW + 32 * kl + 16 * h]) = w;
        }
        if (scaled)
            scale[tid] = sst;
    };

    if (tiles > 0) {
        if (tid == 0)
            some_absent = 0;
        __syncthreads();
        look_up(0);
        if (tiles > kAhead / KT)
            look_up(kAhead);
        __syncthreads();
        fetch_keys(0);
        fetch_values(0);
    }

    f16x8 qh[STEPS], ql[STEPS]; // depths 16 u + 8 half ..
    float to_log2;
    {
        float x[STEPS][8], top = 0.f;
        const float* from = p.q + q_row * p.ldq + (int64_t)head * p.dk;
#pragma unroll
        for (int u = 0; u < STEPS; ++u)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const int d = 16 * u + 8 * half + e;
                f32x4 y = { 0.f, 0.f, 0.f, 0.f };
                if (WIDE) {
                    if (d < p.dk)
                        y = *reinterpret_cast<const f32x4*>(from + d);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (d + i < p.dk)
                            y[i] = from[d + i];
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[u][e + i] = y[i];
                    top = fmaxf(top, fabsf(y[i]));
                }
            }
        const Pow2 sq = pow2_for<1>(exponent(max_halves(top)) + 6); // at most 2^9: scores before to_log2 stay in fp32's range for keys up to 2^100
        to_log2 = sq.down * (p.scale * kLog2e); // 2^-129 or more: -infinity stays what it is
#pragma unroll
        for (int u = 0; u < STEPS; ++u)
            split2x8(x[u], sq.up, qh[u], ql[u]);
    }

    auto mfma = [](f16x8 a, f16x8 b, const f32x16& acc) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0); };
    constexpr f32x16 kZero = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };
    f32x16 oacc[DB], sa[HALVES], sb[HALVES];
#pragma unroll
    for (int d = 0; d < DB; ++d)
        oacc[d] = kZero;
    float m_run = -INFINITY, l_run = 0.f;
    float w_most = 0.f; // the largest probability times scale so far, to within 2^4
    Pow2 power = pow2_for<1>(0); // of the sums
    bool seen = false;

    auto scores = [&](f32x16 (&sc)[HALVES], const unsigned char* ks) {
#pragma unroll
        for (int kb = 0; kb < HALVES; ++kb) {
            sc[kb] = kZero;
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                const f16x8 k = *reinterpret_cast<const f16x8*>(&ks[(2 * u + half) * KBLK + (kb * 32 + c) * 16]);
                sc[kb] = mfma(k, ql[u], sc[kb]);
                sc[kb] = mfma(k, qh[u], sc[kb]);
            }
        }
    };
    // values of four keys for this lane's depth: sixteen lanes address four rows of sixteen depths
    const int v_at = (4 * half + ((c & 15) >> 2)) * VROW + (16 * (c >> 4) + 4 * (c & 3)) * 2;
    auto values = [&](const unsigned char* vs, int key, int d) {
        typedef short s16x4 __attribute__((ext_vector_type(4)));
        struct {
            s16x4 a, b;
        } r;
        r.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vs + v_at + key * VROW + d * 64));
        r.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(vs + v_at + (key + 8) * VROW + d * 64));
        return __builtin_bit_cast(f16x8, r);
    };
    // the products' operands are read from LDS two pairs of products ahead
    auto in_order = [] {
        constexpr int kProducts = 0x8, kReads = 0x100;
        __builtin_amdgcn_sched_group_barrier(kReads, 2, 0);
#pragma unroll
        for (int i = 0; i < HALVES * STEPS; ++i) {
            __builtin_amdgcn_sched_group_barrier(kProducts, 2, 0);
            if (i + 2 < HALVES * STEPS)
                __builtin_amdgcn_sched_group_barrier(kReads, 1, 0);
            else
                __builtin_amdgcn_sched_group_barrier(kReads, 2, 0);
        }
#pragma unroll
        for (int i = 0; i < KT / 16 * DB; ++i) {
            __builtin_amdgcn_sched_group_barrier(kProducts, 2, 0);
            if (i + 2 < KT / 16 * DB)
                __builtin_amdgcn_sched_group_barrier(kReads, 2, 0);
        }
    };
    // tile t: its scores are in sc, its values and scales in vs and scale, the keys of tile t + 1 in ks; registers hold the codes of tile t + 2's
    // keys and of tile t + 1's values
    auto turn = [&](int t, f32x16 (&sc)[HALVES], f32x16 (&next)[HALVES], const unsigned char* ks, const unsigned char* vs, const float* scale,
                    unsigned char* ks_to, unsigned char* vs_to, float* scale_to) {
        const int j0 = k_first + t * KT;
        if (t + 1 < tiles) {
            stage_values(vs_to, scale_to);
            if (t + 2 < tiles) {
                stage_keys(ks_to);
                fetch_values(t + 2);
                if (t + 3 < tiles)
                    fetch_keys(t + 3);
            }
        }
        const int absent = some_absent;
        if ((t * KT & (kAhead - 1)) == 0 && t > 0 && (t + kAhead / KT) < tiles)
            look_up(t * KT + kAhead); // into the half that is done with
        if (j0 < wave_any) { // some row of this wave sees some key of the tile
            const int limit = (visible < k_end ? visible : k_end) - j0; // keys of the tile that this lane's row sees
            const bool some_hidden = j0 + KT > wave_all_see || j0 + KT > k_end, some_gone = __builtin_amdgcn_readfirstlane(absent) != 0;
            auto hidden = [&](int key) { return key >= limit || (some_gone && rows_of[(t * KT + key) & (2 * kAhead - 1)] < 0); };
            // by key i of a set of sixteen, register i of a half; SIXTEENS: such a set has one scale, which then meets its largest score and what scores are
            // multiplied by
            float kf[2 * HALVES], vf[2 * HALVES];
            bool apart = !SIXTEENS;
            if constexpr (SIXTEENS) {
                float most_f = 0.f;
#pragma unroll
                for (int g = 0; g < 2 * HALVES; ++g) {
                    kf[g] = scale[16 * g];
                    vf[g] = scale[KT + 16 * g];
                    most_f = fmaxf(most_f, kf[g]);
                }
                apart = __any(!(most_f * to_log2 < INFINITY)); // products of three numbers in fp32's range, of which two may pass it
            }
            if (apart) {
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 by = *reinterpret_cast<const f32x4*>(scale + kb * 32 + 8 * g + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[kb][4 * g + i] *= by[i];
                    }
#pragma unroll
                for (int g = 0; g < 2 * HALVES; ++g)
                    kf[g] = 1.f;
            }
            if (some_hidden || some_gone) {
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const bool h = hidden(kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3));
                        sc[kb][e] = h ? -INFINITY : sc[kb][e];
                        seen = seen || !h;
                    }
                if constexpr (SIXTEENS) // a scale of NaN is for the rows that see it
#pragma unroll
                    for (int g = 0; g < 2 * HALVES; ++g) {
                        kf[g] = hidden(16 * g) ? 1.f : kf[g];
                        vf[g] = hidden(16 * g) ? 0.f : vf[g];
                    }
            } else {
                seen = true;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < 2 * HALVES; ++g) {
                float of = -INFINITY;
#pragma unroll
                for (int e = 8 * (g & 1); e < 8 * (g & 1) + 8; e += 2)
                    of = fmaxf(fmaxf(of, sc[g >> 1][e]), sc[g >> 1][e + 1]);
                mx = fmaxf(mx, SIXTEENS ? of * kf[g] : of);
                kf[g] = SIXTEENS ? __builtin_elementwise_maximum(kf[g] * to_log2, 0x1p-126f) : to_log2; // above zero for -infinity; NaN stays NaN
            }
            mx = max_halves(mx) * to_log2;
            // The largest score is rounded three times, the exponents' multiply-adds once: up to 2^22 they are less than one apart, of 2^31 further than
            // exponentials reach, and a row would add infinities, or nothing.  From 2^22 on scores are multiplied out first; the largest is one of them.
            if (__builtin_expect(__any(fabsf(mx) >= 0x1p22f && mx > -INFINITY), 0)) {
                mx = -INFINITY;
#pragma unroll
                for (int g = 0; g < 2 * HALVES; ++g) {
#pragma unroll
                    for (int e = 8 * (g & 1); e < 8 * (g & 1) + 8; ++e) {
                        sc[g >> 1][e] *= kf[g];
                        mx = fmaxf(mx, sc[g >> 1][e]);
                    }
                    kf[g] = 1.f;
                }
                mx = max_halves(mx);
            }
            float corr = 1.f;
            if (__any(mx > m_run + 4.f)) {
                const float m_new = mx > m_run + 4.f ? mx : m_run;
                corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
                m_run = m_new;
                l_run *= corr;
                w_most *= corr;
            }
            const float base = m_run == -INFINITY ? 0.f : -m_run; // a row that has seen no key yet adds zeros
            float rs = 0.f, most = 0.f;
#pragma unroll
            for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[kb][e] = __builtin_amdgcn_exp2f(fmaf(sc[kb][e], kf[2 * kb + (e >> 3)], base));
                    rs += sc[kb][e];
                }
            l_run += rs; // the other half of the tile's keys lies in lane + 32: they meet at the end
            if constexpr (SIXTEENS) {
#pragma unroll
                for (int g = 0; g < 2 * HALVES; ++g) {
                    float of = 0.f;
#pragma unroll
                    for (int e = 8 * (g & 1); e < 8 * (g & 1) + 8; e += 2)
                        of = fmaxf(fmaxf(of, sc[g >> 1][e]), sc[g >> 1][e + 1]);
                    most = fmaxf(most, of * vf[g]);
                }
            } else {
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const f32x4 by = *reinterpret_cast<const f32x4*>(scale + KT + kb * 32 + 8 * g + 4 * half);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            sc[kb][4 * g + i] *= by[i];
                    }
                if (some_hidden || some_gone) { // a scale of NaN is for the rows that see it
#pragma unroll
                    for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            sc[kb][e] = hidden(kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3)) ? 0.f : sc[kb][e];
                }
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; e += 2)
                        most = fmaxf(fmaxf(most, sc[kb][e]), sc[kb][e + 1]);
            }
            most = max_halves(most);
            if (__any(most > w_most * 16.f || corr != 1.f)) {
                w_most = fmaxf(w_most, most);
                const Pow2 now = pow2_for<1>(exponent(w_most) + 5); // at most 2^10
                const float by = corr * now.up * power.down; // from the left: the powers' product alone may pass fp32's range
                power = now;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        oacc[d][e] *= by;
            }
            if constexpr (SIXTEENS) {
                float most_f = 0.f;
#pragma unroll
                for (int g = 0; g < 2 * HALVES; ++g)
                    most_f = __builtin_elementwise_maximum(most_f, vf[g]); // NaN stays NaN
                if (__any(!(most_f * power.up < INFINITY))) {
#pragma unroll
                    for (int g = 0; g < 2 * HALVES; ++g) {
#pragma unroll
                        for (int e = 8 * (g & 1); e < 8 * (g & 1) + 8; ++e)
                            sc[g >> 1][e] *= vf[g];
                        vf[g] = 1.f;
                    }
                }
            }
#pragma unroll
            for (int g = 0; g < 2 * HALVES; ++g)
                vf[g] = SIXTEENS ? vf[g] * power.up : power.up;
            __builtin_amdgcn_s_setprio(1); // beside another workgroup's wave that is not at its products (four of 1000 of 3000 keys 391 -> 371 us)
            scores(next, ks);
            // O^T += V^T P^T
#pragma unroll
            for (int u = 0; u < KT / 16; ++u) { // keys of block 2 u + half: registers 8 (u % 2) .. + 7 of accumulator u / 2
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = sc[u >> 1][8 * (u & 1) + j];
                f16x8 ph, pl;
                split2x8(x, vf[u], ph, pl);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const f16x8 v = values(vs, 16 * u, d);
                    oacc[d] = mfma(v, pl, oacc[d]);
                    oacc[d] = mfma(v, ph, oacc[d]);
                }
            }
            in_order();
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
    };
    if (tiles > 0) {
        stage_keys(lds.ks0);
        stage_values(lds.vs0, lds.scale0);
        if (tiles > 1) {
            fetch_keys(1);
            fetch_values(1);
            stage_keys(lds.ks1);
            if (tiles > 2)
                fetch_keys(2);
        }
        __syncthreads();
        scores(sa, lds.ks0);
        __syncthreads(); // ks0 is done with
    }
    for (int t = 0; t < tiles; t += 2) {
        turn(t, sa, sb, lds.ks1, lds.vs0, lds.scale0, lds.ks0, lds.vs1, lds.scale1);
        if (t + 1 < tiles)
            turn(t + 1, sb, sa, lds.ks0, lds.vs1, lds.scale1, lds.ks1, lds.vs0, lds.scale0);
    }

    l_run += __shfl_xor(l_run, 32, 64);
    const uint64_t seen_by = __ballot(seen);
    const bool some = ((seen_by | seen_by >> 32) >> c & 1) != 0;
    const bool in_parts = visible > s.range;
    if (!q_ok || !(in_parts ? k_first < visible : place_in.y == 0))
        return;
    float* to = p.out + q_row * p.ldo + (int64_t)head * p.dv;
    if (in_parts) {
        const int64_t id = part_row(p, s, token, head);
        to = p.tile.out(place_in.y, id, p.dv);
        float* at = p.tile.size(place_in.y, id, p.dv);
        if (half == 0) {
            at[0] = some && m_run == -INFINITY ? -FLT_MAX : m_run;
            at[1] = l_run;
        }
    }
    const float none = some && !in_parts ? NAN : 0.f; // no key: zeros; scores of -infinity only: no softmax
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int depth = 32 * d + 8 * g + 4 * half;
            f32x4 o;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                o[i] = l_run == 0.f ? none : oacc[d][4 * g + i] / l_run * power.down;
            if (WIDE) {
                if (depth < p.dv)
                    *reinterpret_cast<f32x4*>(to + depth) = o;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (depth + i < p.dv)
                        to[depth + i] = o[i];
            }
        }
}

template <int D, int KIND, bool WIDE, bool SIXTEENS>
__global__ __launch_bounds__(256, 2) void paged8_tile_kernel(RaggedParams p, Scales8 scales)
{
    FDX_TILE8_LDS(D, lds);
    tile8_body<D, KIND, WIDE, SIXTEENS>(p, scales, Place { blockIdx.x, blockIdx.y, gridDim.x }, lds);
}

// Both in one launch: what is bound by memory runs beside what is bound by the matrix and vector units.  Tiles, which take longest, come first.
template <int D, int KIND, bool SIXTEENS>
__global__ __launch_bounds__(256, 2) void paged8_mixed_kernel(RaggedParams p, Scales8 scales, Few8 few, unsigned tile_x, unsigned tile_wgs)
{
    FDX_TILE8_LDS(D, lds);
    __shared__ __attribute__((aligned(16))) unsigned char q[2 * D / 32 * 2 * 1024];
    if (blockIdx.x < tile_wgs) {
        tile8_body<D, KIND, true, SIXTEENS>(p, scales, Place { blockIdx.x % tile_x, blockIdx.x / tile_x, tile_x }, lds);
    } else {
        static_assert(16 * (D + 4) * sizeof(float) <= sizeof(lds_ks0) && 16 * (D + 4) * sizeof(float) <= sizeof(lds_vs0)
                && (2 * 4 * 16 + 5 * 64) * sizeof(float) <= sizeof(lds_rows_of), "fits into the tiles' LDS");
        int* rest = lds.rows_of;
        few8_body<D, KIND, true>(p, scales, few, blockIdx.x - tile_wgs,
            Meet8 { reinterpret_cast<float*>(lds.ks0), reinterpret_cast<float*>(lds.ks1), reinterpret_cast<float*>(lds.vs0), reinterpret_cast<float*>(lds.vs1),
                reinterpret_cast<float*>(rest), reinterpret_cast<int (*)[64]>(rest + 2 * 4 * 16), q });
    }
}

// Rows whose keys more than one share, or range, has: sum of 2^(m - M) l o over them, divided by that of 2^(m - M) l.  Eight parts of a head are on
// their way together.  Where there are many rows a wave takes four heads of a row, for which it finds the row's sequence once; where there are few, the four
// waves of a workgroup every fourth part of one head, and their sums meet.  The whole call in us,
// a wave for four heads / a workgroup for each: 32 rows of 64 parts 82.9 / 55.9, of 32 parts 31.1 / 16.5, 192 rows of up to 4 25.8 / 21.5, 1536 of tiles 24.6 /
// 25.8, 2048 of two or three 92.9 / 92.9, 4096 of tiles 35.7 / 41.8.
template <int H>
struct RowSums {
    float top[H], l[H], o0[H], o1[H]; // means of depths lane and 64 + lane
};
// parts first, first + step, ... of H heads
template <int H, class Out, class Size>
__device__ __forceinline__ void sum_parts(const RaggedParams& p, int first, int step, int parts, const Out& out, const Size& size, RowSums<H>& r)
{
    constexpr int W = 8;
    const int lane = threadIdx.x & 63, mine = parts > first ? (parts - first + step - 1) / step : 0;
    auto part = [&](int i) { return first + i * step; };
    float m[H];
#pragma unroll
    for (int h = 0; h < H; ++h) {
        r.top[h] = -INFINITY;
        r.l[h] = r.o0[h] = r.o1[h] = 0.f;
    }
    for (int i0 = 0; i0 < mine; i0 += 64)
#pragma unroll
        for (int h = 0; h < H; ++h)
            if (i0 + lane < mine)
                r.top[h] = fmaxf(r.top[h], size(part(i0 + lane), h)[0]);
#pragma unroll
    for (int h = 0; h < H; ++h) {
        r.top[h] = wave_all<true>(r.top[h]);
        m[h] = r.top[h] == -INFINITY ? 0.f : r.top[h];
    }
    const int d0 = lane < p.dv ? lane : 0, d1 = 64 + lane < p.dv ? 64 + lane : 0;
    auto weight = [&](int i, int h) {
        const float* at = size(part(i), h);
        return at[1] * __builtin_amdgcn_exp2f(at[0] - m[h]);
    };
    for (int i0 = 0; i0 < mine; i0 += 64)
#pragma unroll
        for (int h = 0; h < H; ++h)
            r.l[h] += wave_all<false>(i0 + lane < mine ? weight(i0 + lane, h) : 0.f);
    for (int i0 = 0; i0 < mine; i0 += 64) {
        float w[H]; // parts of the whole: what they multiply may be near fp32's end
#pragma unroll
        for (int h = 0; h < H; ++h)
            w[h] = i0 + lane < mine && r.l[h] != 0.f ? weight(i0 + lane, h) / r.l[h] : 0.f;
        const int count = mine - i0 < 64 ? mine - i0 : 64;
        for (int i = 0; i < count; i += W) {
            float x0[H][W], x1[H][W];
#pragma unroll
            for (int z = 0; z < W; ++z)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const float* from = out(part(i0 + (i + z < count ? i + z : i)), h);
                    x0[h][z] = from[d0];
                    x1[h][z] = from[d1];
                }
#pragma unroll
            for (int z = 0; z < W; ++z)
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w[h]), i + z < count ? i + z : i));
                    r.o0[h] = fmaf(i + z < count ? wi : 0.f, x0[h][z], r.o0[h]);
                    r.o1[h] = fmaf(i + z < count ? wi : 0.f, x1[h][z], r.o1[h]);
                }
        }
    }
}
__device__ __forceinline__ void store_row(const RaggedParams& p, int row, int head, float top, float l, float o0, float o1)
{
    const int lane = threadIdx.x & 63;
    float* to = p.out + (int64_t)row * p.ldo + (int64_t)head * p.dv;
    const float none = top != -INFINITY ? NAN : 0.f; // as finish() has it
    if (lane < p.dv)
        to[lane] = l == 0.f ? none : o0;
    if (64 + lane < p.dv)
        to[64 + lane] = l == 0.f ? none : o1;
}

template <bool FEW>
__global__ __launch_bounds__(256) void paged8_join_kernel(RaggedParams p, Few8 few)
{
    constexpr int H = FEW ? 1 : 4;
    __shared__ float met[FEW ? 4 : 1][4][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const unsigned groups = (unsigned)(p.heads + H - 1) / H, item = FEW ? blockIdx.x : blockIdx.x * 4 + wave;
    const int row = (int)(item / groups), head0 = (int)(item % groups) * H;
    if (row >= p.tokens)
        return;
    const int index = find_row(SearchWave(), p.starts, p.n_seqs, p.tokens, row);
    if (index < 0)
        return;
    const Sequence s = sequence_of<kPagedF32>(p, index, packed_span(p.starts, index, p.tokens));
    const int token = row - s.span.first;
    if (token >= s.span.count)
        return;
    auto head_of = [&](int h) { return head0 + h < p.heads ? head0 + h : p.heads - 1; };
    RowSums<H> r;
    if (!s.few) {
        const int visible = visible_keys(p, s, token);
        if (visible <= s.range)
            return;
        const int64_t first = (int64_t)row * p.heads; // part_row
        sum_parts<H>(p, FEW ? wave : 0, FEW ? 4 : 1, (visible + s.range - 1) / s.range, [&](int i, int h) { return p.tile.out(i, first + head_of(h), p.dv); },
            [&](int i, int h) { return p.tile.size(i, first + head_of(h), p.dv); }, r);
    } else {
        if (few.shares <= 1) // no sequence is shared, and nothing is kept of where they begin
            return;
        const int2 split = few.split[index];
        const int from = split.x, parts = split.y;
        if (parts == 1)
            return;
        auto id = [&](int i, int h) {
            const int head = head_of(h), kv_head = quotient(head, p.by_group);
            return few.row_of(from + i, kv_head, i > 0 ? 0 : 1, token * p.group + head - kv_head * p.group);
        };
        sum_parts<H>(p, FEW ? wave : 0, FEW ? 4 : 1, parts, [&](int i, int h) { return few.out(id(i, h), p.dv); },
            [&](int i, int h) { return few.size(id(i, h), p.dv); }, r);
    }
    if constexpr (FEW) {
        met[wave][0][lane] = r.top[0];
        met[wave][1][lane] = r.l[0];
        met[wave][2][lane] = r.o0[0];
        met[wave][3][lane] = r.o1[0];
        __syncthreads();
        if (wave > 0)
            return;
        const float top = fmaxf(fmaxf(met[0][0][lane], met[1][0][lane]), fmaxf(met[2][0][lane], met[3][0][lane])), m = top == -INFINITY ? 0.f : top;
        float l = 0.f, f[4], o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f[w] = __builtin_amdgcn_exp2f(met[w][0][lane] - m) * met[w][1][lane];
            l += f[w];
        }
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            o0 = fmaf(f[w] / l, met[w][2][lane], o0);
            o1 = fmaf(f[w] / l, met[w][3][lane], o1);
        }
        store_row(p, row, head0, top, l, o0, o1);
    } else {
#pragma unroll
        for (int h = 0; h < H; ++h)
            if (head0 + h < p.heads)
                store_row(p, row, head0 + h, r.top[h], r.l[h], r.o0[h], r.o1[h]);
    }
}

// How a call is cut: paged_plan's tiles; sequences with few rows in as many shares as workgroups fit on the GPU, or as the longest lengths make.
struct Plan8 {
    RaggedPlan tiles;
    Few8 few;
    unsigned few_wgs;
    size_t split_at, few_floats; // where Few8::split is, what all has, in floats
};
static Plan8 plan8(int tokens, int max_new, int heads, const fdx_kv_pages* c)
{
    Plan8 r {};
    r.tiles = paged_plan(tokens, max_new, heads, c);
    if (r.tiles.few_ranges > 0) {
        const int64_t most = (int64_t)c->n_seqs * (((int64_t)c->max_len + 31) / 32), shares = most <= kWhole ? 1 : (most + kLeastShare - 1) / kLeastShare;
        // us with as many as fit, two workgroups a CU or three / with others: 64 of 4000, 32 / 8 heads of 128, 512 118, 768 156; 64 of 100 to 8000, 12 heads of
        // 64, 768 90, 512 and 1024 102
        const int fit = (c->dk <= 64 && c->dv <= 64 ? 768 : 512) / c->kv_heads;
        r.few.shares = fit < 1 ? 1 : (shares < fit ? (int)shares : fit);
        r.few.rows = (int)(r.tiles.few_part / ((int64_t)c->n_seqs * c->kv_heads));
        r.few.unit = 1;
        while (most / r.few.unit + c->n_seqs >= ((int64_t)1 << 30))
            r.few.unit *= 2;
        r.few.kv_heads = c->kv_heads;
        r.few_wgs = (unsigned)(r.few.shares * c->kv_heads);
        if (r.few.shares > 1) {
            r.split_at = ((size_t)r.few_wgs * 2 * r.few.rows * (2 + (size_t)c->dv) + 3) & ~(size_t)3;
            r.few_floats = r.split_at + (((size_t)c->n_seqs * 2 + 3) & ~(size_t)3);
        }
    }
    return r;
}

constexpr int64_t kFewJoins = 1024; // rows that are joined by a workgroup each

template <int D, int KIND>
static void paged8_launch(const RaggedParams& p, const Plan8& plan, const Scales8& scales)
{
    // codes of a row and head are whole 16-byte vectors, those of q and out whole float4; rows start below 2^32 times 16 bytes.  Where one is not so,
    // codes are read byte by byte: 64 sequences of 4000 keys, 16 / 8 heads, 783 us at depth 100, 143 at 112.
    const uintptr_t all = reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.k)
        | reinterpret_cast<uintptr_t>(p.v);
    const int64_t rows = (int64_t)p.n_pages * p.page_size.by, ld = p.ldk > p.ldv ? p.ldk : p.ldv;
    const bool wide = (all & 15) == 0 && ((p.ldq | p.ldo) & 3) == 0 && ((p.dk | p.dv) & 15) == 0 && rows * (ld >> 4) < ((int64_t)1 << 32);
    const unsigned tile_x = (unsigned)plan.tiles.tiles, tile_y = (unsigned)(plan.tiles.tile_ranges > 0 ? plan.tiles.tile_ranges : 1);
    const uint64_t tile_wgs = (uint64_t)tile_x * tile_y, all_wgs = tile_wgs + plan.few_wgs;
    // Blocks of whole sixteens (ranges start at multiples of 64): two multiplications less a score.  us without / with, 128 new tokens of 1000, 12 heads of
    // 64: 25.8 / 23.5; two of 2000 of 3000, 16 / 4 heads of 64, 124.2 / 117.8; four of 1000 of 3000, 32 / 8 heads of 128, 379.8 / 370.8.
    const bool sixteens = scales.block.by % 16 == 0;
    if (wide && tile_wgs > 0 && plan.few_wgs > 0 && all_wgs < (1u << 23)) {
        if (sixteens)
            hipLaunchKernelGGL((paged8_mixed_kernel<D, KIND, true>), dim3((unsigned)all_wgs), dim3(256), 0, stream(), p, scales, plan.few, tile_x, (unsigned)tile_wgs);
        else
            hipLaunchKernelGGL((paged8_mixed_kernel<D, KIND, false>), dim3((unsigned)all_wgs), dim3(256), 0, stream(), p, scales, plan.few, tile_x, (unsigned)tile_wgs);
    } else {
        if (plan.few_wgs > 0) {
            if (wide)
                hipLaunchKernelGGL((paged8_few_kernel<D, KIND, true>), dim3(plan.few_wgs), dim3(256), 0, stream(), p, scales, plan.few);
            else
                hipLaunchKernelGGL((paged8_few_kernel<D, KIND, false>), dim3(plan.few_wgs), dim3(256), 0, stream(), p, scales, plan.few);
        }
        if (tile_wgs > 0) {
            const dim3 grid(tile_x, tile_y);
            if (wide && sixteens)
                hipLaunchKernelGGL((paged8_tile_kernel<D, KIND, true, true>), grid, dim3(256), 0, stream(), p, scales);
            else if (wide)
                hipLaunchKernelGGL((paged8_tile_kernel<D, KIND, true, false>), grid, dim3(256), 0, stream(), p, scales);
            else
                hipLaunchKernelGGL((paged8_tile_kernel<D, KIND, false, false>), grid, dim3(256), 0, stream(), p, scales);
        }
    }
    if (plan.few.shares > 1 || tile_y > 1) {
        const int64_t joined = (int64_t)p.tokens * p.heads, groups = (int64_t)p.tokens * ((p.heads + 3) / 4);
        if (joined <= kFewJoins)
            hipLaunchKernelGGL(paged8_join_kernel<true>, dim3((unsigned)joined), dim3(256), 0, stream(), p, plan.few);
        else
            hipLaunchKernelGGL(paged8_join_kernel<false>, dim3((unsigned)((groups + 3) / 4)), dim3(256), 0, stream(), p, plan.few);
    }
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_mha_paged8_scratch_bytes(int tokens, int max_new, int heads, const fdx_kv_pages8* cache)
{
    const fdx_kv_pages* c = cache ? &cache->pages : nullptr;
    if (!c || tokens <= 0 || max_new <= 0 || heads <= 0 || c->kv_heads <= 0 || heads % c->kv_heads != 0 || c->dk <= 0 || c->dv <= 0 || c->n_seqs <= 0
        || c->max_len <= 0)
        return 0;
    // what the call refuses has no plan, whose numbers would leave their types
    if ((int64_t)tokens * heads > (1 << 25) || (int64_t)c->n_seqs * c->kv_heads > (1 << 22) || c->max_len > (1 << 30) || c->dk > 128 || c->dv > 128)
        return 0;
    const Plan8 plan = plan8(tokens, max_new, heads, c);
    return sizeof(float) * (plan.few_floats + plan.tiles.tile_floats(c->dv));
}

extern "C" fdx_status fdx_mha_paged8_f32(const float* q, int64_t ldq, const int32_t* starts, int tokens, int max_new, int heads,
    const fdx_kv_pages8* cache, float* out, int64_t ldo, void* scratch_dev, int* error_flag_dev)
{
    fdx_status st = check_kv_pages8("mha_paged8", cache);
    if (st != FDX_OK)
        return st;
    const fdx_kv_pages& c = cache->pages;
    RaggedParams p {};
    st = paged_params("mha_paged8", q, ldq, starts, tokens, max_new, heads, &c, out, ldo, scratch_dev,
        fdx_mha_paged8_scratch_bytes(tokens, max_new, heads, cache), error_flag_dev, p);
    if (st != FDX_OK)
        return st;
    Plan8 plan = plan8(tokens, max_new, heads, &c);
    plan.few.parts = static_cast<float*>(scratch_dev);
    plan.few.split = plan.few.shares > 1 ? reinterpret_cast<int2*>(plan.few.parts + plan.split_at) : nullptr;
    p.few_rows = plan.tiles.few_rows;
    p.few = { nullptr, 0, 1, INT_MAX, 0, 0 }; // no ranges: sequences with few rows are cut in shares
    p.tile = { plan.few.parts + plan.few_floats, plan.tiles.tile_part, plan.tiles.tile_ranges, plan.tiles.tile_keys, plan.tiles.tile_whole, 0 };
    const Scales8 scales { cache->k_scale, cache->v_scale, make_divisor(cache->block) };
    const bool small = p.dk <= 64 && p.dv <= 64;
    profile_begin();
    if (c.type == FDX_KV_I8)
        small ? paged8_launch<64, kI8>(p, plan, scales) : paged8_launch<128, kI8>(p, plan, scales);
    else
        small ? paged8_launch<64, kE4M3>(p, plan, scales) : paged8_launch<128, kE4M3>(p, plan, scales);
    profile_end("mha_paged8_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
