// Attention over packed prompts and over paged caches (gfx950), query heads in groups that share a key / value head.
//
//   O = softmax(Q K^T / sqrt(dk)) V a sequence, in one pass over the keys with the running maximum m and sum l of each row:
//   m' = max(m, max s), l' = l 2^(m - m') + sum 2^(s - m'), o' = o 2^(m - m') + sum 2^(s - m') v; out = o / l, s in units of log2.
// Three forms: tiles of 128 rows, split as they are fetched (any batch); the same on tiles that a pass of its own has split (long
// packed prompts); up to 32 rows straight from memory (decode steps).
#include <cfloat>
#include <climits>

#include "bf16_split.hpp"
#include "f16_split.hpp"
#include "ragged_attn.hpp"

namespace fdx {

fdx_status check_kv_pages(const char* who, const fdx_kv_pages* c); // kv_append.hip

// a row by plain sums, into its place
template <int KIND>
__device__ __forceinline__ void store_plain_row(const RaggedParams& p, const Sequence& s, int token, int head, int kv_head, int range, int lane)
{
    const int visible = visible_keys(p, s, token);
    const bool in_parts = visible > s.range;
    const int first = in_parts ? range * s.range : 0;
    if (in_parts ? first >= visible : range > 0)
        return;
    const int last = in_parts && visible - first > s.range ? first + s.range : visible;
    const int64_t row = s.span.first + token;
    float m, l, o[2];
    bool seen, missing;
    plain_row<KIND>(p, s, p.q + row * p.ldq + (int64_t)head * p.dk, kv_head, first, last, m, l, o, seen, missing);
    raise_flag(p, missing);
    float* to = p.out + row * p.ldo + (int64_t)head * p.dv;
    if (in_parts) {
        const PartSums& part = s.few ? p.few : p.tile;
        const int64_t id = part_row(p, s, token, head);
        to = part.out(range, id, p.dv);
        if (lane == 0) {
            float* at = part.size(range, id, p.dv);
            at[0] = seen && m == -INFINITY ? -FLT_MAX : m;
            at[1] = l;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (64 * i + lane < p.dv)
            to[64 * i + lane] = finish(o[i], l, seen && !in_parts);
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
//  * N = D / 16 threads fetch a key's row of either: block N g + l of eight depths holds the 16-byte chunks 2 N g + l and 2 N g + N + l of it,
//    which lane l of the N has.  Keys lie as [plane][depth block][key][16 bytes], which the first product reads as it is; values as
//    [plane][key][depth], and the transposing LDS read gives the second product four keys of a depth at a time.
//  * A query row, a tile's keys and its values are each brought to fp16's range by a power of two.  The sums have the power of the last
//    tile's values that are not all zeros, which changes with one that is another multiple of four.  A tile whose rows are too far apart in
//    size for one power (spread_fits; a row of 10^30 behind the mask) is left to plain sums.
//  * The maximum that a row's exponentials refer to moves only when a score passes it by 2^4, so sums are rescaled a few times a row
//    instead of every tile; exponentials carry 2^10 to stay clear of fp16's small end, at most 2^14.
//  * Bound by the vector units, which split, and the matrix units, whose times still add up for the most part: four sequences that bring 1000
//    tokens to 3000 keys in fp32 pages, 32 / 8 heads of 128, 887 us or 258 TFLOP/s, where three products for one come to 364 at the rate of a
//    large fp16 product; vector instructions 55 % of a busy CU's time, matrix instructions 40 %, LDS 10 %, two waves a SIMD.  64 keys take a
//    workgroup 1.9 us alone on its CU at depth 64.
//  * Rows whose sums are not finite (infinite or NaN operands, whether the row sees them or not, and tiles left out above) or empty though they
//    see keys are taken again by plain_row.
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

// a workgroup's row: its token, the row of q and out, its head (rows behind the last one: the last one's)
struct QueryRow {
    int token, head;
    int64_t row;
};
__device__ __forceinline__ QueryRow row_of(const RaggedParams& p, const Sequence& s, int kv_head, int count, int r)
{
    const int at = r < count ? r : count - 1, token = quotient(at, p.by_group);
    return { token, kv_head * p.group + at - token * p.group, (int64_t)s.span.first + token };
}

constexpr float kShift = 10.f; // exponentials are 2^kShift times the probability's numerator

// where a workgroup stands in its launch
struct Place {
    unsigned x, y, nx;
};

template <int D, int KIND>
struct TileSizes {
    static constexpr int KT = 4096 / D, N = D / 16; // keys of a tile; threads that fetch a key
    static constexpr int KBLK = KT * 16 + 32, VROW = D * 2 + 32; // bytes of a block of keys, of a row of values, offset against each other
    static constexpr int kKeys = 2 * (D / 8) * KBLK, kValues = 2 * KT * VROW; // bytes of a tile
    static constexpr int kAhead = 512; // places of two halves of as many positions are looked up ahead, all threads at once
    static constexpr int kPlaces = KIND == kPackedF32 ? 1 : 2 * kAhead;
};
// its LDS: two tiles, apart so that the compiler sees that what is written is not what is read
struct TileLds {
    unsigned char *ks0, *ks1, *vs0, *vs1;
    Spread (*spread)[4];
    int *rows_of, *some_absent;
};
#define FDX_TILE_LDS(D, KIND, lds)                                                                                          \
    __shared__ __attribute__((aligned(16))) unsigned char lds##_ks0[TileSizes<D, KIND>::kKeys], lds##_ks1[TileSizes<D, KIND>::kKeys]; \
    __shared__ __attribute__((aligned(16))) unsigned char lds##_vs0[TileSizes<D, KIND>::kValues], lds##_vs1[TileSizes<D, KIND>::kValues]; \
    __shared__ Spread lds##_spread[2][4];                                                                                   \
    __shared__ int lds##_rows_of[TileSizes<D, KIND>::kPlaces];                                                              \
    __shared__ int lds##_absent;                                                                                            \
    const TileLds lds { lds##_ks0, lds##_ks1, lds##_vs0, lds##_vs1, lds##_spread, lds##_rows_of, &lds##_absent }

template <int D, int KIND, bool EXACT>
__device__ __forceinline__ void tile_body(const RaggedParams& p, const Place& place_in, const TileLds& lds)
{
    typedef typename KvElement<KIND>::type T;
    typedef TileSizes<D, KIND> S;
    constexpr int KT = S::KT, HALVES = KT / 32, N = S::N, KB = D / 8, STEPS = D / 16, DB = D / 32, KBLK = S::KBLK, VROW = S::VROW, kAhead = S::kAhead;
    constexpr bool kPaged = KIND != kPackedF32;
    unsigned char *ks0 = lds.ks0, *ks1 = lds.ks1, *vs0 = lds.vs0, *vs1 = lds.vs1;
    Spread (*spread)[4] = lds.spread;
    int* rows_of = lds.rows_of;
    int& some_absent = *lds.some_absent;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, half = lane >> 5;
    if (p.error_flag && place_in.x == 0 && place_in.y == 0)
        for (int i = tid; i < p.n_seqs; i += 256) // lengths too: a sequence without new tokens has no tile
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens) || (kPaged && (p.lens[i] < 0 || p.lens[i] > p.max_len)));
    // key heads next to each other: consecutive workgroups go to the eight XCDs in turn, so that an XCD's cache holds few heads'
    // keys; later tiles of a sequence, which see more keys, first
    const int kv_head = place_in.x % p.kv_heads;
    const int64_t number = place_in.x / p.kv_heads;
    const Tile tile = p.causal && p.n_seqs <= 64 ? late_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, p.group, 128, number)
                                                 : find_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, p.group, 128, place_in.nx / p.kv_heads - 1 - number);
    if (tile.seq < 0)
        return;
    const Sequence s = sequence_of<KIND>(p, tile.seq, tile.span);
    if (tid == 0)
        raise_flag(p, s.cut);
    const int count = s.span.count * p.group; // rows
    const int r_first = tile.index * 128;
    if (r_first >= count || (KIND != kPackedF32 && s.few))
        return;
    const int visible = visible_keys(p, s, row_of(p, s, kv_head, count, r_first + wave * 32 + c).token);

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

    // the query: depth block 2 u + half
    f16x8 qh[STEPS], ql[STEPS];
    float q_down;
    {
        float x[STEPS][8], top = 0.f;
        const QueryRow at = row_of(p, s, kv_head, count, r_first + wave * 32 + c);
        const float* from = p.q + at.row * p.ldq + (int64_t)at.head * p.dk;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int blk = 2 * u + half, d0 = 8 * N * (blk / N) + 4 * (blk % N);
            load_depths<float, 4, EXACT>(from, d0, p.dk, p.wide, x[u]);
            load_depths<float, 4, EXACT>(from, d0 + 4 * N, p.dk, p.wide, x[u] + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                top = fmaxf(top, fabsf(x[u][e]));
        }
        const Pow2 sq = pow2_for<1>(exponent(max_halves(top)));
        q_down = sq.down * (p.scale * kLog2e);
#pragma unroll
        for (int u = 0; u < STEPS; ++u)
            split2x8(x[u], sq.up, qh[u], ql[u]);
    }

    const T* kbase = static_cast<const T*>(p.k) + (int64_t)kv_head * p.dk;
    const T* vbase = static_cast<const T*>(p.v) + (int64_t)kv_head * p.dv;
    const int krow = tid / N, kl = tid % N;
    float kst[2][8], vst[2][8];
    // positions behind the range repeat its last one: masked, and as finite as it is
    auto place = [&](int t, int key) -> int64_t {
        if constexpr (kPaged) {
            const int row = rows_of[(t * KT + key) & (2 * kAhead - 1)];
            return row < 0 ? 0 : row;
        } else {
            const int at = k_first + t * KT + key;
            return s.span.first + (at < k_end ? at : k_end - 1);
        }
    };
    auto look_up = [&](int first) { // places of positions first .. first + kAhead - 1 of the range
#pragma unroll
        for (int i = 0; i < kAhead; i += 256) {
            const int at = k_first + first + i + tid;
            const int row = key_row<KIND>(p, s, at < k_end ? at : k_end - 1);
            rows_of[(first + i + tid) & (2 * kAhead - 1)] = row;
            if (row < 0) {
                some_absent = 1;
                raise_flag(p, true);
            }
        }
    };
    auto fetch = [&](int t) {
        const int64_t row = place(t, krow);
        const T *kr = kbase + row * p.ldk, *vr = vbase + row * p.ldv;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            load_depths<T, 4, EXACT>(kr, 4 * N * i + 4 * kl, p.dk, p.wide, kst[i >> 1] + 4 * (i & 1));
            load_depths<T, 4, EXACT>(vr, 4 * N * i + 4 * kl, p.dv, p.wide, vst[i >> 1] + 4 * (i & 1));
        }
    };
    // A turn is shorter than a trip to memory under load: the tile behind the next fetch is brought to the cache, an element of each
    // thread's part of a row (its chunks lie within 64 N bytes), looked at a turn later.
    float asked[2] = { 0.f, 0.f };
    auto ask = [&](int t) {
        asm volatile("" ::"v"(asked[0]), "v"(asked[1]));
        const int64_t row = place(t, krow);
        const int d = 16 * kl; // 16 elements apart
        asked[0] = (float)kbase[row * p.ldk + (EXACT || d < p.dk ? d : 0)];
        asked[1] = (float)vbase[row * p.ldv + (EXACT || d < p.dv ? d : 0)];
    };
    auto measure = [&](int t) { // sizes of the fetched rows, infinities and NaN aside
        float km = 0.f, vm = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            km = max3(km, fabsf(kst[0][e]), fabsf(kst[1][e]));
            vm = max3(vm, fabsf(vst[0][e]), fabsf(vst[1][e]));
        }
        if (__builtin_expect(__any(!(km < INFINITY && vm < INFINITY)), 0)) { // rows that do not see the infinity keep their sums
            km = vm = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    km = fmaxf(km, fabsf(kst[g][e]) < INFINITY ? fabsf(kst[g][e]) : 0.f);
                    vm = fmaxf(vm, fabsf(vst[g][e]) < INFINITY ? fabsf(vst[g][e]) : 0.f);
                }
        }
        km = fmaxf(km, dpp_move<0xB1>(km));
        km = fmaxf(km, dpp_move<0x4E>(km));
        vm = fmaxf(vm, dpp_move<0xB1>(vm));
        vm = fmaxf(vm, dpp_move<0x4E>(vm));
        if (N == 8) {
            km = fmaxf(km, dpp_move<0x141>(km));
            vm = fmaxf(vm, dpp_move<0x141>(vm));
        }
        Spread r = row_spread(km, vm);
        r.top = most_of_wave<N>(r.top);
        r.low = most_of_wave<N>(r.low);
        if (lane == 0)
            spread[t & 1][wave] = r;
    };
    auto mfma = [](f16x8 a, f16x8 b, const f32x16& acc) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, acc, 0, 0, 0); };
    constexpr f32x16 kZero = { 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f };

    f32x16 oacc[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
        oacc[d] = kZero;
    float m_run = -INFINITY, l_run = 0.f;
    // of the tile at work and of the one behind it
    Pow2 sk = pow2_for<1>(0), sk_next = sk, sv_next = pow2_for<4>(0);
    float v_down = 0.f; // of the sums; 0 while all values were zeros
    bool fits = true, fits_next = true;
    auto scale_next = [&](int t) {
        const Spread* r = spread[t & 1];
        const u16x2 top = most(most(r[0].top, r[1].top), most(r[2].top, r[3].top)), low = most(most(r[0].low, r[1].low), most(r[2].low, r[3].low));
        fits_next = spread_fits(top, low);
        sk_next = pow2_for<1>(top[0]);
        sv_next = pow2_for<4>(top[1]);
        sv_next.down = low[1] == 0 ? 0.f : sv_next.down; // values that are all zeros take any power
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
        for (int g = 0; g < 2; ++g) {
            f16x8 h, l;
            split2x8(vst[g], sv_next.up, h, l);
            *reinterpret_cast<f16x8*>(&vs[krow * VROW + (N * g + kl) * 16]) = h;
            *reinterpret_cast<f16x8*>(&vs[(KT + krow) * VROW + (N * g + kl) * 16]) = l;
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
    auto turn = [&](int t, const unsigned char* ks, const unsigned char* vs, unsigned char* ks_next, unsigned char* vs_next) {
        const int j0 = k_first + t * KT;
        const bool work = j0 < wave_any; // some row of this wave sees some key of the tile
        const float f = sv_next.up * v_down, down = sv_next.down;
        sk = sk_next;
        fits = fits_next;
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
        int absent = 0;
        if constexpr (kPaged) {
            absent = some_absent;
            if ((t * KT & (kAhead - 1)) == 0 && t > 0 && (t + kAhead / KT) < tiles)
                look_up(t * KT + kAhead); // into the half that is done with
        }
        if (t + 2 < tiles) {
            fetch(t + 2);
            if (kPaged && t + 3 < tiles)
                ask(t + 3);
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
            if (kPaged && __builtin_amdgcn_readfirstlane(absent)) {
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (rows_of[(t * KT + kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3)) & (2 * kAhead - 1)] < 0)
                            sacc[kb][e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                for (int e = 0; e < 16; e += 2)
                    mx = max3(mx, sacc[kb][e], sacc[kb][e + 1]);
            mx = max_halves(mx);
            const float step = q_down * sk.down, to_log2 = fmaxf(step, 1.17549435e-38f); // above zero: -infinity stays what it is
            mx *= to_log2;
            l_run = fits && step < INFINITY ? l_run : NAN; // an infinite step makes every negative score -infinity
            if (__any(mx > m_run + 4.f) || f != 1.f) {
                const float m_new = mx > m_run + 4.f ? mx : m_run;
                const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
                // NAN: sums that would leave fp32's range
                const float by = down == 0.f || v_down == 0.f ? corr : (f > 1e-18f && f < 1e18f ? corr * f : NAN);
                v_down = down == 0.f ? v_down : down;
                m_run = m_new;
                l_run *= corr;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        oacc[d][e] *= by;
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
                    const f16x8 vh = values(vs, 16 * u, d), vl = values(vs, KT + 16 * u, d);
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
            if (tid == 0)
                some_absent = 0;
            __syncthreads();
            look_up(0);
            if (tiles > kAhead / KT)
                look_up(kAhead);
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
    }
    for (int t = 0; t < tiles; t += 2) {
        turn(t, ks0, vs0, ks1, vs1);
        if (t + 1 < tiles)
            turn(t + 1, ks1, vs1, ks0, vs0);
    }

    int again = r_first + wave * 32 + c; // found out once more, so that no registers hold it during the loop
    asm volatile("" : "+v"(again));
    const bool q_ok = again < count;
    const QueryRow at_row = row_of(p, s, kv_head, count, again);
    const int64_t q_row = at_row.row;
    const int head = at_row.head;
    l_run += __shfl_xor(l_run, 32, 64);
    float size = l_run;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            size += fabsf(oacc[d][e]);
    // a row's two lanes hold half of its depths each; a row that sees keys and has no sum (scores of -infinity, or pages that are not there)
    // is plain_row's to tell apart
    const uint64_t odd_lanes = __ballot(q_ok && (!(size < INFINITY) || (l_run == 0.f && k_first < visible)));
    uint32_t odd = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    const bool in_parts = visible > s.range;
    if (q_ok && !(odd >> c & 1) && (in_parts ? k_first < visible : place_in.y == 0)) {
        const float f = l_run > 0.f ? v_down / l_run : 0.f; // no key: zeros
        float* to = p.out + q_row * p.ldo + (int64_t)head * p.dv;
        if (in_parts) {
            const int64_t id = part_row(p, s, at_row.token, head);
            to = p.tile.out(place_in.y, id, p.dv);
            float* at = p.tile.size(place_in.y, id, p.dv);
            if (half == 0) {
                at[0] = m_run - kShift;
                at[1] = l_run;
            }
        }
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int blk = 4 * d + g, depth = 8 * N * (blk / N) + 4 * N * half + 4 * (blk % N); // what columns 8 blk + 4 half hold
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
        const int t1 = quotient(r1, p.by_group), h1 = kv_head * p.group + r1 - t1 * p.group;
        store_plain_row<KIND>(p, s, t1, h1, kv_head, place_in.y, lane);
    }
}

template <int D, int KIND, bool EXACT>
__global__ __launch_bounds__(256, 2) void ragged_tile_kernel(RaggedParams p)
{
    FDX_TILE_LDS(D, KIND, lds);
    tile_body<D, KIND, EXACT>(p, Place { blockIdx.x, blockIdx.y, gridDim.x }, lds);
}

// ---- packed prompts: keys and values split once, in tiles as the products read them ----
//
// In ragged_tile_kernel the vector units are busier than the matrix units: a third of a wave's issue slots go into splitting keys and
// values, which every workgroup does again for its 128 rows.  Where sequences are long enough to
// fill tiles, ragged_ready_kernel splits them once, into the order that LDS holds: [tile][key head][keys, then values][plane][block][key or
// depth][16 bytes], 16 KB each (as many bytes as fp32), with the powers of two beside them.  ragged_packed_kernel's loads then go from memory to
// LDS past the registers, and the registers hold two tiles' scores: the first product of tile t + 1 runs beside the softmax of tile t.
// Prompts of 8192 and 4001 rows, 32 / 8 heads of 128, causal: 2.02 ms (382 TFLOP/s) on one card and 2.17 (355) on another, bound by the
// matrix units at the clock that the power limit leaves; the pass that splits is 0.04 of it.
__device__ __forceinline__ int64_t ready_tile(const RaggedParams& p, int seq, int first, int keys_a_tile) { return first_tile(first, seq, 1, keys_a_tile); }

template <int D, bool EXACT>
__global__ __launch_bounds__(256) void ragged_ready_kernel(RaggedParams p)
{
    constexpr int KT = 4096 / D, N = D / 16, KB = D / 8, VB = KT / 8;
    __shared__ __attribute__((aligned(16))) unsigned char out[32768];
    __shared__ Spread spread[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kv_head = blockIdx.x % p.kv_heads;
    const int64_t number = blockIdx.x / p.kv_heads;
    const Tile tile = find_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, 1, KT, number);
    if (tile.seq < 0)
        return;
    const int krow = tid / N, kl = tid % N, vblk = tid / (D / 2), vd = tid % (D / 2) * 2;
    const int left = tile.span.count - tile.index * KT; // keys behind the sequence's last are zeros
    const int64_t row = tile.span.first + tile.index * KT;
    const float* kr = static_cast<const float*>(p.k) + (row + (krow < left ? krow : 0)) * p.ldk + (int64_t)kv_head * p.dk;
    const float* vr = static_cast<const float*>(p.v) + row * p.ldv + (int64_t)kv_head * p.dv;
    float k[2][8], v[2][8];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        load_depths<float, 4, EXACT>(kr, 8 * N * g + 4 * kl, p.dk, p.wide, k[g]);
        load_depths<float, 4, EXACT>(kr, 8 * N * g + 4 * N + 4 * kl, p.dk, p.wide, k[g] + 4);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int key = 16 * (vblk >> 1) + 4 * (vblk & 1) + 8 * (j >> 2) + (j & 3);
        float x[2];
        load_depths<float, 2, EXACT>(vr + (key < left ? key : 0) * p.ldv, vd, p.dv, p.wide, x);
        v[0][j] = key < left ? x[0] : 0.f;
        v[1][j] = key < left ? x[1] : 0.f;
    }
    // sizes of the rows, infinities and NaN aside: queries that do not see those keep their sums
    float km = 0.f, vm[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            k[g][e] = krow < left ? k[g][e] : 0.f;
            km = fmaxf(km, fabsf(k[g][e]) < INFINITY ? fabsf(k[g][e]) : 0.f);
        }
        const float a = fabsf(v[0][e]), b = fabsf(v[1][e]);
        vm[e] = fmaxf(a < INFINITY ? a : 0.f, b < INFINITY ? b : 0.f);
    }
    km = N == 4 ? fmaxf(km, dpp_move<0xB1>(km)) : half_row_all<true>(km);
    km = N == 4 ? fmaxf(km, dpp_move<0x4E>(km)) : km;
    Spread r { u16x2 { 0, 0 }, u16x2 { 0, 0 } };
#pragma unroll
    for (int e = 0; e < 8; ++e) { // D / 2 lanes have a row of values
        vm[e] = fmaxf(half_row_all<true>(vm[e]), dpp_move<0x140>(half_row_all<true>(vm[e])));
        vm[e] = fmaxf(vm[e], __shfl_xor(vm[e], 16, 64));
        if (D == 128)
            vm[e] = fmaxf(vm[e], __shfl_xor(vm[e], 32, 64));
        const Spread one = row_spread(km, vm[e]);
        r.top = most(r.top, one.top);
        r.low = most(r.low, one.low);
    }
    r.top = most_of_wave<N>(r.top);
    r.low = most_of_wave<N>(r.low);
    if (lane == 0)
        spread[wave] = r;
    __syncthreads();
    const u16x2 top = most(most(spread[0].top, spread[1].top), most(spread[2].top, spread[3].top));
    const u16x2 low = most(most(spread[0].low, spread[1].low), most(spread[2].low, spread[3].low));
    const Pow2 sk = pow2_for<1>(top[0]), sv = pow2_for<4>(top[1]);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        f16x8 h, l;
        split2x8(k[g], sk.up, h, l);
        *reinterpret_cast<f16x8*>(&out[((N * g + kl) * KT + krow) * 16]) = h;
        *reinterpret_cast<f16x8*>(&out[((KB + N * g + kl) * KT + krow) * 16]) = l;
        split2x8(v[g], sv.up, h, l);
        *reinterpret_cast<f16x8*>(&out[16384 + (vblk * D + vd + g) * 16]) = h;
        *reinterpret_cast<f16x8*>(&out[16384 + ((VB + vblk) * D + vd + g) * 16]) = l;
    }
    if (tid == 0)
        p.powers[blockIdx.x] = { spread_fits(top, low) ? sk.down : NAN, low[1] == 0 ? 0.f : sv.down };
    __syncthreads();
    unsigned char* to = p.ready + (int64_t)blockIdx.x * 32768;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        *reinterpret_cast<f32x4*>(to + (i * 256 + tid) * 16) = *reinterpret_cast<const f32x4*>(&out[(i * 256 + tid) * 16]);
}

// 16 KB from memory to LDS, a kilobyte a wave and instruction
__device__ __forceinline__ void load_to_lds(const unsigned char* from, unsigned char* to, int wave, int lane)
{
#pragma unroll
    for (int i = 0; i < 4; ++i)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + (wave * 4 + i) * 1024 + lane * 16),
            (__attribute__((address_space(3))) void*)(to + (wave * 4 + i) * 1024), 16, 0, 0);
}

template <int D>
__global__ __launch_bounds__(256, 2) void ragged_packed_kernel(RaggedParams p)
{
    constexpr int KT = 4096 / D, HALVES = KT / 32, N = D / 16;
    constexpr int KB = D / 8, VB = KT / 8, STEPS = D / 16, DB = D / 32;
    __shared__ __attribute__((aligned(1024))) unsigned char ks0[16384], ks1[16384], vs0[16384], vs1[16384];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, half = lane >> 5;
    if (p.error_flag && blockIdx.x == 0)
        for (int i = tid; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens));
    const int kv_head = blockIdx.x % p.kv_heads; // the order of ragged_tile_kernel
    const int64_t number = blockIdx.x / p.kv_heads;
    const Tile tile = p.causal && p.n_seqs <= 64 ? late_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, p.group, 128, number)
                                                 : find_tile(SearchWave(), p.starts, p.n_seqs, p.tokens, p.group, 128, gridDim.x / p.kv_heads - 1 - number);
    if (tile.seq < 0)
        return;
    const Sequence s = sequence_of<kPackedF32>(p, tile.seq, tile.span);
    const int count = s.span.count * p.group, r_first = tile.index * 128;
    const int r = r_first + wave * 32 + c;
    const bool q_ok = r < count;
    const int token = quotient(q_ok ? r : count - 1, p.by_group), head = kv_head * p.group + (q_ok ? r : count - 1) - token * p.group;
    const int64_t q_row = s.span.first + token;
    const int visible = visible_keys(p, s, token);
    const int r_last = r_first + 128 < count ? r_first + 127 : count - 1;
    const int tiles = (visible_keys(p, s, quotient(r_last, p.by_group)) + KT - 1) / KT; // at least one
    const int w_first = r_first + wave * 32, w_last = w_first + 31 < count ? w_first + 31 : count - 1;
    const int wave_all_see = visible_keys(p, s, quotient(w_first < count ? w_first : count - 1, p.by_group));
    const int wave_any = visible_keys(p, s, quotient(w_last, p.by_group));

    const int64_t tile0 = ready_tile(p, tile.seq, s.span.first, KT) * p.kv_heads + kv_head;
    const unsigned char* ready = p.ready + tile0 * 32768;
    const f32x2_pow* powers = p.powers + tile0;
    const int64_t tile_bytes = (int64_t)p.kv_heads * 32768;
    load_to_lds(ready, ks0, wave, lane);
    load_to_lds(ready + 16384, vs0, wave, lane);
    if (tiles > 1)
        load_to_lds(ready + tile_bytes, ks1, wave, lane);

    f16x8 qh[STEPS], ql[STEPS]; // depth block 2 u + half
    float q_down;
    {
        float x[STEPS][8], top = 0.f;
        const float* from = p.q + q_row * p.ldq + (int64_t)head * p.dk;
#pragma unroll
        for (int u = 0; u < STEPS; ++u) {
            const int blk = 2 * u + half, d0 = 8 * N * (blk / N) + 4 * (blk % N);
            load_depths<float, 4, false>(from, d0, p.dk, p.wide, x[u]);
            load_depths<float, 4, false>(from, d0 + 4 * N, p.dk, p.wide, x[u] + 4);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                top = fmaxf(top, fabsf(x[u][e]));
        }
        const Pow2 sq = pow2_for<1>(exponent(max_halves(top)));
        q_down = sq.down * (p.scale * kLog2e);
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
    float v_down = 0.f; // what takes the sums' power back: that of the last tile with a value that is not zero

    auto scores = [&](f32x16 (&sc)[HALVES], const unsigned char* ks) {
#pragma unroll
        for (int kb = 0; kb < HALVES; ++kb) {
            sc[kb] = kZero;
#pragma unroll
            for (int u = 0; u < STEPS; ++u) {
                const f16x8 kh = *reinterpret_cast<const f16x8*>(&ks[((2 * u + half) * KT + kb * 32 + c) * 16]);
                const f16x8 kw = *reinterpret_cast<const f16x8*>(&ks[((KB + 2 * u + half) * KT + kb * 32 + c) * 16]);
                sc[kb] = mfma(kw, qh[u], sc[kb]);
                sc[kb] = mfma(kh, ql[u], sc[kb]);
                sc[kb] = mfma(kh, qh[u], sc[kb]);
            }
        }
    };
    // tile t: its scores are in sc; ks holds the keys of tile t + 1 and vs the values of tile t; the keys of tile t + 2 go to ks_to, the values of
    // tile t + 1 to vs_to
    auto turn = [&](int t, f32x16 (&sc)[HALVES], f32x16 (&next)[HALVES], const unsigned char* ks, const unsigned char* vs, unsigned char* ks_to,
                    unsigned char* vs_to) {
        const int j0 = t * KT;
        if (t + 1 < tiles)
            load_to_lds(ready + (t + 1) * tile_bytes + 16384, vs_to, wave, lane);
        if (t + 2 < tiles)
            load_to_lds(ready + (t + 2) * tile_bytes, ks_to, wave, lane);
        const f32x2_pow down = powers[(int64_t)t * p.kv_heads];
        if (j0 < wave_any) { // some row of this wave sees some key of the tile
            const int limit = visible - j0; // keys of the tile that this lane's row sees
            if (j0 + KT > wave_all_see) {
#pragma unroll
                for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (kb * 32 + 8 * (e >> 2) + 4 * half + (e & 3) >= limit)
                            sc[kb][e] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                for (int e = 0; e < 16; e += 2)
                    mx = max3(mx, sc[kb][e], sc[kb][e + 1]);
            const float step = q_down * down.k_down, to_log2 = fmaxf(step, 1.17549435e-38f); // above zero: -infinity stays what it is
            mx = max_halves(mx) * to_log2;
            l_run = step < INFINITY ? l_run : NAN; // NaN: a tile that is left to plain sums; an infinite step makes every negative score -infinity
            if (__any(mx > m_run + 4.f) || down.v_down != v_down) {
                const float m_new = mx > m_run + 4.f ? mx : m_run;
                const float corr = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
                const float f = v_down / down.v_down;
                // NAN: sums that would leave fp32's range
                const float by = down.v_down == 0.f || v_down == 0.f ? corr : (f > 1e-18f && f < 1e18f ? corr * f : NAN);
                m_run = m_new;
                v_down = down.v_down == 0.f ? v_down : down.v_down;
                l_run *= corr;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        oacc[d][e] *= by;
            }
            const float base = kShift - (m_run == -INFINITY ? 0.f : m_run);
            float rs = 0.f;
#pragma unroll
            for (int kb = 0; kb < HALVES; ++kb)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    sc[kb][e] = __builtin_amdgcn_exp2f(fmaf(sc[kb][e], to_log2, base));
                    rs += sc[kb][e];
                }
            l_run += rs;
            scores(next, ks);
#pragma unroll
            for (int u = 0; u < KT / 16; ++u) { // keys of block 2 u + half: registers 8 (u % 2) .. + 7 of accumulator u / 2
                float x[8];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    x[j] = sc[u >> 1][8 * (u & 1) + j];
                f16x8 ph, pl;
                split2x8(x, ph, pl);
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const f16x8 vh = *reinterpret_cast<const f16x8*>(&vs[((2 * u + half) * D + d * 32 + c) * 16]);
                    const f16x8 vl = *reinterpret_cast<const f16x8*>(&vs[((VB + 2 * u + half) * D + d * 32 + c) * 16]);
                    oacc[d] = mfma(vl, ph, oacc[d]);
                    oacc[d] = mfma(vh, pl, oacc[d]);
                    oacc[d] = mfma(vh, ph, oacc[d]);
                }
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // this wave's part of the tiles is in LDS
    __syncthreads();
    scores(sa, ks0);
    __syncthreads(); // ks0 is done with
    for (int t = 0; t < tiles; t += 2) {
        turn(t, sa, sb, ks1, vs0, ks0, vs1);
        if (t + 1 < tiles)
            turn(t + 1, sb, sa, ks0, vs1, ks1, vs0);
    }

    l_run += __shfl_xor(l_run, 32, 64);
    float size = l_run;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e)
            size += fabsf(oacc[d][e]);
    // a row's two lanes hold half of its depths each
    const uint64_t odd_lanes = __ballot(q_ok && (!(size < INFINITY) || l_run == 0.f));
    uint32_t odd = (uint32_t)odd_lanes | (uint32_t)(odd_lanes >> 32);
    if (q_ok && !(odd >> c & 1)) {
        const float f = v_down / l_run;
        float* to = p.out + q_row * p.ldo + (int64_t)head * p.dv;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int depth = 32 * d + 8 * g + 4 * half;
                const f32x4 o = { oacc[d][4 * g] * f, oacc[d][4 * g + 1] * f, oacc[d][4 * g + 2] * f, oacc[d][4 * g + 3] * f };
                if (p.wide && depth < p.dv) {
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
        const int t1 = quotient(r1, p.by_group), h1 = kv_head * p.group + r1 - t1 * p.group;
        store_plain_row<kPackedF32>(p, s, t1, h1, kv_head, 0, lane);
    }
}

// ---- few query rows: keys and values pass once, straight from memory to the matrix instructions ----
//
// A workgroup takes the rows that a sequence brings to one key head, over one range of its keys.  Up to sixteen rows: its four waves take every
// fourth block of 16 keys; up to thirty-two: two waves for either half of the rows take every second block, and the later one of two that load
// the same keys finds them in the CU's cache (20 rows each of 32 sequences of 3000 keys, 32 / 8 heads of 128, 231 us with fp32 pages; a
// workgroup for either half 291).  Waves have sums of their own, which meet at the end.  Bound by memory: a lane's loads are the operands of the
// products, nothing is staged, and a block's loads are on their way while the block before is worked on.  A token each for 64 sequences of
// 4000, 32 / 8 heads of 128: 368 us with fp32 pages (5.7 TB/s), 226 with bf16 pages (4.6 TB/s); 12 heads of 64, 64 sequences of 2000: 165 and
// 87 us (4.8 and 4.5 TB/s).  One of 201 keys, 12 heads of 64: 8.5 us, a chain of dependent trips to memory.
//  * S^T = K Q^T: lane (c, g) of 16 x 4 loads chunks of key c, chunk i at depth 4 W i + W g (W elements are 16 bytes), and has scores of keys
//    4 g .. 4 g + 3 of row c.
//  * O^T = V^T P^T: lane (c, g) loads depths V c .. V c + V - 1 of keys 4 g .. + 3, so the probabilities it has are the operand, and gets
//    depths V (4 g + i) + e of row c.
//  * fp32 pages: the 16x16x4 fp32 products, 32 cycles per 16 keys, 16 rows and 4 depths, which is half of what the memory's share of a CU needs
//    for the keys.  bf16 pages bring twice the keys in that time: the bf16 products take them as they are, queries and probabilities as the
//    exact sum of three bf16 values (bf16_split.hpp), 576 cycles instead of 2048 for 16 keys at depth 128.
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

template <int D, int KIND, bool WIDE>
__device__ __forceinline__ void few_body(const RaggedParams& p, const Place& place_in, float* meet_01, float* meet_23, float* meet_ml)
{
    typedef typename KvElement<KIND>::type T;
    constexpr int W = 16 / (int)sizeof(T), NK = D / (4 * W); // elements of a key chunk, chunks of a lane
    constexpr int DL = D / 16, VW = DL < W ? DL : W, NV = DL / VW; // depths of a lane, in NV loads of VW
    constexpr bool kBf16 = KIND == kPagedBf16;
    typedef T kvec __attribute__((ext_vector_type(W)));
    typedef T vvec __attribute__((ext_vector_type(VW)));
    struct Block {
        kvec k[NK];
        vvec v[4][NV];
        int row;
    };
    // [wave][row][depth] of the sums o, two waves each, and [wave][row] of m, then of l
    float (*meet_m)[16] = reinterpret_cast<float (*)[16]>(meet_ml), (*meet_l)[16] = meet_m + 4;
    auto meet_o = [&](int w, int row) { return (w < 2 ? meet_01 : meet_23) + ((w & 1) * 16 + row) * (D + 4); };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int seq = place_in.x / p.kv_heads, kv_head = place_in.x % p.kv_heads;
    if (p.error_flag && place_in.x == 0 && place_in.y == 0)
        for (int i = tid; i < p.n_seqs; i += 256)
            raise_flag(p, !packed_start_ok(p.starts, i, p.tokens));
    const Sequence s = sequence_of<KIND>(p, seq, packed_span(p.starts, seq, p.tokens));
    if (tid == 0)
        raise_flag(p, s.cut);
    const int count = s.span.count * p.group;
    if (count == 0 || !s.few)
        return;
    const bool halves = count > 16;
    const int step = halves ? 2 : 4, slot = halves ? wave & 1 : wave, r_first = halves ? (wave >> 1) * 16 : 0; // of this wave
    int k_end = visible_keys(p, s, s.span.count - 1);
    const int64_t k_from = (int64_t)place_in.y * s.range;
    if (place_in.y > 0 && k_from >= k_end)
        return;
    const int k_first = (int)k_from;
    if (k_end - k_first > s.range)
        k_end = k_first + s.range;
    const int blocks = k_end > k_first ? (k_end - k_first + 15) / 16 : 0;

    const T* kbase = static_cast<const T*>(p.k) + (int64_t)kv_head * p.dk;
    const T* vbase = static_cast<const T*>(p.v) + (int64_t)kv_head * p.dv;
    auto look_up = [&](int blk) { // the place of key c of a block; positions behind the range repeat its last one
        int first = k_first + blk * 16;
        asm("" : "+s"(first)); // no register keeps a part of the sum for the next time
        const int at = first + c;
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
    if (slot < blocks) {
        const int row_a = look_up(slot);
        row_b = look_up(slot + step);
        fetch(a, row_a);
    }

    float q[kBf16 ? 1 : NK][W];
    bf16x8 q3[kBf16 ? NK : 1][3];
    const bool q_ok = r_first + c < count;
    const int q_token = quotient(q_ok ? r_first + c : 0, p.by_group);
    const int visible = q_ok ? visible_keys(p, s, q_token) : 0;
    {
        const float* from = p.q + (int64_t)(s.span.first + q_token) * p.ldq
            + (int64_t)(kv_head * p.group + (q_ok ? r_first + c : 0) - q_token * p.group) * p.dk;
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            float y[W];
#pragma unroll
            for (int h = 0; h < W; h += 4) {
                const f32x4 x = load_chunk<float, 4, WIDE>(from, 4 * W * i + W * g + h, p.dk);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    y[h + e] = x[e] * (p.scale * kLog2e);
            }
            if constexpr (kBf16) {
                uint32_t w[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    split3(y[2 * e], y[2 * e + 1], w[0][e], w[1][e], w[2][e]);
#pragma unroll
                for (int z = 0; z < 3; ++z)
                    q3[i][z] = __builtin_bit_cast(bf16x8, (u32x4 { w[z][0], w[z][1], w[z][2], w[z][3] }));
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    q[i][e] = y[e];
            }
        }
    }
    float m_run = -INFINITY, l_run = 0.f;
    f32x4 oacc[DL];
#pragma unroll
    for (int e = 0; e < DL; ++e)
        oacc[e] = f32x4 { 0.f, 0.f, 0.f, 0.f };
    // keys that the first row sees are seen by all
    const int first_sees = visible_keys(p, s, quotient(r_first, p.by_group)), all_see = first_sees < k_end ? first_sees : k_end;
    bool missing = false;
    auto work = [&](const Block& x, int blk) {
        f32x4 sc = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
        for (int i = 0; i < NK; ++i) {
            if constexpr (kBf16) {
#pragma unroll
                for (int z = 2; z >= 0; --z) // small ones first
                    sc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[i]), q3[i][z], sc, 0, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    sc = __builtin_amdgcn_mfma_f32_16x16x4f32(x.k[i][e], q[i][e], sc, 0, 0, 0);
            }
        }
        const int at = k_first + blk * 16;
        if (at + 16 > all_see) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (at + 4 * g + i >= (visible < k_end ? visible : k_end))
                    sc[i] = -INFINITY;
        }
        if (__any(x.row < 0)) {
            missing = true;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sc[i] = __shfl(x.row, 4 * g + i, 64) < 0 ? -INFINITY : sc[i];
        }
        float mx = fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3]));
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = max_halves(mx);
        if (__any(mx > m_run + 8.f)) { // the maximum moves when a score passes it by 2^8
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
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sc[i] = __builtin_amdgcn_exp2f(sc[i] - base);
            l_run += sc[i];
        }
        if constexpr (kBf16) {
            typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
            u32x2 pr[3];
            uint32_t w[3][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                split3(sc[2 * i], sc[2 * i + 1], w[0][i], w[1][i], w[2][i]);
#pragma unroll
            for (int z = 0; z < 3; ++z)
                pr[z] = u32x2 { w[z][0], w[z][1] };
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    const bf16x4 v4 = { x.v[0][j][e], x.v[1][j][e], x.v[2][j][e], x.v[3][j][e] };
#pragma unroll
                    for (int z = 2; z >= 0; --z)
                        oacc[j * VW + e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, v4), __builtin_bit_cast(s16x4, pr[z]),
                            oacc[j * VW + e], 0, 0, 0);
                }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < VW; ++e)
                        oacc[j * VW + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.v[i][j][e], sc[i], oacc[j * VW + e], 0, 0, 0);
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
    if (g == 0) {
        meet_m[wave][c] = m_run;
        meet_l[wave][c] = l_run;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < VW; ++e)
                meet_o(wave, c)[16 * VW * j + VW * (4 * g + i) + e] = oacc[j * VW + e][i];
    __syncthreads();
    // found out anew, so that no register keeps it through the loop
    const int lane2 = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0)), tid2 = wave * 64 + lane2;
    const int at = tid2 >> 4, d0 = (tid2 & 15) * DL;
    uint32_t odd = 0; // of this wave's four rows, and of the four behind the next sixteen
    for (int half = 0; half <= (halves ? 1 : 0); ++half) {
        const int w_first = 2 * half, w_last = halves ? w_first + 1 : 3; // the waves that have these rows
        float top = -INFINITY;
        for (int w = w_first; w <= w_last; ++w)
            top = fmaxf(top, meet_m[w][at]);
        const float m = top == -INFINITY ? 0.f : top;
        float l = 0.f, o[DL];
#pragma unroll
        for (int e = 0; e < DL; ++e)
            o[e] = 0.f;
        for (int w = w_first; w <= w_last; ++w) {
            const float f = __builtin_amdgcn_exp2f(meet_m[w][at] - m);
            l += f * meet_l[w][at];
#pragma unroll
            for (int e = 0; e < DL; ++e)
                o[e] += f * meet_o(w, at)[d0 + e];
        }
        float size = l;
#pragma unroll
        for (int e = 0; e < DL; ++e)
            size += fabsf(o[e]);
        const int r = 16 * half + at;
        const bool there = r < count;
        const int token = quotient(there ? r : 0, p.by_group), head = kv_head * p.group + (there ? r : 0) - token * p.group;
        const int sees = visible_keys(p, s, token);
        const bool in_parts = sees > s.range, mine = there && (in_parts ? k_first < sees : place_in.y == 0);
        // rows whose sums are not finite, or empty though there are keys; a row's 16 threads agree
        const uint64_t bad = __ballot(mine && (!(size < INFINITY) || (l == 0.f && k_first < sees)));
        if (mine && (bad >> (lane2 & 48) & 0xffff) == 0) {
            const float f = l > 0.f ? 1.f / l : 0.f; // no key: zeros
            float* to = p.out + (int64_t)(s.span.first + token) * p.ldo + (int64_t)head * p.dv;
            if (in_parts) {
                const int64_t id = part_row(p, s, token, head);
                to = p.few.out(place_in.y, id, p.dv);
                float* size_at = p.few.size(place_in.y, id, p.dv);
                if ((tid2 & 15) == 0) {
                    size_at[0] = top;
                    size_at[1] = l;
                }
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
        for (int k = 0; k < 4; ++k)
            if (bad >> (16 * k) & 0xffff)
                odd |= 1u << (16 * half + 4 * wave + k);
    }
    if (__builtin_expect(odd == 0, 1))
        return;
#pragma clang loop unroll(disable)
    while (odd) {
        const int r1 = __builtin_ctz(odd);
        odd &= odd - 1;
        const int t1 = quotient(r1, p.by_group);
        store_plain_row<KIND>(p, s, t1, kv_head * p.group + r1 - t1 * p.group, kv_head, place_in.y, lane2);
    }
}

template <int D, int KIND, bool WIDE>
__global__ __launch_bounds__(256, WIDE ? 2 : 1) void ragged_few_kernel(RaggedParams p)
{
    __shared__ float meet[2][2 * 16 * (D + 4)], meet_ml[2 * 4 * 16];
    few_body<D, KIND, WIDE>(p, Place { blockIdx.x, blockIdx.y, gridDim.x }, meet[0], meet[1], meet_ml);
}

// Both in one launch: what is bound by memory runs beside what is bound by the matrix and vector units.  Tiles, which take longest, come first.
// Twelve sequences of 400 to 12 000 keys that bring 1 to 1024 tokens, 32 / 8 heads of 128, fp32 pages: 350 us, one launch behind the other 417,
// few-row workgroups spread among the tiles 483.
template <int D, int KIND>
__global__ __launch_bounds__(256, 2) void ragged_mixed_kernel(RaggedParams p, unsigned tile_x, unsigned tile_wgs, unsigned few_x)
{
    FDX_TILE_LDS(D, KIND, lds);
    if (blockIdx.x < tile_wgs) {
        tile_body<D, KIND, true>(p, Place { blockIdx.x % tile_x, blockIdx.x / tile_x, tile_x }, lds);
    } else {
        static_assert(2 * 16 * (D + 4) * sizeof(float) <= sizeof(lds_ks0) && 2 * 4 * 16 * sizeof(float) <= sizeof(lds_vs0), "fits into the tiles' LDS");
        const unsigned at = blockIdx.x - tile_wgs;
        few_body<D, KIND, true>(p, Place { at % few_x, at / few_x, few_x }, reinterpret_cast<float*>(lds.ks0), reinterpret_cast<float*>(lds.ks1),
            reinterpret_cast<float*>(lds.vs0));
    }
}

// Rows that more than one range of keys was summed for: sum of 2^(m - M) l o over the ranges, divided by that of 2^(m - M) l.
template <int KIND>
__global__ __launch_bounds__(256) void ragged_join_kernel(RaggedParams p)
{
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t item = (int64_t)blockIdx.x * 4 + wave;
    const int row = (int)((uint64_t)item / (uint32_t)p.heads), head = (int)(item - (int64_t)row * p.heads);
    if (row >= p.tokens)
        return;
    const int index = find_row(SearchWave(), p.starts, p.n_seqs, p.tokens, row);
    if (index < 0)
        return;
    const Sequence s = sequence_of<KIND>(p, index, packed_span(p.starts, index, p.tokens));
    const int token = row - s.span.first;
    if (token >= s.span.count)
        return;
    const int visible = visible_keys(p, s, token);
    if (visible <= s.range)
        return;
    const int parts = (visible + s.range - 1) / s.range;
    const PartSums& part = s.few ? p.few : p.tile;
    const int64_t id = part_row(p, s, token, head);
    // a lane a range for the sizes, then all lanes a range at a time for the rows, four of them on their way together
    float top = -INFINITY;
    for (int i0 = 0; i0 < parts; i0 += 64)
        if (i0 + lane < parts)
            top = fmaxf(top, part.size(i0 + lane, id, p.dv)[0]);
    top = wave_all<true>(top);
    const float m = top == -INFINITY ? 0.f : top;
    float l = 0.f, o0 = 0.f, o1 = 0.f;
    for (int i0 = 0; i0 < parts; i0 += 64) {
        float w = 0.f;
        if (i0 + lane < parts) {
            const float* at = part.size(i0 + lane, id, p.dv);
            w = at[1] * __builtin_amdgcn_exp2f(at[0] - m);
        }
        l += wave_all<false>(w);
        const int count = parts - i0 < 64 ? parts - i0 : 64;
        for (int i = 0; i < count; i += 4) {
            float x0[4], x1[4];
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const float* from = part.out(i0 + (i + z < count ? i + z : i), id, p.dv);
                x0[z] = from[lane < p.dv ? lane : 0];
                x1[z] = from[64 + lane < p.dv ? 64 + lane : 0];
            }
#pragma unroll
            for (int z = 0; z < 4; ++z) {
                const float wi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i + z < count ? i + z : i));
                o0 = fmaf(i + z < count ? wi : 0.f, x0[z], o0);
                o1 = fmaf(i + z < count ? wi : 0.f, x1[z], o1);
            }
        }
    }
    float* to = p.out + (int64_t)row * p.ldo + (int64_t)head * p.dv;
    if (lane < p.dv)
        to[lane] = finish(o0, l, top != -INFINITY);
    if (64 + lane < p.dv)
        to[64 + lane] = finish(o1, l, top != -INFINITY);
}

// How a call is cut: sequences of few rows (up to `few_rows`) go to ragged_few_kernel in ranges of up to few_keys keys, the others to
// ragged_tile_kernel in ranges of up to tile_keys.
struct RaggedPlan {
    int few_rows, few_ranges, few_keys; // few_ranges 0: no such launch
    int tile_ranges, tile_keys, tile_whole;
    int64_t few_part, tile_part; // rows whose sums may be kept
    int64_t tiles;
    int64_t ready; // tiles of split keys and values, for all key heads; 0: none are laid out
    size_t ready_bytes() const { return (size_t)ready * (32768 + sizeof(f32x2_pow)); }
    size_t few_floats(int dv) const { return few_ranges > 1 ? ((size_t)few_ranges * few_part * (2 + (size_t)dv) + 3) & ~(size_t)3 : 0; }
    size_t tile_floats(int dv) const { return tile_ranges > 1 ? (size_t)tile_ranges * tile_part * (2 + (size_t)dv) : 0; }
};

static int ranges_of(int keys, int64_t most, int* range_keys)
{
    *range_keys = (int)(most > keys ? keys : (most + 63) & ~(int64_t)63);
    return (keys + *range_keys - 1) / *range_keys;
}

static RaggedPlan paged_plan(int tokens, int max_new, int heads, const fdx_kv_pages* c)
{
    RaggedPlan r {};
    const int group = heads / c->kv_heads;
    const int64_t most = (int64_t)(max_new < tokens ? max_new : tokens) * group; // rows of a sequence
    r.few_rows = most <= 16 ? 16 : 32;
    if (group <= r.few_rows) {
        const int64_t items = (int64_t)c->n_seqs * c->kv_heads;
        // Ranges enough for some 4096 workgroups when every sequence is as long as the longest (max_len in all figures here: what a longer
        // max_len costs stands at fdx_kv_pages), which leaves those of shorter ones to fill gaps; 256 keys or more, and 64 ranges or fewer, which one
        // pass of ragged_join_kernel takes.  us with at least 128 / 192 / 256 / 384 / 512
        // keys, fp32: one sequence of 8000, 32 / 8 heads of 128, 28.4 / 29.9 / 26.0 / 28.0 / 31.7; 16 of 1000, 12 heads of 64, 28.1 / 29.2 / 26.4 / 28.9 /
        // 28.9; one of 2000, 12.9 / 13.0 / 13.9 / 16.4 / 18.8; four of 32 000, 8 / 1 heads of 128, 60.9 / 56.3 / 46.7 / 48.0 / 41.0.
        // Where 512 keys make 768 workgroups or more, 512: with 256 / 512, 32 / 8 heads of 128, 64 sequences of 1000 112 / 105 (bf16 pages 58.8 / 52.7),
        // of 100 to 2000 92.3 / 86.7 (50.8 / 43.3), 32 of 3000 with 5 tokens each 237 / 220 (134 / 114); below, eight of 200 to 4000 43.2 / 44.6.
        const int64_t all = c->max_len * items, least = all >= 512 * 768 ? 512 : 256;
        const int64_t keys = all / 4096 < least ? least : all / 4096;
        const int64_t share = ((int64_t)c->max_len + 63) / 64;
        r.few_ranges = ranges_of(c->max_len, keys < share ? share : keys, &r.few_keys);
        r.few_part = items * (most < r.few_rows ? most : r.few_rows);
    }
    if (r.few_ranges == 0)
        r.few_rows = 0;
    if (most > r.few_rows) {
        r.tiles = tile_numbers(tokens, c->n_seqs, group, 128) * c->kv_heads;
        const int64_t full = ((int64_t)tokens * group + 127) / 128 * c->kv_heads;
        // Ranges while there are fewer tiles than the 512 workgroups that the GPU takes at once, of 192 (deep heads: 128) to 4096 keys.  us with at
        // least 128 / 192 / 256 / 512 keys, fp32 pages: 128 new tokens of 1000, 12 heads of 64 (12 tiles), 19.6 / 20.9 / 22.5 / 30.9; 512 of 1000 (48 tiles)
        // 30.0 / 28.8 / 27.7 / 34.3; 471 of 1211, 8 / 1 heads of 128 (30 tiles), 35.4 / 37.6 / 40.0 / 52.1; 32 / 8 heads of 128, 128 of 2000 (32 tiles)
        // 44.7 / 45.8 / 49.2 / 55.8, 128 of 8000 93.8 / 91.3 / 89.8 / 88.4, four times 128 of 1000 (128 tiles) 62.8 / 62.8 / 62.8 / 75.4.  With at most 512 /
        // 1024 / 2048 / 4096: twice 2000 of 3000, 16 / 4 heads of 64 (500 tiles) 206 / 197 / 190 / 166; four times 1000 of 4000 (1000 tiles) 1087 / 982 /
        // 957 / 887.  A sequence of up to eight turns of a tile stays whole, the join costs what ranges save: ten of 386 keys, 16 / 4 heads of 64 (124
        // tiles), 25.9 whole and 28.8 in two; 16 decode steps of 1000 keys beside a prompt of 256, 12 heads of 64, 37.7 and 38.9 (35.3 with a grid for ranges of 512, of which fewer are empty).
        const bool deep = c->dk > 64 || c->dv > 64;
        const int64_t least = deep ? 128 : 192;
        r.tile_whole = deep ? 256 : 512;
        int64_t keys = full < 512 ? c->max_len / (512 / full) : c->max_len;
        keys = keys < least ? least : (keys > 4096 ? 4096 : keys);
        // At most 16 ranges, and 16 384 workgroups of tiles and ranges: every range keeps sums of all rows, so scratch memory ends at 2^21 rows of
        // them, 1.02 GiB at depth 128.  Without and with that limit, 32 / 8 heads of 128: twice 4096 new tokens of 131 072 55.4 / 55.2 ms (2.2 / 1.1 GB); 128
        // of 131 072 beside 16 prompts of 512, whose sums nobody needs, 1.77 / 2.24 ms (2.3 / 1.0 GB).
        const int64_t ranges = 16384 / full < 1 ? 1 : (16384 / full < 16 ? 16384 / full : 16), share = (c->max_len + ranges - 1) / ranges;
        r.tile_ranges = ranges_of(c->max_len, keys < share ? share : keys, &r.tile_keys);
        r.tile_part = (int64_t)tokens * heads;
    }
    return r;
}

static RaggedPlan packed_plan(int tokens, int n_seqs, int heads, int kv_heads, int dk, int dv, int causal)
{
    RaggedPlan r {};
    const int keys_a_tile = dk <= 64 && dv <= 64 ? 64 : 32, length = tokens / n_seqs;
    r.tiles = tile_numbers(tokens, n_seqs, heads / kv_heads, 128) * kv_heads;
    r.tile_ranges = 1;
    r.tile_keys = 0x7fffffff;
    // A few long prompts: ranges of 256 keys or more while there are tiles for half the CUs or fewer (three quarters with a mask, which leaves
    // half of the ranges to nobody); the join is a launch and reads what they wrote.  us without ranges / with: no mask, 4 heads of 64, one prompt
    // of 600 26.5 / 20.0, 1000 39.0 / 22.8, 4000 (128 tiles) 116 / 79.4, two of 1000 38.6 / 31.2; causal, 12 heads, one of 600 27.7 / 23.6, 1000
    // 40.0 / 33.3, 2000 (192 tiles) 72.0 / 54.6.  They lose with prompts of 300 to 500 (12 heads, four of 500 causal 24.2 / 38.3) and with
    // more tiles (12 heads, two of 2000 causal, 384 tiles, 76.2 / 88.5; one of 2000 without a mask, 192 tiles, 72.1 / 75.1).
    const int64_t full = ((int64_t)tokens * (heads / kv_heads) + 127) / 128 * kv_heads;
    if (length >= 512 && full <= (causal ? 192 : 128)) {
        int64_t keys = length / (512 / full);
        keys = keys < 256 ? 256 : keys;
        const int64_t share = ((int64_t)tokens + 15) / 16; // at most 16 ranges, whose sums take scratch memory
        keys = keys < share ? share : keys;
        if (keys < length) {
            r.tile_ranges = ranges_of(tokens, keys, &r.tile_keys);
            r.tile_part = (int64_t)tokens * heads;
            return r;
        }
    }
    // The pass of its own moves a tile's 32 KB twice more (of 8192 tokens, 16 heads of 64: 18 us), every 128 rows that use the tile then take a
    // fifth less time.  8192 tokens in sequences of one length, one pass against two in us: no mask, 512 / 1024 / 2048 rows a sequence
    // and key head, 76.7 / 87.4, 133 / 134, 248 / 230 at depth 64 and 144 / 165, 252 / 255, 476 / 439 at 128; causal, 1024 / 2048 / 4096 rows,
    // 81.7 / 94.7, 143 / 144, 266 / 249 and 157 / 182, 274 / 274, 519 / 466.
    if ((int64_t)tokens * (heads / kv_heads) >= (int64_t)n_seqs * (causal ? 2048 : 1024) && tokens >= (int64_t)n_seqs * keys_a_tile)
        r.ready = tile_numbers(tokens, n_seqs, 1, keys_a_tile) * kv_heads;
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
    p.wide = WIDE;
    const bool exact = WIDE && p.dk == D && p.dv == D;
    const dim3 block(256);
    if constexpr (KIND == kPackedF32) {
        if (plan.ready > 0) {
            if (exact)
                hipLaunchKernelGGL((ragged_ready_kernel<D, true>), dim3((unsigned)plan.ready), block, 0, stream(), p);
            else
                hipLaunchKernelGGL((ragged_ready_kernel<D, false>), dim3((unsigned)plan.ready), block, 0, stream(), p);
            hipLaunchKernelGGL(ragged_packed_kernel<D>, dim3((unsigned)plan.tiles), block, 0, stream(), p);
            return;
        }
    }
    const unsigned tile_x = (unsigned)plan.tiles, tile_y = (unsigned)(plan.tile_ranges > 0 ? plan.tile_ranges : 1);
    bool mixed = false;
    if constexpr (KIND != kPackedF32) {
        const unsigned few_x = (unsigned)(p.n_seqs * p.kv_heads);
        const uint64_t few_wgs = (uint64_t)few_x * plan.few_ranges, tile_wgs = (uint64_t)tile_x * tile_y;
        mixed = exact && few_wgs > 0 && tile_wgs > 0 && few_wgs + tile_wgs < (1u << 23);
        if (mixed)
            hipLaunchKernelGGL((ragged_mixed_kernel<D, KIND>), dim3((unsigned)(few_wgs + tile_wgs)), block, 0, stream(), p, tile_x, (unsigned)tile_wgs,
                few_x);
        else if (few_wgs > 0)
            hipLaunchKernelGGL((ragged_few_kernel<D, KIND, WIDE>), dim3(few_x, (unsigned)plan.few_ranges), block, 0, stream(), p);
    }
    if (!mixed && plan.tiles > 0) {
        const dim3 grid(tile_x, tile_y);
        if (exact)
            hipLaunchKernelGGL((ragged_tile_kernel<D, KIND, true>), grid, block, 0, stream(), p);
        else
            hipLaunchKernelGGL((ragged_tile_kernel<D, KIND, false>), grid, block, 0, stream(), p);
    }
    if (plan.few_ranges > 1 || plan.tile_ranges > 1)
        hipLaunchKernelGGL(ragged_join_kernel<KIND>, dim3((unsigned)(((int64_t)p.tokens * p.heads + 3) / 4)), block, 0, stream(), p);
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
    FDX_REQUIRE((int64_t)p.tokens * p.heads <= (1 << 25) && (int64_t)p.n_seqs * p.kv_heads <= (1 << 22),
        "%s: tokens * heads or sequences * key heads too many for one launch", who);
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
    if (tokens <= 0 || n_seqs <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dk <= 0 || dv <= 0)
        return 0;
    size_t most = 0;
    for (int causal = 0; causal < 2; ++causal) {
        const RaggedPlan plan = packed_plan(tokens, n_seqs, heads, kv_heads, dk, dv, causal);
        const size_t need = plan.ready_bytes() + sizeof(float) * plan.tile_floats(dv);
        most = need > most ? need : most;
    }
    return most;
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
    p.by_group = make_divisor(p.group);
    profile_begin();
    const RaggedPlan plan = packed_plan(tokens, n_seqs, heads, kv_heads, dk, dv, causal);
    p.ready = static_cast<unsigned char*>(scratch_dev);
    p.powers = reinterpret_cast<f32x2_pow*>(p.ready + plan.ready * 32768);
    p.tile = { static_cast<float*>(scratch_dev), plan.tile_part, plan.tile_ranges, plan.tile_keys, plan.tile_whole, 0 };
    ragged_dispatch<kPackedF32>(p, plan);
    profile_end("mha_packed_f32", 0.0, 4.0 * tokens * ((double)heads + kv_heads) * (dk + dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}

extern "C" size_t fdx_mha_paged_scratch_bytes(int tokens, int max_new, int heads, const fdx_kv_pages* c)
{
    if (!c || tokens <= 0 || max_new <= 0 || heads <= 0 || c->kv_heads <= 0 || heads % c->kv_heads != 0 || c->dk <= 0 || c->dv <= 0 || c->n_seqs <= 0
        || c->max_len <= 0)
        return 0;
    const RaggedPlan plan = paged_plan(tokens, max_new, heads, c);
    return sizeof(float) * (plan.few_floats(c->dv) + plan.tile_floats(c->dv));
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
    p.page_size = make_divisor(cache->page_size); p.max_len = cache->max_len; p.max_new = max_new < tokens ? max_new : tokens;
    p.error_flag = error_flag_dev;
    st = check_ragged("mha_paged", p, scratch_dev, fdx_mha_paged_scratch_bytes(tokens, max_new, heads, cache));
    if (st != FDX_OK)
        return st;
    p.scale = (float)(1.0 / std::sqrt((double)p.dk));
    const RaggedPlan plan = paged_plan(tokens, max_new, heads, cache);
    float* part = static_cast<float*>(scratch_dev);
    p.by_group = make_divisor(p.group);
    p.few_rows = plan.few_rows;
    p.few = { part, plan.few_part, plan.few_ranges, plan.few_keys, 0, (int)(plan.few_part / ((int64_t)p.n_seqs * p.kv_heads)) };
    p.tile = { part + plan.few_floats(p.dv), plan.tile_part, plan.tile_ranges, plan.tile_keys, plan.tile_whole, 0 };
    profile_begin();
    if (cache->type == FDX_KV_F32)
        ragged_dispatch<kPagedF32>(p, plan);
    else
        ragged_dispatch<kPagedBf16>(p, plan);
    profile_end("mha_paged_f32", 0.0, 4.0 * tokens * heads * (double)(p.dk + p.dv));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
