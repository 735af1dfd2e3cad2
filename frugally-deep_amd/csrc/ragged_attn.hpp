// Shared parts of the attention kernels for packed rows and paged caches (ragged_attn.hip).
#pragma once
#include <cmath>
#include <cstdint>

#include "common.hpp"
#include "kv_pages.hpp"

namespace fdx {

// what calls ask of their caches (kv_append.hip)
fdx_status check_kv_pages(const char* who, const fdx_kv_pages* c);
fdx_status check_kv_pages8(const char* who, const fdx_kv_pages8* c);

typedef float f32x4 __attribute__((ext_vector_type(4)));

// where keys and values come from
enum { kPackedF32 = 0, kPagedF32 = 1, kPagedBf16 = 2 };

// Rows that see more keys than one workgroup takes: their sums over each range of keys, for ragged_join_kernel.  [range][row][depth] of
// o / l, then [range][row][m, l].  m is -infinity where the range has no key, -FLT_MAX where all its scores are -infinity.
struct PartSums {
    float* at;
    int64_t rows;
    int ranges, keys; // of the longest sequence; keys: what a range has at most
    int whole;        // sequences of up to so many keys have one range
    int a_head;       // few rows: rows of a sequence and key head

    __device__ __forceinline__ float* out(int range, int64_t row, int dv) const { return at + (range * rows + row) * dv; }
    __device__ __forceinline__ float* size(int range, int64_t row, int dv) const { return at + ranges * rows * dv + 2 * (range * rows + row); }
};

struct f32x2_pow {
    float k_down, v_down; // what takes a tile's powers of two back; k_down NaN: a tile for plain sums, v_down 0: values of zeros
};

struct RaggedParams {
    const float* q;
    float* out;
    int64_t ldq, ldo;
    const void *k, *v;    // rows of kv_heads * dk keys / kv_heads * dv values, ldk / ldv elements apart
    int64_t ldk, ldv;
    const int32_t* starts;
    int n_seqs, tokens, heads, kv_heads, group, dk, dv, causal;
    Divisor by_group, page_size;
    float scale;
    const int32_t *table, *lens; // paged only
    int table_width, n_pages, max_len, max_new;
    int* error_flag;
    PartSums few, tile;   // of the launch for few rows and of the one for tiles
    int few_rows;         // sequences that bring up to this many rows to a key head are ragged_few_kernel's, others ragged_tile_kernel's
    int wide;             // rows of every tensor lie on 16-byte vectors, and depths are whole ones
    unsigned char* ready; // packed prompts: tiles of split keys and values, [tile][key head][32 KB], and their powers [tile][key head]
    f32x2_pow* powers;
};

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

// of a call on a paged cache: how it is cut, and its parameters after its arguments have been checked (ragged_attn.hip)
RaggedPlan paged_plan(int tokens, int max_new, int heads, const fdx_kv_pages* c);
fdx_status paged_params(const char* who, const float* q, int64_t ldq, const int32_t* starts, int tokens, int max_new, int heads,
    const fdx_kv_pages* cache, float* out, int64_t ldo, const void* scratch_dev, size_t scratch_bytes, int* error_flag_dev, RaggedParams& p);

// where a workgroup stands in its launch
struct Place {
    unsigned x, y, nx;
};

template <int KIND>
struct KvElement {
    typedef float type;
};
template <>
struct KvElement<kPagedBf16> {
    typedef __bf16 type;
};

// one sequence of a call: its new rows, its keys
struct Sequence {
    Span span;    // rows of q and out
    int keys;     // positions that its last new token sees (all of them without a causal mask)
    int ahead;    // position of its first new token; may be negative: tokens that see nothing
    int index;
    bool few;     // its rows are few enough for ragged_few_kernel
    int range;    // keys of a range: as many ranges as its keys need, of the same length
    bool cut;     // lens or the number of new tokens beyond what the call was told
};

template <int KIND>
__device__ __forceinline__ Sequence sequence_of(const RaggedParams& p, int index, Span span)
{
    Sequence s { span, span.count, 0, index, false, 0x7fffffff, false };
    if constexpr (KIND != kPackedF32) {
        const int len = p.lens[index];
        s.keys = len < 0 ? 0 : (len > p.max_len ? p.max_len : len);
        s.ahead = s.keys - span.count;
        s.cut = len != s.keys || span.count > p.max_new;
        if (span.count > p.max_new)
            s.span.count = p.max_new;
        s.few = s.span.count * p.group <= p.few_rows;
    }
    const int most = s.few ? p.few.keys : p.tile.keys;
    if (s.keys > most && s.keys > (s.few ? p.few.whole : p.tile.whole)) {
        const int parts = (s.keys + most - 1) / most;
        s.range = ((s.keys + parts - 1) / parts + 63) & ~63;
    }
    return s;
}

// where the sums of a row are kept, rows as the launches number them
__device__ __forceinline__ int64_t part_row(const RaggedParams& p, const Sequence& s, int token, int head)
{
    if (!s.few)
        return (int64_t)(s.span.first + token) * p.heads + head;
    const int kv_head = quotient(head, p.by_group);
    return ((int64_t)s.index * p.kv_heads + kv_head) * p.few.a_head + token * p.group + head - kv_head * p.group;
}

// row of a position in k and v, -1 for one that is not there
template <int KIND>
__device__ __forceinline__ int key_row(const RaggedParams& p, const Sequence& s, int pos)
{
    if constexpr (KIND == kPackedF32)
        return s.span.first + pos;
    else
        return page_row(p.table + (int64_t)s.index * p.table_width, p.table_width, p.n_pages, p.page_size, pos);
}

// positions 0 .. visible - 1 are what a new token sees
__device__ __forceinline__ int visible_keys(const RaggedParams& p, const Sequence& s, int token)
{
    if (!p.causal)
        return s.keys;
    const int n = s.ahead + token + 1;
    return n < 0 ? 0 : n;
}

// the wave that searches, for the functions of kv_pages.hpp
struct SearchWave {
    struct Kept {
        int mine;
        __device__ __forceinline__ int at(int) const { return mine; }
    };
    int lane = threadIdx.x & 63;
    template <class F>
    __device__ __forceinline__ Kept kept(const F& f) const { return { f(lane) }; }
    template <class F>
    __device__ __forceinline__ uint64_t mask(const F& f) const { return __ballot(f(lane)); }
    template <class F>
    __device__ __forceinline__ int count(const F& f) const { return __builtin_popcountll(mask(f)); }
    template <class F>
    __device__ __forceinline__ float sum(const F& f) const { return wave_all<false>(f(lane)); }
    template <class F>
    __device__ __forceinline__ float most(const F& f) const { return wave_all<true>(f(lane)); }
};

// exponentials are taken to base two on scores that carry log2(e)
constexpr float kLog2e = 1.44269504088896340736f;

// One query row over the keys first .. last - 1 by one whole wave, in fp32: a lane has a key's score, then depths lane and
// 64 + lane of the output.  m - 24 is the largest score in units of log2, l the sum of 2^(score - m), o the weighted values: with 2^-24 in every
// weight the sums of values near fp32's end stay below it.
template <int KIND>
__device__ __forceinline__ void plain_row(const RaggedParams& p, const Sequence& s, const float* q, int kv_head, int first, int last, float& m,
    float& l, float (&o)[2], bool& seen, bool& missing)
{
    typedef typename KvElement<KIND>::type T;
    const int lane = threadIdx.x & 63;
    const T* kb = static_cast<const T*>(p.k) + (int64_t)kv_head * p.dk;
    const T* vb = static_cast<const T*>(p.v) + (int64_t)kv_head * p.dv;
    const float scale = p.scale * kLog2e;
    m = -INFINITY;
    l = o[0] = o[1] = 0.f;
    seen = missing = false;
#pragma clang loop unroll(disable)
    for (int j0 = first; j0 < last; j0 += 64) {
        const int row = j0 + lane < last ? key_row<KIND>(p, s, j0 + lane) : -1;
        seen = seen || __any(row >= 0);
        missing = missing || __any(j0 + lane < last && row < 0);
        float sc = -INFINITY;
        if (row >= 0) {
            const T* kr = kb + (int64_t)row * p.ldk;
            float dot = 0.f;
            for (int d = 0; d < p.dk; ++d)
                dot = fmaf(q[d], (float)kr[d], dot);
            sc = dot * scale;
        }
        float mx = sc;
        for (int w = 32; w > 0; w >>= 1)
            mx = fmaxf(mx, __shfl_xor(mx, w, 64));
        const float m_new = fmaxf(m, mx + 24.f), m_use = m_new == -INFINITY ? 0.f : m_new, corr = __builtin_amdgcn_exp2f(m - m_use);
        const float pr = row >= 0 ? __builtin_amdgcn_exp2f(sc - m_use) : 0.f;
        float rs = pr;
        for (int w = 32; w > 0; w >>= 1)
            rs += __shfl_xor(rs, w, 64);
        l = l * corr + rs;
        m = m_new;
        o[0] *= corr;
        o[1] *= corr;
        const int count = last - j0 < 64 ? last - j0 : 64;
#pragma clang loop unroll(disable)
        for (int j = 0; j < count; ++j) {
            const int r = __shfl(row, j, 64);
            const float pj = __shfl(pr, j, 64);
            if (r < 0)
                continue;
            const T* vr = vb + (int64_t)r * p.ldv;
            if (lane < p.dv)
                o[0] = fmaf(pj, (float)vr[lane], o[0]);
            if (64 + lane < p.dv)
                o[1] = fmaf(pj, (float)vr[64 + lane], o[1]);
        }
    }
}

// what a row's sums come to: a row that sees no key gets zeros, one whose scores are all -infinity (infinite operands) has no
// softmax, as in the formula
__device__ __forceinline__ float finish(float o, float l, bool sees) { return l == 0.f ? (sees ? NAN : 0.f) : o / l; }

__device__ __forceinline__ void raise_flag(const RaggedParams& p, bool on)
{
    if (on && p.error_flag)
        *p.error_flag = 1;
}

} // namespace fdx
