// Log probabilities of given tokens, entropy and the likeliest tokens of each row of logits.
//
//   m = max x, Z = sum e^(x - m), W = sum e^(x - m) (x - m);  log p[i] = x[i] - m - log Z,  H = log Z - W / Z
// Both terms of H are at least zero, so nothing cancels.  Bound by memory: every logit is read once and stays in registers for all
// that is asked of it.
//
// A workgroup takes a row, or a part of one where rows are few, in chunks of 4 E vectors a thread; waves keep sums of their own, which
// meet at the end (exp(m_w - m) each).  The likeliest `top` tokens of a wave are a sorted list in LDS.  Of a chunk, every lane finds its own
// best token; the top-th best of these 64 is a threshold that no fewer than `top` tokens of the chunk reach, and only `top` lanes can hold
// tokens that do: on random logits about as many as are asked for, and never more than fit.  Those and the list so far are
// ordered by counting, for each, the better ones.  Lists of waves and of parts meet in pairs, an item's place being its place in its
// own list plus the number of better ones in the other.
#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace fdx {

constexpr int kMostTop = 32, kMostParts = 64;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4))); // rows start at any multiple of four bytes
constexpr float kLog2e = 1.44269504088896340736f;

struct ScoreParams {
    const float* x;
    int64_t ld, rows;
    int vocab, top;
    const int32_t* ids;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_ids;
    int* error_flag;
    uint64_t* part_keys; // [row][part][top]
    f32x4* part_sums;    // [row][part]: m, Z, W
    int parts, part_len; // part_len: logits of a part, a multiple of 1024
};

// Order of the likeliest tokens: descending logit (NaN as -infinity), then ascending id.  Larger keys come first, 0 is no token.
__device__ __forceinline__ uint64_t score_key(float x, int id)
{
    uint32_t b = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x); // -0 and +0 are equal logits
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)b << 32 | (uint32_t)~id;
}
__device__ __forceinline__ float key_score(uint64_t key)
{
    const uint32_t b = (uint32_t)(key >> 32);
    return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b);
}

struct Sums {
    float m, z, w;
};
__device__ __forceinline__ void add_sums(Sums& a, float m, float z, float w)
{
    const float top = fmaxf(a.m, m), use = top == -INFINITY ? 0.f : top;
    // a sum without a finite logit has z = w = 0, and its distance is taken as finite so that the products are 0
    const float da = fmaxf(a.m - use, -1e30f), db = fmaxf(m - use, -1e30f);
    const float fa = __builtin_amdgcn_exp2f(da * kLog2e), fb = __builtin_amdgcn_exp2f(db * kLog2e);
    a.w = fa * (a.w + a.z * da) + fb * (w + z * db);
    a.z = fa * a.z + fb * z;
    a.m = top;
}

__device__ __forceinline__ void wave_lds_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// `lists` sorted lists of `top` keys, one behind the other in `from`, become one at the returned place (`from` or `to`, both in LDS)
__device__ __forceinline__ uint64_t* join_lists(uint64_t* from, uint64_t* to, int lists, int top)
{
    while (lists > 1) {
        const int left = (lists + 1) / 2;
        __syncthreads();
        for (int i = threadIdx.x; i < lists * top; i += 256) {
            const int list = i / top, place = i - list * top, other = list ^ 1;
            const uint64_t key = from[i];
            int better = 0;
            if (other < lists)
                for (int step = 32; step > 0; step >>= 1) // how many of the other list are larger
                    if (better + step <= top && from[other * top + better + step - 1] > key)
                        better += step;
            // equal keys are empty places: those of the second list go behind
            if (other < lists && key == 0 && (list & 1))
                better = top;
            if (place + better < top)
                to[(list >> 1) * top + place + better] = key;
        }
        uint64_t* t = from;
        from = to;
        to = t;
        lists = left;
    }
    __syncthreads();
    return from;
}

// what is asked of a row, from its sums and its list
__device__ __forceinline__ void score_results(const ScoreParams& p, int64_t row, const Sums& s, const uint64_t* list)
{
    const float m = s.m == -INFINITY ? 0.f : s.m;
    const float lz = s.z == 0.f ? 0.f : logf(s.z); // NaN where the row holds one, or an infinity
    const int tid = threadIdx.x;
    if (tid < p.top) {
        const uint64_t key = list[tid];
        p.top_ids[row * p.top + tid] = (int)~(uint32_t)key;
        p.top_logprobs[row * p.top + tid] = (key_score(key) - m) - lz;
    }
    if (tid == 64 && p.ids) {
        const int id = p.ids[row];
        float r = 0.f;
        if (id >= p.vocab) {
            r = NAN;
            if (p.error_flag)
                *p.error_flag = 1;
        } else if (id >= 0) {
            r = (p.x[row * p.ld + id] - m) - lz;
        }
        p.logprobs[row] = r;
    }
    if (tid == 128 && p.entropy)
        p.entropy[row] = s.z == 0.f ? 0.f : lz - s.w / s.z;
}

template <int E, bool TOP>
__global__ __launch_bounds__(256) void token_scores_kernel(ScoreParams p)
{
    extern __shared__ __attribute__((aligned(16))) uint64_t lds[]; // a wave: two lists, the chunk's candidates
    __shared__ Sums met[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    const int first = part * p.part_len, last = p.vocab - first < p.part_len ? p.vocab : first + p.part_len;
    const float* x = p.x + row * p.ld;
    uint64_t* list = lds + wave * 2 * p.top;
    uint64_t* spare = list + p.top;
    uint64_t* found = lds + 8 * p.top + wave * 4 * E * p.top;
    uint64_t worst = 0; // of a full list
    if (TOP && lane < p.top)
        list[lane] = 0;
    Sums s { -INFINITY, 0.f, 0.f };
    for (int c0 = first; c0 < last; c0 += 1024 * E) {
        f32x4 v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int at = c0 + (j * 256 + tid) * 4;
            v[j] = f32x4 { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
            if (at + 3 < last) {
                v[j] = *reinterpret_cast<const f32x4_any*>(x + at);
            } else {
#pragma unroll
                for (int e = 0; e < 3; ++e)
                    if (at + e < last)
                        v[j][e] = x[at + e];
            }
        }
        float best = -INFINITY;
        int where = 0x7fffffff;
#pragma unroll
        for (int j = 0; j < E; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (TOP) {
                    const int at = c0 + (j * 256 + tid) * 4 + e;
                    where = v[j][e] > best ? at : where;
                }
                best = fmaxf(best, v[j][e]);
            }
        const float m = wave_all<true>(best), use = m == -INFINITY ? 0.f : m;
        float z = 0.f, w = 0.f;
#pragma unroll
        for (int j = 0; j < E; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float d = fmaxf(v[j][e] - use, -1e30f); // finite, so that 0 times it is 0
                const float f = __builtin_amdgcn_exp2f((v[j][e] - use) * kLog2e);
                z += f;
                w = fmaf(f, d, w);
            }
        add_sums(s, m, wave_all<false>(z), wave_all<false>(w));
        if constexpr (TOP) {
            // a lane of nothing but -infinity and NaN: its first token that there is
            if (where == 0x7fffffff && c0 + tid * 4 < last)
                where = c0 + tid * 4;
            const uint64_t mine = where == 0x7fffffff ? 0 : score_key(best, where);
            int better = 0;
#pragma unroll 8
            for (int i = 0; i < 64; ++i) {
                const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), i) << 32
                    | (uint32_t)__builtin_amdgcn_readlane((int)mine, i);
                better += o > mine;
            }
            const uint64_t is_cut = __ballot(better == p.top - 1 && mine != 0);
            uint64_t cut = worst + 1;
            if (is_cut) {
                const int l = __builtin_ctzll(is_cut);
                const uint64_t o = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), l) << 32
                    | (uint32_t)__builtin_amdgcn_readlane((int)mine, l);
                cut = o > cut ? o : cut;
            }
            const float cut_score = cut >> 32 ? key_score(cut) : -INFINITY; // no token below it is better
            int count = 0;
#pragma unroll
            for (int j = 0; j < E; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float score = fmaxf(v[j][e], -INFINITY); // NaN as -infinity
                    if (__any(score >= cut_score)) {
                        const int at = c0 + (j * 256 + tid) * 4 + e;
                        const uint64_t key = at < last ? score_key(score, at) : 0;
                        const uint64_t in = __ballot(key >= cut && key != 0);
                        if (key >= cut && key != 0)
                            found[count + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0))] = key;
                        count += __builtin_popcountll(in);
                    }
                }
            if (count) {
                wave_lds_fence();
                for (int i = lane; i < p.top; i += 64)
                    spare[i] = 0;
                wave_lds_fence();
                for (int i = lane; i < p.top + count; i += 64) {
                    const uint64_t key = i < p.top ? list[i] : found[i - p.top];
                    int place = 0;
                    for (int k = 0; k < p.top; ++k)
                        place += list[k] > key;
                    for (int k = 0; k < count; ++k)
                        place += found[k] > key;
                    if (key != 0 && place < p.top)
                        spare[place] = key;
                }
                wave_lds_fence();
                uint64_t* t = list;
                list = spare;
                spare = t;
                worst = list[p.top - 1];
                worst = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(worst >> 32)) << 32
                    | (uint32_t)__builtin_amdgcn_readfirstlane((int)worst);
            }
        }
    }
    if (lane == 0)
        met[wave] = s;
    uint64_t* all = lds + 8 * p.top;
    if constexpr (TOP) {
        __syncthreads(); // candidates are done with
        if (lane < p.top)
            all[wave * p.top + lane] = list[lane];
        all = join_lists(all, all + 4 * p.top, 4, p.top);
    } else {
        __syncthreads();
    }
    s = met[0];
#pragma unroll
    for (int i = 1; i < 4; ++i)
        add_sums(s, met[i].m, met[i].z, met[i].w);
    if (p.parts == 1) {
        score_results(p, row, s, all);
    } else {
        if (tid < p.top)
            p.part_keys[(int64_t)blockIdx.x * p.top + tid] = all[tid];
        if (tid == 64)
            p.part_sums[blockIdx.x] = f32x4 { s.m, s.z, s.w, 0.f };
    }
}

__global__ __launch_bounds__(256) void token_scores_join_kernel(ScoreParams p)
{
    extern __shared__ __attribute__((aligned(16))) uint64_t lds[]; // lists of all parts, twice
    const int64_t row = blockIdx.x;
    for (int i = threadIdx.x; i < p.parts * p.top; i += 256)
        lds[i] = p.part_keys[row * p.parts * p.top + i];
    Sums s { -INFINITY, 0.f, 0.f };
    for (int i = 0; i < p.parts; ++i) {
        const f32x4 o = p.part_sums[row * p.parts + i];
        add_sums(s, o[0], o[1], o[2]);
    }
    const uint64_t* list = join_lists(lds, lds + p.parts * p.top, p.parts, p.top);
    score_results(p, row, s, list);
}

// Rows are cut in parts while there are fewer workgroups than the GPU takes at once.
struct ScorePlan {
    int parts, part_len;
    size_t keys, sums; // bytes
};
static ScorePlan score_plan(int64_t rows, int vocab, int top)
{
    int64_t parts = 1024 / rows, most = (vocab + 4095) / 4096;
    parts = parts < 1 ? 1 : (parts > most ? most : parts);
    parts = parts > kMostParts ? kMostParts : parts;
    ScorePlan r {};
    r.part_len = (int)((vocab + parts * 1024 - 1) / (parts * 1024) * 1024);
    r.parts = (vocab + r.part_len - 1) / r.part_len;
    if (r.parts > 1) {
        r.keys = ((size_t)rows * r.parts * top * sizeof(uint64_t) + 15) & ~(size_t)15;
        r.sums = (size_t)rows * r.parts * sizeof(f32x4);
    }
    return r;
}

template <int E>
static void score_launch(const ScoreParams& p)
{
    const dim3 grid((unsigned)(p.rows * p.parts));
    const size_t lds = sizeof(uint64_t) * p.top * (8 + 16 * E);
    if (p.top > 0)
        hipLaunchKernelGGL((token_scores_kernel<E, true>), grid, dim3(256), lds, stream(), p);
    else
        hipLaunchKernelGGL((token_scores_kernel<E, false>), grid, dim3(256), 0, stream(), p);
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_token_logprobs_scratch_bytes(int64_t rows, int vocab, int top)
{
    if (rows <= 0 || vocab <= 0 || top < 0)
        return 0;
    const ScorePlan plan = score_plan(rows, vocab, top);
    return plan.keys + plan.sums;
}

extern "C" fdx_status fdx_token_logprobs_f32(const float* logits, int64_t ld, int64_t rows, int vocab, const int32_t* ids, int top,
    float* logprobs, float* entropy, int32_t* top_ids, float* top_logprobs, void* scratch_dev, int* error_flag_dev)
{
    FDX_REQUIRE(logits, "token_logprobs: null pointer");
    FDX_REQUIRE(rows > 0 && rows <= (1 << 23) && vocab > 0 && vocab <= (1 << 24), "token_logprobs: 1 to 2^23 rows of 1 to 2^24 logits");
    FDX_REQUIRE(ld >= vocab, "token_logprobs: rows overlap");
    FDX_REQUIRE((ids != nullptr) == (logprobs != nullptr), "token_logprobs: ids and logprobs go together");
    FDX_REQUIRE(top >= 0 && top <= kMostTop && top <= vocab, "token_logprobs: 0 to 32 alternatives, no more than the vocabulary has");
    FDX_REQUIRE((top > 0) == (top_ids != nullptr) && (top > 0) == (top_logprobs != nullptr), "token_logprobs: top_ids and top_logprobs go with top");
    FDX_REQUIRE(logprobs || entropy || top > 0, "token_logprobs: nothing asked for");
    const size_t need = fdx_token_logprobs_scratch_bytes(rows, vocab, top);
    FDX_REQUIRE(need == 0 || (scratch_dev && (reinterpret_cast<uintptr_t>(scratch_dev) & 15) == 0),
        "token_logprobs: scratch missing or not 16-byte aligned");
    const ScorePlan plan = score_plan(rows, vocab, top);
    char* scratch = static_cast<char*>(scratch_dev);
    const ScoreParams p { logits, ld, rows, vocab, top, ids, logprobs, entropy, top_logprobs, top_ids, error_flag_dev,
        reinterpret_cast<uint64_t*>(scratch), reinterpret_cast<f32x4*>(scratch + plan.keys), plan.parts, plan.part_len };
    profile_begin();
    if (plan.part_len <= 4096)
        score_launch<4>(p);
    else
        score_launch<12>(p);
    if (plan.parts > 1)
        hipLaunchKernelGGL(token_scores_join_kernel, dim3((unsigned)rows), dim3(256), 2 * sizeof(uint64_t) * plan.parts * top, stream(), p);
    profile_end("token_logprobs_f32", 5.0 * rows * vocab, 4.0 * rows * ((double)vocab + 3 + 2 * top));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
