// Log probabilities of given tokens, entropy and the likeliest tokens of each row of logits.
//
//   m = max x, t = (x - m) log2(e), Z = sum 2^t, W = sum 2^t t;  log p[i] = x[i] - m - ln2 log2 Z,  H = ln2 (log2 Z - W / Z)
// Both terms of H are at least zero, so nothing cancels.  Bound by memory: every logit is read once and stays in registers for all
// that is asked of it (2048 rows of 50 257: 76 us, 5.4 TB/s, without alternatives, 102 us, 4.0 TB/s, with 20, where ordering them takes the
// vector units; 16 rows with 5: 11 us, two dependent launches).
//
// A workgroup takes a row, or a part of one, in chunks of 4 E logits a thread; waves keep sums of their own, which meet at the end.  The likeliest
// `top` tokens of a wave are a sorted list in LDS.  Of a chunk, `top` lanes' largest logits are a threshold that no fewer than `top` tokens
// reach: it is found bit by bit with votes on the lanes' largest, and stops as soon as not many more lanes than that pass.  On
// random logits about as many tokens pass as are asked for; they and the list so far are ordered by counting, for each, the better ones.
// Where more pass than there is room for (equal logits), the best are taken one at a time.  Only finite logits are listed: places that stay
// empty are those of ruled-out tokens, the lowest ids that are not listed.  Lists of waves and of parts meet in pairs, an item's place being its
// place in its own list plus the number of better ones in the other.
#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace fdx {

constexpr int kMostTop = 32, kMostParts = 64, kFound = 192;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4))); // rows start at any multiple of four bytes
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

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
    int parts, part_len, chunk; // logits of a part, and of a chunk: multiples of what the workgroup's threads load at once
};

// Order of the likeliest tokens: descending logit, then ascending id.  Larger keys come first, 0 is no token.
__device__ __forceinline__ uint32_t score_bits(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f); // -0 and +0 are equal logits
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bits_score(uint32_t b) { return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b); }

struct Sums {
    float m, z, w; // w in units of log2
};
__device__ __forceinline__ void add_sums(Sums& a, float m, float z, float w)
{
    const float top = fmaxf(a.m, m), use = top == -INFINITY ? 0.f : top;
    // a sum without a finite logit has z = w = 0, and its distance is taken as finite so that the products are 0
    const float da = fmaxf((a.m - use) * kLog2e, -1e30f), db = fmaxf((m - use) * kLog2e, -1e30f);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
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
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v)
{
    for (int w = 32; w > 0; w >>= 1) {
        const uint32_t lo = __shfl_xor((int)(uint32_t)v, w, 64), hi = __shfl_xor((int)(v >> 32), w, 64);
        const uint64_t o = (uint64_t)hi << 32 | lo;
        v = o > v ? o : v;
    }
    return v;
}
__device__ __forceinline__ uint64_t uniform_key(uint64_t v)
{
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// `lists` sorted lists of `top` keys, one behind the other in `from`, become one at the returned place (`from` or `to`, both in LDS)
__device__ __forceinline__ uint64_t* join_lists(uint64_t* from, uint64_t* to, int lists, int top)
{
    while (lists > 1) {
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
        lists = (lists + 1) / 2;
    }
    __syncthreads();
    return from;
}

// what is asked of a row, from its sums and its list
__device__ __forceinline__ void score_results(const ScoreParams& p, int64_t row, const Sums& s, const uint64_t* list)
{
    const float m = s.m == -INFINITY ? 0.f : s.m;
    const float lz = s.z == 0.f ? 0.f : __log2f(s.z); // NaN where the row holds one, or an infinity
    auto logprob = [&](float x) { return (x - m) - lz * kLn2; };
    const int tid = threadIdx.x;
    if (tid < p.top) {
        uint64_t key = list[tid];
        int id = (int)~(uint32_t)key;
        float x = bits_score((uint32_t)(key >> 32));
        if (key == 0) { // the place of a token that is ruled out: of the ids that are not listed, the lowest come first
            int listed = 0;
            while (listed < tid && list[listed] != 0)
                ++listed;
            int left = tid - listed;
            for (id = 0;; ++id) {
                bool in = false;
                for (int i = 0; i < listed; ++i)
                    in = in || (int)~(uint32_t)list[i] == id;
                if (!in && left-- == 0)
                    break;
            }
            x = -INFINITY;
        }
        p.top_ids[row * p.top + tid] = id;
        p.top_logprobs[row * p.top + tid] = logprob(x);
    }
    if (tid == 64 && p.ids) {
        const int id = p.ids[row];
        float r = 0.f;
        if (id >= p.vocab) {
            r = NAN;
            if (p.error_flag)
                *p.error_flag = 1;
        } else if (id >= 0) {
            r = logprob(p.x[row * p.ld + id]);
        }
        p.logprobs[row] = r;
    }
    if (tid == 128 && p.entropy)
        p.entropy[row] = s.z == 0.f ? 0.f : (lz - s.w / s.z) * kLn2;
}

template <int E, bool TOP>
__global__ __launch_bounds__(256) void token_scores_kernel(ScoreParams p)
{
    __shared__ __attribute__((aligned(16))) uint64_t lists[TOP ? 8 * kMostTop : 1]; // a wave: its list and a spare one
    __shared__ __attribute__((aligned(16))) uint64_t found_by[TOP ? 4 : 1][TOP ? kFound : 1];
    __shared__ Sums met[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    const int first = part * p.part_len, last = p.vocab - first < p.part_len ? p.vocab : first + p.part_len;
    const float* x = p.x + row * p.ld;
    uint64_t* list = lists + wave * 2 * kMostTop;
    uint64_t* spare = list + kMostTop;
    uint64_t* found = found_by[TOP ? wave : 0];
    uint32_t worst = 0; // logit of a full list's last token
    if (TOP && lane < p.top)
        list[lane] = 0;
    Sums s { -INFINITY, 0.f, 0.f };
    for (int c0 = first; c0 < last; c0 += p.chunk) {
        const int end = last - c0 < p.chunk ? last : c0 + p.chunk;
        f32x4 v[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const int at = c0 + (j * 256 + tid) * 4;
            v[j] = f32x4 { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
            if (c0 + j * 256 * 4 < end) { // the same for the workgroup
                if (at + 3 < end) {
                    v[j] = *reinterpret_cast<const f32x4_any*>(x + at);
                } else {
#pragma unroll
                    for (int e = 0; e < 3; ++e)
                        if (at + e < end)
                            v[j][e] = x[at + e];
                }
            }
        }
        float best = -INFINITY;
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (c0 + j * 256 * 4 < end)
                best = fmaxf(fmaxf(fmaxf(best, v[j][0]), fmaxf(v[j][1], v[j][2])), v[j][3]);
        const float m = wave_all<true>(best), use = m == -INFINITY ? 0.f : m;
        float z[2] = { 0.f, 0.f }, w[2] = { 0.f, 0.f };
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (c0 + j * 256 * 4 < end) {
#pragma unroll
                for (int e = 0; e < 4; ++e) { // finite, so that 0 times it is 0; NaN stays NaN
                    const float t = __builtin_elementwise_maximum((v[j][e] - use) * kLog2e, -1e30f), f = __builtin_amdgcn_exp2f(t);
                    z[e & 1] += f;
                    w[e & 1] = fmaf(f, t, w[e & 1]);
                }
            }
        add_sums(s, m, wave_all<false>(z[0] + z[1]), wave_all<false>(w[0] + w[1]));
        if constexpr (TOP) {
            const uint32_t mine = best > -INFINITY ? score_bits(best) : 0;
            if (__ballot(mine > worst)) {
                uint32_t cut = worst + 1; // equal logits: those of lower ids are in the list already
                if (worst == 0) {
                    cut = 0;
                    for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                        const int pass = __builtin_popcountll(__ballot(mine >= (cut | bit)));
                        cut = pass >= p.top ? cut | bit : cut;
                        if (pass >= p.top && pass <= p.top + 4)
                            break;
                    }
                }
                const float cut_score = bits_score(cut > 0x00800000u ? cut : 0x00800000u); // no less than -FLT_MAX
                int count = 0;
#pragma unroll
                for (int j = 0; j < E; ++j)
                    if (c0 + j * 256 * 4 < end) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint64_t in = __ballot(v[j][e] >= cut_score);
                            if (in) {
                                const int at = count + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
                                if (v[j][e] >= cut_score && at < kFound)
                                    found[at] = (uint64_t)score_bits(v[j][e]) << 32 | (uint32_t)~(c0 + (j * 256 + tid) * 4 + e);
                                count += __builtin_popcountll(in);
                            }
                        }
                    }
                if (count > kFound) { // the best ones, one at a time
                    uint64_t before = ~(uint64_t)0;
                    count = 0;
                    while (count < p.top) {
                        uint64_t most = 0;
#pragma unroll
                        for (int j = 0; j < E; ++j)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const uint64_t key = (uint64_t)score_bits(v[j][e]) << 32 | (uint32_t)~(c0 + (j * 256 + tid) * 4 + e);
                                most = v[j][e] >= cut_score && key < before && key > most ? key : most;
                            }
                        before = uniform_key(wave_max_key(most));
                        if (before == 0)
                            break;
                        if (lane == 0)
                            found[count] = before;
                        ++count;
                    }
                }
                if (count > 0) {
                    wave_lds_fence();
                    if (lane < p.top)
                        spare[lane] = 0;
                    wave_lds_fence();
                    for (int i = lane; i < p.top + count; i += 64) {
                        const uint64_t key = i < p.top ? list[i] : found[i - p.top];
                        int place = 0;
#pragma unroll 4
                        for (int k = 0; k < p.top; ++k)
                            place += list[k] > key;
#pragma unroll 4
                        for (int k = 0; k < count; ++k)
                            place += found[k] > key;
                        if (key != 0 && place < p.top)
                            spare[place] = key;
                    }
                    wave_lds_fence();
                    uint64_t* t = list;
                    list = spare;
                    spare = t;
                    worst = (uint32_t)(uniform_key(list[p.top - 1]) >> 32);
                }
            }
        }
    }
    if (lane == 0)
        met[wave] = s;
    const uint64_t* all = nullptr;
    if constexpr (TOP) {
        uint64_t* flat = found_by[0]; // candidates are done with
        __syncthreads();
        if (lane < p.top)
            flat[wave * p.top + lane] = list[lane];
        all = join_lists(flat, flat + 4 * p.top, 4, p.top);
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
    __shared__ uint64_t lds[2 * kMostParts * kMostTop];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63;
    f32x4 o = { -INFINITY, 0.f, 0.f, 0.f }; // a lane a part
    if (lane < p.parts)
        o = p.part_sums[row * p.parts + lane];
    for (int i = threadIdx.x; i < p.parts * p.top; i += 256)
        lds[i] = p.part_keys[row * p.parts * p.top + i];
    Sums s { wave_all<true>(o[0]), 0.f, 0.f };
    const float d = fmaxf((o[0] - (s.m == -INFINITY ? 0.f : s.m)) * kLog2e, -1e30f), f = __builtin_amdgcn_exp2f(d);
    s.z = wave_all<false>(f * o[1]);
    s.w = wave_all<false>(f * (o[2] + o[1] * d));
    const uint64_t* list = join_lists(lds, lds + p.parts * p.top, p.parts, p.top);
    score_results(p, row, s, list);
}

// Rows are cut in one part for 4096 logits, or fewer parts, while that makes no more workgroups than two for each CU; all but the last part are
// whole thousands (of 1024), three at least.
struct ScorePlan {
    int parts, part_len, chunk;
    size_t keys, sums; // bytes
};
// A chunk's vectors a thread: chunks cost some 300 instructions each whatever their length, registers cost waves.  2048 rows of 50 257 and 1000 of
// 131 072 with 20 alternatives, in us: 7 vectors 107 / 118, 8 102 / 118, 9 108 / 115, 13 127 / 168, 17 118 / 145.
constexpr int kScoreE = 8;
static ScorePlan score_plan(int64_t rows, int vocab, int top)
{
    ScorePlan r {};
    auto thousands = [&](int64_t n, int64_t into) { return (int)((n + into * 1024 - 1) / (into * 1024) * 1024); };
    const int64_t most = ((int64_t)vocab + 4095) / 4096;
    int64_t parts = 512 / rows < most ? 512 / rows : most;
    parts = parts < 1 ? 1 : (parts > kMostParts ? kMostParts : parts);
    r.part_len = thousands(vocab, parts);
    r.parts = (vocab + r.part_len - 1) / r.part_len;
    r.chunk = thousands(r.part_len, (r.part_len + 1024 * kScoreE - 1) / (1024 * kScoreE)); // chunks of a part are of one length
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
    if (p.top > 0)
        hipLaunchKernelGGL((token_scores_kernel<E, true>), grid, dim3(256), 0, stream(), p);
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
        reinterpret_cast<uint64_t*>(scratch), reinterpret_cast<f32x4*>(scratch + plan.keys), plan.parts, plan.part_len, plan.chunk };
    profile_begin();
    if (plan.chunk <= 4096)
        score_launch<4>(p);
    else
        score_launch<kScoreE>(p);
    if (plan.parts > 1)
        hipLaunchKernelGGL(token_scores_join_kernel, dim3((unsigned)rows), dim3(256), 0, stream(), p);
    profile_end("token_logprobs_f32", 5.0 * rows * vocab, 4.0 * rows * ((double)vocab + 3 + 2 * top));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
