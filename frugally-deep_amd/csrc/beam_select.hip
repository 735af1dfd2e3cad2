// The best continuations of a sequence's beams over the vocabulary.
//
//   total(b, t) = score_b + (x[b, t] - m_b) - log sum exp(x[b, :] - m_b), the best `keep` of beams * vocab
// A row's order is its logits', so its `keep` likeliest are all that can be among the best.  Two launches: a workgroup reads a row, or a part of one,
// once, and leaves its sum and its list (score_lists.hpp); then a workgroup a sequence brings the lists together.
//  * Totals of different beams decide an order, so sums are held in 64 bits (a thread's chunk in 32: some 20 terms of one size) and totals are taken in
//    64 bits: two rows' sums are off by some 5e-8, not by the 5e-7 of fp32 totals of ten or so.  What a term costs more is one multiply-add for
//    log2(e)'s second half.
//  * Of the lists' heads, one or more of each so that they are about twice as many as are kept, the `keep`-th best is a threshold: no fewer
//    continuations reach it, and of a list whose first is behind it none does.  Those that reach it, twice as many as are kept on random logits and
//    keep * keep at most, are ordered by counting the better ones of each.  32 sequences of 16 beams, 32 kept of 50 257 tokens, 32 lists:
//    282 us where all of 32 lists were ordered, 53 so.
// 64 sequences of 8 beams over 50 257 tokens, a sixth of which have ended (86 MB): rows 27 us, 3.2 TB/s, the selection 7; four rows take the same 7 each, two
// launches of dependent steps.
// The next chunk's logits on their way take registers: 35 -> 39 us, with half the chunk 38.
#include "score_lists.hpp"
#include "kv_pages.hpp"

namespace fdx {

constexpr int kMostBeams = 32, kBeamLists = 128, kBeamE = 8; // lists of a sequence

struct BeamParams {
    const float* x;
    int64_t ld;
    int beams, vocab, keep;
    const float* scores;
    const int32_t* done;
    int end_id;
    int32_t *parents, *tokens, *new_done;
    float* new_scores;
    int* error_flag;
    uint64_t* part_keys; // [row][part][keep]
    double* part_sums;   // [row][part][m, z]
    int parts, part_len, chunk;
    int width; // a power of two, not less than parts
    Divisor by_parts, by_keep, by_deep;
};

// beams that have ended, or have no score, are not read
__device__ __forceinline__ bool beam_reads(const BeamParams& p, int64_t row)
{
    const float score = p.scores[row];
    return !(p.done && p.done[row]) && score > -INFINITY && score < INFINITY;
}

template <int E>
__global__ __launch_bounds__(256) void beam_rows_kernel(BeamParams p)
{
    __shared__ __attribute__((aligned(16))) uint64_t lists[8 * kMostTop]; // a wave: its list and a spare one
    __shared__ __attribute__((aligned(16))) uint64_t found_by[4][kFound];
    __shared__ double met[4][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t row = blockIdx.x / p.parts;
    const int part = blockIdx.x % p.parts;
    if (!beam_reads(p, row))
        return;
    const int first = part * p.part_len, last = p.vocab - first < p.part_len ? p.vocab : first + p.part_len;
    const float* x = p.x + row * p.ld;
    TopList t { lists + wave * 2 * kMostTop, lists + wave * 2 * kMostTop + kMostTop, found_by[wave], 0 };
    if (lane < p.keep)
        t.list[lane] = 0;
    float m = -INFINITY;
    double z = 0.0;
    for (int c0 = first; c0 < last; c0 += p.chunk) {
        const int end = last - c0 < p.chunk ? last : c0 + p.chunk;
        f32x4 v[E];
        load_chunk(x, c0, end, v);
        const float best = most_of_chunk(v, c0, end);
        const float top = fmaxf(m, wave_all<true>(best)), use = top == -INFINITY ? 0.f : top;
        constexpr float kHigh = 0x1.715476p+0f, kLow = 0x1.4ae0cp-26f; // log2(e) = kHigh + kLow
        float sum[2] = { 0.f, 0.f };
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (c0 + j * 256 * 4 < end) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float d = __builtin_elementwise_maximum(v[j][e] - use, -1e30f); // finite, so that the halves do not cancel; NaN stays NaN
                    sum[e & 1] += __builtin_amdgcn_exp2f(fmaf(d, kHigh, d * kLow));
                }
            }
        if (top > m && m > -INFINITY) // a few times a row
            z *= exp((double)m - (double)top);
        z += (double)(sum[0] + sum[1]);
        m = top;
        add_chunk(t, p.keep, v, c0, end, best);
    }
    for (int w = 32; w > 0; w >>= 1)
        z += __shfl_xor(z, w, 64);
    if (lane == 0) {
        met[wave][0] = m;
        met[wave][1] = z;
    }
    uint64_t* flat = found_by[0]; // candidates are done with
    __syncthreads();
    if (lane < p.keep)
        flat[wave * p.keep + lane] = t.list[lane];
    const uint64_t* all = join_lists(flat, flat + 4 * p.keep, 4, p.keep);
    if (tid < p.keep)
        p.part_keys[(int64_t)blockIdx.x * p.keep + tid] = all[tid];
    if (tid == 64) {
        const double most = fmax(fmax(met[0][0], met[1][0]), fmax(met[2][0], met[3][0]));
        double sum = 0.0;
        for (int i = 0; i < 4; ++i)
            sum += met[i][0] == -INFINITY ? met[i][1] : met[i][1] * exp(met[i][0] - most);
        p.part_sums[(int64_t)blockIdx.x * 2] = most;
        p.part_sums[(int64_t)blockIdx.x * 2 + 1] = sum;
    }
}

// continuations in their order: the larger key of a beam is the larger logit, or the lower token of equal ones
struct Continuation {
    double total;
    uint64_t key;
    int beam;
};
__device__ __forceinline__ bool better(const Continuation& a, const Continuation& b)
{
    return a.total > b.total || (a.total == b.total && (a.beam < b.beam || (a.beam == b.beam && a.key > b.key)));
}
// a set of them in LDS
template <int N>
struct Continuations {
    double total[N];
    uint64_t key[N];
    int beam[N];

    __device__ __forceinline__ Continuation at(int i) const { return { total[i], key[i], beam[i] }; }
    __device__ __forceinline__ void put(int i, const Continuation& c)
    {
        total[i] = c.total;
        key[i] = c.key;
        beam[i] = c.beam;
    }
    // how many of the first n are better than c, the me-th; those that are the same (empty) by their places.  Eight totals are on their way together.
    __device__ __forceinline__ int in_front(int n, const Continuation& c, int me) const
    {
        static_assert(N % 8 == 0, "whole eights");
        int count = 0;
        for (int k0 = 0; k0 < n; k0 += 8) {
            double t[8];
#pragma unroll
            for (int z = 0; z < 8; ++z)
                t[z] = total[k0 + z];
            bool same = false;
#pragma unroll
            for (int z = 0; z < 8; ++z) {
                const bool there = k0 + z < n;
                count += there && t[z] > c.total;
                same = same || (there && t[z] == c.total && k0 + z != me);
            }
            if (__builtin_expect(same, 0)) // of one total
                for (int k = k0; k < n && k < k0 + 8; ++k)
                    if (k != me && total[k] == c.total)
                        count += better(at(k), c) || (beam[k] == c.beam && key[k] == c.key && k < me);
        }
        return count;
    }
};

__global__ __launch_bounds__(256) void beam_select_kernel(BeamParams p)
{
    __shared__ Continuations<kMostTop * kMostTop> items;
    __shared__ Continuations<kBeamLists> heads; // of each list the first `deep`
    __shared__ double before_of[kMostBeams], most_of[kMostBeams]; // a beam's score less its sum's logarithm, its largest logit
    __shared__ int ended_of[kMostBeams], count;
    __shared__ Continuation threshold;
    const int tid = threadIdx.x;
    const int64_t s = blockIdx.x, row0 = s * p.beams;
    const int lists = p.beams * p.parts;
    const uint64_t* keys = p.part_keys + row0 * p.parts * p.keep;
    if (tid == 0) {
        count = 0;
        threshold = { -INFINITY, 0, kMostBeams };
    }
    const int head_list = quotient(tid, p.by_deep), deep = (int)p.by_deep.by, n_heads = lists * deep; // up to kBeamLists
    const uint64_t first_key = tid < n_heads ? keys[head_list * p.keep + tid - head_list * deep] : 0; // on its way beside the sums (rows that are not read have left anything)
    const uint64_t my_key = tid < lists * p.keep ? keys[tid] : 0;
    // the rows' sums: p.width threads a beam, one a part
    for (int b = tid / p.width; b < p.beams; b += 256 / p.width) {
        const int64_t row = row0 + b;
        const int part = tid & (p.width - 1);
        const float score = p.scores[row];
        const bool done = p.done && p.done[row], finite = score > -INFINITY && score < INFINITY, reads = finite && !done;
        double m = -INFINITY, z = 0.0;
        if (part < p.parts) {
            m = p.part_sums[(row * p.parts + part) * 2];
            z = p.part_sums[(row * p.parts + part) * 2 + 1];
        }
        double most = m;
        for (int w = p.width / 2; w > 0; w >>= 1)
            most = fmax(most, __shfl_xor(most, w, 64));
        z = m == -INFINITY || m == most ? z : z * exp(m - most);
        for (int w = p.width / 2; w > 0; w >>= 1)
            z += __shfl_xor(z, w, 64);
        if (part == 0) {
            const bool bad = !(score < INFINITY) || (reads && !(z < INFINITY)); // a NaN or an infinity: no continuation
            // The largest logit stays apart: beside one of 10^12 or more the logarithm has no room, beside fp32's lowest value, which masks are made of, none at all.
            const bool sums = reads && z > 0.0;
            before_of[b] = bad || !finite || (reads && z == 0.0) ? -INFINITY : sums ? (double)score - log(z) : (double)score;
            most_of[b] = sums ? most : 0.0;
            ended_of[b] = finite && done;
            if (bad && p.error_flag)
                *p.error_flag = 1;
        }
    }
    __syncthreads();
    auto listed = [&](int list, int j, uint64_t key) -> Continuation { // an ended beam has one continuation, in its first list
        const int b = quotient(list, p.by_parts);
        const double before = before_of[b];
        if (ended_of[b])
            return list == b * p.parts && j == 0 ? Continuation { before, 1, b } : Continuation { -INFINITY, 0, b };
        if (key == 0 || before == -INFINITY)
            return { -INFINITY, 0, b };
        return { before + ((double)bits_score((uint32_t)(key >> 32)) - most_of[b]), key, b };
    };
    if (tid < n_heads)
        heads.put(tid, listed(head_list, tid - head_list * deep, first_key));
    __syncthreads();
    if (tid < n_heads) {
        const Continuation mine = heads.at(tid);
        if (heads.in_front(n_heads, mine, tid) == p.keep - 1)
            threshold = mine;
    }
    __syncthreads();
    const Continuation least = threshold;
    for (int i = tid; i < lists * p.keep; i += 256) {
        const int list = quotient(i, p.by_keep);
        if (better(least, heads.at(list * deep)))
            continue;
        const Continuation c = listed(list, i - list * p.keep, i == tid ? my_key : keys[i]);
        if (c.total > -INFINITY && !better(least, c))
            items.put(atomicAdd(&count, 1), c);
    }
    __syncthreads();
    const int found = count;
    for (int i = tid; i < found; i += 256) {
        const Continuation mine = items.at(i);
        const int place = items.in_front(found, mine, i);
        if (place < p.keep) {
            const int64_t at = s * p.keep + place;
            const bool ended = ended_of[mine.beam];
            const int token = ended ? p.end_id : (int)~(uint32_t)mine.key;
            p.parents[at] = (int)(row0 + mine.beam);
            p.tokens[at] = token;
            p.new_scores[at] = (float)mine.total;
            if (p.new_done)
                p.new_done[at] = ended || token == p.end_id;
        }
    }
    if (tid < p.keep && tid >= found) { // places that are left over
        const int64_t at = s * p.keep + tid;
        p.parents[at] = p.tokens[at] = -1;
        p.new_scores[at] = -INFINITY;
        if (p.new_done)
            p.new_done[at] = 0;
    }
}

// Rows are cut in one part for 4096 logits, or fewer parts, while that makes no more workgroups than kBeamGroups and no more lists of a sequence than
// kBeamLists; all but the last part are whole thousands (of 1024).  us with 512 / 1024 / 2048 workgroups: 64 sequences of 8 beams, 50 257 tokens, 46.0 / 35.4 /
// 40.6; 100 of 5, 10 000 tokens, 19.5 / 18.2 / 18.3; level for fewer rows.
constexpr int kBeamGroups = 1024;
struct BeamPlan {
    int parts, part_len, chunk;
    size_t keys, all; // bytes
};
static BeamPlan beam_plan(int64_t rows, int beams, int vocab, int keep)
{
    BeamPlan r {};
    auto thousands = [&](int64_t n, int64_t into) { return (int)((n + into * 1024 - 1) / (into * 1024) * 1024); };
    const int64_t most = ((int64_t)vocab + 4095) / 4096;
    int64_t parts = kBeamGroups / rows < most ? kBeamGroups / rows : most;
    parts = parts < kBeamLists / beams ? parts : kBeamLists / beams;
    parts = parts < 1 ? 1 : (parts > 64 ? 64 : parts);
    r.part_len = thousands(vocab, parts);
    r.parts = (vocab + r.part_len - 1) / r.part_len;
    r.chunk = thousands(r.part_len, (r.part_len + 1024 * kBeamE - 1) / (1024 * kBeamE)); // chunks of a part are of one length
    r.keys = ((size_t)rows * r.parts * keep * sizeof(uint64_t) + 15) & ~(size_t)15;
    r.all = r.keys + (size_t)rows * r.parts * 2 * sizeof(double);
    return r;
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_beam_select_scratch_bytes(int n_seqs, int beams, int vocab, int keep)
{
    if (n_seqs <= 0 || beams <= 0 || vocab <= 0 || keep <= 0)
        return 0;
    return beams <= kMostBeams ? beam_plan((int64_t)n_seqs * beams, beams, vocab, keep).all : 0;
}

extern "C" fdx_status fdx_beam_select_f32(const float* logits, int64_t ld, int n_seqs, int beams, int vocab, const float* scores, const int32_t* done,
    int end_id, int keep, int32_t* parents, int32_t* tokens, float* new_scores, int32_t* new_done, void* scratch_dev, int* error_flag_dev)
{
    FDX_REQUIRE(logits && scores && parents && tokens && new_scores, "beam_select: null pointer");
    FDX_REQUIRE(n_seqs > 0 && beams > 0 && beams <= kMostBeams && (int64_t)n_seqs * beams <= (1 << 23), "beam_select: 1 to 32 beams, up to 2^23 rows");
    FDX_REQUIRE(vocab > 0 && vocab <= (1 << 24), "beam_select: 1 to 2^24 logits a row");
    FDX_REQUIRE(ld >= vocab, "beam_select: rows overlap");
    FDX_REQUIRE(keep > 0 && keep <= kMostTop && keep <= (int64_t)beams * vocab, "beam_select: 1 to 32 continuations, no more than there are");
    FDX_REQUIRE(end_id < vocab && (end_id >= 0 || (!done && !new_done)), "beam_select: end_id is no token");
    FDX_REQUIRE(scratch_dev && (reinterpret_cast<uintptr_t>(scratch_dev) & 15) == 0, "beam_select: scratch missing or not 16-byte aligned");
    const int64_t rows = (int64_t)n_seqs * beams;
    const size_t in_bytes = 4 * (size_t)rows, out_bytes = 4 * (size_t)n_seqs * keep, x_bytes = 4 * ((size_t)(rows - 1) * ld + vocab);
    const void* const outs[] = { new_scores, new_done, parents, tokens }; // the first two may take the place of what a sequence's workgroup has read
    const void* const ins[] = { scores, done };
    for (int i = 0; i < 4; ++i) {
        if (!outs[i])
            continue;
        bool meets = overlap(outs[i], out_bytes, logits, x_bytes);
        for (int j = 0; j < 2; ++j)
            meets = meets || (ins[j] && !(i == j && outs[i] == ins[j] && keep == beams) && overlap(outs[i], out_bytes, ins[j], in_bytes));
        for (int j = i + 1; j < 4; ++j)
            meets = meets || overlap(outs[i], out_bytes, outs[j], out_bytes);
        FDX_REQUIRE(!meets, "beam_select: results overlap an input or each other");
    }
    const BeamPlan plan = beam_plan(rows, beams, vocab, keep);
    int width = 1;
    while (width < plan.parts)
        width *= 2;
    // heads enough for twice as many as are kept, which are fewer than kBeamLists: 2 keep + lists for fewer lists than 2 keep
    const int lists = beams * plan.parts, twice = (2 * keep + lists - 1) / lists, deep = twice < keep ? twice : keep;
    char* scratch = static_cast<char*>(scratch_dev);
    const BeamParams p { logits, ld, beams, vocab, keep, scores, done, end_id, parents, tokens, new_done, new_scores, error_flag_dev,
        reinterpret_cast<uint64_t*>(scratch), reinterpret_cast<double*>(scratch + plan.keys), plan.parts, plan.part_len, plan.chunk, width,
        make_divisor(plan.parts), make_divisor(keep), make_divisor(deep) };
    const dim3 grid((unsigned)(rows * plan.parts));
    profile_begin();
    if (plan.chunk <= 4096)
        hipLaunchKernelGGL(beam_rows_kernel<4>, grid, dim3(256), 0, stream(), p);
    else
        hipLaunchKernelGGL(beam_rows_kernel<kBeamE>, grid, dim3(256), 0, stream(), p);
    hipLaunchKernelGGL(beam_select_kernel, dim3((unsigned)n_seqs), dim3(256), 0, stream(), p);
    profile_end("beam_select_f32", 4.0 * rows * vocab, 4.0 * rows * (double)vocab);
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
