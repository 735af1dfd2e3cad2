// The best continuations of a sequence's beams over the vocabulary.
#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace fdx {

constexpr int kMostKeep = 32, kMostBeams = 32;

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
    double* sums;   // [row]: log of the sum of exponentials
    uint64_t* keys; // [row][keep]
};

// Order of a row's tokens: descending logit, then ascending id.  Larger keys come first, 0 is no token.
__device__ __forceinline__ uint32_t logit_bits(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f); // -0 and +0 are equal logits
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bits_logit(uint32_t b) { return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b); }

// A workgroup takes a row: its sum, then its best tokens one after another.
__global__ __launch_bounds__(256) void beam_rows_kernel(BeamParams p)
{
    __shared__ double sum_of[256];
    __shared__ uint64_t best_of[256];
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x;
    const float* x = p.x + row * p.ld;
    if (p.done && p.done[row])
        return;
    float m = -INFINITY;
    bool odd = false;
    for (int i = tid; i < p.vocab; i += 256) {
        m = fmaxf(m, x[i]);
        odd = odd || !(x[i] < INFINITY);
    }
    odd = __syncthreads_or(odd);
    sum_of[tid] = m;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if (tid < w)
            sum_of[tid] = fmax(sum_of[tid], sum_of[tid + w]);
        __syncthreads();
    }
    m = (float)sum_of[0];
    __syncthreads();
    double z = 0.0;
    for (int i = tid; i < p.vocab; i += 256)
        z += exp((double)x[i] - (double)m);
    sum_of[tid] = z;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if (tid < w)
            sum_of[tid] += sum_of[tid + w];
        __syncthreads();
    }
    if (tid == 0) {
        p.sums[row] = (double)m + log(sum_of[0]);
        if (odd && p.error_flag)
            *p.error_flag = 1;
    }
    uint64_t before = ~(uint64_t)0;
    for (int j = 0; j < p.keep; ++j) {
        uint64_t best = 0;
        for (int i = tid; i < p.vocab; i += 256) {
            const uint64_t key = (uint64_t)logit_bits(x[i]) << 32 | (uint32_t)~i;
            best = x[i] > -INFINITY && !odd && key < before && key > best ? key : best;
        }
        __syncthreads();
        best_of[tid] = best;
        __syncthreads();
        for (int w = 128; w > 0; w >>= 1) {
            if (tid < w && best_of[tid + w] > best_of[tid])
                best_of[tid] = best_of[tid + w];
            __syncthreads();
        }
        before = best_of[0];
        if (tid == 0)
            p.keys[row * p.keep + j] = before;
    }
}

// A wave takes a sequence: the best of its beams' next ones, one after another.
__global__ __launch_bounds__(64) void beam_select_kernel(BeamParams p)
{
    const int s = blockIdx.x, lane = threadIdx.x;
    const int64_t row = (int64_t)s * p.beams + lane;
    bool ended = false, live = lane < p.beams;
    double before = 0.0, log_sum = 0.0;
    if (live) {
        before = p.scores[row];
        ended = p.done && p.done[row];
        const bool odd = !(before < INFINITY);
        if (odd && p.error_flag)
            *p.error_flag = 1;
        live = before > -INFINITY && !odd;
        log_sum = ended ? 0.0 : p.sums[row];
    }
    int next = 0;
    for (int j = 0; j < p.keep; ++j) {
        double total = -INFINITY;
        int token = -1;
        if (live && ended) {
            token = p.end_id;
            total = next == 0 ? before : -INFINITY;
        } else if (live && next < p.keep) {
            const uint64_t key = p.keys[row * p.keep + next];
            token = (int)~(uint32_t)key;
            total = key ? before + ((double)bits_logit((uint32_t)(key >> 32)) - log_sum) : -INFINITY;
        }
        double best = total;
        int who = lane;
        for (int w = 32; w > 0; w >>= 1) {
            const double o = __shfl_xor(best, w, 64);
            const int ow = __shfl_xor(who, w, 64);
            if (o > best || (o == best && ow < who)) {
                best = o;
                who = ow;
            }
        }
        const bool there = best > -INFINITY;
        if (lane == who) {
            const int64_t at = (int64_t)s * p.keep + j;
            p.parents[at] = there ? (int)row : -1;
            p.tokens[at] = there ? token : -1;
            p.new_scores[at] = (float)best;
            if (p.new_done)
                p.new_done[at] = there && (ended || token == p.end_id);
            ++next;
        }
    }
}

} // namespace fdx

using namespace fdx;

static size_t beam_sums(int64_t rows) { return ((size_t)rows * sizeof(double) + 15) & ~(size_t)15; }

extern "C" size_t fdx_beam_select_scratch_bytes(int n_seqs, int beams, int vocab, int keep)
{
    if (n_seqs <= 0 || beams <= 0 || vocab <= 0 || keep <= 0)
        return 0;
    const int64_t rows = (int64_t)n_seqs * beams;
    return beam_sums(rows) + (size_t)rows * keep * sizeof(uint64_t);
}

extern "C" fdx_status fdx_beam_select_f32(const float* logits, int64_t ld, int n_seqs, int beams, int vocab, const float* scores, const int32_t* done,
    int end_id, int keep, int32_t* parents, int32_t* tokens, float* new_scores, int32_t* new_done, void* scratch_dev, int* error_flag_dev)
{
    FDX_REQUIRE(logits && scores && parents && tokens && new_scores, "beam_select: null pointer");
    FDX_REQUIRE(n_seqs > 0 && beams > 0 && beams <= kMostBeams && (int64_t)n_seqs * beams <= (1 << 23), "beam_select: 1 to 32 beams, up to 2^23 rows");
    FDX_REQUIRE(vocab > 0 && vocab <= (1 << 24), "beam_select: 1 to 2^24 logits a row");
    FDX_REQUIRE(ld >= vocab, "beam_select: rows overlap");
    FDX_REQUIRE(keep > 0 && keep <= kMostKeep && keep <= (int64_t)beams * vocab, "beam_select: 1 to 32 continuations, no more than there are");
    FDX_REQUIRE(end_id < vocab && (end_id >= 0 || (!done && !new_done)), "beam_select: end_id is no token");
    FDX_REQUIRE(scratch_dev && (reinterpret_cast<uintptr_t>(scratch_dev) & 15) == 0, "beam_select: scratch missing or not 16-byte aligned");
    const int64_t rows = (int64_t)n_seqs * beams;
    char* scratch = static_cast<char*>(scratch_dev);
    const BeamParams p { logits, ld, beams, vocab, keep, scores, done, end_id, parents, tokens, new_done, new_scores, error_flag_dev,
        reinterpret_cast<double*>(scratch), reinterpret_cast<uint64_t*>(scratch + beam_sums(rows)) };
    profile_begin();
    hipLaunchKernelGGL(beam_rows_kernel, dim3((unsigned)rows), dim3(256), 0, stream(), p);
    hipLaunchKernelGGL(beam_select_kernel, dim3((unsigned)n_seqs), dim3(64), 0, stream(), p);
    profile_end("beam_select_f32", 4.0 * rows * vocab, 4.0 * rows * (double)vocab);
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
