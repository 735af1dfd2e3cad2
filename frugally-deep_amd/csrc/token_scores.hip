// Log probabilities of given tokens, entropy and the likeliest tokens of each row of logits.
//
//   m = max x, Z = sum e^(x - m), log p[i] = x[i] - m - log Z, H = log Z - sum e^(x - m) (x - m) / Z
// Both terms of H are at least zero, so nothing cancels.
#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace fdx {

constexpr int kMostTop = 32;

struct ScoreParams {
    const float* x;
    int64_t ld, rows;
    int vocab, top;
    const int32_t* ids;
    float *logprobs, *entropy, *top_logprobs;
    int32_t* top_ids;
    int* error_flag;
};

// Order of the likeliest tokens: descending logit, NaN below all, then ascending id.  Larger keys come first; no two are equal.
__device__ __forceinline__ uint64_t score_key(float x, int id)
{
    uint32_t b = __builtin_bit_cast(uint32_t, x == 0.f ? 0.f : x); // -0 and +0 are equal logits
    b = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)(x != x ? 0u : b) << 32 | (uint32_t)~id;
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

// a workgroup a row, a pass for each thing
__global__ __launch_bounds__(256) void token_scores_kernel(ScoreParams p)
{
    __shared__ float red[3][4];
    __shared__ uint64_t best[4];
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, wave = tid >> 6;
    const float* x = p.x + r * p.ld;
    float m = -INFINITY;
    bool odd = false;
    for (int i = tid; i < p.vocab; i += 256) {
        m = fmaxf(m, x[i]);
        odd = odd || !(x[i] < INFINITY);
    }
    m = wave_all<true>(m);
    if ((tid & 63) == 0)
        red[0][wave] = m;
    odd = __syncthreads_or(odd);
    m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    const float m_use = m == -INFINITY ? 0.f : m;
    float z = 0.f, w = 0.f;
    for (int i = tid; i < p.vocab; i += 256) {
        const float d = x[i] - m_use, e = expf(d);
        z += e;
        w += e > 0.f ? e * d : 0.f;
    }
    z = wave_all<false>(z);
    w = wave_all<false>(w);
    if ((tid & 63) == 0) {
        red[1][wave] = z;
        red[2][wave] = w;
    }
    __syncthreads();
    z = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    w = red[2][0] + red[2][1] + red[2][2] + red[2][3];
    const float lz = odd ? NAN : (z > 0.f ? logf(z) : 0.f);
    if (tid == 0) {
        if (p.ids) {
            const int id = p.ids[r];
            p.logprobs[r] = id < 0 ? 0.f : (id >= p.vocab ? NAN : (x[id] - m_use) - lz);
            if (id >= p.vocab && p.error_flag)
                *p.error_flag = 1;
        }
        if (p.entropy)
            p.entropy[r] = odd ? NAN : (z > 0.f ? lz - w / z : 0.f);
    }
    uint64_t last = ~(uint64_t)0;
    for (int j = 0; j < p.top; ++j) {
        uint64_t b = 0;
        for (int i = tid; i < p.vocab; i += 256) {
            const uint64_t key = score_key(x[i], i);
            if (key < last && key > b)
                b = key;
        }
        b = wave_max_key(b);
        __syncthreads();
        if ((tid & 63) == 0)
            best[wave] = b;
        __syncthreads();
        for (int i = 0; i < 4; ++i)
            b = best[i] > b ? best[i] : b;
        last = b;
        if (tid == 0) {
            const int id = (int)~(uint32_t)b;
            p.top_ids[r * p.top + j] = id;
            p.top_logprobs[r * p.top + j] = (x[id] - m_use) - lz;
        }
    }
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_token_logprobs_scratch_bytes(int64_t rows, int vocab, int top)
{
    (void)rows; (void)vocab; (void)top;
    return 0;
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
    const ScoreParams p { logits, ld, rows, vocab, top, ids, logprobs, entropy, top_logprobs, top_ids, error_flag_dev };
    profile_begin();
    hipLaunchKernelGGL(token_scores_kernel, dim3((unsigned)rows), dim3(256), 0, stream(), p);
    profile_end("token_logprobs_f32", 5.0 * rows * vocab, 4.0 * rows * ((double)vocab + 3 + 2 * top));
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}
