// The likeliest tokens of rows of logits, for kernels whose workgroups of 256 threads take a row, or a part of one, in chunks.
//
// The best `top` tokens of a wave are a sorted list in LDS.  Of a chunk, `top` lanes' largest logits are a threshold that no fewer than `top` tokens
// reach: it is found bit by bit with votes on the lanes' largest, and stops as soon as not many more lanes than that pass.  On
// random logits about as many tokens pass as are asked for; they and the list so far are ordered by counting, for each, the better ones.
// Where more pass than there is room for (equal logits), the best are taken one at a time.  Only finite logits are listed.  Lists of waves and of
// parts meet in pairs, an item's place being its place in its own list plus the number of better ones in the other.
#pragma once
#include <cmath>
#include <cstdint>

#include "common.hpp"

namespace fdx {

constexpr int kMostTop = 32, kFound = 192;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4))); // rows start at any multiple of four bytes

// Order of the likeliest tokens: descending logit, then ascending id.  Larger keys come first, 0 is no token.
__device__ __forceinline__ uint32_t score_bits(float x)
{
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f); // -0 and +0 are equal logits
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float bits_score(uint32_t b) { return __builtin_bit_cast(float, b & 0x80000000u ? b & 0x7fffffffu : ~b); }

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

// a chunk's logits c0 .. end - 1, 4 E a thread, -infinity behind them
template <int E>
__device__ __forceinline__ void load_chunk(const float* x, int c0, int end, f32x4 (&v)[E])
{
    const int tid = threadIdx.x;
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
}
// the largest of a thread's logits
template <int E>
__device__ __forceinline__ float most_of_chunk(const f32x4 (&v)[E], int c0, int end)
{
    float best = -INFINITY;
#pragma unroll
    for (int j = 0; j < E; ++j)
        if (c0 + j * 256 * 4 < end)
            best = fmaxf(fmaxf(fmaxf(best, v[j][0]), fmaxf(v[j][1], v[j][2])), v[j][3]);
    return best;
}

// A wave's list and a spare one behind it, room for a chunk's candidates, and the logit of a full list's last token (0: it is not full).
struct TopList {
    uint64_t *list, *spare, *found;
    uint32_t worst;
};
// adds a chunk to it; best: the thread's largest logit
template <int E>
__device__ __forceinline__ void add_chunk(TopList& t, int top, const f32x4 (&v)[E], int c0, int end, float best)
{
    const int tid = threadIdx.x, lane = tid & 63;
    const uint32_t mine = best > -INFINITY ? score_bits(best) : 0;
    if (__ballot(mine > t.worst)) {
        uint32_t cut = t.worst + 1; // equal logits: those of lower ids are in the list already
        if (t.worst == 0) {
            cut = 0;
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                const int pass = __builtin_popcountll(__ballot(mine >= (cut | bit)));
                cut = pass >= top ? cut | bit : cut;
                if (pass >= top && pass <= top + 4)
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
                            t.found[at] = (uint64_t)score_bits(v[j][e]) << 32 | (uint32_t)~(c0 + (j * 256 + tid) * 4 + e);
                        count += __builtin_popcountll(in);
                    }
                }
            }
        if (count > kFound) { // the best ones, one at a time
            uint64_t before = ~(uint64_t)0;
            count = 0;
            while (count < top) {
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
                    t.found[count] = before;
                ++count;
            }
        }
        if (count > 0) {
            wave_lds_fence();
            if (lane < top)
                t.spare[lane] = 0;
            wave_lds_fence();
            for (int i = lane; i < top + count; i += 64) {
                const uint64_t key = i < top ? t.list[i] : t.found[i - top];
                int place = 0;
#pragma unroll 4
                for (int k = 0; k < top; ++k)
                    place += t.list[k] > key;
#pragma unroll 4
                for (int k = 0; k < count; ++k)
                    place += t.found[k] > key;
                if (key != 0 && place < top)
                    t.spare[place] = key;
            }
            wave_lds_fence();
            uint64_t* const was = t.list;
            t.list = t.spare;
            t.spare = was;
            t.worst = (uint32_t)(uniform_key(t.list[top - 1]) >> 32);
        }
    }
}

} // namespace fdx
