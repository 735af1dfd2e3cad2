// The page table after a selection: sequences go on as copies of others, full pages are shared, partly filled ones get copies.
//
// Which pages are kept is a bit each; the free ones are then the zeros, taken from the lowest on by ranks: of the sequences' needs (a prefix
// sum) and of the zeros (prefix sums over the words' counts), so nothing depends on the order in which threads arrive.  A chain of a dozen
// dependent steps, bound by their latency: one workgroup takes them all where its LDS holds a number for each sequence and a bit for each page
// (64 groups of eight beams, 24 000 entries of the table: 14 us), so that the steps meet at barriers instead of launches.  Larger tables are marked
// by a launch of their own (kSmallEntries).  The copies follow in a launch, at the memory's rate (33 MB read and written 8 us).  Of the 14 us nine are the
// table's passage: more loads of a thread at once, the next ones beside the marks, or a wave's lanes on one sequence took 16 to 20.
#include <climits>

#include "kv8.hpp"

namespace fdx {

struct ForkParams {
    const int32_t *table, *lens, *parents, *grow;
    int32_t *new_table, *new_lens, *free_pages;
    int n_seqs, width, n_pages, max_len;
    Divisor page_size, by_width;
    uint32_t* used;   // a bit a page (these three: of large tables only)
    int32_t* owner;   // of a partly filled page: the first sequence that goes on in it
    int32_t* list;    // free pages that are taken
    int4* plan;       // a sequence: its partly filled page (-1: none), its copy's page (-1: none), filled rows
    int* error_flag;
};

struct Fork {
    int parent, length, want; // positions that it goes on from, and has room for
};
__device__ __forceinline__ Fork fork_of(const ForkParams& p, int i, bool& odd)
{
    const int parent = p.parents[i], more = p.grow ? p.grow[i] : 0;
    odd = parent >= p.n_seqs;
    if (odd || parent < 0)
        return { -1, 0, 0 };
    const int len = p.lens[parent];
    Fork f { parent, len < 0 ? 0 : (len > p.max_len ? p.max_len : len), 0 };
    f.want = more < 0 || more > p.max_len - f.length ? f.length : f.length + more;
    odd = f.length != len || f.want - f.length != more;
    return f;
}

// sum over the workgroup's threads in front of this one, and over all
__device__ __forceinline__ int before_me(int v, int* lds, int& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int sum = wave_prefix(v);
    __syncthreads();
    if (lane == 63)
        lds[wave] = sum;
    __syncthreads();
    int front = 0;
    total = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) {
        front += w < wave ? lds[w] : 0;
        total += lds[w];
    }
    return front + sum - v;
}

__device__ __forceinline__ int agent_load(const int32_t* at) { return __hip_atomic_load(at, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void agent_store(int32_t* at, int v) { __hip_atomic_store(at, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

constexpr int kForkThreads = 1024;
// what a workgroup's LDS is laid out for: a sequence a thread, and a hash table of twice as many pages
constexpr int kSmallSeqs = kForkThreads, kSmallWords = 4096, kHash = 2 * kSmallSeqs;
// Entries of a table (sequences times its width, capacity that nobody uses too) that one workgroup walks, 8192 in some 3 us; marks by a launch of their own
// cost two more launches and dependent loads.  us of the call in one workgroup / through memory: 512 sequences, 6144 entries 14.5 / 21.6, 24 064 18.2 / 30.5,
// 40 960 24.2 / 31.6, 60 416 31.4 / 31.6, 81 920 38.4 / 34.5, 131 072 57.8 / 36.8; 1024 sequences, 61 440 33.7 / 36.9, 131 072 59.6 / 41.4, 260 096 104.3 / 50.9.
constexpr int64_t kSmallEntries = 1 << 16;

// entry j of a sequence in the table: the page that it shares, -1 if none
__device__ __forceinline__ int checked_page(const ForkParams& p, int at, bool& odd)
{
    if (at >= 0 && at < p.n_pages)
        return at;
    odd = true;
    return -1;
}

// where a sequence's new pages begin and end among its entries
struct Entries {
    int full, part, begin, end;
};
__device__ __forceinline__ Entries entries_of(const ForkParams& p, const Fork& f, int page, bool kept)
{
    Entries e;
    e.full = quotient(f.length, p.page_size);
    e.part = f.length - e.full * (int)p.page_size.by;
    e.end = quotient(f.want, p.page_size);
    e.end += f.want > e.end * (int)p.page_size.by;
    e.begin = e.full + (e.part > 0 && (kept || page < 0)); // a partly filled page that is none of the cache has no copy
    return e;
}
__device__ __forceinline__ void write_entries(const ForkParams& p, int i, const Entries& e, int page, bool kept, int rank, int there, const int32_t* list)
{
    int32_t* row = p.new_table + (int64_t)i * p.width;
    if (e.part > 0 && (kept || page < 0))
        row[e.full] = page;
    const int copy = e.part > 0 && !kept && page >= 0 && rank < there ? list[rank] : -1;
    for (int j = e.begin; j < e.end; ++j, ++rank)
        row[j] = rank < there ? list[rank] : -1;
    p.plan[i] = int4 { page, copy, e.part, 0 };
}

// All of it, for up to kSmallSeqs sequences (no more than the workgroup has threads) and 32 kSmallWords pages.
__global__ __launch_bounds__(kForkThreads) void kv_fork_small_kernel(ForkParams p)
{
    __shared__ uint32_t used[kSmallWords];
    __shared__ int32_t parent_of[kSmallSeqs], length_of[kSmallSeqs], page_of[kSmallSeqs], hashed[2 * kHash];
    __shared__ int sums[kForkThreads / 64];
    int32_t *pages = hashed, *first = hashed + kHash; // who is the first to go on in a page
    const int tid = threadIdx.x, threads = blockDim.x, words = (p.n_pages + 31) / 32;
    const bool mine = tid < p.n_seqs;
    bool odd = false;
    Fork f { -1, 0, 0 };
    if (mine) {
        f = fork_of(p, tid, odd);
        parent_of[tid] = f.parent;
        length_of[tid] = f.length;
        page_of[tid] = -1;
        p.new_lens[tid] = f.want;
    }
    for (int w = tid; w < words; w += threads)
        used[w] = 0;
    for (int w = tid; w < kHash; w += threads) {
        pages[w] = -1;
        first[w] = INT_MAX;
    }
    __syncthreads();
    const int entries = p.n_seqs * p.width;
    constexpr int W = 8; // loads of a thread that are on their way together
    struct Entry {
        int seq, at, filled; // rows from this entry's first on
    };
    auto entry = [&](int e) {
        const int seq = quotient(e, p.by_width), at = e - seq * p.width;
        const int64_t left = length_of[seq] - (int64_t)at * (int)p.page_size.by; // tables may be far wider than max_len
        return Entry { seq, at, left > 0 ? (int)left : 0 };
    };
    for (int e0 = tid; e0 < entries; e0 += W * threads) {
        int there[W];
#pragma unroll
        for (int z = 0; z < W; ++z) {
            const int i = e0 + z * threads;
            there[z] = -1;
            if (i < entries) {
                const Entry e = entry(i);
                if (e.filled > 0)
                    there[z] = p.table[(int64_t)parent_of[e.seq] * p.width + e.at];
            }
        }
#pragma unroll
        for (int z = 0; z < W; ++z) {
            const int i = e0 + z * threads;
            if (i >= entries)
                break;
            const Entry e = entry(i);
            const int page = e.filled > 0 ? checked_page(p, there[z], odd) : -1;
            const bool full = e.filled >= (int)p.page_size.by;
            if (full && page >= 0)
                atomicOr(used + (page >> 5), 1u << (page & 31));
            if (e.filled > 0 && !full)
                page_of[e.seq] = page;
            p.new_table[i] = full ? page : -1;
        }
    }
    __syncthreads();
    const int page = mine ? page_of[tid] : -1;
    int slot = 0;
    if (page >= 0) {
        slot = (int)((uint32_t)page * 2654435761u >> 16) & (kHash - 1);
        for (;;) { // half of the places are free
            const int was = atomicCAS(pages + slot, -1, page);
            if (was == -1 || was == page)
                break;
            slot = (slot + 1) & (kHash - 1);
        }
        atomicMin(first + slot, tid);
    }
    __syncthreads();
    // who keeps one: no full page of another's, and the first; the bits are set when all have looked
    const bool kept = page >= 0 && first[slot] == tid && !(used[page >> 5] >> (page & 31) & 1);
    const Entries e = entries_of(p, f, page, kept);
    int needed;
    const int rank = before_me(mine ? e.end - e.begin : 0, sums, needed);
    if (kept)
        atomicOr(used + (page >> 5), 1u << (page & 31));
    __syncthreads();
    // the free pages, by rank, into what the hash table had if they fit
    int32_t* list = needed <= 2 * kHash ? hashed : p.list;
    int ranked = 0;
    for (int w0 = 0; w0 < words; w0 += threads) {
        const int w = w0 + tid;
        uint32_t zeros = w < words ? ~used[w] : 0;
        if (w == words - 1 && p.n_pages % 32)
            zeros &= (1u << (p.n_pages % 32)) - 1;
        int total;
        int r = ranked + before_me(__builtin_popcount(zeros), sums, total);
        ranked += total;
        for (; zeros && r < needed; zeros &= zeros - 1)
            list[r++] = w * 32 + __builtin_ctz(zeros);
    }
    __syncthreads();
    const int there = needed < ranked ? needed : ranked;
    if (mine)
        write_entries(p, tid, e, page, kept, rank, there, list);
    if ((odd || needed > ranked) && p.error_flag)
        *p.error_flag = 1;
    if (tid == 0 && p.free_pages)
        *p.free_pages = ranked - there;
}

// The same for tables of any size, through memory: the bits are cleared, the shared pages marked by as many workgroups as there are entries for, and one
// workgroup does the rest.
__global__ __launch_bounds__(256) void kv_fork_clear_kernel(ForkParams p)
{
    const int64_t w = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (w < (p.n_pages + 31) / 32)
        p.used[w] = 0;
}

__global__ __launch_bounds__(256) void kv_fork_mark_kernel(ForkParams p)
{
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= (int64_t)p.n_seqs * p.width)
        return;
    const int i = quotient((int)e, p.by_width), j = (int)(e - (int64_t)i * p.width);
    bool odd, bad = false;
    const Fork f = fork_of(p, i, odd);
    int at = -1;
    if (j < quotient(f.length, p.page_size)) {
        at = checked_page(p, p.table[(int64_t)f.parent * p.width + j], bad);
        if (at >= 0)
            atomicOr(p.used + (at >> 5), 1u << (at & 31));
    }
    p.new_table[e] = at;
    if (bad && p.error_flag)
        *p.error_flag = 1;
}

__global__ __launch_bounds__(kForkThreads) void kv_fork_rest_kernel(ForkParams p)
{
    __shared__ int sums[kForkThreads / 64];
    const int tid = threadIdx.x, words = (p.n_pages + 31) / 32;
    int32_t* bits = reinterpret_cast<int32_t*>(p.used);
    bool odd = false;
    for (int i = tid; i < p.n_seqs; i += kForkThreads) {
        bool bad;
        const Fork f = fork_of(p, i, bad);
        odd = odd || bad;
        const int full = quotient(f.length, p.page_size);
        int at = -1;
        if (f.length > full * (int)p.page_size.by) {
            at = checked_page(p, p.table[(int64_t)f.parent * p.width + full], odd);
            if (at >= 0)
                agent_store(p.owner + at, INT_MAX);
        }
        p.plan[i].x = at;
        p.new_lens[i] = f.want;
    }
    __syncthreads();
    for (int i = tid; i < p.n_seqs; i += kForkThreads)
        if (p.plan[i].x >= 0)
            atomicMin(p.owner + p.plan[i].x, i);
    __syncthreads();
    for (int i = tid; i < p.n_seqs; i += kForkThreads) {
        const int at = p.plan[i].x;
        p.plan[i].w = at >= 0 && agent_load(p.owner + at) == i && !(agent_load(bits + (at >> 5)) >> (at & 31) & 1);
    }
    __syncthreads();
    int needed = 0;
    for (int i0 = 0; i0 < p.n_seqs; i0 += kForkThreads) {
        const int i = i0 + tid;
        int need = 0;
        if (i < p.n_seqs) {
            bool bad;
            const Entries e = entries_of(p, fork_of(p, i, bad), p.plan[i].x, p.plan[i].w);
            need = e.end - e.begin;
            if (p.plan[i].w)
                atomicOr(p.used + (p.plan[i].x >> 5), 1u << (p.plan[i].x & 31));
        }
        int total;
        const int front = before_me(need, sums, total);
        if (i < p.n_seqs)
            p.plan[i].z = needed + front;
        needed += total;
    }
    __syncthreads();
    int ranked = 0;
    for (int w0 = 0; w0 < words; w0 += kForkThreads) {
        const int w = w0 + tid;
        uint32_t zeros = w < words ? ~(uint32_t)agent_load(bits + w) : 0;
        if (w == words - 1 && p.n_pages % 32)
            zeros &= (1u << (p.n_pages % 32)) - 1;
        int total;
        int r = ranked + before_me(__builtin_popcount(zeros), sums, total);
        ranked += total;
        for (; zeros && r < needed; zeros &= zeros - 1)
            p.list[r++] = w * 32 + __builtin_ctz(zeros);
    }
    __syncthreads();
    const int there = needed < ranked ? needed : ranked;
    for (int i = tid; i < p.n_seqs; i += kForkThreads) {
        bool bad;
        const int4 plan = p.plan[i];
        write_entries(p, i, entries_of(p, fork_of(p, i, bad), plan.x, plan.w), plan.x, plan.w, plan.z, there, p.list);
    }
    if ((odd || needed > ranked) && p.error_flag)
        *p.error_flag = 1;
    if (tid == 0 && p.free_pages)
        *p.free_pages = ranked - there;
}

struct ForkCopyParams {
    const int4* plan;
    char *k, *v;
    float *k_scale, *v_scale;
    int64_t k_row, v_row;      // bytes
    int page_size, block, kv_heads; // block 0: no scales
    int wide;                  // rows are whole 16-byte vectors
};

constexpr int kCopyThreads = 256, kCopyBytes = 16384;

// `bytes` bytes in vectors of T, four of a thread on their way together
template <typename T>
__device__ __forceinline__ void copy_bytes(const char* from, char* to, int bytes)
{
    constexpr int W = 4, kStep = kCopyThreads * (int)sizeof(T);
    for (int at = threadIdx.x * (int)sizeof(T); at < bytes; at += W * kStep) {
        T x[W];
#pragma unroll
        for (int i = 0; i < W; ++i)
            x[i] = *reinterpret_cast<const T*>(from + (at + i * kStep < bytes ? at + i * kStep : at));
#pragma unroll
        for (int i = 0; i < W; ++i)
            if (at + i * kStep < bytes)
                *reinterpret_cast<T*>(to + at + i * kStep) = x[i];
    }
}

// A workgroup takes 16 KB of the filled rows of one sequence's page, of keys (z 0) or values (z 1).
__global__ __launch_bounds__(kCopyThreads) void kv_fork_copy_kernel(ForkCopyParams p)
{
    const int4 plan = p.plan[blockIdx.x];
    if (plan.y < 0 || plan.x < 0 || plan.z <= 0)
        return;
    const bool values = blockIdx.z > 0;
    const int64_t row = values ? p.v_row : p.k_row, all = plan.z * row;
    const int64_t from = (int64_t)plan.x * p.page_size * row, to = (int64_t)plan.y * p.page_size * row;
    char* base = values ? p.v : p.k;
    for (int64_t first = (int64_t)blockIdx.y * kCopyBytes; first < all; first += (int64_t)gridDim.y * kCopyBytes) {
        const int bytes = all - first < kCopyBytes ? (int)(all - first) : kCopyBytes;
        if (p.wide)
            copy_bytes<f32x4>(base + from + first, base + to + first, bytes);
        else
            copy_bytes<char>(base + from + first, base + to + first, bytes);
    }
    if (p.block > 0 && blockIdx.y == 0) {
        float* scales = values ? p.v_scale : p.k_scale;
        const int64_t a_page = (int64_t)(p.page_size / p.block) * p.kv_heads, count = (int64_t)((plan.z + p.block - 1) / p.block) * p.kv_heads;
        for (int64_t i = threadIdx.x; i < count; i += kCopyThreads)
            scales[plan.y * a_page + i] = scales[plan.x * a_page + i];
    }
}

struct ForkScratch {
    size_t used, owner, list, plan, all;
};
static ForkScratch fork_scratch(const fdx_kv_pages* c)
{
    auto round = [](size_t n) { return (n + 15) & ~(size_t)15; };
    ForkScratch r;
    r.used = 0;
    r.owner = round(((size_t)c->n_pages + 31) / 32 * 4);
    r.list = r.owner + round((size_t)c->n_pages * 4);
    r.plan = r.list + round((size_t)c->n_pages * 4);
    r.all = r.plan + (size_t)c->n_seqs * sizeof(int4);
    return r;
}

static fdx_status fork_launch(const char* who, const fdx_kv_pages* c, size_t size, const fdx_kv_pages8* eight, const int32_t* parents,
    const int32_t* grow, int32_t* new_table, int32_t* new_lens, int32_t* free_pages, void* scratch_dev, int* error_flag_dev)
{
    FDX_REQUIRE(parents && new_table && new_lens, "%s: null pointer", who);
    FDX_REQUIRE(c->n_seqs <= (1 << 23), "%s: more than 2^23 sequences", who);
    FDX_REQUIRE((int64_t)c->n_seqs * c->table_width < ((int64_t)1 << 31), "%s: a table of more than 2^31 entries", who);
    FDX_REQUIRE(scratch_dev && (reinterpret_cast<uintptr_t>(scratch_dev) & 15) == 0, "%s: scratch missing or not 16-byte aligned", who);
    const size_t table_bytes = (size_t)c->n_seqs * c->table_width * 4, lens_bytes = (size_t)c->n_seqs * 4;
    const struct {
        const void* at;
        size_t bytes;
    } tensors[] = { { new_table, table_bytes }, { new_lens, lens_bytes }, { free_pages, free_pages ? 4u : 0u }, { c->table, table_bytes },
        { c->lens, lens_bytes }, { parents, lens_bytes }, { grow, grow ? lens_bytes : 0 } };
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 7; ++j)
            FDX_REQUIRE(!overlap(tensors[i].at, tensors[i].bytes, tensors[j].at, tensors[j].bytes),
                "%s: the new table, the new lengths or free_pages overlap an input or each other", who);
    const ForkScratch at = fork_scratch(c);
    char* scratch = static_cast<char*>(scratch_dev);
    const ForkParams p { c->table, c->lens, parents, grow, new_table, new_lens, free_pages, c->n_seqs, c->table_width, c->n_pages, c->max_len,
        make_divisor(c->page_size), make_divisor(c->table_width), reinterpret_cast<uint32_t*>(scratch + at.used),
        reinterpret_cast<int32_t*>(scratch + at.owner), reinterpret_cast<int32_t*>(scratch + at.list), reinterpret_cast<int4*>(scratch + at.plan),
        error_flag_dev };
    const int64_t k_row = (int64_t)c->kv_heads * c->dk * (int64_t)size, v_row = (int64_t)c->kv_heads * c->dv * (int64_t)size;
    const bool wide = ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v) | (uintptr_t)k_row | (uintptr_t)v_row) & 15) == 0;
    const ForkCopyParams copy { p.plan, static_cast<char*>(c->k), static_cast<char*>(c->v), eight ? eight->k_scale : nullptr,
        eight ? eight->v_scale : nullptr, k_row, v_row, c->page_size, eight ? eight->block : 0, c->kv_heads, wide };
    const int64_t parts = ((k_row > v_row ? k_row : v_row) * c->page_size + kCopyBytes - 1) / kCopyBytes;
    profile_begin();
    const int64_t entries = (int64_t)c->n_seqs * c->table_width;
    if (c->n_seqs <= kSmallSeqs && c->n_pages <= 32 * kSmallWords && entries <= kSmallEntries) {
        const int threads = entries <= 2048 && c->n_seqs <= 256 ? 256 : kForkThreads; // barriers of four waves take less
        hipLaunchKernelGGL(kv_fork_small_kernel, dim3(1), dim3(threads), 0, stream(), p);
    } else {
        hipLaunchKernelGGL(kv_fork_clear_kernel, dim3((unsigned)(((int64_t)c->n_pages + 31) / 32 + 255) / 256), dim3(256), 0, stream(), p);
        hipLaunchKernelGGL(kv_fork_mark_kernel, dim3((unsigned)((entries + 255) / 256)), dim3(256), 0, stream(), p);
        hipLaunchKernelGGL(kv_fork_rest_kernel, dim3(1), dim3(kForkThreads), 0, stream(), p);
    }
    hipLaunchKernelGGL(kv_fork_copy_kernel, dim3((unsigned)c->n_seqs, (unsigned)(parts < 64 ? parts : 64), 2), dim3(kCopyThreads), 0, stream(), copy);
    profile_end("kv_fork", 0.0, 2.0 * table_bytes);
    FDX_LAUNCH_CHECK();
    return FDX_OK;
}

} // namespace fdx

using namespace fdx;

extern "C" size_t fdx_kv_fork_scratch_bytes(const fdx_kv_pages* cache)
{
    return cache && cache->n_pages > 0 && cache->n_seqs > 0 ? fork_scratch(cache).all : 0;
}
extern "C" size_t fdx_kv8_fork_scratch_bytes(const fdx_kv_pages8* cache) { return cache ? fdx_kv_fork_scratch_bytes(&cache->pages) : 0; }

extern "C" fdx_status fdx_kv_fork(const fdx_kv_pages* cache, const int32_t* parents, const int32_t* grow, int32_t* new_table, int32_t* new_lens,
    int32_t* free_pages, void* scratch_dev, int* error_flag_dev)
{
    const fdx_status st = check_kv_pages("kv_fork", cache);
    return st != FDX_OK ? st : fork_launch("kv_fork", cache, cache->type == FDX_KV_BF16 ? 2 : 4, nullptr, parents, grow, new_table, new_lens,
        free_pages, scratch_dev, error_flag_dev);
}

extern "C" fdx_status fdx_kv8_fork(const fdx_kv_pages8* cache, const int32_t* parents, const int32_t* grow, int32_t* new_table, int32_t* new_lens,
    int32_t* free_pages, void* scratch_dev, int* error_flag_dev)
{
    const fdx_status st = check_kv_pages8("kv8_fork", cache);
    return st != FDX_OK ? st : fork_launch("kv8_fork", &cache->pages, 1, cache, parents, grow, new_table, new_lens, free_pages, scratch_dev,
        error_flag_dev);
}
