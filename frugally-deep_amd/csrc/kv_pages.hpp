// Where the rows of ragged batches lie: spans of packed rows, tiles of them, places in a paged cache.  Plain integer
// arithmetic on numbers that device memory holds and nobody has checked: whatever they are, what comes out is in range.
#pragma once
#include <cstdint>

#if defined(__HIPCC__)
#define FDX_HD __host__ __device__ __forceinline__
#else
#define FDX_HD inline
#endif

namespace fdx {

// Quotients by a number that a launch does not change, as a product: with 2^l >= by, mul = floor(2^(31+l) / by) + 1 is off from 2^(31+l) / by
// by at most 1, so n mul / 2^(31+l) from n / by by less than 1 / by for n < 2^31.
struct Divisor {
    uint32_t by, mul;
    int shift;
};
inline Divisor make_divisor(int by)
{
    int l = 0;
    while (((int64_t)1 << l) < by)
        ++l;
    return { (uint32_t)by, (uint32_t)(((uint64_t)1 << (31 + l)) / (uint32_t)by + 1), 31 + l };
}
FDX_HD int quotient(int n, const Divisor& d) { return (int)((uint64_t)(uint32_t)n * d.mul >> d.shift); }

struct Span {
    int first, count;
};

// rows starts[i] .. starts[i + 1] - 1, cut to 0 .. tokens - 1
FDX_HD Span packed_span(const int32_t* starts, int i, int tokens)
{
    int a = starts[i], b = starts[i + 1];
    a = a < 0 ? 0 : (a > tokens ? tokens : a);
    b = b < a ? a : (b > tokens ? tokens : b);
    return { a, b - a };
}

FDX_HD bool packed_start_ok(const int32_t* starts, int i, int tokens)
{
    return starts[i] >= 0 && starts[i] <= starts[i + 1] && starts[i + 1] <= tokens;
}

// Tiles of `rows` rows over sequences that bring `per_token` rows a token, without a pass that adds up lengths: sequence i owns
// the numbers from starts[i] * per_token / rows + i up to the next sequence's, which are at least as many as it has tiles
// (floor(x + y) + 1 - floor(x) >= ceil(y)).  The numbers that are left over are no tile.
FDX_HD int64_t first_tile(int start, int i, int per_token, int rows) { return (int64_t)start * per_token / rows + i; }

FDX_HD int64_t tile_numbers(int tokens, int n_seqs, int per_token, int rows) { return first_tile(tokens, n_seqs, per_token, rows); }

struct Tile {
    int seq, index; // sequence (-1: no tile), tile inside it
    Span span;
};

// The searches are a wave's: sixty-four places are looked at together, where a binary search waits for memory once a step.  Wave has
// count(f), mask(f), sum(f) and most(f) over f(0) .. f(63), and kept(f), numbers that each lane has worked out once.
//
// how many of the places 0 .. n - 1 are not above, where those are the first ones; whatever they are, 0 .. n
template <class Wave, class NotAbove>
FDX_HD int not_above(const Wave& wave, int n, const NotAbove& f)
{
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 63) >> 6, from = lo, to = hi;
        const int count = wave.count([&](int lane) { return from + lane * step < to && f(from + lane * step); });
        const int next = lo + count * step;
        if (step == 1)
            return next;
        hi = next < hi ? next : hi;
        lo = count > 0 ? next - step + 1 : hi;
    }
    return lo;
}

template <class Wave>
FDX_HD Tile find_tile(const Wave& wave, const int32_t* starts, int n_seqs, int tokens, int per_token, int rows, int64_t number)
{
    Tile t { not_above(wave, n_seqs,
                 [&](int i) {
                     const int a = starts[i];
                     return first_tile(a < 0 ? 0 : (a > tokens ? tokens : a), i, per_token, rows) <= number;
                 }) - 1,
        0, { 0, 0 } };
    if (t.seq < 0)
        return t;
    t.span = packed_span(starts, t.seq, tokens);
    const int64_t index = number - first_tile(t.span.first, t.seq, per_token, rows);
    if (index < 0 || index * rows >= (int64_t)t.span.count * per_token)
        t.seq = -1;
    t.index = (int)index;
    return t;
}

// find_tile for up to sixty-four sequences, numbered the other way: tiles furthest inside their sequences first, which see most keys.
// before(j) = tiles of index j and more; the tile with `number` tiles in front of it has the index j with before(j + 1) <= number < before(j).
template <class Wave>
FDX_HD Tile late_tile(const Wave& wave, const int32_t* starts, int n_seqs, int tokens, int per_token, int rows, int64_t number)
{
    const auto kept = wave.kept([&](int lane) {
        return lane < n_seqs ? (int)(((int64_t)packed_span(starts, lane, tokens).count * per_token + rows - 1) / rows) : 0;
    });
    // exact below 2^24: tokens * heads is at most 2^25
    auto before = [&](int j) { return (int64_t)wave.sum([&](int lane) { return (float)(kept.at(lane) > j ? kept.at(lane) - j : 0); }); };
    Tile t { -1, 0, { 0, 0 } };
    if (number >= before(0))
        return t;
    int lo = 0, hi = (int)wave.most([&](int lane) { return (float)kept.at(lane); }); // before(lo) > number >= before(hi)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (before(mid) > number)
            lo = mid;
        else
            hi = mid;
    }
    uint64_t of = wave.mask([&](int lane) { return kept.at(lane) > lo; });
    for (int skip = (int)(number - before(lo + 1)); skip > 0 && of; --skip)
        of &= of - 1;
    if (of == 0) // sequences that overlap: more tiles than there are rows, too many to count
        return t;
    t.seq = __builtin_ctzll(of);
    t.index = lo;
    t.span = packed_span(starts, t.seq, tokens);
    return t;
}

// the sequence that row `row` belongs to, -1 if none
template <class Wave>
FDX_HD int find_row(const Wave& wave, const int32_t* starts, int n_seqs, int tokens, int row)
{
    const int i = not_above(wave, n_seqs, [&](int at) { return starts[at] <= row; }) - 1;
    if (i < 0)
        return -1;
    const Span s = packed_span(starts, i, tokens);
    return row >= s.first && row - s.first < s.count ? i : -1;
}

// row of position `pos` among the rows of all pages, -1 if the table does not reach it or names no page of the cache
FDX_HD int page_row(const int32_t* table_row, int table_width, int n_pages, const Divisor& page_size, int pos)
{
    if (pos < 0)
        return -1;
    const int at = quotient(pos, page_size);
    if (at >= table_width)
        return -1;
    const int page = table_row[at];
    return page < 0 || page >= n_pages ? -1 : page * (int)page_size.by + (pos - at * (int)page_size.by);
}

} // namespace fdx
