// The arithmetic of ragged batches and page tables on host memory, with whatever numbers a caller's device memory might hold: run
// under the address sanitizer, every array exactly as long as the device's.
#include <algorithm>
#include <climits>
#include <cstdio>
#include <random>
#include <vector>

#include "kv_pages.hpp"

using namespace fdx;

#define CHECK(c)                                                                                                                          \
    do {                                                                                                                                  \
        if (!(c)) {                                                                                                                       \
            std::printf("failed at line %d: %s\n", __LINE__, #c);                                                                         \
            return 1;                                                                                                                     \
        }                                                                                                                                 \
    } while (0)

// a wave's sixty-four lanes, one after another
struct HostWave {
    struct Kept {
        std::vector<int> all;
        int at(int lane) const { return all[lane]; }
    };
    template <class F>
    Kept kept(const F& f) const
    {
        Kept k;
        for (int lane = 0; lane < 64; ++lane)
            k.all.push_back(f(lane));
        return k;
    }
    template <class F>
    uint64_t mask(const F& f) const
    {
        uint64_t m = 0;
        for (int lane = 0; lane < 64; ++lane)
            m |= (uint64_t)(f(lane) ? 1 : 0) << lane;
        return m;
    }
    template <class F>
    int count(const F& f) const { return __builtin_popcountll(mask(f)); }
    template <class F>
    float sum(const F& f) const
    {
        float s = 0.f;
        for (int lane = 0; lane < 64; ++lane)
            s += f(lane);
        return s;
    }
    template <class F>
    float most(const F& f) const
    {
        float m = f(0);
        for (int lane = 1; lane < 64; ++lane)
            m = std::max(m, f(lane));
        return m;
    }
};

int main()
{
    std::mt19937 rng(7);
    auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
    // ascending starts: every tile of every sequence has exactly one number, every row its sequence
    for (int round = 0; round < 3000; ++round) {
        const bool many = round % 50 == 0;
        const int n = 1 + upto(many ? 9000 : round % 5 == 0 ? 80 : 9), per_token = 1 + upto(7), rows = 1 << upto(7);
        std::vector<int32_t> starts(n + 1);
        starts[0] = upto(3) == 0 ? upto(20) : 0;
        for (int i = 0; i < n; ++i)
            starts[i + 1] = starts[i] + (upto(2) == 0 ? 0 : upto(1 << upto(many ? 1 : round % 5 == 0 ? 4 : 9)));
        const int tokens = starts[n] + (upto(1) ? upto(30) : 0);
        std::vector<std::vector<int>> seen(n);
        for (int i = 0; i < n; ++i)
            seen[i].assign((((int64_t)starts[i + 1] - starts[i]) * per_token + rows - 1) / rows, 0);
        for (int64_t number = 0; number < tile_numbers(tokens, n, per_token, rows); ++number) {
            const Tile t = find_tile(HostWave(), starts.data(), n, tokens, per_token, rows, number);
            if (t.seq >= 0) {
                CHECK(t.index >= 0 && t.index < (int)seen[t.seq].size());
                CHECK(t.span.first == starts[t.seq] && t.span.count == starts[t.seq + 1] - starts[t.seq]);
                ++seen[t.seq][t.index];
            }
        }
        for (const auto& s : seen)
            for (int count : s)
                CHECK(count == 1);
        for (int64_t number = 0, index = INT_MAX; n <= 64 && number < tile_numbers(tokens, n, per_token, rows); ++number) {
            const Tile t = late_tile(HostWave(), starts.data(), n, tokens, per_token, rows, number);
            if (t.seq >= 0) {
                CHECK(t.index >= 0 && t.index <= index && t.index < (int)seen[t.seq].size());
                CHECK(t.span.first == starts[t.seq] && t.span.count == starts[t.seq + 1] - starts[t.seq]);
                CHECK(--seen[t.seq][t.index] == 0);
                index = t.index;
            }
        }
        for (const auto& s : seen)
            for (int count : s)
                CHECK(count == (n <= 64 ? 0 : 1));
        for (int row = 0; row < tokens; ++row) {
            const int s = find_row(HostWave(), starts.data(), n, tokens, row);
            bool any = false;
            for (int i = 0; i < n; ++i)
                any = any || (row >= starts[i] && row < starts[i + 1]);
            CHECK(any == (s >= 0));
            if (s >= 0)
                CHECK(row >= starts[s] && row < starts[s + 1]);
        }
        for (int i = 0; i < n; ++i)
            CHECK(packed_start_ok(starts.data(), i, tokens));
    }
    // any starts at all: what comes out lies in the tensors
    const int32_t odd[] = { INT_MIN, -1, 0, 1, 5, 17, 64, 65, 1000, INT_MAX };
    for (int round = 0; round < 20000; ++round) {
        const int n = 1 + upto(round % 20 == 0 ? 200 : 5), per_token = 1 + upto(7), rows = 1 << upto(7), tokens = 1 + upto(70);
        std::vector<int32_t> starts(n + 1);
        for (auto& s : starts)
            s = odd[upto(9)];
        for (int64_t number = 0; number < tile_numbers(tokens, n, per_token, rows); ++number) {
            for (int late = 0; late <= (n <= 64 ? 1 : 0); ++late) {
                const Tile t = late ? late_tile(HostWave(), starts.data(), n, tokens, per_token, rows, number)
                                    : find_tile(HostWave(), starts.data(), n, tokens, per_token, rows, number);
                if (t.seq < 0)
                    continue;
                CHECK(t.seq < n && t.index >= 0 && t.span.first >= 0 && t.span.count > 0 && t.span.first + t.span.count <= tokens);
                CHECK((int64_t)t.index * rows < (int64_t)t.span.count * per_token);
            }
        }
        for (int row = 0; row < tokens; ++row) {
            const int s = find_row(HostWave(), starts.data(), n, tokens, row);
            CHECK(s < n);
            if (s >= 0) {
                const Span span = packed_span(starts.data(), s, tokens);
                CHECK(row >= span.first && row < span.first + span.count && span.first + span.count <= tokens);
            }
        }
    }
    // quotients: every divisor's multiples and their neighbours, small and large
    for (int round = 0; round < 200000; ++round) {
        const int by = round < 3000 ? round + 1 : 1 + (int)(rng() % (upto(3) == 0 ? 2147483647u : 100000u));
        const Divisor d = make_divisor(by);
        const int64_t multiple = (int64_t)by * (1 + (int64_t)(rng() % (2147483647u / (unsigned)by)));
        for (int64_t n : { (int64_t)0, (int64_t)by - 1, (int64_t)by, multiple - 1, multiple, multiple + 1, (int64_t)2147483647, (int64_t)(rng() >> 1) })
            if (n >= 0 && n <= 2147483647)
                CHECK(quotient((int)n, d) == (int)(n / by));
    }
    // any page numbers and positions: a row of the cache or -1
    for (int round = 0; round < 20000; ++round) {
        const int width = 1 + upto(6), page_size = 1 + upto(70), n_pages = 1 + upto(9);
        std::vector<int32_t> table(width);
        for (auto& t : table)
            t = upto(3) == 0 ? odd[upto(9)] : upto(n_pages);
        const int32_t positions[] = { INT_MIN, -1, 0, page_size - 1, page_size, width * page_size - 1, width * page_size, INT_MAX, upto(500) };
        for (int pos : positions) {
            const int row = page_row(table.data(), width, n_pages, make_divisor(page_size), pos);
            const bool there = pos >= 0 && pos / page_size < width && table[pos / page_size] >= 0 && table[pos / page_size] < n_pages;
            CHECK(there == (row >= 0));
            if (there)
                CHECK(row == table[pos / page_size] * page_size + pos % page_size && row < n_pages * page_size);
        }
    }
    // the largest cache
    const int32_t last[] = { (1 << 27) - 1 };
    CHECK(page_row(last, 1, (1 << 27) - 1 + 1, make_divisor(15), 14) == (int)(((int64_t)(1 << 27) - 1) * 15 + 14));
    std::printf("kv_pages done\n");
    return 0;
}
