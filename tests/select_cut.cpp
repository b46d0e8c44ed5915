// Host check of csrc/select_cut.h: lists of keys as the kernel makes them from a cut, against the keys sorted, for every row
// of a few scores that small and for longer random ones.  Prints how many lists were made; one that has other keys than the
// sorted ones, or more than it has room for, ends the program with a message.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

#include <algorithm>
#include <random>
#include <vector>

#include "select_cut.h"

using Keys = std::vector<uint64_t>;
static uint32_t hi(uint64_t k) { return (uint32_t)(k >> 32); }

// Numbers of the listed keys, ascending, as the kernel lists them.
static std::vector<int> listed(const Keys &key, int n_sel)
{
    const int n = (int)key.size();
    std::vector<uint32_t> low(n);   // lower halves of the keys that need them
    SelectCut cut = {1, 0, true, 0};
    if (n > n_sel) {
        uint32_t largest = 0;
        for (uint64_t k : key)
            if (hi(k) != ~0u) largest = std::max(largest, hi(k));
        cut = select_cut(
            n, n_sel, largest, [&](uint32_t from) { return (int)std::count_if(key.begin(), key.end(), [&](uint64_t k) { return hi(k) >= from; }); },
            [&](uint32_t upper) {
                for (int i = 0; i < n; i++) low[i] = hi(key[i]) == upper ? std::max((uint32_t)key[i], 1u) : 0;
            },
            [&](uint32_t from) { return (int)std::count_if(low.begin(), low.end(), [&](uint32_t l) { return l >= from; }); });
    }
    std::vector<int> out;
    int eq = 0;
    for (int i = 0; i < n; i++) {
        const bool tied = cut.tied(hi(key[i]), low[i]);
        if (cut.above(hi(key[i]), low[i]) || (tied && eq < cut.ties)) out.push_back(i);
        eq += tied;
    }
    return out;
}

static void check(const Keys &key, int n_sel)
{
    std::vector<int> want;
    for (int i = 0; i < (int)key.size(); i++)
        if (key[i] != KEY_NONE) want.push_back(i);
    std::stable_sort(want.begin(), want.end(), [&](int a, int b) { return key[a] > key[b]; });
    if ((int)want.size() > n_sel) want.resize(n_sel);
    std::sort(want.begin(), want.end());
    const std::vector<int> got = listed(key, n_sel);
    if (got == want) return;
    fprintf(stderr, "a list of %d has %zu keys, not %zu, or others; keys", n_sel, got.size(), want.size());
    for (size_t i = 0; i < key.size() && i < 64; i++) fprintf(stderr, " %016llx", (unsigned long long)key[i]);
    fprintf(stderr, "\n");
    exit(1);
}

int main()
{
    long made = 0;
    const double inf = INFINITY;
    // scores whose keys end in ones or zeros, beside ordinary ones; the last is a block without a page
    const std::vector<double> some = {-1.0, -2.0, nextafter(2.0, 0.0), 0.0, -1.25, -inf, NAN, 3.5, -nextafter(1.0, 2.0)};
    auto key = [&](int i) { return i < (int)some.size() ? score_key(some[i]) : KEY_NONE; };
    const int kinds = (int)some.size() + 1;
    // every row of up to 5 of them, the first n_first and last n_last of which are always taken
    for (int n = 1; n <= 5; n++) {
        long all = 1;
        for (int i = 0; i < n; i++) all *= kinds;
        for (long x = 0; x < all; x++) {
            Keys k(n);
            long y = x;
            for (uint64_t &v : k) {
                v = key((int)(y % kinds));
                y /= kinds;
            }
            for (int n_last = 1; n_last <= n; n_last++)
                for (int n_first = 0; n_first + n_last <= n; n_first++)
                    for (int n_sel = n_first + n_last; n_sel <= n; n_sel++) {
                        Keys f = k;
                        for (int i = 0; i < n; i++)
                            if ((i < n_first || i >= n - n_last) && f[i] != KEY_NONE) f[i] = KEY_ALWAYS;
                        check(f, n_sel);
                        made++;
                    }
        }
    }
    // longer rows: scores of one kind, of a few, of few upper halves, of any size
    std::mt19937_64 g(1);
    auto below = [&](int n) { return (int)(g() % (unsigned)n); };
    std::normal_distribution<double> normal;
    for (int t = 0; t < 200000; t++) {
        const int n = 1 + below(t % 100 ? 60 : 700), n_sel = 1 + below(n + 2), n_last = 1 + below(n_sel);
        const int n_first = below(3) ? below(n_sel - n_last + 1) : n_sel - n_last, kind = below(5), same = below(kinds);
        const double base = ldexp(below(2) ? 1.0 : -1.0, below(40) - 20);
        Keys k(n);
        for (int i = 0; i < n; i++) {
            k[i] = kind == 0   ? key(same)
                   : kind == 1 ? key(below(kinds))
                   : kind == 2 ? score_key(base * (1.0 + ldexp(below(9) - 4, -below(52))))
                   : kind == 3 ? (below(4) ? g() % ~0ull : KEY_NONE)
                               : score_key(normal(g));
            if ((i < n_first || i >= n - n_last) && k[i] != KEY_NONE) k[i] = KEY_ALWAYS;
        }
        check(k, n_sel);
        made++;
    }
    printf("%ld\n", made);
    return 0;
}
