// Host check of csrc/paged_rows.h: the search and the walk over value blocks as the kernels run them, a wave's 64
// lanes one after the other, over every small q_start and over long ones with wrong entries.  Prints how many arrays
// were walked; a walk that does not end, a row or position that is not its sequence's, or (where q_start does not
// decrease) a row left out or taken twice ends the program with a message.
#include <stdio.h>
#include <stdlib.h>

#include <random>
#include <vector>

#include "paged_rows.h"

struct Batch {
    std::vector<int> q, kv;   // q_start, kv_len
    int n_rows, max_q, max_kv;
    int n_seq() const { return (int)kv.size(); }
    PagedSeq seq(int s) const { return paged_checked(q[s], q[s + 1], kv[s], n_rows, max_q, max_kv); }
    int find(int row) const
    {
        return paged_steps(n_seq(), [&](int lo, int len, int stride) {
            int n = 0;
            for (int lane = 0; lane < 64; lane++) {
                const int i = (lane + 1) * stride - 1;
                n += i < len && q[lo + i + 1] <= row;
            }
            return n;
        });
    }
    void bad(const char *what, int row) const
    {
        fprintf(stderr, "%s at row %d; n_rows %d, max_q %d, q_start", what, row, n_rows, max_q);
        for (int v : q) fprintf(stderr, " %d", v);
        fprintf(stderr, "\nkv_len");
        for (int v : kv) fprintf(stderr, " %d", v);
        fprintf(stderr, "\n");
        exit(1);
    }
};

static void check(const Batch &b)
{
    bool sorted = b.q[0] >= 0;
    for (int s = 0; s < b.n_seq(); s++) sorted = sorted && b.q[s] <= b.q[s + 1];
    // keys and queries: a row's place
    for (int row = 0; row < b.n_rows; row++) {
        const int s = b.find(row);
        if (s < 0 || s > b.n_seq()) b.bad("no sequence", row);
        if (sorted) {
            int first = 0;
            while (first < b.n_seq() && b.q[first + 1] <= row) first++;
            if (s != first) b.bad("not the row's sequence", row);
        }
        if (s == b.n_seq()) continue;
        const PagedSeq q = b.seq(s);
        if (q.holds(row) && (row < b.q[s] || row >= b.q[s + 1])) b.bad("a row of no sequence", row);
        if (q.holds(row) && (q.position(row) >= b.kv[s] || q.position(row) >= b.max_kv)) b.bad("a position behind the sequence", row);
    }
    // values: the blocks of every unit
    for (int unit : {2, 8}) {
        std::vector<int> taken(b.n_rows, 0);
        std::vector<std::vector<char>> stored(b.n_seq());
        for (int s = 0; s < b.n_seq(); s++) stored[s].assign(b.seq(s).q_len > 0 ? b.kv[s] : 0, 0);
        for (int first = 0; first < b.n_rows; first += unit) {
            const int last = first + unit < b.n_rows ? first + unit : b.n_rows;
            int finds = 0;
            paged_blocks(
                first, last, b.n_seq(),
                [&](int row) {
                    if (++finds > unit) b.bad("a walk that does not end", row);
                    return b.find(row);
                },
                [&](int s) { return b.seq(s); },
                [&](int s, int row, int pos, int n) {
                    if (n < 1 || n > 8 - (pos & 7)) b.bad("rows of two blocks", row);
                    for (int k = 0; k < n; k++) {
                        const PagedSeq q = b.seq(s);
                        if (!q.holds(row + k) || q.position(row + k) != pos + k || pos + k < 0 || pos + k >= b.kv[s])
                            b.bad("a value that is not its sequence's", row + k);
                        if (stored[s][pos + k]++) b.bad("a position stored twice", row + k);
                        taken[row + k]++;
                    }
                });
        }
        for (int row = 0; sorted && row < b.n_rows; row++) {
            const int s = b.find(row);
            const bool want = s < b.n_seq() && b.seq(s).holds(row) && b.seq(s).position(row) >= 0;
            if (taken[row] != want) b.bad("a value left out or taken twice", row);
        }
    }
}

int main()
{
    long walked = 0;
    // every array of up to 4 sequences over up to 9 rows, entries from -1 to one past the end
    for (int n_rows : {4, 9})
        for (int n_seq = 1; n_seq <= 4; n_seq++) {
            const int base = n_rows + 3;
            long all = 1;
            for (int i = 0; i <= n_seq; i++) all *= base;
            for (long x = 0; x < all; x++) {
                Batch b = {std::vector<int>(n_seq + 1), {}, n_rows, n_rows, 40};
                long y = x;
                for (int &v : b.q) {
                    v = (int)(y % base) - 1;
                    y /= base;
                }
                const int kv[] = {40, 2, 11, 0};
                for (int s = 0; s < n_seq; s++) b.kv.push_back(kv[(s + x) % 4]);
                check(b);
                walked++;
            }
        }
    // long ones: lengths of 0 to 12 rows, then one to four entries anything
    std::mt19937 g(1);
    auto below = [&](int n) { return (int)(g() % (unsigned)n); };
    for (int t = 0; t < 6000; t++) {
        Batch b;
        const int n_seq = 1 + below(t % 50 == 0 ? 5000 : 300), most = 1 + below(13);
        b.q.push_back(0);
        for (int s = 0; s < n_seq; s++) {
            const int n = below(most);
            b.q.push_back(b.q.back() + n);
            b.kv.push_back(below(4) ? n + below(30) : below(n + 1));
        }
        b.n_rows = b.q.back() + below(3) + 1;
        b.max_q = most;
        b.max_kv = 45;
        for (int i = t % 5; i > 0; i--) b.q[below(n_seq + 1)] = below(8) ? below(b.n_rows + 1) : (int)g();
        check(b);
        walked++;
    }
    // the arrays that were found first
    for (std::vector<int> q : {std::vector<int>{0, 10, 2, 4, 8}, {0, 9, 2, 5}, {0, 10, 2, 6}, {0, 4, 6, 9, 13, 14, 20, 18, 19, 20}}) {
        Batch b = {q, std::vector<int>(q.size() - 1, 100), 20, 20, 100};
        check(b);
        walked++;
    }
    printf("%ld\n", walked);
    return 0;
}
