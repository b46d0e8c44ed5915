// Which sequence a row of a batch belongs to (x100_paged.h), for any contents of q_start and kv_len.  Constexpr
// functions without HIP: kernels call them, and a test walks every small array through them on the host.
//
// q_start is device memory that the host cannot check.  Where it decreases, the search below ends at some sequence,
// not always at one that holds the row: whoever takes its answer asks holds() first.
#pragma once

struct PagedSeq {
    int q0, q_len, kv_len;   // first row, rows, cached positions (q_len < 0: the sequence is refused)
    constexpr bool holds(int row) const { return q_len > 0 && row >= q0 && row - q0 < q_len; }
    // of a row that it holds: 0 .. kv_len - 1, or below 0
    constexpr int position(int row) const { return kv_len - q_len + (row - q0); }
};

// A sequence with rows q0 .. q1 - 1 and kv positions, checked against the host's bounds.
constexpr PagedSeq paged_checked(int q0, int q1, int kv, int n_rows, int max_q, int max_kv)
{
    const bool ok = q0 >= 0 && q1 >= q0 && q1 <= n_rows && q1 - q0 <= max_q && kv >= 0 && kv <= max_kv;
    return {q0, ok ? q1 - q0 : -1, kv};
}

// The first of 0 .. n - 1 that does not lie below (n if there is none; they lie below up to some place and not behind
// it).  count(lo, len, stride): how many of the 64 entries lo + (i + 1) * stride - 1 within the next len lie below.
template <class Count> constexpr int paged_steps(int n, Count &&count)
{
    int lo = 0, len = n;
    while (len > 0) {
        const int stride = (len + 63) / 64;
        const int below = count(lo, len, stride) * stride;   // entries known to lie below
        if (stride == 1) return lo + below;
        lo += below;
        len = stride - 1 < len - below ? stride - 1 : len - below;   // the next entry probed does not
    }
    return lo;
}

// The blocks of 8 positions that rows first .. last - 1 begin: visit(s, row, pos, n) for n rows from `row` on, at
// positions pos .. pos + n - 1 of one block of sequence s.  A block begins at its sequence's first row and at every
// position 8 k; its rows may lie behind `last`.  find(row): the search's sequence, seq(s): that one, checked.  Every
// turn moves the row on, whatever the search gives.
template <class Find, class Seq, class Visit>
constexpr void paged_blocks(int first, int last, int n_seq, Find &&find, Seq &&seq, Visit &&visit)
{
    for (int row = first; row < last;) {
        const int s = find(row);
        if (s >= n_seq) return;
        const PagedSeq q = seq(s);
        if (!q.holds(row)) {
            row++;
            continue;
        }
        const int end = q.q0 + q.q_len, stop = last < end ? last : end;
        while (row < stop) {
            const int pos = q.position(row);
            if (pos < 0) {   // on to position 0
                row = stop - row < -pos ? stop : row - pos;
                continue;
            }
            const int into = pos & 7, left = end - row, n = 8 - into < left ? 8 - into : left;
            if (into == 0 || row == q.q0) visit(s, row, pos, n);
            row += n;
        }
    }
}
