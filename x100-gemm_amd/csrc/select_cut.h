// Keys of scores, and the cut that makes a list of some of them (sparse.hip).  Constexpr functions without HIP: a kernel
// calls them, and a test walks them through many arrays on the host.
#pragma once
#include <stdint.h>

// Keys are compared as unsigned numbers, in the order of the scores.  0: not to be selected; all ones: always.
constexpr uint64_t KEY_NONE = 0, KEY_ALWAYS = ~0ull;
constexpr uint64_t score_key(double s)
{
    if (!(s == s)) s = -__builtin_inf();
    s += 0.0;   // -0 is 0
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    return u >> 63 ? ~u : u | 1ull << 63;
}

// Keys in two halves.  Selected are those with upper halves from `upper` on (exact), or those with upper halves above it, those
// that have it and a lower half above `lower`, and the first `ties` that are both.
struct SelectCut {
    uint32_t upper, lower;
    bool exact;
    int ties;
    constexpr bool tied(uint32_t u, uint32_t l) const { return !exact && u == upper && l == lower; }
    constexpr bool above(uint32_t u, uint32_t l) const { return exact ? u >= upper : u > upper || (u == upper && l > lower); }
};

// The cut of more keys than n_sel, of which n_sel at most are KEY_ALWAYS, one bit at a time until as many keys are left as the
// list takes.  largest: the largest upper half that is not KEY_ALWAYS's (0: none); count(from): upper halves from `from` on.  Where
// keys with the cut's upper half are in the list and others are not (their scores differ by less than 1e-6, one row in thousands,
// or are equal), lowers(upper) makes these keys' lower halves (1 or more; 0 for the other keys), and count_low(from)
// counts those from `from` > 0 on.
template <class Count, class Lowers, class CountLow>
constexpr SelectCut select_cut(int n, int n_sel, uint32_t largest, Count &&count, Lowers &&lowers, CountLow &&count_low)
{
    uint32_t yh = 0, yl = 0;
    bool exact = false;
    // The upper 12 bits (a score's sign and exponent) lie at or little below those of the largest: these few values first,
    // instead of 12 bits.
    int top = 31;
    uint32_t from = largest & 0xfff00000u;
    for (int k = 0; k < 4 && from; k++, from -= 0x00100000u) {
        const int c = count(from);
        exact = c == n_sel;
        if (c >= n_sel) {
            yh = from;
            top = 19;
            break;
        }
    }
    for (int bit = top; bit >= 0 && !exact; bit--) {
        const uint32_t next = yh | 1u << bit;
        const int c = count(next);
        if (c >= n_sel) yh = next;
        exact = c == n_sel;
    }
    if (yh == 0) return {1, 0, true, 0};   // fewer keys than the list takes
    if (exact) return {yh, 0, true, 0};
    // yh is not all ones: those keys are no more than n_sel.  Where the keys that are always taken fill the list, the search may
    // have ended at the largest other one's upper half, and takes none of those.
    const int need = n_sel - count(yh + 1);
    if (need == 0) return {yh + 1, 0, true, 0};
    lowers(yh);
    int c = 0;
    for (int bit = 31; bit >= 0 && c != need; bit--) {
        const uint32_t next = yl | 1u << bit;
        c = count_low(next);
        if (c >= need) yl = next;
    }
    return {yh, yl, false, c == need ? n : need - (yl == ~0u ? 0 : count_low(yl + 1))};
}
