// The paged KV cache (x100_paged.h) as its kernels see it: the batch, pages and the 4-bit format.
#pragma once
#include "paged_rows.h"
#include "rows_load.h"
#include "x100_paged.h"

// Sequence s of the batch, every entry checked against the host's bounds (x100_paged.h).
X100_DEV PagedSeq paged_seq(const x100_kv_batch &b, int s)
{
    return paged_checked(b.q_start[s], b.q_start[s + 1], b.kv_len[s], b.n_rows, b.max_q, b.max_kv);
}

// Page of position p (0 <= p < max_kv) of sequence s, or -1 outside 0 .. n_pages - 1.
X100_DEV int paged_page(const x100_kv_cfg &c, const x100_kv_batch &b, int s, int p)
{
    const int g = b.block_table[(size_t)s * b.table_ld + (p >> __builtin_ctz(c.page))];
    return g >= 0 && g < c.n_pages ? g : -1;
}

// The first s of 0 .. n - 1 for which below(s + 1) does not hold (n if there is none; below holds up to some
// place and not behind it), by the whole wave, 64 entries per step.
template <class F> X100_DEV int paged_search(int n_seq, F &&below)
{
    const int lane = threadIdx.x & 63;
    return paged_steps(n_seq, [&](int lo, int len, int stride) __attribute__((always_inline)) {
        const int i = (lane + 1) * stride - 1;
        return __popcll(__ballot(i < len && below(lo + i + 1)));
    });
}
// The sequence of row r: the first s with q_start[s + 1] > r (n_seq if there is none; any, where q_start decreases).
X100_DEV int paged_find(const x100_kv_batch &b, int r)
{
    return paged_search(b.n_seq, [&](int s) { return b.q_start[s] <= r; });
}

// Bytes of one head's part of a page, K or V.
template <int HD, bool Q4> X100_DEV constexpr int page_head_bytes(int page) { return Q4 ? page * HD * 5 / 8 : page * HD * 2; }

// 4-bit codes: number e of 8 at bit 16 (e % 2) + 4 (e / 2) of the word.
X100_DEV constexpr int q4_shift(int e) { return 16 * (e & 1) + 4 * (e >> 1); }

// d, m of a group from its smallest and largest value (fp16 bits; d = m = NaN where bad, or where either is past
// fp16's range) and 1 / d.  d is mostly rounded to nearest; where that would take the largest code's value past fp16's
// range (0 .. 65504: d = 4368, 15 d = 65520), the fp16 below it, 15 of whose steps end at the largest value or below.
struct Q4Scale {
    uint16_t d, m;
    float inv, mf;
    bool bad;
};
X100_DEV Q4Scale q4_scale(float lo, float hi, bool bad)
{
    bad |= !(lo >= -65504.0f) || !(hi <= 65504.0f);
    const _Float16 m = f2h_rne(lo);
    _Float16 d = f2h_rne((hi - lo) * (1.0f / 15.0f));
    if (__builtin_fmaf16((_Float16)15.0f, d, m) > (_Float16)65504.0f)
        d = __builtin_bit_cast(_Float16, (uint16_t)(__builtin_bit_cast(uint16_t, d) - 1));
    const float df = (float)d, mf = (float)m;
    Q4Scale s;
    s.d = bad ? 0x7e00 : __builtin_bit_cast(uint16_t, d);
    s.m = bad ? 0x7e00 : __builtin_bit_cast(uint16_t, m);
    s.inv = !bad && df > 0.0f ? 1.0f / df : 0.0f;
    s.mf = mf;
    s.bad = bad;
    return s;
}
X100_DEV uint32_t q4_code(const Q4Scale &s, float x)
{
    const float n = rintf((x - s.mf) * s.inv);
    return s.bad ? 0u : (uint32_t)fminf(fmaxf(n, 0.0f), 15.0f);
}

// The 8 numbers of a word as fp16 codes 0 .. 15, pairs (0,1), (2,3), (4,5), (6,7): a code under the
// exponent of 1024 reads as 1024 + n (low nibble of a byte) or 1024 + 16 n (high), both exact.  The
// exponent is kept in a vector register: with it v_and_or_b32 takes a mask and it in one instruction.
X100_DEV void q4_unpack(uint32_t w, v2h (&n)[4])
{
    uint32_t ex;
    asm("v_mov_b32 %0, 0x64006400" : "=v"(ex));
    const v2h k1024 = {(_Float16)1024.0f, (_Float16)1024.0f};
    const v2h k16 = {(_Float16)0.0625f, (_Float16)0.0625f}, k64 = {(_Float16)-64.0f, (_Float16)-64.0f};
    const uint32_t w8 = w >> 8;
    n[0] = as_h2((w & 0x000f000fu) | ex) - k1024;
    n[1] = __builtin_elementwise_fma(as_h2((w & 0x00f000f0u) | ex), k16, k64);
    n[2] = as_h2((w8 & 0x000f000fu) | ex) - k1024;
    n[3] = __builtin_elementwise_fma(as_h2((w8 & 0x00f000f0u) | ex), k16, k64);
}
// A V word's 8 positions as fp16 values, d and m of the 8 positions.
X100_DEV v4u q4_v(uint32_t w, v4u d, v4u m)
{
    v2h n[4];
    q4_unpack(w, n);
    v4u r;
#pragma unroll
    for (int e = 0; e < 4; e++) r[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n[e], as_h2(d[e]), as_h2(m[e])));
    return r;
}
