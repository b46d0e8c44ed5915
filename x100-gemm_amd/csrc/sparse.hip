// Which blocks of the paged cache a query attends to (x100_sparse.h): mean keys of full pages, and the selection.
//
// The score of block b for a row and KV head is (the sum of the KV head's queries) . (the block's mean key), which is the
// mean of their scores with the block's keys.  It is summed in fp64 (a product of two 16-bit numbers is exact there): two
// blocks change places only where their scores differ by 1e-16 of their terms, so the lists do not depend on an order
// of sums, and equal blocks tie.
#include <algorithm>

#include "paged.h"
#include "select_cut.h"
#include "x100_internal.h"

namespace {

template <int CTRL> X100_DEV double dpp_d(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp_i<CTRL>(0, (int)(uint32_t)u), hi = dpp_i<CTRL>(0, (int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
X100_DEV double xor16_d(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)xor16_u((uint32_t)(u >> 32)) << 32 | xor16_u((uint32_t)u));
}
X100_DEV double xor32_d(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)xor32_u((uint32_t)(u >> 32)) << 32 | xor32_u((uint32_t)u));
}
// sum over each group of L = 4, 8 or 16 lanes, in all of them
template <int L> X100_DEV double sum_lanes(double v)
{
    v += dpp_d<0xB1>(v);
    v += dpp_d<0x4E>(v);
    if constexpr (L > 4) v += dpp_d<0x141>(v);
    if constexpr (L == 16) v += dpp_d<0x140>(v);
    return v;
}

// 8 elements of a head row as floats: as they are stored, or the 4-bit numbers' values (d2, m2: d and m twice).
template <int AT> X100_DEV void elems16(v4u u, float (&v)[8])
{
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[2 * e] = act2f<AT>(u[e] & 0xffffu);
        v[2 * e + 1] = act2f<AT>(u[e] >> 16);
    }
}
X100_DEV void elems_q4(uint32_t w, uint32_t dm, float (&v)[8])
{
    const v2h d2 = as_h2((dm & 0xffffu) * 0x10001u), m2 = as_h2((dm >> 16) * 0x10001u);
    v2h n[4];
    q4_unpack(w, n);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const v2h x = __builtin_elementwise_fma(n[e], d2, m2);
        v[2 * e] = (float)x[0];
        v[2 * e + 1] = (float)x[1];
    }
}

// Mean keys.  A block looks at 16 rows of the batch and one KV head.  Its lanes look the rows up side by side: by how many of
// 64 sequences end before them, from the first row's on (one search) where there are more.  A single page (a
// prompt's, or one of a batch of single tokens) is shared by the block's waves, of several each wave takes every fourth.  Lane l
// has the elements 8 (l % L) .. + 7 of every (64 / L)-th row of its part (L lanes per row), 4 loads on their way.
// Bound by the chain row -> sequence -> page -> keys for single tokens, by the keys' bytes for prompts.
constexpr int MEAN_ROWS = 16;
template <int HD, int AT, bool Q4>
__global__ __launch_bounds__(256) void k_kv_means(const x100_kv_cfg c, const x100_kv_batch b, const uint8_t *kp, uint16_t *means)
{
    constexpr int L = HD / 8, RS = 64 / L;   // lanes of a row, rows of a step
    __shared__ double s_sum[3][HD];
    const int lane = threadIdx.x & 63, w = wave_id(), kvh = blockIdx.x % c.n_head_kv, row0 = blockIdx.x / c.n_head_kv * MEAN_ROWS;
    // lane i < 16: page of row row0 + i, if that row is the last of a page (else -1)
    const int s0 = b.n_seq <= 64 ? 0 : paged_find(b, row0);
    if (s0 >= b.n_seq) return;
    const int row = row0 + min(lane, MEAN_ROWS - 1);
    // sequence s0 + lane, and by its end the sequence of each row
    const int i0 = min(s0 + lane, b.n_seq - 1);
    const int start = b.q_start[i0], end = b.q_start[i0 + 1], kv = b.kv_len[i0];
    int s = s0;
#pragma unroll
    for (int i = 0; i < MEAN_ROWS; i++) {
        const int past = __popcll(__ballot(s0 + lane < b.n_seq && end <= row0 + i));
        if (row == row0 + i) s = s0 + past;
    }
    const int from = min(s - s0, 63);
    PagedSeq q = paged_checked(__shfl(start, from, 64), __shfl(end, from, 64), __shfl(kv, from, 64), b.n_rows, b.max_q, b.max_kv);
    // more than 64 sequences without rows in between, or q_start in disorder: each row by itself
    if (__any(s < b.n_seq && (s - s0 >= 64 || !q.holds(row)))) {
        for (int i = 0; i < MEAN_ROWS; i++) {
            PagedSeq f;
            const int at = paged_find(b, row0 + i, f);
            if (row == row0 + i) {
                s = at;
                q = f;
            }
        }
    }
    int page = -1;
    if (lane < MEAN_ROWS && s < b.n_seq) {
        const int pos = q.holds(row) ? q.position(row) : -1;
        if (pos >= 0 && (pos & (c.page - 1)) == c.page - 1) page = paged_page(c, b, s, pos);
    }
    uint64_t todo = __ballot(page >= 0);
    const bool one = __popcll(todo) == 1;
    const int r0 = one ? w * (c.page / 4) : 0, r1 = one ? r0 + c.page / 4 : c.page;   // rows of the page
    for (int n = 0; todo; n++) {
        const int i = __ffsll((unsigned long long)todo) - 1, pg = __shfl(page, i, 64);
        todo &= todo - 1;
        if (!one && (n & 3) != w) continue;
        const uint8_t *kb = kp + ((size_t)pg * c.n_head_kv + kvh) * page_head_bytes<HD, Q4>(c.page);
        double sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int e0 = lane % L;
        for (int r = r0 + lane / L; r < r1; r += 4 * RS) {   // a part has at least 4 rows: some lanes' steps may lie behind it
            float v[4][8];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int rr = min(r + u * RS, r1 - 1);
                if constexpr (!Q4) elems16<AT>(*(const v4u *)(kb + ((size_t)rr * HD + 8 * e0) * 2), v[u]);
                else
                    elems_q4(((const uint32_t *)kb)[rr * L + e0],
                             ((const uint32_t *)(kb + c.page * HD / 2))[rr * (HD / 32) + e0 / 4], v[u]);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (r + u * RS >= r1) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] += (double)v[u][e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (L == 8) sum[e] += dpp_d<0x128>(sum[e]);   // rows of lanes l and l ^ 8 too
            sum[e] += xor16_d(sum[e]);
            sum[e] += xor32_d(sum[e]);
        }
        if (one) {   // every wave comes here, once
            if (w > 0 && lane < L) {
#pragma unroll
                for (int e = 0; e < 8; e++) s_sum[w - 1][8 * lane + e] = sum[e];
            }
            __syncthreads();
            if (w > 0) return;
            if (lane < L) {
#pragma unroll
                for (int k = 0; k < 3; k++)
#pragma unroll
                    for (int e = 0; e < 8; e++) sum[e] += s_sum[k][8 * lane + e];
            }
        }
        if (lane < L) {
            const double f = 1.0 / c.page;   // a power of two
            v4u o;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = f2act<AT>((float)(sum[2 * e] * f)) | f2act<AT>((float)(sum[2 * e + 1] * f)) << 16;
            *(v4u *)(means + ((size_t)pg * c.n_head_kv + kvh) * HD + 8 * e0) = o;
        }
    }
}

// ---- selection -----------------------------------------------------------------------------------

struct SelectArgs {
    x100_kv_cfg c;
    x100_kv_batch b;
    x100_kv_sel pick;
    const uint16_t *q;
    int64_t ldq;
    const uint16_t *means;
    int *sel;
    bool apart;   // sequences of MANY rows are k_attn_select_rows's, the others k_attn_select's
    bool by_seq;  // k_attn_select's units are MANY - 1 rows of each sequence (else the batch's rows)
    unsigned block0;   // first block of this launch
};

// Sequences of so many rows in a batch go to the kernel that takes rows together, the others' rows are taken one by one.
constexpr int MANY = 8;

// ---- one row of few: a block per row and KV head

template <int NT, int CAP> struct SelectLds {
    uint64_t key[CAP];           // first the pages
    double q[128];               // the sum of the queries
    int hist[256];
    int bin, above, same;        // the digit of the list's last key, keys above it, keys with it
    int gt[NT / 64], eq[NT / 64];
};

// The list of n keys (n > 0): the n_sel largest that are not KEY_NONE, lowest index first among equal ones, ascending.  The
// smallest of them is found 8 bits at a time, until a digit's keys are all in or all digits are known.
template <int NT, int CAP> X100_DEV void select_keys(SelectLds<NT, CAP> &sh, int n, int n_sel, int *out)
{
    const uint64_t *k = sh.key;
    const int t = threadIdx.x, lane = t & 63, w = wave_id();
    uint64_t low = 1;      // selected: keys >= low,
    int ties = 0;          // or, if ties > 0, keys > low and the first `ties` keys that are low
    if (n > n_sel) {
        uint64_t prefix = 0, mask = 0;
        int need = n_sel;
        for (int shift = 56; shift >= 0; shift -= 8) {
            if (t < 256) sh.hist[t] = 0;
            __syncthreads();
            for (int i = t; i < n; i += NT)
                if ((k[i] & mask) == prefix) atomicAdd(&sh.hist[(int)(k[i] >> shift) & 255], 1);
            __syncthreads();
            if (w == 0) {   // lane l: bins 255 - 4 l .. 252 - 4 l
                int c[4], s = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) s += c[e] = sh.hist[255 - 4 * lane - e];
                int upto = s;   // of the lanes up to this one
                upto += dpp_i<0x111>(0, upto);
                upto += dpp_i<0x112>(0, upto);
                upto += dpp_i<0x114>(0, upto);
                upto += dpp_i<0x118>(0, upto);
                upto += dpp_i<0x142, 0xa>(0, upto);
                upto += dpp_i<0x143, 0xc>(0, upto);
                int before = upto - s;
                if (before < need && need <= upto) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        if (before < need && need <= before + c[e]) {
                            sh.bin = 255 - 4 * lane - e;
                            sh.above = before;
                            sh.same = c[e];
                        }
                        before += c[e];
                    }
                }
            }
            __syncthreads();   // the next pass's first barrier lies behind these reads
            prefix |= (uint64_t)sh.bin << shift;
            mask |= 255ull << shift;
            need -= sh.above;
            low = prefix;
            if (sh.same == need) break;   // all keys with these digits
            if (shift == 0) ties = need;
        }
        if (low == KEY_NONE) {   // blocks without a page would be among them
            low = 1;
            ties = 0;
        }
    }
    // wave w has the w-th part of the keys, in order
    constexpr int NW = NT / 64;
    const int part = (n + NT - 1) / NT * 64, i0 = min(n, w * part), i1 = min(n, i0 + part);
    int gt = 0, eq = 0;
    for (int i = i0 + lane; i - lane < i1; i += 64) {
        const uint64_t x = i < i1 ? k[i] : 0;
        gt += __popcll(__ballot(i < i1 && (ties > 0 ? x > low : x >= low)));
        eq += __popcll(__ballot(i < i1 && x == low));
    }
    if (lane == 0) {
        sh.gt[w] = gt;
        sh.eq[w] = eq;
    }
    __syncthreads();
    int at = 0, eq0 = 0, total = 0;
#pragma unroll
    for (int v = 0, e = 0; v < NW; v++) {
        const int take = sh.gt[v] + (ties > 0 ? min(max(ties - e, 0), sh.eq[v]) : 0);
        if (v == w) eq0 = e;
        if (v < w) at += take;
        total += take;
        e += sh.eq[v];
    }
    const uint64_t below = (1ull << lane) - 1;
    for (int i = i0 + lane; i - lane < i1; i += 64) {
        const uint64_t x = i < i1 ? k[i] : 0;
        const uint64_t bq = __ballot(i < i1 && x == low);
        const bool take = i < i1 && (ties > 0 ? x > low || (x == low && eq0 + __popcll(bq & below) < ties) : x >= low);
        const uint64_t bt = __ballot(take);
        if (take) out[at + __popcll(bt & below)] = i;
        at += __popcll(bt);
        eq0 += __popcll(bq);
    }
    for (int i = total + t; i < n_sel; i += NT) out[i] = -1;
}

// L lanes have a mean, 16 elements each, 64 / L means of a wave at a time, U times on their way; each row and KV head reads its
// own means.  Bound by latency (row -> sequence -> pages -> means -> digits) and, on the few CUs that few rows keep busy, by
// fp64: 16 rows of up to 938 blocks 17.4 us (8 elements per lane and a longer sum over lanes 19.1), of which 4 to the
// position and 4 for the lists.  Scores in fp32 by the 16-bit matrix cores with bounds of their error, and fp64 for what the bounds
// leave, were no faster (20).
template <int HD, int AT, int NT, int CAP, int U> __global__ __launch_bounds__(NT) void k_attn_select(const SelectArgs a)
{
    constexpr int L = HD / 16, NG = NT / L;
    __shared__ SelectLds<NT, CAP> sh;
    const int t = threadIdx.x, lane = t & 63, l = lane % L, n_kv = a.c.n_head_kv, unit = (a.block0 + blockIdx.x) / n_kv;
    const int kvh = (a.block0 + blockIdx.x) % n_kv, G = a.c.n_head / n_kv, psh = __builtin_ctz(a.c.page);
    int row = unit, s = 0;
    PagedSeq q;
    if (a.by_seq) {
        s = unit / (MANY - 1);
        q = paged_seq(a.b, s);
        row = q.q0 + unit % (MANY - 1);
        if (!q.holds(row) || q.q_len >= MANY) return;
    }
    for (int e = t; e < HD; e += NT) {   // the sum of the queries
        double y = 0.0;
        for (int h = 0; h < G; h++) y += (double)act2f<AT>(a.q[(size_t)row * a.ldq + (size_t)(kvh * G + h) * HD + e]);
        sh.q[e] = y;
    }
    if (!a.by_seq) {
        s = paged_find(a.b, row, q);
        if (!q.holds(row) || (a.apart && q.q_len >= MANY)) return;
    }
    const int pos = q.position(row), own = pos >> psh;   // below 0: no position
    int *out = a.sel + ((size_t)row * n_kv + kvh) * a.pick.n_sel;
    if (pos < 0) {
        for (int i = t; i < a.pick.n_sel; i += NT) out[i] = -1;
        return;
    }
    const int *tab = a.b.block_table + (size_t)s * a.b.table_ld;
    for (int i = t; i <= own; i += NT) sh.key[i] = (uint32_t)tab[i];
    __syncthreads();
    double x[16];
#pragma unroll
    for (int e = 0; e < 16; e++) x[e] = sh.q[16 * l + e];
    const v4u *means = (const v4u *)(a.means + (size_t)kvh * HD) + 2 * l;
    for (int b0 = t / L; b0 - lane / L <= own; b0 += U * NG) {   // the lanes of a wave together
        v4u m[U][2];
        int pg[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (b0 - lane / L + u * NG > own) continue;   // all lanes'
            pg[u] = b0 + u * NG <= own ? (int)(uint32_t)sh.key[b0 + u * NG] : -1;
            if (pg[u] < 0 || pg[u] >= a.c.n_pages) pg[u] = -1;
            m[u][0] = means[(size_t)max(pg[u], 0) * n_kv * (HD / 8)];
            m[u][1] = means[(size_t)max(pg[u], 0) * n_kv * (HD / 8) + 1];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int b = b0 + u * NG;
            if (b - lane / L > own) continue;
            float v[8];
            elems16<AT>(m[u][0], v);
            double y = 0.0, z = 0.0;
#pragma unroll
            for (int e = 0; e < 8; e++) y = __builtin_fma(x[e], (double)v[e], y);
            elems16<AT>(m[u][1], v);
#pragma unroll
            for (int e = 0; e < 8; e++) z = __builtin_fma(x[8 + e], (double)v[e], z);
            y += z;
            y = sum_lanes<L>(y);
            const bool always = b < a.pick.n_first || b > own - a.pick.n_last;
            if (l == 0 && b <= own) sh.key[b] = pg[u] < 0 ? KEY_NONE : (always ? KEY_ALWAYS : score_key(y));
        }
    }
    __syncthreads();
    select_keys(sh, own + 1, a.pick.n_sel, out);
}

// ---- rows of a prompt: a block per R rows and KV head

typedef double v4d __attribute__((ext_vector_type(4)));
constexpr int RT = 512;   // threads

// The list of a row by one wave from the upper halves of its n keys, key i in lane i % 64 (select_cut.h).  Counts are kept per
// lane and summed once per bit (a ballot and a scalar count per key cost three times as much).  low(i, upper) gives the lower
// halves that are needed, which take the places of the upper ones.  put(place, key's number, or -1).
template <int CAP, class Low, class Put> X100_DEV void select_row(uint32_t *key, int n, int n_sel, Low &&low, Put &&put)
{
    constexpr int KL = CAP / 64;
    const int lane = threadIdx.x & 63, used = (n + 63) >> 6;
    uint32_t kh[KL];
#pragma unroll
    for (int u = 0; u < KL; u++) kh[u] = 64 * u + lane < n ? key[64 * u + lane] : (uint32_t)(KEY_NONE >> 32);
    auto count = [&](uint32_t from) __attribute__((always_inline)) {   // keys >= from
        int c = 0;
#pragma unroll
        for (int u = 0; u < KL; u++) c += kh[u] >= from ? 1 : 0;
        return wave_sum_u(c);
    };
    SelectCut cut = {1, 0, true, 0};
    if (n > n_sel) {
        uint32_t mx = 0;
#pragma unroll
        for (int u = 0; u < KL; u++) mx = kh[u] != ~0u ? max(mx, kh[u]) : mx;
        mx = (uint32_t)wave_max_iu((int)(mx ^ 0x80000000u)) ^ 0x80000000u;
        cut = select_cut(
            n, n_sel, mx, count,
            [&](uint32_t upper) __attribute__((always_inline)) {   // a lower half is at least 1 here, 0: not one of these keys
                for (int i = lane; i < n; i += 64) key[i] = key[i] == upper ? max(low(i, upper), 1u) : 0;
            },
            [&](uint32_t from) __attribute__((always_inline)) {
                int c = 0;
                for (int i = lane; i < n; i += 64) c += key[i] >= from ? 1 : 0;
                return wave_sum_u(c);
            });
    }
    int at_out = 0, eq = 0;
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int u = 0; u < KL; u++) {
        if (u >= used) continue;
        bool take = kh[u] >= cut.upper;
        if (!cut.exact) {
            const uint32_t l = 64 * u + lane < n ? key[64 * u + lane] : 0;
            const bool tied = cut.tied(kh[u], l);
            const uint64_t bq = __ballot(tied);
            take = cut.above(kh[u], l) || (tied && eq + __popcll(bq & below) < cut.ties);
            eq += __popcll(bq);
        }
        const uint64_t bt = __ballot(take);
        if (take) put(at_out + __popcll(bt & below), 64 * u + lane);
        at_out += __popcll(bt);
    }
    for (int i = at_out + lane; i < n_sel; i += 64) put(i, -1);
}

// Scores of 16 blocks and 16 rows by the fp64 matrix instruction, 4 elements each time: lane (c, g) has elements HD / 4 * g ..
// of row c's query sum (in registers) and of block c's mean; every sum adds its terms in the same order.  Waves take every
// eighth tile of blocks, the next one's means on their way, then every eighth row's list.  The upper halves of the keys are kept:
// whole ones of more than 1024 blocks would leave no room for 16 rows, and the rest of the 16 columns idle (2000 rows on 1032 /
// 2063 blocks, 4 KV heads: 80 / 241 us, with whole keys 134 / 576).  2001 rows on 500 blocks: 40 us, of which 8 to the
// query sums (21 where each wave makes its own), 22 scores (13 of them the matrix instructions'), 10 lists (all scores equal: 200;
// whole keys 40).
template <int HD, int AT, int R, int CAP> __global__ __launch_bounds__(RT) void k_attn_select_rows(const SelectArgs a)
{
    constexpr int KS = HD / 4, LD = CAP + 1, NW = RT / 64;   // steps; keys of a row, off the banks of the one before
    constexpr int E = 16 * HD / RT, LQ = HD + 2;             // a thread's elements of the query sums, and their rows in LDS
    static_assert(E == 2 || E == 4, "");
    __shared__ uint32_t key[R * LD];   // upper halves
    __shared__ double qsum[R * LQ];
    const int lane = threadIdx.x & 63, w = wave_id(), c = lane & 15, g = lane >> 4;
    const int n_kv = a.c.n_head_kv, kvh = blockIdx.x % n_kv, row0 = blockIdx.x / n_kv * R;
    const int G = a.c.n_head / n_kv, psh = __builtin_ctz(a.c.page), rows = min(R, a.b.n_rows - row0);
    for (int j = 0; j < rows;) {
        PagedSeq q;
        const int s = paged_find(a.b, row0 + j, q);
        if (s >= a.b.n_seq) return;
        if (!q.holds(row0 + j)) {
            j++;
            continue;
        }
        const int n = min(rows - j, q.q0 + q.q_len - (row0 + j)), first = row0 + j;   // rows of this sequence
        j += n;
        if (a.apart && q.q_len < MANY) continue;
        const int own_last = q.position(first + n - 1) >> psh;   // the last row's own block (below 0: no position)
        const int own = q.position(first + min(c, n - 1)) >> psh;
        const int *tab = a.b.block_table + (size_t)s * a.b.table_ld;
        const uint16_t *means = a.means + (size_t)kvh * HD + KS * g;
        auto page = [&](int t) __attribute__((always_inline)) {
            const int b = 16 * t + c, pg = b <= own_last ? tab[b] : -1;
            return pg >= 0 && pg < a.c.n_pages ? pg : -1;
        };
        v4u m[KS / 8];
        auto load = [&](int pg) __attribute__((always_inline)) {
            const v4u *p = (const v4u *)(means + (size_t)max(pg, 0) * n_kv * HD);
#pragma unroll
            for (int i = 0; i < KS / 8; i++) m[i] = p[i];
        };
        int pg = page(w), pn = page(w + NW);
        load(pg);
        // the sums of the queries, by all threads
        __syncthreads();   // the lists of the rows before are made
        if (const int qr = threadIdx.x / (HD / E), e0 = threadIdx.x % (HD / E) * E; qr < n) {
            const uint16_t *p = a.q + (size_t)(first + qr) * a.ldq + (size_t)kvh * G * HD + e0;
            double y[E];
#pragma unroll
            for (int e = 0; e < E; e++) y[e] = 0.0;
#pragma unroll 4
            for (int h = 0; h < G; h++, p += HD) {
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const uint32_t u = ((const uint32_t *)p)[e / 2];
                    y[e] += (double)act2f<AT>(u & 0xffffu);
                    y[e + 1] += (double)act2f<AT>(u >> 16);
                }
            }
#pragma unroll
            for (int e = 0; e < E; e++) qsum[qr * LQ + e0 + e] = y[e];
        }
        __syncthreads();
        double x[KS];
#pragma unroll
        for (int e = 0; e < KS; e++) x[e] = qsum[min(c, n - 1) * LQ + KS * g + e];
        for (int t = w; 16 * t <= own_last; t += NW) {
            const uint64_t ok = __ballot(pg >= 0);
            v4u now[KS / 8];
#pragma unroll
            for (int i = 0; i < KS / 8; i++) now[i] = m[i];
            load(pn);
            pg = pn;
            pn = page(t + 2 * NW);
            v4d y[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};   // two sums, so that an instruction need not wait for the one before
#pragma unroll
            for (int i = 0; i < KS / 8; i++) {
                float v[8];
                elems16<AT>(now[i], v);
#pragma unroll
                for (int e = 0; e < 8; e++) y[e & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64((double)v[e], x[8 * i + e], y[e & 1], 0, 0, 0);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {   // blocks 4 e + g, row c
                const int b = 16 * t + 4 * e + g;
                const bool always = b < a.pick.n_first || b > own - a.pick.n_last;
                const double z = y[0][e] + y[1][e];
                if (c < n && b < CAP) key[c * LD + b] = (uint32_t)((!(ok >> (4 * e + g) & 1) ? KEY_NONE : (always ? KEY_ALWAYS : score_key(z))) >> 32);
            }
        }
        __syncthreads();
        for (int r = w; r < n; r += NW) {
            const int pos = q.position(first + r);
            int *out = a.sel + ((size_t)(first + r) * n_kv + kvh) * a.pick.n_sel;
            if (pos < 0) {
                for (int i = lane; i < a.pick.n_sel; i += 64) out[i] = -1;
            } else {
                // the lower half of block b's key; its upper half, summed in another order, may be the next one to yh
                auto low = [&](int b, uint32_t yh) {
                    const v4u *p = (const v4u *)(a.means + ((size_t)tab[b] * n_kv + kvh) * HD);
                    double y = 0.0;
                    for (int i = 0; i < HD / 8; i++) {
                        float v[8];
                        elems16<AT>(p[i], v);
#pragma unroll
                        for (int e = 0; e < 8; e++) y = __builtin_fma(qsum[r * LQ + 8 * i + e], (double)v[e], y);
                    }
                    const uint64_t x = score_key(y);
                    const uint32_t h = (uint32_t)(x >> 32);
                    return h == yh ? (uint32_t)x : (h > yh ? ~0u : 0u);
                };
                select_row<CAP>(key + r * LD, (pos >> psh) + 1, a.pick.n_sel, low, [&](int i, int k) __attribute__((always_inline)) { out[i] = k; });
            }
        }
    }
}

template <int HD, int AT, int R, int CAP> hipError_t select_rows(const SelectArgs &a, hipStream_t s)
{
    const unsigned grid = (unsigned)(((int64_t)a.b.n_rows + R - 1) / R * a.c.n_head_kv);
    k_attn_select_rows<HD, AT, R, CAP><<<grid, RT, 0, s>>>(a);
    return hipGetLastError();
}

// Which kernels a batch takes: rows together, where a sequence can have MANY (and their keys find room in LDS); one by one,
// where none can.  Where the bounds leave room for both, both run and leave the other's sequences alone (with few sequences,
// the second looks at MANY - 1 rows of each: by rows of the batch, 2 x 1000 rows on 1563 blocks took 65 us more); where every
// sequence may have max_q rows, the first takes whatever there is.  2000 rows on 4096 blocks together: 433 us; on 4097, one by
// one: 1142, on 8000 1955, on 16384 4000.
template <int HD, int AT> hipError_t select_by_size(SelectArgs a, hipStream_t s)
{
    const int n = (a.b.max_kv - 1) / a.c.page + 1;
    if (a.b.max_q >= MANY && n <= 4096) {
        a.apart = (int64_t)a.b.n_seq * a.b.max_q > a.b.n_rows;
        const hipError_t e = n <= 512 ? select_rows<HD, AT, 16, 512>(a, s) : n <= 1024 ? select_rows<HD, AT, 16, 1024>(a, s) : n <= 2048 ? select_rows<HD, AT, 16, 2048>(a, s) : select_rows<HD, AT, 8, 4096>(a, s);
        if (e != hipSuccess || !a.apart) return e;
    }
    a.by_seq = a.apart && (int64_t)a.b.n_seq * (MANY - 1) < a.b.n_rows;
    const unsigned grid = (unsigned)((int64_t)(a.by_seq ? a.b.n_seq * (MANY - 1) : a.b.n_rows) * a.c.n_head_kv);
    // few rows: more waves for each (16 rows of 938 blocks, 8 elements per lane: 19 / 26 us with 16 / 4 waves)
    if (n <= 1024 && grid <= 512) k_attn_select<HD, AT, 1024, 1024, 2><<<grid, 1024, 0, s>>>(a);
    else if (n <= 1024) k_attn_select<HD, AT, 256, 1024, 2><<<grid, 256, 0, s>>>(a);
    else
        for (constexpr unsigned MOST = 1u << 21; a.block0 < grid; a.block0 += MOST)   // launches of less than 2^32 threads
            k_attn_select<HD, AT, 1024, X100_SPARSE_MAX_BLOCKS, 4><<<std::min(MOST, grid - a.block0), 1024, 0, s>>>(a);
    return hipGetLastError();
}

template <int HD, int AT> hipError_t means_as(const x100_kv_cfg &c, const x100_kv_batch &b, const void *kp, void *means, hipStream_t s)
{
    const unsigned grid = (unsigned)(((int64_t)b.n_rows + MEAN_ROWS - 1) / MEAN_ROWS * c.n_head_kv);
    if (c.kv_type == X100_KV_Q4) k_kv_means<HD, AT, true><<<grid, 256, 0, s>>>(c, b, (const uint8_t *)kp, (uint16_t *)means);
    else k_kv_means<HD, AT, false><<<grid, 256, 0, s>>>(c, b, (const uint8_t *)kp, (uint16_t *)means);
    return hipGetLastError();
}

}  // namespace

hipError_t x100_kv_means_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *kp, void *means, hipStream_t s)
{
    if (c.head_dim == 64)
        return c.act_type == X100_T_F16 ? means_as<64, X100_T_F16>(c, b, kp, means, s) : means_as<64, X100_T_BF16>(c, b, kp, means, s);
    return c.act_type == X100_T_F16 ? means_as<128, X100_T_F16>(c, b, kp, means, s) : means_as<128, X100_T_BF16>(c, b, kp, means, s);
}

hipError_t x100_attn_select_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const x100_kv_sel &pick, const void *q,
                                   int64_t ldq, const void *means, int *sel, hipStream_t s)
{
    const SelectArgs a = {c, b, pick, (const uint16_t *)q, ldq, (const uint16_t *)means, sel, false, false, 0};
    if (c.head_dim == 64) return c.act_type == X100_T_F16 ? select_by_size<64, X100_T_F16>(a, s) : select_by_size<64, X100_T_BF16>(a, s);
    return c.act_type == X100_T_F16 ? select_by_size<128, X100_T_F16>(a, s) : select_by_size<128, X100_T_BF16>(a, s);
}
