// Which blocks of the paged cache a query attends to (x100_sparse.h): mean keys of full pages, and the selection.
//
// The score of block b for a row and KV head is (the sum of the KV head's queries) . (the block's mean key), which is the
// mean of their scores with the block's keys.  It is summed in fp64 (a product of two 16-bit numbers is exact there): two
// blocks change places only where their scores differ by 1e-16 of their terms, so the lists do not depend on an order
// of sums, and equal blocks tie.
#include "paged.h"
#include "x100_internal.h"

namespace {

X100_DEV double xor_d(double v, int m)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    uint32_t lo = (uint32_t)u, hi = (uint32_t)(u >> 32);
    lo = m == 32 ? xor32_u(lo) : xor16_u(lo);
    hi = m == 32 ? xor32_u(hi) : xor16_u(hi);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
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

// Mean keys.  A block looks at 16 rows of the batch; a wave takes every fourth of those that end a page.  Lane l has the
// elements 8 (l % L) .. + 7 of rows l / L, l / L + 64 / L, ... of the page (L lanes per row), 8 loads on their way.
// Bound by the chain row -> sequence -> page -> keys for single tokens, by the keys' bytes for prompts.
constexpr int MEAN_ROWS = 16;
template <int HD, int AT, bool Q4>
__global__ __launch_bounds__(256) void k_kv_means(const x100_kv_cfg c, const x100_kv_batch b, const uint8_t *kp, uint16_t *means)
{
    constexpr int L = HD / 8, RS = 64 / L;   // lanes of a row, rows of a step
    const int lane = threadIdx.x & 63, w = wave_id(), kvh = blockIdx.x % c.n_head_kv, row0 = blockIdx.x / c.n_head_kv * MEAN_ROWS;
    const int psh = __builtin_ctz(c.page);
    // lane i: page of row row0 + i, if that row is the last of a page
    int pg = -1;
    for (int i = 0; i < MEAN_ROWS && row0 + i < b.n_rows; i += 1) {
        if ((i & 3) != w) continue;
        const int row = row0 + i, s = paged_find(b, row);
        if (s >= b.n_seq) break;
        const PagedSeq q = paged_seq(b, s);
        if (!q.holds(row)) continue;
        const int pos = q.position(row);
        if (pos < 0 || (pos & (c.page - 1)) != c.page - 1) continue;
        pg = paged_page(c, b, s, pos);
        if (pg < 0) continue;
        const uint8_t *kb = kp + ((size_t)pg * c.n_head_kv + kvh) * page_head_bytes<HD, Q4>(c.page);
        double sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        const int r0 = lane / L, e0 = lane % L;
        for (int r = r0; r < c.page; r += 4 * RS) {   // a page has at least 16 rows: some lanes' steps may lie behind it
            float v[4][8];
#pragma unroll
            for (int u = 0; u < 4; u++) {
                const int rr = min(r + u * RS, c.page - 1);
                if constexpr (!Q4) elems16<AT>(*(const v4u *)(kb + ((size_t)rr * HD + 8 * e0) * 2), v[u]);
                else
                    elems_q4(((const uint32_t *)kb)[rr * L + e0],
                             ((const uint32_t *)(kb + c.page * HD / 2))[rr * (HD / 32) + e0 / 4], v[u]);
            }
#pragma unroll
            for (int u = 0; u < 4; u++) {
                if (r + u * RS >= c.page) continue;
#pragma unroll
                for (int e = 0; e < 8; e++) sum[e] += (double)v[u][e];
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            if constexpr (L == 8) {   // rows of lanes l and l ^ 8 too
                const uint64_t u = __builtin_bit_cast(uint64_t, sum[e]);
                const uint32_t lo = dpp_i<0x128>(0, (int)(uint32_t)u), hi = dpp_i<0x128>(0, (int)(uint32_t)(u >> 32));
                sum[e] += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
            }
            sum[e] += xor_d(sum[e], 16);
            sum[e] += xor_d(sum[e], 32);
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

// Keys are compared as unsigned numbers, in the order of the scores.  0: not to be selected; all ones: always.
constexpr uint64_t KEY_NONE = 0, KEY_ALWAYS = ~0ull;
X100_DEV uint64_t score_key(double s)
{
    if (!(s == s)) s = -__builtin_inf();
    s += 0.0;   // -0 is 0
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    return u >> 63 ? ~u : u | 1ull << 63;
}

struct SelectArgs {
    x100_kv_cfg c;
    x100_kv_batch b;
    x100_kv_sel pick;
    const uint16_t *q;
    int64_t ldq;
    const uint16_t *means;
    int *sel;
};

constexpr int ST = 256;   // threads of a block

template <int HD, int R, int CAP> struct SelectLds {
    uint64_t key[R][CAP];
    double q[R][HD];
    int hist[256];
    int bin, above, same;        // the digit of the list's last key, keys above it, keys with it
    int gt[ST / 64], eq[ST / 64];
};

// The list of the n keys k (n > 0): the n_sel largest that are not KEY_NONE, lowest index first among equal ones,
// ascending.  The smallest of them is found 8 bits at a time, until a digit's keys are all in or all digits are known.
template <class Lds> X100_DEV void select_keys(Lds &sh, const uint64_t *k, int n, int n_sel, int *out)
{
    const int t = threadIdx.x, lane = t & 63, w = wave_id();
    uint64_t low = 1;      // selected: keys >= low,
    int ties = 0;          // or, if ties > 0, keys > low and the first `ties` keys that are low
    if (n > n_sel) {
        uint64_t prefix = 0, mask = 0;
        int need = n_sel;
        for (int shift = 56; shift >= 0; shift -= 8) {
            sh.hist[t] = 0;
            __syncthreads();
            for (int i = t; i < n; i += ST)
                if ((k[i] & mask) == prefix) atomicAdd(&sh.hist[(int)(k[i] >> shift) & 255], 1);
            __syncthreads();
            if (w == 0) {   // lane l: bins 255 - 4 l .. 252 - 4 l
                int c[4], s = 0;
#pragma unroll
                for (int e = 0; e < 4; e++) s += c[e] = sh.hist[255 - 4 * lane - e];
                int upto = s;   // of the lanes up to this one
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int y = __shfl_up(upto, d, 64);
                    if (lane >= d) upto += y;
                }
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
            __syncthreads();
            prefix |= (uint64_t)sh.bin << shift;
            mask |= 255ull << shift;
            need -= sh.above;
            const bool all = sh.same == need;
            __syncthreads();   // bin, above and same are read
            if (all) {
                low = prefix;
                break;
            }
            if (shift == 0) {
                low = prefix;
                ties = need;
            }
        }
        if (low == KEY_NONE) {   // blocks without a page would be among them
            low = 1;
            ties = 0;
        }
    }
    // wave w has the w-th quarter of the keys, in order
    const int part = (n + 4 * 64 - 1) / (4 * 64) * 64, i0 = min(n, w * part), i1 = min(n, i0 + part);
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
    for (int v = 0, e = 0; v < ST / 64; v++) {
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
    for (int i = total + t; i < n_sel; i += ST) out[i] = -1;
}

// A block: R rows of the batch and one KV head.  Rows of one sequence read its means together: thread t has blocks t, t +
// 256, ... of the sequence, whose mean it loads once for the rows.  Bound by the means' bytes for single tokens
// (each row and KV head reads its own), by the fp64 unit for prompts.
template <int HD, int AT, int R, int CAP> __global__ __launch_bounds__(ST) void k_attn_select(const SelectArgs a)
{
    __shared__ SelectLds<HD, R, CAP> sh;
    const int t = threadIdx.x, n_kv = a.c.n_head_kv, kvh = blockIdx.x % n_kv, row0 = blockIdx.x / n_kv * R;
    const int G = a.c.n_head / n_kv, psh = __builtin_ctz(a.c.page), rows = min(R, a.b.n_rows - row0);
    for (int j = 0; j < rows;) {
        const int s = paged_find(a.b, row0 + j);
        if (s >= a.b.n_seq) return;
        const PagedSeq q = paged_seq(a.b, s);
        if (!q.holds(row0 + j)) {
            j++;
            continue;
        }
        const int n = min(rows - j, q.q0 + q.q_len - (row0 + j));   // rows of this sequence
        const int own_last = q.position(row0 + j + n - 1) >> psh;   // the last row's own block (below 0: no position)
        __syncthreads();   // the rows before are done with sh
        for (int u = t; u < n * HD; u += ST) {
            const int r = u / HD, e = u % HD;
            const uint16_t *x = a.q + (size_t)(row0 + j + r) * a.ldq + (size_t)kvh * G * HD + e;
            double y = 0.0;
            for (int h = 0; h < G; h++) y += (double)act2f<AT>(x[h * HD]);
            sh.q[r][e] = y;
        }
        __syncthreads();
        const int *tab = a.b.block_table + (size_t)s * a.b.table_ld;
        for (int blk = t; blk <= own_last; blk += ST) {
            const int pg = tab[blk];
            const bool ok = pg >= 0 && pg < a.c.n_pages;
            double y[R];
#pragma unroll
            for (int r = 0; r < R; r++) y[r] = 0.0;
            if (ok) {
                const v4u *m = (const v4u *)(a.means + ((size_t)pg * n_kv + kvh) * HD);
                v4u x[HD / 8];
#pragma unroll
                for (int i = 0; i < HD / 8; i++) x[i] = m[i];
#pragma unroll
                for (int i = 0; i < HD / 8; i++) {
                    float v[8];
                    elems16<AT>(x[i], v);
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const double d = (double)v[e];
#pragma unroll
                        for (int r = 0; r < R; r++) y[r] = __builtin_fma(sh.q[r][8 * i + e], d, y[r]);
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < R; r++) {
                if (r >= n) continue;
                const int own = q.position(row0 + j + r) >> psh;
                const bool always = blk < a.pick.n_first || blk > own - a.pick.n_last;
                sh.key[r][blk] = !ok ? KEY_NONE : (always ? KEY_ALWAYS : score_key(y[r]));
            }
        }
        __syncthreads();
        for (int r = 0; r < n; r++) {
            const int pos = q.position(row0 + j + r);
            int *out = a.sel + ((size_t)(row0 + j + r) * n_kv + kvh) * a.pick.n_sel;
            if (pos < 0) {
                for (int i = t; i < a.pick.n_sel; i += ST) out[i] = -1;
                continue;
            }
            if (r) __syncthreads();   // the counts of the row before are read
            select_keys(sh, sh.key[r], (pos >> psh) + 1, a.pick.n_sel, out);
        }
        j += n;
    }
}

template <int HD, int AT, int R, int CAP> hipError_t select(const SelectArgs &a, hipStream_t s)
{
    const unsigned grid = (unsigned)(((int64_t)a.b.n_rows + R - 1) / R * a.c.n_head_kv);
    k_attn_select<HD, AT, R, CAP><<<grid, ST, 0, s>>>(a);
    return hipGetLastError();
}

// Rows of a block by whether sequences have several, and what their keys take in LDS.
template <int HD, int AT> hipError_t select_by_size(const SelectArgs &a, hipStream_t s)
{
    const int n = (a.b.max_kv - 1) / a.c.page + 1;
    if (a.b.max_q >= 4 && n <= 1024) return select<HD, AT, 4, 1024>(a, s);
    if (a.b.max_q >= 4 && n <= 4096) return select<HD, AT, 4, 4096>(a, s);
    if (n <= 1024) return select<HD, AT, 1, 1024>(a, s);
    return select<HD, AT, 1, X100_SPARSE_MAX_BLOCKS>(a, s);
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
    const SelectArgs a = {c, b, pick, (const uint16_t *)q, ldq, (const uint16_t *)means, sel};
    if (c.head_dim == 64) return c.act_type == X100_T_F16 ? select_by_size<64, X100_T_F16>(a, s) : select_by_size<64, X100_T_BF16>(a, s);
    return c.act_type == X100_T_F16 ? select_by_size<128, X100_T_F16>(a, s) : select_by_size<128, X100_T_BF16>(a, s);
}
