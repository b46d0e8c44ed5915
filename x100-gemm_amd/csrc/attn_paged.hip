// Attention over the paged KV cache (x100_paged.h).
//
// o = sum_p softmax_p(scale q.K_p) V_p over the positions p <= the row's own, online: running maximum
// m and sum l per row, O rescaled when m rises.  The query heads of a KV head are rows of one tile:
// row i of a sequence and KV head is token i / G, head i % G (G query heads per KV head), so that a
// K and V row is read once for all of them.
//
// Scores come transposed, S^T = K Q^T (a lane holds one query row and several positions), which is the
// operand layout of O^T = V^T P^T: the weights go from the first product to the second in the
// registers they were made in.  The cache keeps V in blocks of 8 positions per element for the same
// reason: a lane's operand of V^T is one 16-byte load (16 bits) or one word (4 bits).
//
// The weights are rounded to 16 bits for the second product, which takes no more; their sum is of the rounded ones, so
// that they still sum to one.  Against 64 bits the results' distance (2-norm, relative) grows from the result's own
// rounding, 0.0016 in bf16 and 0.00021 in f16, to 0.0018-0.0021 and 0.00028.  A second product with what the rounding left
// would cost single tokens nothing, but make a NaN of every infinity in V whose weight 16 bits hold exactly.
//
// Here: k_attn_tile for sequences of few rows (bound by the cache's bytes) and for rows with lists of blocks
// (x100_sparse.h), k_attn_join, which merges split results, and a call's layout.  attn_prompt.hip has the kernel of many rows (bound by the matrix cores).
#include <algorithm>

#include "paged_attn.h"
#include "x100_internal.h"
#include "x100_sparse.h"

namespace {

constexpr float NEG_INF = X100_NEG_INF;
using AttnArgs = PagedAttnArgs;
constexpr int TILE_ROWS = 16;     // rows (token, head) of a block of the tile kernel
constexpr int TILE_PAGES = 512;   // most pages of a split of the tile kernel (their list is in LDS)

// What a lane reads of a tile of 32 positions, as the cache holds it: K rows 8 (c / 4) + 4 h + c % 4 (h = 0,
// 1), V block 8 g .. 8 g + 7.
template <int HD, bool Q4> struct TileRegs;
template <int HD> struct TileRegs<HD, false> {
    v4u k[2][HD / 32], v[HD / 16];
    bool ok;             // the page of the V block (and of the scores' positions) is one
};
template <int HD> struct TileRegs<HD, true> {
    uint32_t k[2][HD / 32], ks[2];
    v4u v[HD / 64], vd[HD / 64], vm[HD / 64];
    bool ok;
};

// One block: 16 rows (token, head) of a sequence and KV head, one split of the positions; its four waves
// take tiles of 32 positions in turn and merge at the end.
// Lane (c = lane % 16, g = lane / 16): query row c; of a tile the positions 8 g .. 8 g + 7.
// The loop is bound by memory as long as loads are always in flight: K and V of the next tile are requested
// as soon as their registers are free, the pages come from a list in LDS.  63 sequences of 4096 positions, 32 heads on 4 of
// 128, bf16: 91 us, 5.8 TB/s (a read of 2 GiB: 6.1); 16 of up to 60001 in 4 bits: 94 us, 4.8 TB/s, where unpacking
// takes half of the issue slots.  One of 1024: 6.5 us, the chain of loads lengths -> pages -> K -> V.
//
// SP (x100_sparse.h): a tile is one token's rows, with a list of blocks of its own.  The list's pages in order are a
// sequence to the rest of the kernel: its positions are counted through them, and only the last block can be the token's
// own, of which the positions behind it are left out.
template <int HD, int AT, bool Q4, bool SP> __global__ __launch_bounds__(256, Q4 || HD == 64 ? 4 : 3) void k_attn_tile(const AttnArgs a)
{
    constexpr int MT = Q4 ? X100_T_F16 : AT;   // type on the matrix cores
    constexpr int NW = 4;                      // waves
    constexpr int KS = HD / 32, NJ = HD / 16;  // steps of K Q^T, element tiles of V^T P^T
    __shared__ union {
        int pg[TILE_PAGES];                     // pages of the split, -1 where there is none
        float o[NW][16][HD + 4];               // at the end
    } sh;
    __shared__ float s_m[NW][16], s_l[NW][16];
    const int lane = threadIdx.x & 63, w = wave_id(), c = lane & 15, g = lane >> 4;
    const int n_kv = a.c.n_head_kv, G = a.c.n_head / n_kv, page = a.c.page, psh = __builtin_ctz(page);
    int sp, kvh, s, i0, row0, kv_len, n_rows, pos0, vis, ns, per, pg0;   // row0: token 0's row, pos0: its position
    auto valid = [&](int pg) __attribute__((always_inline)) { return pg >= 0 && pg < a.c.n_pages ? pg : -1; };
    if constexpr (SP) {
        const int unit = blockIdx.x;
        kvh = unit % n_kv;
        sp = unit / n_kv % a.tile.n;
        row0 = unit / (n_kv * a.tile.n);
        i0 = 0;
        n_rows = G;
        const int *list = a.sel + ((size_t)row0 * n_kv + kvh) * a.n_sel;
        constexpr int LE = X100_SPARSE_MAX_SEL / (64 * NW);   // entries of a thread: on their way beside the search
        int entry[LE], before[LE];
#pragma unroll
        for (int k = 0; k < LE; k++) {
            const int i = threadIdx.x + 64 * NW * k;
            entry[k] = i < a.n_sel ? list[i] : -1;
            before[k] = i < a.n_sel && i ? list[i - 1] : -1;
        }
        PagedSeq q;
        s = paged_find(a.b, row0, q);
        if (!q.holds(row0)) return;
        const int at = q.position(row0), own = at >> psh;   // below 0: no block
        const int *tab = a.b.block_table + (size_t)s * a.b.table_ld;
        // the list's pages, up to the first entry that breaks its order
        __shared__ int s_cnt[NW], s_own[NW];
        int end = a.n_sel, own_at = a.n_sel;
#pragma unroll
        for (int k = 0; k < LE; k++) {
            const int i = threadIdx.x + 64 * NW * k, e = entry[k];
            if (i >= a.n_sel) continue;
            const bool ok = e > before[k] && e >= 0 && e <= own;
            if (!ok) end = min(end, i);
            if (ok && e == own) own_at = min(own_at, i);
            sh.pg[i] = ok ? valid(tab[e]) : -1;
        }
        end = -wave_max_iu(-end);
        own_at = -wave_max_iu(-own_at);
        if (lane == 0) {
            s_cnt[w] = end;
            s_own[w] = own_at;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NW; k++) end = min(end, s_cnt[k]);
        vis = end * page;
#pragma unroll
        for (int k = 0; k < NW; k++)   // entries ascend up to the end, so only the last one, and a wave's first such, can be the own block
            if (s_own[k] == end - 1) vis = end * page - (page - 1 - (at & (page - 1)));
        kv_len = vis;
        pos0 = vis - 1;
        per = a.tile.positions(a.n_sel << psh);
        ns = a.tile.n;
        pg0 = 0;
    } else {
        // Units (sequence, KV head, split) in runs of a.run, each run with all its tiles (plan_of)
        const int unit = blockIdx.x / (a.run * a.tiles) * a.run + blockIdx.x % a.run, tile = blockIdx.x / a.run % a.tiles;
        sp = unit % a.tile.n;
        kvh = unit / a.tile.n % n_kv;
        s = unit / (a.tile.n * n_kv);
        if (s >= a.b.n_seq) return;
        i0 = tile * 16;
        // A short table's pages are read here, beside the lengths; a long one's when the split is known.
        const int *tab = a.b.block_table + (size_t)s * a.b.table_ld;
        const int n_all = (a.b.max_kv + page - 1) >> psh;
        const bool all = n_all <= TILE_PAGES;
        auto list = [&](int first, int n) {
            for (int i = threadIdx.x; i < n; i += 64 * NW) sh.pg[i] = valid(tab[first + i]);
        };
        if (all) list(0, n_all);
        const PagedSeq q = paged_seq(a.b, s);
        row0 = q.q0;
        kv_len = q.kv_len;
        n_rows = q.q_len * G;
        if (i0 >= n_rows || n_rows > a.few) return;
        pos0 = kv_len - q.q_len;
        vis = pos0 + (min(i0 + 15, n_rows - 1)) / G + 1;   // positions that the tile's last row sees
        per = a.tile.positions(kv_len);
        ns = max(1, (vis + per - 1) / per);
        if (sp >= ns) return;
        const int t0 = sp * per, t1 = min(t0 + per, vis);
        pg0 = all ? 0 : t0 >> psh;                         // first page of the list
        if (!all) list(pg0, t1 > t0 ? ((t1 - 1) >> psh) - (t0 >> psh) + 1 : 0);
    }
    const int t0 = sp * per, t1 = min(t0 + per, vis);
    const int n_pg = t1 > t0 ? ((t1 - 1) >> psh) - (t0 >> psh) + 1 : 0;

    const int i = min(i0 + c, n_rows - 1), tok = SP ? 0 : i / G, head = kvh * G + i % G;
    const int pos = pos0 + tok;
    const int pos_lo = pos0 + (SP ? 0 : i0 / G);               // the tile's first row's
    const size_t head_bytes = page_head_bytes<HD, Q4>(page);
    // positions up to here are seen by every row, on pages that are
    __syncthreads();
    bool none = false;
    for (int i = lane; i < n_pg; i += 64) none |= sh.pg[(t0 >> psh) - pg0 + i] < 0;
    const int whole = __any(none) ? t0 : min(t1, pos_lo + 1);

    // K, and V, of tile t into registers
    TileRegs<HD, Q4> R;
    const uint8_t *kp = a.kp + (size_t)kvh * head_bytes, *vp = a.vp + (size_t)kvh * head_bytes;
    auto load_k = [&](int t) __attribute__((always_inline)) {
        const int kb = t + 8 * (c >> 2);
        const int pg = kb < t1 ? sh.pg[(kb >> psh) - pg0] : -1;
        const uint8_t *kpage = kp + (size_t)max(pg, 0) * n_kv * head_bytes;
        const int koff = (kb & (page - 1)) + (c & 3);
        if constexpr (!Q4) {
            const uint16_t *kr = (const uint16_t *)kpage + koff * HD + 8 * g;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int j = 0; j < KS; j++) R.k[h][j] = *(const v4u *)(kr + 4 * h * HD + 32 * j);
        } else {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t *kr = (const uint32_t *)kpage + (koff + 4 * h) * (HD / 8) + g * KS;
                if constexpr (KS == 4) {
                    const v4u x = __builtin_nontemporal_load((const v4u *)kr);
#pragma unroll
                    for (int j = 0; j < 4; j++) R.k[h][j] = x[j];
                } else {
                    const v2u x = *(const v2u *)kr;
                    R.k[h][0] = x[0];
                    R.k[h][1] = x[1];
                }
                R.ks[h] = ((const uint32_t *)(kpage + page * HD / 2))[(koff + 4 * h) * (HD / 32) + g * HD / 128];
            }
        }
    };
    auto load_v = [&](int t) __attribute__((always_inline)) {
        const int vb = t + 8 * g;
        const int pg = vb < t1 ? sh.pg[(vb >> psh) - pg0] : -1;
        R.ok = pg >= 0;
        const uint8_t *vpage = vp + (size_t)max(pg, 0) * n_kv * head_bytes;
        const int vblk = (vb & (page - 1)) >> 3;
        if constexpr (!Q4) {
            const uint16_t *vr = (const uint16_t *)vpage + vblk * (HD * 8) + 8 * c;
#pragma unroll
            for (int j = 0; j < NJ; j++) R.v[j] = *(const v4u *)(vr + 128 * j);
        } else {
            const uint32_t *vr = (const uint32_t *)vpage + vblk * HD + 4 * c;
            const uint8_t *vs = vpage + page * HD / 2 + (vblk * (HD / 32) + (c >> 3)) * 32;
#pragma unroll
            for (int u = 0; u < HD / 64; u++) {   // elements 64 u + 4 c .. + 3, of group 2 u + c / 8
                R.v[u] = __builtin_nontemporal_load((const v4u *)(vr + 64 * u));
                R.vd[u] = *(const v4u *)(vs + 64 * u);
                R.vm[u] = *(const v4u *)(vs + 64 * u + 16);
            }
        }
    };
    const int tw = t0 + 32 * w;
    if (tw < t1) {
        load_k(tw);
        load_v(tw);
    }

    v4u qf[KS];
    float sc2 = a.scale2;
    {
        const uint16_t *qr = a.q + (size_t)(row0 + tok) * a.ldq + (size_t)head * HD;
#pragma unroll
        for (int j = 0; j < KS; j++) qf[j] = *(const v4u *)(qr + (Q4 ? g * (HD / 4) + 8 * j : 32 * j + 8 * g));
        if constexpr (Q4 && AT == X100_T_BF16) {
            float mx = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    mx = fmaxf(mx, fmaxf(fabsf(bf2f(qf[j][e] & 0xffffu)), fabsf(__uint_as_float(qf[j][e] & 0xffff0000u))));
            mx = fmaxf(mx, xor16_f(mx));
            mx = fmaxf(mx, xor32_f(mx));
            const int ex = row_exponent(mx);
            sc2 = ldexpf(sc2, ex);
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    qf[j][e] = pack2<X100_T_F16>(ldexpf(bf2f(qf[j][e] & 0xffffu), -ex),
                                                 ldexpf(__uint_as_float(qf[j][e] & 0xffff0000u), -ex));
        }
    }

    v4f o[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) o[j] = v4f{0, 0, 0, 0};
    float m = NEG_INF, msub = 0.0f, l = 0.0f;

    // S^T: tile row r of half h is position 8 (r / 4) + 4 h + r % 4, so that lane (c, g) receives
    // positions 8 g + 4 h .. + 3 of row c
    v4f sc[2];
    auto scores = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v4f y = {0, 0, 0, 0};
            if constexpr (!Q4) {
#pragma unroll
                for (int j = 0; j < KS; j++) y = Mfma16<MT>::mul(R.k[h][j], qf[j], y);
            } else {
                const v2h d2 = as_h2((R.ks[h] & 0xffffu) * 0x10001u), m2 = as_h2((R.ks[h] >> 16) * 0x10001u);
#pragma unroll
                for (int j = 0; j < KS; j++) {
                    v2h n[4];
                    q4_unpack(R.k[h][j], n);
                    v4u k;
#pragma unroll
                    for (int e = 0; e < 4; e++) k[e] = __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(n[e], d2, m2));
                    y = Mfma16<MT>::mul(k, qf[j], y);
                }
            }
            sc[h] = y;
        }
    };
    // The weights p, relative to m (tile_lift), which may stay up to 8 (a factor of 256) behind.
    v4u p;
    auto weights = [&]() __attribute__((always_inline)) {
        float mx = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
        for (int e = 1; e < 4; e++) mx = fmaxf(fmaxf(mx, sc[0][e]), sc[1][e]);
        mx = __builtin_fmaf(mx, sc2, -tile_lift<MT>());
        if (__any(mx > m + 8.0f)) {
            mx = fmaxf(mx, xor16_f(mx));
            mx = fmaxf(mx, xor32_f(mx));
            const float mn = fmaxf(m, mx);
            const float f = __builtin_amdgcn_exp2f(mn == NEG_INF ? 0.0f : m - mn);
            m = mn;
            msub = mn == NEG_INF ? 0.0f : mn;
            l *= f;
#pragma unroll
            for (int j = 0; j < NJ; j++) o[j] *= f;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e >> 1][2 * (e & 1)], sc2, -msub));
            const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e >> 1][2 * (e & 1) + 1], sc2, -msub));
            p[e] = pack2<MT>(p0, p1);
            l = add2<MT>(p[e], l);
        }
    };

    int t = tw;
    for (; t + 32 <= whole; t += 32 * NW) {
        const int tn = t + 32 * NW;
        scores();
        if (tn < t1) load_k(tn);
        weights();
        // O^T += V^T P^T
        if constexpr (!Q4) {
#pragma unroll
            for (int j = 0; j < NJ; j++) o[j] = Mfma16<MT>::mul(R.v[j], p, o[j]);
        } else {
#pragma unroll
            for (int u = 0; u < HD / 64; u++)
#pragma unroll
                for (int k = 0; k < 4; k++) o[4 * u + k] = Mfma16<MT>::mul(q4_v(R.v[u][k], R.vd[u], R.vm[u]), p, o[4 * u + k]);
        }
        if (tn < t1) load_v(tn);
    }
    // Tiles that not every row sees whole, one element tile of V per turn, the accumulators and operands
    // moving up (unrolled, this would cost the loop above its registers).
    for (; t < t1; t += 32 * NW) {
        const int vb = t + 8 * g;
        scores();
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (!(R.ok && vb + e <= pos)) sc[e >> 2][e & 3] = NEG_INF;
        weights();
        // positions that no row of the sequence has, and those of a page that is none: V as zeros
        uint32_t keep[4];
        const int n = R.ok ? kv_len - vb : 0;
#pragma unroll
        for (int e = 0; e < 4; e++) keep[e] = n >= 2 * e + 2 ? ~0u : (n == 2 * e + 1 ? 0xffffu : 0u);
#pragma unroll 1
        for (int turn = 0; turn < NJ; turn++) {
            v4u vf;
            if constexpr (!Q4) {
                vf = R.v[0];
#pragma unroll
                for (int j = 0; j + 1 < NJ; j++) R.v[j] = R.v[j + 1];
            } else {
                vf = q4_v(R.v[0][0], R.vd[0], R.vm[0]);
#pragma unroll
                for (int j = 0; j + 1 < NJ; j++) R.v[j >> 2][j & 3] = R.v[(j + 1) >> 2][(j + 1) & 3];
                if (turn == 3) {
                    R.vd[0] = R.vd[HD / 64 - 1];
                    R.vm[0] = R.vm[HD / 64 - 1];
                }
            }
            // An element that is not finite, in a position that only some of the tile's rows see, must
            // not meet the others' zero weights: such elements are taken out, and added as infinities
            // (both signs: a NaN) to the rows that see them.
            constexpr uint32_t EXP = MT == X100_T_F16 ? 0x7c00u : 0x7f80u, ONE = MT == X100_T_F16 ? 0x3c00u : 0x3f80u;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t y = vf[e] & keep[e];
                vf[e] = y;
                odd |= (y & EXP) == EXP || (y & (EXP << 16)) == EXP << 16;
            }
            if (__any(odd)) {
                v4u up = {0, 0, 0, 0}, dn = {0, 0, 0, 0}, see = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    uint32_t y = vf[e], uu = 0, dd = 0;
#pragma unroll
                    for (int b = 0; b < 32; b += 16) {
                        const uint32_t z = y >> b & 0xffffu;
                        if ((z & EXP) == EXP) {
                            const bool nan = (z & 0x7fffu) != EXP;
                            if (nan || !(z & 0x8000u)) uu |= ONE << b;
                            if (nan || (z & 0x8000u)) dd |= ONE << b;
                            y &= ~(0xffffu << b);
                        }
                    }
                    vf[e] = y;
                    up[e] = uu;
                    dn[e] = dd;
                    see[e] = (R.ok && vb + 2 * e <= pos ? ONE : 0u) | (R.ok && vb + 2 * e + 1 <= pos ? ONE << 16 : 0u);
                }
                const v4f z4 = {0, 0, 0, 0};
                const v4f nu = Mfma16<MT>::mul(up, see, z4), nd = Mfma16<MT>::mul(dn, see, z4);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    if (nu[e] > 0.0f) o[0][e] += __builtin_inff();
                    if (nd[e] > 0.0f) o[0][e] -= __builtin_inff();
                }
            }
            const v4f first = Mfma16<MT>::mul(vf, p, o[0]);
#pragma unroll
            for (int j = 0; j + 1 < NJ; j++) o[j] = o[j + 1];
            o[NJ - 1] = first;
        }
        if (t + 32 * NW < t1) {
            load_k(t + 32 * NW);
            load_v(t + 32 * NW);
        }
    }

    // the 4 lane groups hold parts of l; then the waves' m, l, O are merged
    l += xor16_f(l);
    l += xor32_f(l);
    if (g == 0) {
        s_m[w][c] = m;
        s_l[w][c] = l;
    }
    __syncthreads();   // the page list is done with
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int el = Q4 ? 4 * (4 * g + e) + (j & 3) + 64 * (j >> 2) : 16 * j + 4 * g + e;
            sh.o[w][c][el] = o[j][e];
        }
    __syncthreads();
    for (int u = threadIdx.x; u < 16 * (HD / 2); u += 64 * NW) {
        const int r = u / (HD / 2), el = u % (HD / 2) * 2;
        if (i0 + r >= n_rows) continue;
        float mm = NEG_INF;
#pragma unroll
        for (int k = 0; k < NW; k++) mm = fmaxf(mm, s_m[k][r]);
        const float ms = mm == NEG_INF ? 0.0f : mm;
        float ls = 0.0f, y0 = 0.0f, y1 = 0.0f;
#pragma unroll
        for (int k = 0; k < NW; k++) {
            // a wave without weights has no O; one whose every score is NaN has no maximum either, but a NaN as l
            const float f = __builtin_amdgcn_exp2f(s_m[k][r] - ms);
            if (s_l[k][r] == 0.0f) continue;
            ls = __builtin_fmaf(s_l[k][r], f, ls);
            y0 = __builtin_fmaf(sh.o[k][r][el], f, y0);
            y1 = __builtin_fmaf(sh.o[k][r][el + 1], f, y1);
        }
        const int tk = SP ? 0 : (i0 + r) / G, hh = kvh * G + (i0 + r) % G;
        if (ns == 1) {
            const float f = ls == 0.0f ? 0.0f : 1.0f / ls;
            const uint32_t b = ls == 0.0f ? 0u : f2act<AT>(y0 * f) | f2act<AT>(y1 * f) << 16;
            *(uint32_t *)(a.out + (size_t)(row0 + tk) * a.ldo + (size_t)hh * HD + el) = b;
        } else {
            const size_t at = (SP ? sparse_part(a, row0, kvh, r) : tile_part(a, s, kvh, i0 + r)) + sp;
            *(float2 *)(a.part_o + at * HD + el) = make_float2(y0, y1);
            if (el == 0) a.part_ml[at] = make_float2(mm, ls);
        }
    }
}

// Merges the splits of rows that have more than one: HD / 4 lanes per (row, head), 4 elements each; x = row, or
// (where only the tile kernel has splits) sequence and token, y = the heads of a block.  WIDE: the whole block takes
// one head, its lane groups every 256 / (HD / 4)-th split (64 splits: 8 turns of dependent loads become one).
// SP: rows with lists, whose splits are all there.
template <int HD, int AT, bool WIDE, bool SP> __global__ __launch_bounds__(256) void k_attn_join(const AttnArgs a)
{
    constexpr int L = HD / 4, GR = 256 / L;
    __shared__ float4 s_o[WIDE ? GR : 1][L];
    __shared__ float s_l[WIDE ? GR : 1];
    const int G = a.c.n_head / a.c.n_head_kv, gr = threadIdx.x / L, l4 = threadIdx.x % L;
    const int head = WIDE ? blockIdx.y : blockIdx.y * GR + gr;
    const bool rows = SP || a.prompt.n > 1;
    const int tokens = a.tile_rows / G;
    const int s = rows ? paged_find(a.b, blockIdx.x) : blockIdx.x / tokens;
    if (s >= a.b.n_seq) return;
    const PagedSeq q = paged_seq(a.b, s);
    const int row = rows ? blockIdx.x : q.q0 + blockIdx.x % tokens;
    if (!q.holds(row) || (!rows && q.q_len * G > a.few)) return;
    const int hd = min(head, a.c.n_head - 1), kvh = hd / G, i = (SP ? 0 : row - q.q0) * G + hd % G;
    const bool few = SP || q.q_len * G <= a.few;
    const int tr = few ? TILE_ROWS : PROMPT_ROWS, per = (few ? a.tile : a.prompt).positions(q.kv_len);
    const int vis = q.kv_len - q.q_len + min(i / tr * tr + tr - 1, q.q_len * G - 1) / G + 1;
    const int ns = SP ? a.tile.n : (vis + per - 1) / per;
    if (ns <= 1 || head >= a.c.n_head) return;   // the lanes of a head together
    const size_t at = SP ? sparse_part(a, row, kvh, i) : few ? tile_part(a, s, kvh, i) : prompt_part(a, q.q0, kvh, i);
    const float2 *ml = a.part_ml + at;
    const float4 *po = (const float4 *)(a.part_o + at * HD) + l4;
    float m = NEG_INF;
    for (int k = l4; k < ns; k += L) m = fmaxf(m, ml[k].x);
#pragma unroll
    for (int d = 1; d < L; d <<= 1) m = fmaxf(m, __shfl_xor(m, d, L));
    const float ms = m == NEG_INF ? 0.0f : m;
    float l = 0.0f;
    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int ST = WIDE ? GR : 1;
    for (int k0 = WIDE ? gr : 0; k0 < ns; k0 += 8 * ST) {   // eight at a time on their way
        float2 v[8];
        float4 b[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int k = min(k0 + u * ST, ns - 1);
            v[u] = ml[k];
            b[u] = po[(size_t)k * L];
        }
#pragma unroll
        for (int u = 0; u < 8; u++) {
            if (k0 + u * ST >= ns || v[u].y == 0.0f) continue;   // a split without weights has no O
            const float f = __builtin_amdgcn_exp2f(v[u].x - ms);
            l = __builtin_fmaf(v[u].y, f, l);
            y.x = __builtin_fmaf(b[u].x, f, y.x);
            y.y = __builtin_fmaf(b[u].y, f, y.y);
            y.z = __builtin_fmaf(b[u].z, f, y.z);
            y.w = __builtin_fmaf(b[u].w, f, y.w);
        }
    }
    if constexpr (WIDE) {
        s_o[gr][l4] = y;
        if (l4 == 0) s_l[gr] = l;
        __syncthreads();
        if (gr != 0) return;
        for (int k = 1; k < GR; k++) {
            const float4 z = s_o[k][l4];
            y.x += z.x;
            y.y += z.y;
            y.z += z.z;
            y.w += z.w;
            l += s_l[k];
        }
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    v2u o = {0, 0};
    if (l != 0.0f) o = v2u{pack2<AT>(y.x * f, y.y * f), pack2<AT>(y.z * f, y.w * f)};
    *(v2u *)(a.out + (size_t)row * a.ldo + (size_t)head * HD + 4 * l4) = o;
}

// How a call is laid out: sequences of up to `few` rows (token, head) go to the tile kernel, longer ones to the
// prompt kernel; the positions in splits, so that the blocks fill the chip.
constexpr int FEW = 32, FEW_Q4 = 64;   // us with 32 / 64: 64 sequences of 64 rows at 2048 positions, 16 bits 45 / 86,
                                       // 4 bits 62 / 60; of 40 rows 44 / 66 and 60 / 48
constexpr int WIDE_SPLITS = 8;   // more splits than this are joined by a block per head

struct Plan {
    PagedSplit tile, prompt;   // n == 0: the kernel is not launched
    size_t tile_parts, prompt_parts;   // split results
    int few, tile_rows, tiles, run;    // rows of a sequence and their tiles, tile kernel; units of a run of blocks
};

Plan plan_of(const x100_kv_cfg &c, const x100_kv_batch &b)
{
    Plan p = {};
    p.run = 8;
    const int G = c.n_head / c.n_head_kv;
    const int64_t rows = (int64_t)b.max_q * G, kv = b.max_kv;   // of the longest sequence
    // Prompts beside single tokens (the sequences but one have less than a quarter of max_q on average) take both
    // kernels: 63 tokens at 4096 positions and 512 at 4608, 290 / 165 us (each alone 91 and 57).  A batch of prompts
    // takes the prompt kernel alone, which is right for any rows: the other launch costs 2 us.
    const int few = c.kv_type == X100_KV_Q4 ? FEW_Q4 : FEW;
    const bool prompts = rows > few;
    const bool both = prompts && b.n_seq > 1 && ((int64_t)b.n_rows - b.max_q) * 4 <= (int64_t)(b.n_seq - 1) * b.max_q;
    if (!prompts || both) {
        // A block per CU where rows of 16 bits are read (256 blocks of four waves keep HBM busy: 64 sequences of
        // up to 4096 positions, us with 256 / 512 / 1024 blocks wanted: 70.6 / 78.6 / 77.2), three where 4-bit
        // codes have to be unpacked (16 of up to 60001: 115.8 / 113.9 / 101.8, 768: 98.4).  Up to 512 positions
        // one block is faster than two and their join (9.6 / 12.6 us); behind that 128 positions, a tile per wave, are
        // the least (one sequence of 1024: 10.7 us at 256, 9.8 at 128).
        const int64_t most = (int64_t)TILE_PAGES * c.page;
        p.few = few;
        p.tile_rows = (int)std::min<int64_t>(rows, few);
        p.tiles = (p.tile_rows + TILE_ROWS - 1) / TILE_ROWS;
        const int64_t base = (int64_t)(both ? 1 : p.tiles) * std::min(b.n_seq, b.n_rows) * c.n_head_kv;
        const int64_t want = kv <= 512 ? 1 : std::max<int64_t>(1, (c.kv_type == X100_KV_Q4 ? 768 : 256) / base);
        p.tile = {(int)std::max(std::min(want, (kv + 127) / 128), (kv + most - 1) / most), 128};
        // Runs of eight, one per XCD, where most sequences have their last tile: the tiles of a unit share an L2 (64
        // sequences of 32 rows at 2048 positions, 48 us; all first tiles before all second ones 80).  Else of 256, a
        // block per CU: empty tiles between others leave CUs without work (63 tokens beside a prompt, every other
        // block or eight blocks empty, 125 / 91 us).
        if (both || (int64_t)b.n_rows * G <= (int64_t)b.n_seq * TILE_ROWS * (p.tiles - 1)) p.run = 256;
        if (p.tile.n > 1) p.tile_parts = (size_t)b.n_seq * p.tile_rows * c.n_head_kv * p.tile.n;
    }
    if (prompts) {
        // One block per CU at a time, so rounds of 256 blocks: the number of splits with the least sum over the
        // rounds of a block's positions and its own start and end (as long as 512 positions), the join besides.
        const int64_t tiles = (rows + PROMPT_ROWS - 1) / PROMPT_ROWS;
        // tiles that have rows (of one sequence, the others single tokens, or of all)
        const int64_t full = both ? std::max(1, b.n_rows - b.n_seq + 1) * (int64_t)G / PROMPT_ROWS : (int64_t)b.n_rows * G / PROMPT_ROWS + b.n_seq;
        const int64_t base = std::max<int64_t>(1, std::min(tiles * b.n_seq, full)) * c.n_head_kv;
        const int64_t most = (int64_t)PROMPT_PAGES * c.page;
        int64_t best = 0;
        for (int64_t n = (kv + most - 1) / most, n0 = n; n == n0 || (n <= 16 && n * 512 < kv + 512); n++) {
            const int64_t cost = (base * n + 255) / 256 * (kv / n + 512) + (n > 1 ? 512 : 0);
            if (n == n0 || cost < best) {
                best = cost;
                p.prompt = {(int)n, 512};
            }
        }
        if (p.prompt.n > 1) p.prompt_parts = (size_t)b.n_rows * c.n_head * p.prompt.n;
    }
    return p;
}

int64_t tile_blocks(const Plan &p, const x100_kv_cfg &c, const x100_kv_batch &b)
{
    return ((int64_t)b.n_seq * c.n_head_kv * p.tile.n + p.run - 1) / p.run * p.run * p.tiles;
}

template <int HD, int AT> hipError_t attn_as(const AttnArgs &a, const Plan &p, hipStream_t s)
{
    if (p.prompt.n) {
        const hipError_t e = x100_attn_prompt_launch(a, s);
        if (e != hipSuccess) return e;
    }
    if (p.tile.n) {
        const unsigned blocks = (unsigned)tile_blocks(p, a.c, a.b);
        if (a.c.kv_type == X100_KV_Q4) k_attn_tile<HD, AT, true, false><<<blocks, 256, 0, s>>>(a);
        else k_attn_tile<HD, AT, false, false><<<blocks, 256, 0, s>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.tile.n <= 1 && p.prompt.n <= 1) return hipSuccess;
    constexpr int heads = 256 / (HD / 4);
    const unsigned rows = p.prompt.n > 1 ? a.b.n_rows : (unsigned)a.b.n_seq * (a.tile_rows / (a.c.n_head / a.c.n_head_kv));
    if (p.tile.n > WIDE_SPLITS && p.prompt.n <= 1) k_attn_join<HD, AT, true, false><<<dim3(rows, a.c.n_head), 256, 0, s>>>(a);
    else k_attn_join<HD, AT, false, false><<<dim3(rows, (a.c.n_head + heads - 1) / heads), 256, 0, s>>>(a);
    return hipGetLastError();
}

// Rows with lists: a block per row, KV head and split of the list, splits as for single tokens (their counts there).
PagedSplit sparse_split(const x100_kv_cfg &c, const x100_kv_batch &b, int n_sel)
{
    const int64_t kv = (int64_t)n_sel * c.page, base = (int64_t)b.n_rows * c.n_head_kv;
    const int64_t want = kv <= 512 ? 1 : std::max<int64_t>(1, (c.kv_type == X100_KV_Q4 ? 768 : 256) / base);
    return {(int)std::min(want, (kv + 127) / 128), 128};
}

template <int HD, int AT> hipError_t sparse_as(const AttnArgs &a, hipStream_t s)
{
    const unsigned blocks = (unsigned)((int64_t)a.b.n_rows * a.c.n_head_kv * a.tile.n);
    if (a.c.kv_type == X100_KV_Q4) k_attn_tile<HD, AT, true, true><<<blocks, 256, 0, s>>>(a);
    else k_attn_tile<HD, AT, false, true><<<blocks, 256, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.tile.n <= 1) return e;
    constexpr int heads = 256 / (HD / 4);
    if (a.tile.n > WIDE_SPLITS) k_attn_join<HD, AT, true, true><<<dim3(a.b.n_rows, a.c.n_head), 256, 0, s>>>(a);
    else k_attn_join<HD, AT, false, true><<<dim3(a.b.n_rows, (a.c.n_head + heads - 1) / heads), 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

bool x100_attn_sparse_workspace(const x100_kv_cfg &c, const x100_kv_batch &b, int n_sel, size_t *bytes)
{
    const PagedSplit p = sparse_split(c, b, n_sel);
    if ((int64_t)b.n_rows * c.n_head_kv * p.n >= 1 << 24) return false;
    *bytes = p.n > 1 ? (size_t)b.n_rows * c.n_head * p.n * (c.head_dim + 2) * sizeof(float) : 0;
    return true;
}

hipError_t x100_attn_sparse_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *q, int64_t ldq,
                                   const void *kp, const void *vp, float scale, const int *sel, int n_sel, void *out,
                                   int64_t ldo, void *ws, hipStream_t s)
{
    AttnArgs a = {};
    a.c = c;
    a.b = b;
    a.q = (const uint16_t *)q;
    a.ldq = ldq;
    a.kp = (const uint8_t *)kp;
    a.vp = (const uint8_t *)vp;
    a.scale2 = scale * 1.4426950408889634f;
    a.out = (uint16_t *)out;
    a.ldo = ldo;
    a.tile = sparse_split(c, b, n_sel);
    a.tile_rows = c.n_head / c.n_head_kv;   // the join's rows of a token
    a.part_o = (float *)ws;
    a.part_ml = (float2 *)(a.part_o + (size_t)b.n_rows * c.n_head * a.tile.n * c.head_dim);
    a.sel = sel;
    a.n_sel = n_sel;
    if (c.head_dim == 64) return c.act_type == X100_T_F16 ? sparse_as<64, X100_T_F16>(a, s) : sparse_as<64, X100_T_BF16>(a, s);
    return c.act_type == X100_T_F16 ? sparse_as<128, X100_T_F16>(a, s) : sparse_as<128, X100_T_BF16>(a, s);
}

bool x100_attn_paged_workspace(const x100_kv_cfg &c, const x100_kv_batch &b, size_t *bytes)
{
    const Plan p = plan_of(c, b);
    if (tile_blocks(p, c, b) >= 1 << 24 || x100_attn_prompt_blocks(c, b, p.prompt.n) >= 1 << 23) return false;
    *bytes = (p.tile_parts + p.prompt_parts) * (c.head_dim + 2) * sizeof(float);
    return true;
}

hipError_t x100_attn_paged_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *q, int64_t ldq,
                                  const void *kp, const void *vp, float scale, void *out, int64_t ldo, void *ws,
                                  hipStream_t s)
{
    const Plan p = plan_of(c, b);
    AttnArgs a = {};
    a.c = c;
    a.b = b;
    a.q = (const uint16_t *)q;
    a.ldq = ldq;
    a.kp = (const uint8_t *)kp;
    a.vp = (const uint8_t *)vp;
    a.scale2 = scale * 1.4426950408889634f;
    a.out = (uint16_t *)out;
    a.ldo = ldo;
    a.part_o = (float *)ws;
    a.part_ml = (float2 *)(a.part_o + (p.prompt_parts + p.tile_parts) * c.head_dim);
    a.few = p.few;
    a.tile = p.tile;
    a.prompt = p.prompt;
    a.tile_at = p.prompt_parts;
    a.tile_rows = p.tile_rows;
    a.tiles = p.tiles;
    a.run = p.run;
    if (c.head_dim == 64)
        return c.act_type == X100_T_F16 ? attn_as<64, X100_T_F16>(a, p, s) : attn_as<64, X100_T_BF16>(a, p, s);
    return c.act_type == X100_T_F16 ? attn_as<128, X100_T_F16>(a, p, s) : attn_as<128, X100_T_BF16>(a, p, s);
}
