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
#include <algorithm>

#include "paged_attn.h"
#include "x100_internal.h"

namespace {

constexpr float NEG_INF = X100_NEG_INF;
using AttnArgs = PagedAttnArgs;
constexpr int TILE_SPLIT = 8192;   // most positions of a split of the tile kernel (its page list is in LDS)

// Positions of a split of the tile kernel: a sequence's positions in n_split equal parts, so that the blocks
// of a batch of unequal sequences are as equal as its lengths let them be; 256 or more, whole turns of
// four waves.
X100_DEV int few_split(const AttnArgs &a, int kv_len)
{
    return max(256, ((kv_len + a.n_split - 1) / a.n_split + 127) & ~127);
}

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

// One block: 16 rows (token, head) of a sequence and KV head, one split of the positions; its NW waves
// take tiles of 32 positions in turn and merge at the end.
// Lane (c = lane % 16, g = lane / 16): query row c; of a tile the positions 8 g .. 8 g + 7.
// The loop is bound by memory as long as loads are always in flight: K and V of the next tile are requested
// as soon as their registers are free, the pages come from a list in LDS.
template <int HD, int AT, bool Q4, int NW> __global__ __launch_bounds__(64 * NW, Q4 || HD == 64 ? 4 : 3) void k_attn_tile(const AttnArgs a)
{
    constexpr int MT = Q4 ? X100_T_F16 : AT;   // type on the matrix cores
    constexpr int KS = HD / 32, NJ = HD / 16;  // steps of K Q^T, element tiles of V^T P^T
    __shared__ union {
        int pg[TILE_SPLIT / 16];               // pages of the split, -1 where there is none
        float o[NW][16][HD + 4];               // at the end
    } sh;
    __shared__ float s_m[NW][16], s_l[NW][16];
    const int lane = threadIdx.x & 63, w = wave_id(), c = lane & 15, g = lane >> 4;
    const int sp = blockIdx.x % a.n_split, tile = blockIdx.x / a.n_split, kvh = blockIdx.y, s = blockIdx.z;
    const int n_kv = a.c.n_head_kv, G = a.c.n_head / n_kv, page = a.c.page, psh = __builtin_ctz(page);
    const int i0 = tile * 16;
    // A short table's pages are read here, beside the lengths; a long one's when the split is known.
    const int *tab = a.b.block_table + (size_t)s * a.b.table_ld;
    const int n_all = (a.b.max_kv + page - 1) >> psh;
    const bool all = n_all <= TILE_SPLIT / 16;
    auto list = [&](int first, int n) {
        for (int i = threadIdx.x; i < n; i += 64 * NW) {
            const int pg = tab[first + i];
            sh.pg[i] = pg >= 0 && pg < a.c.n_pages ? pg : -1;
        }
    };
    if (all) list(0, n_all);
    const PagedSeq q = paged_seq(a.b, s);
    const int n_rows = q.q_len * G;
    if (i0 >= n_rows || n_rows > a.few) return;
    const int pos0 = q.kv_len - q.q_len;                       // position of token 0
    const int vis = pos0 + (min(i0 + 15, n_rows - 1)) / G + 1;  // positions that the tile's last row sees
    const int per = few_split(a, q.kv_len);
    const int ns = max(1, (vis + per - 1) / per);
    if (sp >= ns) return;
    const int t0 = sp * per, t1 = min(t0 + per, vis);
    const int pg0 = all ? 0 : t0 >> psh;                       // first page of the list
    const int n_pg = t1 > t0 ? ((t1 - 1) >> psh) - (t0 >> psh) + 1 : 0;
    if (!all) list(pg0, n_pg);

    const int i = min(i0 + c, n_rows - 1), tok = i / G, head = kvh * G + i % G;
    const int pos = pos0 + tok;
    const int pos_lo = pos0 + i0 / G;                          // the tile's first row's
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
        const uint16_t *qr = a.q + (size_t)(q.q0 + tok) * a.ldq + (size_t)head * HD;
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
    // The weights p.  The maximum may stay up to 8 (a factor of 256) behind: every sum is relative to it.
    v4u p;
    auto weights = [&]() __attribute__((always_inline)) {
        float mx = fmaxf(sc[0][0], sc[1][0]);
#pragma unroll
        for (int e = 1; e < 4; e++) mx = fmaxf(fmaxf(mx, sc[0][e]), sc[1][e]);
        mx *= sc2;
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
        const int n = R.ok ? q.kv_len - vb : 0;
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
            const float f = __builtin_amdgcn_exp2f(s_m[k][r] - ms);
            if (s_m[k][r] == NEG_INF) continue;
            ls = __builtin_fmaf(s_l[k][r], f, ls);
            y0 = __builtin_fmaf(sh.o[k][r][el], f, y0);
            y1 = __builtin_fmaf(sh.o[k][r][el + 1], f, y1);
        }
        const int tk = (i0 + r) / G, hh = kvh * G + (i0 + r) % G;
        if (ns == 1) {
            const float f = ls == 0.0f ? 0.0f : 1.0f / ls;
            const uint32_t b = ls == 0.0f ? 0u : f2act<AT>(y0 * f) | f2act<AT>(y1 * f) << 16;
            *(uint32_t *)(a.out + (size_t)(q.q0 + tk) * a.ldo + (size_t)hh * HD + el) = b;
        } else {
            const size_t at = part_few(a, s, kvh, i0 + r) + sp;
            *(float2 *)(a.o_few + at * HD + el) = make_float2(y0, y1);
            if (el == 0) a.ml_few[at] = make_float2(mm, ls);
        }
    }
}

// Merges the splits of rows that have more than one: a wave per row (token, head), HD / 64 elements per
// lane.  FEW: the tile kernel's rows, blockIdx.x = sequence, y = KV head and four rows; else the prompt
// kernel's, x = token row, y = four heads.
template <int HD, int AT, bool FEW> __global__ __launch_bounds__(256) void k_attn_join(const AttnArgs a)
{
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63, w = wave_id(), G = a.c.n_head / a.c.n_head_kv;
    int s, i, kvh;
    PagedSeq q;
    if constexpr (FEW) {
        const int per = (a.few_rows + 3) / 4;
        s = blockIdx.x;
        kvh = blockIdx.y / per;
        i = blockIdx.y % per * 4 + w;
        q = paged_seq(a.b, s);
        if (i >= q.q_len * G || q.q_len * G > a.few) return;
    } else {
        const int row = blockIdx.x, head = blockIdx.y * 4 + w;
        if (head >= a.c.n_head) return;
        s = paged_find(a.b, row);
        if (s >= a.b.n_seq) return;
        q = paged_seq(a.b, s);
        if (q.q_len * G <= a.few || row < q.q0) return;
        kvh = head / G;
        i = (row - q.q0) * G + head % G;
    }
    const int tr = FEW ? 16 : PROMPT_ROWS, split = FEW ? few_split(a, q.kv_len) : a.split_p;
    const int vis = q.kv_len - q.q_len + min(i / tr * tr + tr - 1, q.q_len * G - 1) / G + 1;
    const int ns = (vis + split - 1) / split;
    if (ns <= 1) return;
    const size_t at = FEW ? part_few(a, s, kvh, i) : part_prompt(a, q.q0, kvh, i);
    const float2 *ml = (FEW ? a.ml_few : a.ml_p) + at;
    const float *po = (FEW ? a.o_few : a.o_p) + at * HD + lane * E;
    // (m, l) by lane, up to 64 splits at a time; the splits' O eight at a time
    float m = NEG_INF;
    for (int k = lane; k < ns; k += 64) m = fmaxf(m, ml[k].x);
    m = wave_max_u(m);
    const float ms = m == NEG_INF ? 0.0f : m;
    float l = 0.0f, y[E] = {};
    for (int k0 = 0; k0 < ns; k0 += 64) {
        const float2 v = k0 + lane < ns ? ml[k0 + lane] : make_float2(NEG_INF, 0.0f);
        const float fl = __builtin_amdgcn_exp2f(v.x - ms);   // 0 where a split has no position
        l += wave_sum_uf(v.x == NEG_INF ? 0.0f : v.y * fl);
        const int n = min(64, ns - k0);
        for (int k = 0; k < n; k += 8) {
            float b[8][E];
#pragma unroll
            for (int u = 0; u < 8; u++)
#pragma unroll
                for (int e = 0; e < E; e++) b[u][e] = po[(size_t)(k0 + min(k + u, n - 1)) * HD + e];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(fl), k + u));
                if (k + u < n && f != 0.0f)   // a split without positions has no O
#pragma unroll
                    for (int e = 0; e < E; e++) y[e] = __builtin_fmaf(b[u][e], f, y[e]);
            }
        }
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    uint16_t *o = a.out + (size_t)(q.q0 + i / G) * a.ldo + (size_t)(kvh * G + i % G) * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = l == 0.0f ? 0 : (uint16_t)f2act<AT>(y[e] * f);
}

// How a call is laid out.  Sequences of up to `few` rows (token, head) go to the tile kernel, longer ones
// to the prompt kernel; positions are split so that the blocks fill the chip.
struct Plan {
    int few, few_rows, tiles, split, n_split;   // tile kernel
    int tiles_p, split_p, n_split_p;            // prompt kernel (tiles_p 0: not launched)
    // split results that the kernels keep
    size_t results_few(const x100_kv_cfg &c, const x100_kv_batch &b) const
    {
        return n_split == 1 ? 0 : (size_t)b.n_seq * c.n_head_kv * few_rows * n_split;
    }
    size_t results_prompt(const x100_kv_cfg &c, const x100_kv_batch &b) const
    {
        return n_split_p == 1 ? 0 : (size_t)b.n_rows * c.n_head * n_split_p;
    }
};

// Splits of max_kv positions for `want` of them, each of `least` positions or more and a multiple of 128.
void split_of(int64_t max_kv, int64_t want, int64_t least, int64_t most, int &split, int &n_split)
{
    int64_t s = (max_kv + want - 1) / want;
    s = std::min(most, std::max(least, (s + 127) / 128 * 128));
    s = std::min<int64_t>(s, (max_kv + 127) / 128 * 128);
    split = (int)s;
    n_split = (int)((max_kv + s - 1) / s);
}

Plan plan_of(const x100_kv_cfg &c, const x100_kv_batch &b)
{
    Plan p = {};
    const int G = c.n_head / c.n_head_kv;
    const int64_t rows = (int64_t)b.max_q * G;   // of the longest sequence
    p.few = 32;
    p.split = p.split_p = 128;
    p.n_split = p.n_split_p = 1;
    p.few_rows = (int)std::min<int64_t>(rows, p.few);
    p.tiles = (p.few_rows + 15) / 16;
    const int64_t base = (int64_t)p.tiles * std::min(b.n_seq, b.n_rows) * c.n_head_kv;
    // A block per CU where rows of 16 bits are read (256 blocks of four waves keep HBM busy: 64 sequences of up
    // to 4096 positions, us with 256 / 512 / 1024 blocks wanted: 70.6 / 78.6 / 77.2), three where 4-bit codes have
    // to be unpacked (16 of up to 60001: 115.8 / 113.9 / 101.8, 768: 98.4).  Up to 512 positions one block is
    // faster than two and their join (9.6 / 12.6 us).
    const int64_t blocks = c.kv_type == X100_KV_Q4 ? 768 : 256;
    split_of(b.max_kv, b.max_kv <= 512 ? 1 : std::max<int64_t>(1, blocks / base), 256, TILE_SPLIT, p.split, p.n_split);
    if (rows > p.few) {
        p.tiles_p = (int)((rows + PROMPT_ROWS - 1) / PROMPT_ROWS);
        // tiles that have rows: no more than one per sequence besides the full ones
        const int64_t full = (int64_t)b.n_rows * G / PROMPT_ROWS + 1;
        const int64_t base_p = std::min<int64_t>((int64_t)p.tiles_p * b.n_seq, full + b.n_seq) * c.n_head_kv;
        split_of(b.max_kv, std::max<int64_t>(1, 512 / base_p), 512, PROMPT_SPLIT, p.split_p, p.n_split_p);
    }
    return p;
}

template <int HD, int AT> hipError_t attn_as(const AttnArgs &a, const Plan &p, hipStream_t s)
{
    if (p.tiles) {
        const dim3 grid((unsigned)(p.tiles * p.n_split), a.c.n_head_kv, a.b.n_seq);
        if (a.c.kv_type == X100_KV_Q4) k_attn_tile<HD, AT, true, 4><<<grid, 256, 0, s>>>(a);
        else k_attn_tile<HD, AT, false, 4><<<grid, 256, 0, s>>>(a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (p.n_split > 1) {
            k_attn_join<HD, AT, true><<<dim3(a.b.n_seq, a.c.n_head_kv * ((a.few_rows + 3) / 4)), 256, 0, s>>>(a);
            const hipError_t e2 = hipGetLastError();
            if (e2 != hipSuccess) return e2;
        }
    }
    if (p.tiles_p) {
        const hipError_t e = x100_attn_prompt_launch(a, p.tiles_p, s);
        if (e != hipSuccess) return e;
        if (p.n_split_p > 1) k_attn_join<HD, AT, false><<<dim3(a.b.n_rows, (a.c.n_head + 3) / 4), 256, 0, s>>>(a);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace

size_t x100_attn_paged_workspace(const x100_kv_cfg &c, const x100_kv_batch &b)
{
    const Plan p = plan_of(c, b);
    return (p.results_few(c, b) + p.results_prompt(c, b)) * (c.head_dim + 2) * sizeof(float);
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
    const size_t n_few = p.results_few(c, b), n_p = p.results_prompt(c, b);
    a.o_few = (float *)ws;
    a.o_p = a.o_few + n_few * c.head_dim;
    a.ml_few = (float2 *)(a.o_p + n_p * c.head_dim);
    a.ml_p = a.ml_few + n_few;
    a.split = p.split;
    a.n_split = p.n_split;
    a.few = p.few;
    a.few_rows = p.few_rows;
    a.split_p = p.split_p;
    a.n_split_p = p.n_split_p;
    if (c.head_dim == 64)
        return c.act_type == X100_T_F16 ? attn_as<64, X100_T_F16>(a, p, s) : attn_as<64, X100_T_BF16>(a, p, s);
    return c.act_type == X100_T_F16 ? attn_as<128, X100_T_F16>(a, p, s) : attn_as<128, X100_T_BF16>(a, p, s);
}
