// Attention over the paged KV cache for many rows (x100_paged.h): prompts and pieces of prompts.
//
// One block: 256 rows (token, head) of a sequence and KV head, eight waves of 32 rows (two per SIMD), and
// one split of the positions in tiles of 32.  As in attn_paged.hip the scores come transposed, S^T = K Q^T
// (v_mfma 32x32x16), and go as the operand P^T into O^T += V^T P^T in the registers they were made in.
//
// A step holds three tiles that do not depend on each other: the products of tile i - 1, the weights of
// tile i, the scores of tile i + 1.  Behind each matrix instruction stand a few vector instructions of the
// weights and the read of an operand for four instructions later, so that the matrix cores, the vector
// unit and LDS all work all the time; two waves, because one alone issues an instruction only every
// 2.4 ns.  K and V come 64 positions at a time by asynchronous copies from the cache into LDS (4-bit
// pages: through registers, where they become fp16), read by all waves, with one barrier for two tiles.
//
// The running maximum m is taken from the first tile and then only followed where a weight would leave
// its 16 bits: the weights' sum, which is needed anyway, says so, and the tile's weights are made again.
//
// 4 x 4000 rows of 32 heads on 4 of 128, bf16: 485 us, 1080 TFLOP/s counted over the visible half (an 8192^3 product
// of the library: 1216); in a step of 32 positions the matrix instructions take 512 cycles of a wave, the weights'
// vector instructions 380.  Heads of 64 have half the former for the same weights and are bound by the latter: 4096
// rows of 32 heads 750 TFLOP/s; twelve waves of 168 registers instead of eight 450.  4 bits: unpacking once per
// block costs 14% more (2 x 4096 rows 248 / 283 us).
#include "paged_attn.h"
#include "x100_internal.h"

namespace {

constexpr float NEG_INF = X100_NEG_INF;

// sum over the wave's lanes up to this one
X100_DEV int prefix_sum(int v)
{
    v += dpp_i<0x111>(0, v);
    v += dpp_i<0x112>(0, v);
    v += dpp_i<0x114>(0, v);
    v += dpp_i<0x118>(0, v);
    v += dpp_i<0x142, 0xa>(0, v);
    v += dpp_i<0x143, 0xc>(0, v);
    return v;
}

// LDS of every wave written and read up to here
X100_DEV void lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int HD, int AT, bool Q4> __global__ __launch_bounds__(512, 2) void k_attn_prompt(const PagedAttnArgs a)
{
    constexpr int MT = Q4 ? X100_T_F16 : AT;
    constexpr int NT = 512;
    constexpr int KS = HD / 16, NJ = HD / 32;
    constexpr int KB = 32 * HD * 2;       // bytes of a K (or V) tile of 32 positions
    constexpr int ND = 2 * KB / 8192;     // copies of 1 KiB per wave and pair of tiles
    __shared__ __attribute__((aligned(1024))) uint8_t s_k[3][2 * KB], s_v[3][2 * KB];   // pairs of tiles
    __shared__ int s_pg[PROMPT_PAGES];
    __shared__ int s_inf[2][HD], s_odd;
    const int lane = threadIdx.x & 63, w = wave_id(), c = lane & 31, h = lane >> 5;
    const int n_kv = a.c.n_head_kv, G = a.c.n_head / n_kv, page = a.c.page, psh = __builtin_ctz(page);
    const int ns_max = a.prompt.n, kvh = blockIdx.x % n_kv, u = blockIdx.x / n_kv, sp = u % ns_max;
    // Item u / ns_max of the sequences' tiles of rows, counted by each wave, 64 sequences at a time.  (A grid of the
    // longest sequence's tiles for every sequence: 64 of 16 rows under a bound of 4096, 200 / 24 us; blocks without work
    // among the others leave a shader engine a block more than it has CUs for: 16 of 32 rows, 80 / 56 us.)
    const int item = u / ns_max, n_seq = a.b.n_seq;
    auto first = [&](int s) { return (int64_t)a.b.q_start[s] * G / PROMPT_ROWS + s; };
    int s = 0, place = item;
    if (n_seq > 512) {
        // more sequences: s has the items from q_start[s] G / 256 + s on, which leaves room for its tiles whatever the
        // rows before it
        s = paged_search(n_seq, [&](int s) { return first(s) <= item; });
        if (s >= n_seq) return;
        place = (int)max(min(item - first(s), (int64_t)INT_MAX), (int64_t)-1);
    } else if (n_seq > 1) {
        for (int before = 0; s < n_seq; s += 64) {
            int mine = 0;
            if (s + lane < n_seq) {
                const int rows = paged_seq(a.b, s + lane).q_len * G;
                if (rows > a.few) mine = (rows + PROMPT_ROWS - 1) / PROMPT_ROWS;
            }
            const int incl = before + prefix_sum(mine);   // tiles up to this lane's sequence
            const uint64_t over = __ballot(incl > item);
            if (over) {
                const int k = __builtin_ctzll(over);
                place = item - __builtin_amdgcn_readlane(incl - mine, k);
                s += k;
                break;
            }
            before = __builtin_amdgcn_readlane(incl, 63);
        }
        if (s >= n_seq) return;
    }
    const PagedSeq q = paged_seq(a.b, s);
    const int n_rows = q.q_len * G, tiles = (n_rows + PROMPT_ROWS - 1) / PROMPT_ROWS;
    if (n_rows <= a.few || place < 0 || place >= tiles) return;
    const int i0 = (tiles - 1 - place) * PROMPT_ROWS, pos0 = q.kv_len - q.q_len;   // the longest first
    const int vis = pos0 + min(i0 + PROMPT_ROWS - 1, n_rows - 1) / G + 1;
    const int per = a.prompt.positions(q.kv_len), ns = max(1, (vis + per - 1) / per);
    if (sp >= ns) return;
    const int t0 = sp * per, t1 = min(t0 + per, vis);
    const int n = max(0, (t1 - t0 + 31) >> 5);   // tiles

    const int iw = i0 + 32 * w;
    // query row iw + c
    int pos;
    float sc2 = a.scale2;
    v4u qf[KS];
    {
        const int i = min(iw + c, n_rows - 1), tok = i / G, head = kvh * G + i % G;
        pos = pos0 + tok;
        const uint16_t *qr = a.q + (size_t)(q.q0 + tok) * a.ldq + (size_t)head * HD + 8 * h;
#pragma unroll
        for (int j = 0; j < KS; j++) qf[j] = *(const v4u *)(qr + 16 * j);
        if constexpr (Q4 && AT == X100_T_BF16) {
            float mx = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    mx = fmaxf(mx, fmaxf(fabsf(bf2f(qf[j][e] & 0xffffu)), fabsf(__uint_as_float(qf[j][e] & 0xffff0000u))));
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

    // pages of the split; one that is none sends every tile through the masked step
    const int *tab = a.b.block_table + (size_t)s * a.b.table_ld + (t0 >> psh);
    const int pg0 = t0 >> psh, n_pg = n > 0 ? ((t1 - 1) >> psh) - pg0 + 1 : 0;
    bool bad = false;
    for (int i = threadIdx.x; i < n_pg; i += NT) {
        const int g = tab[i];
        const bool ok = g >= 0 && g < a.c.n_pages;
        s_pg[i] = ok ? g : -1;
        bad |= !ok;
    }
    bad = __syncthreads_or(bad);
    // Tiles that every row of the block sees whole; that the wave's rows see whole; that they see at all.
    const int nw = bad ? 0 : max(0, min(n, (pos0 + i0 / G + 1 - t0) >> 5));
    const int ww = bad ? 0 : max(0, min(n, (pos0 + min(iw, n_rows - 1) / G + 1 - t0) >> 5));
    const int wn = iw >= n_rows ? 0 : max(0, min(n, (pos0 + min(iw + 31, n_rows - 1) / G + 1 - t0 + 31) >> 5));

    // ---- pairs of tiles into LDS -------------------------------------------------------------------
    // K: [64 positions][HD], the 16-byte pieces of a row exchanged by an XOR with the position, so that
    // 16 lanes that read one piece of 16 positions meet different banks.  V: [8][HD][8] as in the cache.
    // Wave w copies positions 8 w .. 8 w + 7, which lie on one page; their bytes begin at the same place of the
    // K and of the V pool.
    constexpr int RC = HD / 8;   // pieces of a row
    auto swz = [](int tok) { return HD == 128 ? tok & 15 : (tok >> 1) & 7; };
    const size_t head_bytes = page_head_bytes<HD, Q4>(page);
    const int np = (n + 1) >> 1;   // pairs
    auto page_at = [&](int pp) {   // entry of the page list for the wave's positions of pair pp
        const int t = t0 + 64 * pp + 8 * w;
        return s_pg[((t < t1 ? t : t0) >> psh) - pg0];
    };
    auto bytes_at = [&](int pp, int pg) -> size_t {
        const int t = t0 + 64 * pp + 8 * w;
        return (size_t)(max(__builtin_amdgcn_readfirstlane(pg), 0) * n_kv + kvh) * head_bytes + (t & (page - 1)) * (HD * 2);
    };
    uint32_t kvoff[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) {
        const int tok = (1024 * d) / (HD * 2) + lane / RC;
        kvoff[d] = (uint32_t)tok * (HD * 2) + (uint32_t)((lane % RC) ^ swz(8 * w + tok)) * 16;
    }
    const uint32_t lk = lds_addr(s_k) + w * (KB / 4), lv = lds_addr(s_v) + w * (KB / 4);
    auto load_k = [&](size_t at, int slot, int d) __attribute__((always_inline)) {
        dma16s(kvoff[d], a.kp + at, lk + slot * (2 * KB) + d * 1024);
    };
    auto load_v = [&](size_t at, int slot, int d) __attribute__((always_inline)) {
        dma16s(16u * lane + 1024u * d, a.vp + at, lv + slot * (2 * KB) + d * 1024);
    };
    // 4 bits: a thread takes HD / 8 elements of a K position, and HD / 64 elements of a V block of 8 positions.
    constexpr int W4 = HD / 64;
    uint32_t rk_w[W4], rk_s, rv_w[W4];
    v4u rv_d, rv_m;
    const int x4 = threadIdx.x;
    auto base4 = [&](const uint8_t *pool, int pp, int &off) {
        const int pg = max(s_pg[((pp < t1 ? pp : t0) >> psh) - pg0], 0);
        off = pp & (page - 1);
        return pool + ((size_t)pg * n_kv + kvh) * head_bytes;
    };
    auto words4 = [&](const uint32_t *p, uint32_t (&r)[W4]) __attribute__((always_inline)) {
        if constexpr (W4 == 2) {
            const v2u v = *(const v2u *)p;
            r[0] = v[0];
            r[1] = v[1];
        } else {
            r[0] = p[0];
        }
    };
    auto load4 = [&](int pk, int pv) __attribute__((always_inline)) {   // K of pair pk, V of pair pv
        int off;
        const uint8_t *kb = base4(a.kp, t0 + 64 * min(pk, np - 1) + (x4 >> 3), off);
        words4((const uint32_t *)kb + off * (HD / 8) + (x4 & 7) * W4, rk_w);
        rk_s = ((const uint32_t *)(kb + page * HD / 2))[off * (HD / 32) + (x4 & 7) * HD / 256];
        const uint8_t *vb = base4(a.vp, t0 + 64 * min(pv, np - 1) + 8 * (x4 >> 6), off);
        words4((const uint32_t *)vb + (off >> 3) * HD + (x4 & 63) * W4, rv_w);
        const v4u *vs = (const v4u *)(vb + page * HD / 2 + ((off >> 3) * (HD / 32) + (x4 & 63) * W4 / 32) * 32);
        rv_d = vs[0];
        rv_m = vs[1];
    };
    auto store_k4 = [&](int slot, int k) __attribute__((always_inline)) {   // what load4 fetched, as fp16
        const uint32_t d = (rk_s & 0xffffu) * 0x10001u, m = (rk_s >> 16) * 0x10001u;
        *(v4u *)(s_k[slot] + (x4 >> 3) * (HD * 2) + (((x4 & 7) * W4 + k) ^ swz(x4 >> 3)) * 16) =
            q4_v(rk_w[k], v4u{d, d, d, d}, v4u{m, m, m, m});
    };
    auto store_v4 = [&](int slot, int k) __attribute__((always_inline)) {
        *(v4u *)(s_v[slot] + (x4 * W4 + k) * 16) = q4_v(rv_w[k], rv_d, rv_m);
    };

    // ---- products --------------------------------------------------------------------------------
    // K operand: row r of the tile's 32 is position 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4, so
    // that lane (c, h) receives positions 16 s + 8 h + 0 .. 7 of row c in registers 8 s .. 8 s + 7.
    const int ktok = 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3);
    uint32_t kad[KS];
#pragma unroll
    for (int j = 0; j < KS; j++) kad[j] = ktok * (HD * 2) + (((2 * j + h) ^ swz(ktok)) * 16);
    const uint32_t vad = h * (HD * 16) + c * 16;

    v16f S, T, O[NJ];
    v4u P[2];      // weights of tile i - 1
    v4u f[4];      // operands of the next four matrix instructions
    float m = NEG_INF, msub = 0.0f, l = 0.0f, lt = 0.0f;
#pragma unroll
    for (int j = 0; j < NJ; j++) O[j] = v16f{};
    P[0] = P[1] = v4u{0, 0, 0, 0};
    // Matrix instruction g of a step: products (V of tile i - 1) for g < 2 NJ, then scores (K of tile i + 1).
    constexpr int NM = 2 * NJ + KS, PER = 16 / NM;
    auto operand = [&](int g, const uint8_t *v, const uint8_t *k) __attribute__((always_inline)) {
        return *(const v4u *)(g < 2 * NJ ? v + vad + (g / NJ) * (2 * HD * 16) + (g % NJ) * 512 : k + kad[(g - 2 * NJ) % KS]);
    };
    auto maximum = [&](const v16f &X) __attribute__((always_inline)) {
        float y = fmaxf(X[0], X[1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2) y = fmaxf(fmaxf(y, X[e]), X[e + 1]);
        // The lift makes the instruction 4 bytes longer; 4 more leave the step behind, 8 bytes per instruction, where
        // it was (3 x 509 rows behind 16384 in 4 bits, heads of 64: 206 us without this, 198 with it or without lift).
        if constexpr (prompt_lift<MT>() != 0.0f) asm volatile("s_nop 0");
        return __builtin_fmaf(y, sc2, -prompt_lift<MT>());
    };
    // m rises to the tile's maximum (less the lift), O and l go to the new unit (no weights in flight)
    auto rescale = [&](const v16f &X) __attribute__((always_inline)) {
        const float mx = maximum(X), y = fmaxf(mx, xor32_f(mx));
        const float mn = y > m ? y : m;
        const float r = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        msub = mn == NEG_INF ? 0.0f : mn;
        l *= r;
#pragma unroll
        for (int j = 0; j < NJ; j++) O[j] *= r;
    };
    // After a step: its weights are good as long as their sum is below prompt_most, so that fp16 holds each (an
    // infinity among them shows in the sum) and sums over bf16 V up to 2^100 stay finite (a row that has no maximum
    // yet: not good).  Else m follows.
    auto settle = [&](const v16f &X) __attribute__((always_inline)) {
        if (__any(!(lt < prompt_most<MT>()) || m == NEG_INF)) {
            rescale(X);
            lt = 0.0f;
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(X[8 * k + 2 * e], sc2, -msub));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(X[8 * k + 2 * e + 1], sc2, -msub));
                    P[k][e] = pack2<MT>(p0, p1);
                    lt = add2<MT>(P[k][e], lt);
                }
        }
        l += lt;
    };
    // Scores Y of tile i + 1 (K at k), products of tile i - 1 (V at v), weights of tile i from X; the last four
    // operands read are the first of the next step's (V at vn).  copy(g) is run behind instruction g.
    auto mix = [&](const v16f &X, v16f &Y, const uint8_t *v, const uint8_t *k, const uint8_t *vn, auto &&copy) __attribute__((always_inline)) {
        float x[16], y = 0.0f;
        uint32_t p[8];
        // Each result is pinned where it is made: the compiler would move it behind all matrix instructions.
        auto fma1 = [&](int e) __attribute__((always_inline)) {
            if (e >= 16) return;
            x[e] = __builtin_fmaf(X[e], sc2, -msub);
            asm volatile("" : "+v"(x[e]));
        };
        auto exp1 = [&](int e) __attribute__((always_inline)) {
            if (e >= 16) return;
            x[e] = __builtin_amdgcn_exp2f(x[e]);
            asm volatile("" : "+v"(x[e]));
        };
#pragma unroll
        for (int e = 0; e <= PER; e++) fma1(e);
#pragma unroll
        for (int e = 0; e < PER; e++) exp1(e);
        v16f sn = v16f{};
#pragma unroll
        for (int g = 0; g < NM; g++) {
            __builtin_amdgcn_sched_barrier(0);
            if (g < 2 * NJ) O[g % NJ] = mfma32<MT>(f[g & 3], P[g / NJ], O[g % NJ]);
            else sn = mfma32<MT>(f[g & 3], qf[g - 2 * NJ], sn);
            f[g & 3] = g + 4 < NM ? operand(g + 4, v, k) : operand(g + 4 - NM, vn, k);
#pragma unroll
            for (int u = 0; u < PER; u++) {
                const int e = PER * g + u;   // scores up to e are through exp2 (of the slot before)
                if (e & 1) {
                    p[e >> 1] = pack2<MT>(x[e - 1], x[e]);
                    asm volatile("" : "+v"(p[e >> 1]));
                } else if (e) {
                    y = add2<MT>(p[(e >> 1) - 1], y);
                    asm volatile("" : "+v"(y));
                }
                fma1(e + PER + 1);
                exp1(e + PER);
            }
            copy(g);
        }
        y = add2<MT>(p[7], y);
        __builtin_amdgcn_sched_barrier(0);
        Y = sn;
        lt = y;
        P[0] = v4u{p[0], p[1], p[2], p[3]};
        P[1] = v4u{p[4], p[5], p[6], p[7]};
    };
    // Validity of the tile's two groups of 16 positions (their pages).
    auto ok16 = [&](int i, int k) {
        const int t = t0 + 32 * i + 16 * k;
        return t < t1 && s_pg[(t >> psh) - pg0] >= 0;
    };
    auto mask = [&](int i, v16f &X) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const bool ok = ok16(i, k);
            const int p = t0 + 32 * i + 16 * k + 8 * h;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (!(ok && p + e <= pos)) X[8 * k + e] = NEG_INF;
        }
    };
    // V of a tile that not every row sees whole, before its products: the positions that no row has as
    // zeros, and elements that are not finite taken out, because 0 times such an element would reach the
    // rows that do not see it.  Rows see a prefix of the positions, so the first place of each element
    // where it is +inf, and where it is -inf (a NaN: both), says at the end which rows take it.
    auto clean = [&](int i, uint8_t *vt) __attribute__((always_inline)) {
        constexpr uint32_t EXP = MT == X100_T_F16 ? 0x7c00u : 0x7f80u;
        for (int x = threadIdx.x; x < KB / 16; x += NT) {
            const int blk = x / HD, el = x % HD, p = t0 + 32 * i + 8 * blk;
            const int left = ok16(i, blk >> 1) ? q.kv_len - p : 0;
            uint16_t *v = (uint16_t *)(vt + x * 16);
            for (int e = 0; e < 8; e++) {
                const uint32_t y = v[e];
                if (e < left && (y & EXP) != EXP) continue;
                v[e] = 0;
                if (e >= left) continue;
                const bool nan = (y & 0x7fffu) != EXP;
                if (nan || !(y & 0x8000u)) atomicMin(&s_inf[0][el], p + e);
                if (nan || (y & 0x8000u)) atomicMin(&s_inf[1][el], p + e);
                s_odd = 1;
            }
        }
        lds_sync();
    };

    // Step i: see the head of this file.  vt: V of tile i, v: of tile i - 1, k: K of tile i + 1.
    auto step = [&](int i, v16f &X, v16f &Y, uint8_t *vt, const uint8_t *v, const uint8_t *k, auto &&copy) __attribute__((always_inline)) {
        if (i >= nw) clean(i, vt);
        if (i >= ww) mask(i, X);
        mix(X, Y, v, k, vt, copy);
        settle(X);
    };

    if (n > 0) {
        size_t at = 0;   // where the wave's positions of the next V pair are
        int pg = 0;      // page of the next K pair
        if constexpr (!Q4) {
            const size_t a0 = bytes_at(0, page_at(0));
            at = bytes_at(min(1, np - 1), page_at(min(1, np - 1)));
#pragma unroll
            for (int d = 0; d < ND; d++) {
                load_k(a0, 0, d);
                load_v(a0, 0, d);
                load_k(at, 1, d);
            }
            pg = page_at(min(2, np - 1));
        } else {
            load4(0, 0);
#pragma unroll
            for (int k = 0; k < W4; k++) {
                store_k4(0, k);
                store_v4(0, k);
            }
            load4(1, 1);
#pragma unroll
            for (int k = 0; k < W4; k++) store_k4(1, k);
            load4(2, 1);
        }
        // step 0 multiplies the tile before the first (second of V pair 2's place) by zero weights
        for (int x = threadIdx.x; x < KB / 16; x += NT) *(v4u *)(s_v[2] + KB + x * 16) = v4u{0, 0, 0, 0};
        for (int x = threadIdx.x; x < 2 * HD; x += NT) s_inf[x / HD][x % HD] = INT_MAX;
        if (threadIdx.x == 0) s_odd = 0;
        if constexpr (!Q4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_sync();
        S = v16f{};
#pragma unroll
        for (int j = 0; j < KS; j++) S = mfma32<MT>(*(const v4u *)(s_k[0] + kad[j]), qf[j], S);
#pragma unroll
        for (int g = 0; g < 4; g++) f[g] = v4u{0, 0, 0, 0};
        if (ww == 0) mask(0, S);
        rescale(S);
        // Pair pp: K of pairs pp and pp + 1 and V of pairs pp - 1 and pp are in LDS for every wave, the places of K
        // pair pp - 1 and V pair pp - 2 free.
        const int npw = (wn + 1) >> 1;   // pairs with tiles that the wave's rows see
        int r = 0, pp = 0;               // r = pp % 3: the place of pair pp
        for (; pp < npw; pp++) {
            const int r1 = r == 2 ? 0 : r + 1, r2 = r1 == 2 ? 0 : r1 + 1;
            // The copies go out one by one behind matrix instructions of the pair's first tile: all at once they
            // would hold the waves up.
            uint8_t *v0 = s_v[r];
            const uint8_t *k1 = s_k[r] + KB;
            if constexpr (!Q4) {
                asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                const size_t av = at;
                at = bytes_at(min(pp + 2, np - 1), pg);
                step(2 * pp, S, T, v0, s_v[r2] + KB, k1, [&](int g) {
                    if (g % 2 == 1 && g / 2 < ND) load_v(av, r1, g / 2);
                    if (g % 2 == 1 && g / 2 >= ND && g / 2 < 2 * ND) load_k(at, r2, g / 2 - ND);
                });
                pg = page_at(min(pp + 3, np - 1));
            } else {
                lds_sync();
                step(2 * pp, S, T, v0, s_v[r2] + KB, k1, [&](int g) {
                    if (g % 2 == 1 && g / 2 < W4) store_v4(r1, g / 2);
                    if (g % 2 == 1 && g / 2 >= W4 && g / 2 < 2 * W4) store_k4(r2, g / 2 - W4);
                });
                load4(pp + 3, pp + 2);
            }
            // tile 2 pp + 1: behind the last tile all of it is masked
            step(2 * pp + 1, T, S, v0 + KB, v0, s_k[r1], [](int) {});
            r = r1;
        }
        // the products of the wave's last tile
        if (npw > 0) {
            const uint8_t *v = s_v[r == 0 ? 2 : r - 1] + KB;
#pragma unroll
            for (int g = 0; g < 2 * NJ; g++) O[g % NJ] = mfma32<MT>(operand(g, v, v), P[g / NJ], O[g % NJ]);
        }
        // pairs that only other waves' rows see
        for (; pp < np; pp++) {
            const int r1 = r == 2 ? 0 : r + 1, r2 = r1 == 2 ? 0 : r1 + 1;
            if constexpr (!Q4) {
                asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
#pragma unroll
                for (int d = 0; d < ND; d++) load_v(at, r1, d);
                at = bytes_at(min(pp + 2, np - 1), pg);
#pragma unroll
                for (int d = 0; d < ND; d++) load_k(at, r2, d);
                pg = page_at(min(pp + 3, np - 1));
            } else {
                lds_sync();
#pragma unroll
                for (int k = 0; k < W4; k++) {
                    store_v4(r1, k);
                    store_k4(r2, k);
                }
                load4(pp + 3, pp + 2);
            }
            for (int i = 2 * pp; i < 2 * pp + 2; i++)
                if (i >= nw) clean(i, s_v[r] + (i & 1) * KB);
            r = r1;
        }
        if constexpr (!Q4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every copy into this block's LDS
        if (s_odd) {
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    const int el = 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
                    if (pos >= s_inf[0][el]) O[j][e] += __builtin_inff();
                    if (pos >= s_inf[1][el]) O[j][e] -= __builtin_inff();
                }
        }
    }

    // ---- results -----------------------------------------------------------------------------------
    // Through LDS, so that a store instruction writes whole rows: a lane holds 4 elements here and there (stored from
    // the registers, 1 x 4096 rows of bf16: pieces of 8 bytes 141 us, of 16 136; on another card 16 132.4, so 131.4, and
    // split results, 512 rows behind 8192, 81.4, so 79.3).  Each wave has 32 rows of 2 HD bytes, a row's 16-byte pieces
    // exchanged by an XOR with its number.
    constexpr int NP = HD / 8;
    l += xor32_f(l);
    lds_sync();   // the last tiles are read
    uint8_t *st = (w < 4 ? s_k[0] : s_v[0]) + (w & 3) * KB;
    auto at = [&](int r, int p) __attribute__((always_inline)) { return (v4u *)(st + r * (2 * HD) + ((p ^ (r & (NP - 1))) * 16)); };
    const uint32_t inv_g = (1u << 31) / G + 1;   // i / G = i inv_g / 2^31 for i < 2^27
    // row and piece of the lane in the t-th store; the row's number among the sequence's, token and head
    auto rows = [&](auto &&store) __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // other lanes' pieces
#pragma unroll
        for (int t = 0; t < NP / 2; t++) {
            const int r = (64 * t + lane) / NP, p = lane % NP, i = iw + r;
            const int tok = __umulhi(2 * i, inv_g);
            if (i < n_rows) store(*at(r, p), i, tok, kvh * G + i - tok * G, p);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    };
    if (ns == 1) {
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        // Lanes c and c + 32 have halves of 8 elements each; of two such pieces each lane takes one.
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                v4u y;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t p0 = pack2<AT>(O[j][e + 2 * k] * r, O[j][e + 2 * k + 1] * r);
                    const uint32_t p1 = pack2<AT>(O[j][e + 4 + 2 * k] * r, O[j][e + 5 + 2 * k] * r);
                    const auto sw = __builtin_amdgcn_permlane32_swap(p0, p1, false, false);
                    y[k] = sw[0];
                    y[2 + k] = sw[1];
                }
                if (l == 0.0f) y = v4u{0, 0, 0, 0};
                *at(c, 4 * j + e / 4 + h) = y;
            }
        rows([&](v4u y, int, int tok, int head, int p) __attribute__((always_inline)) {
            *(v4u *)(a.out + (size_t)(q.q0 + tok) * a.ldo + (size_t)head * HD + 8 * p) = y;
        });
    } else {
#pragma unroll
        for (int half = 0; half < 2; half++) {   // of the elements
#pragma unroll
            for (int j = 0; j < NJ / 2; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const v16f &o = O[half * (NJ / 2) + j];
                    *at(c, 8 * j + 2 * e + h) = v4u{__float_as_uint(o[4 * e]), __float_as_uint(o[4 * e + 1]),
                                                    __float_as_uint(o[4 * e + 2]), __float_as_uint(o[4 * e + 3])};
                }
            rows([&](v4u y, int i, int, int, int p) __attribute__((always_inline)) {
                *(v4u *)(a.part_o + (prompt_part(a, q.q0, kvh, i) + sp) * HD + half * (HD / 2) + 4 * p) = y;
            });
        }
        if (h == 0 && iw + c < n_rows) a.part_ml[prompt_part(a, q.q0, kvh, iw + c) + sp] = make_float2(m, l);
    }
}

template <int HD, int AT> hipError_t prompt_as(const PagedAttnArgs &a, hipStream_t s)
{
    const unsigned blocks = (unsigned)x100_attn_prompt_blocks(a.c, a.b, a.prompt.n);
    if (a.c.kv_type == X100_KV_Q4) k_attn_prompt<HD, AT, true><<<blocks, 512, 0, s>>>(a);
    else k_attn_prompt<HD, AT, false><<<blocks, 512, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

int64_t x100_attn_prompt_blocks(const x100_kv_cfg &c, const x100_kv_batch &b, int splits)
{
    return ((int64_t)b.n_rows * (c.n_head / c.n_head_kv) / PROMPT_ROWS + b.n_seq) * splits * c.n_head_kv;
}

hipError_t x100_attn_prompt_launch(const PagedAttnArgs &a, hipStream_t s)
{
    if (a.c.head_dim == 64) return a.c.act_type == X100_T_F16 ? prompt_as<64, X100_T_F16>(a, s) : prompt_as<64, X100_T_BF16>(a, s);
    return a.c.act_type == X100_T_F16 ? prompt_as<128, X100_T_F16>(a, s) : prompt_as<128, X100_T_BF16>(a, s);
}
