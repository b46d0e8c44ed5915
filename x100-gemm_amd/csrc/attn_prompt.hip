// Attention over the paged KV cache for many rows (x100_paged.h): prompts and pieces of prompts.
//
// One block: 256 rows (token, head) of a sequence and KV head, four waves of 64 rows (two column
// blocks of 32), and one split of the positions in tiles of 32.  As in attn_paged.hip the scores come
// transposed, S^T = K Q^T (v_mfma 32x32x16), and go as the operand P^T into O^T += V^T P^T in the
// registers they were made in.
//
// The two column blocks run half a step apart, so that matrix cores and vector unit always have work that
// does not depend on the other's:
//   first half    weights of block 0, tile i        beside scores of block 1, tile i, and its products of tile i - 1
//   second half   weights of block 1, tile i        beside scores of block 0, tile i + 1, and its products of tile i
// The operands of K and V are read from LDS once per tile, in the first half (as soon as the last ones have been
// used), and kept for both blocks.  K and V come 64 positions at a time by asynchronous copies from the
// cache into LDS (4-bit pages: through registers, where they become fp16), read by all four waves, with one
// barrier for two tiles.
//
// The running maximum m is taken from the first tile and then only followed where a weight would leave
// its 16 bits: the weights' sum, which is needed anyway, says so, and the tile's weights are made again.
#include "paged_attn.h"
#include "x100_internal.h"

namespace {

constexpr float NEG_INF = X100_NEG_INF;

// 16 bytes per lane from sbase + voff to lds_base + 16 * lane; not counted by the compiler.
X100_DEV void dma16s(uint32_t voff, const void *sbase, uint32_t lds_base)
{
    asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds_base) : "memory");
}

// LDS of every wave written and read up to here
X100_DEV void lds_sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int HD, int AT, bool Q4> __global__ __launch_bounds__(256, 1) void k_attn_prompt(const PagedAttnArgs a)
{
    constexpr int MT = Q4 ? X100_T_F16 : AT;
    constexpr int KS = HD / 16, NJ = HD / 32;
    constexpr int KB = 32 * HD * 2;       // bytes of a K (or V) tile of 32 positions
    constexpr int ND = 2 * KB / 4096;     // copies of 1 KiB per wave and pair of tiles
    __shared__ __attribute__((aligned(1024))) uint8_t s_k[3][2 * KB], s_v[2][2 * KB];   // pairs of tiles
    __shared__ int s_pg[PROMPT_SPLIT / 16];
    __shared__ int s_inf[2][HD], s_odd;
    const int lane = threadIdx.x & 63, w = wave_id(), c = lane & 31, h = lane >> 5;
    const int n_kv = a.c.n_head_kv, G = a.c.n_head / n_kv, page = a.c.page, psh = __builtin_ctz(page);
    const int kvh = blockIdx.x % n_kv, u = blockIdx.x / n_kv, sp = u % a.n_split_p;
    const int tile = gridDim.x / (n_kv * a.n_split_p) - 1 - u / a.n_split_p, s = blockIdx.y;   // longest first
    const PagedSeq q = paged_seq(a.b, s);
    const int n_rows = q.q_len * G, i0 = tile * PROMPT_ROWS;
    if (i0 >= n_rows || n_rows <= a.few) return;
    const int pos0 = q.kv_len - q.q_len;
    const int vis = pos0 + min(i0 + PROMPT_ROWS - 1, n_rows - 1) / G + 1;
    const int ns = max(1, (vis + a.split_p - 1) / a.split_p);
    if (sp >= ns) return;
    const int t0 = sp * a.split_p, t1 = min(t0 + a.split_p, vis);
    const int n = max(0, (t1 - t0 + 31) >> 5);   // tiles

    // pages of the split; one that is none sends every tile through the masked step
    const int *tab = a.b.block_table + (size_t)s * a.b.table_ld + (t0 >> psh);
    const int n_pg = n > 0 ? ((t1 - 1) >> psh) - (t0 >> psh) + 1 : 0;
    bool bad = false;
    for (int i = threadIdx.x; i < n_pg; i += 256) {
        const int g = tab[i];
        const bool ok = g >= 0 && g < a.c.n_pages;
        s_pg[i] = ok ? g : -1;
        bad |= !ok;
    }
    bad = __syncthreads_or(bad);
    const int nw = bad ? 0 : max(0, min(n, (pos0 + i0 / G + 1 - t0) >> 5));   // tiles that every row sees whole

    // queries: rows 64 w + 32 b + c
    int pos[2];
    float sc2[2];
    v4u qf[2][KS];
#pragma unroll
    for (int b = 0; b < 2; b++) {
        const int i = min(i0 + 64 * w + 32 * b + c, n_rows - 1), tok = i / G, head = kvh * G + i % G;
        pos[b] = pos0 + tok;
        sc2[b] = a.scale2;
        const uint16_t *qr = a.q + (size_t)(q.q0 + tok) * a.ldq + (size_t)head * HD + 8 * h;
#pragma unroll
        for (int j = 0; j < KS; j++) qf[b][j] = *(const v4u *)(qr + 16 * j);
        if constexpr (Q4 && AT == X100_T_BF16) {
            float mx = 0.0f;
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    mx = fmaxf(mx, fmaxf(fabsf(bf2f(qf[b][j][e] & 0xffffu)), fabsf(__uint_as_float(qf[b][j][e] & 0xffff0000u))));
            mx = fmaxf(mx, xor32_f(mx));
            const int ex = row_exponent(mx);
            sc2[b] = ldexpf(sc2[b], ex);
#pragma unroll
            for (int j = 0; j < KS; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    qf[b][j][e] = pack2<X100_T_F16>(ldexpf(bf2f(qf[b][j][e] & 0xffffu), -ex),
                                                    ldexpf(__uint_as_float(qf[b][j][e] & 0xffff0000u), -ex));
        }
    }

    // ---- pairs of tiles into LDS -------------------------------------------------------------------
    // K: [64 positions][HD], the 16-byte pieces of a row exchanged by an XOR with the position, so that
    // 16 lanes that read one piece of 16 positions meet different banks.  V: [8][HD][8] as in the cache.
    // Wave w copies positions 16 w .. 16 w + 15, which lie on one page; their bytes begin at the same place of
    // the K and of the V pool.
    constexpr int RC = HD / 8;   // pieces of a row
    auto swz = [](int tok) { return HD == 128 ? tok & 15 : (tok >> 1) & 7; };
    const size_t head_bytes = page_head_bytes<HD, Q4>(page);
    const int np = (n + 1) >> 1;   // pairs
    auto page_at = [&](int pp) {   // entry of the page list for the wave's positions of pair pp
        const int t = t0 + 64 * pp + 16 * w;
        return s_pg[((t < t1 ? t : t0) >> psh) - (t0 >> psh)];
    };
    auto place = [&](int pp, int pg) -> size_t {
        const int t = t0 + 64 * pp + 16 * w;
        return (size_t)(max(__builtin_amdgcn_readfirstlane(pg), 0) * n_kv + kvh) * head_bytes + (t & (page - 1)) * (HD * 2);
    };
    uint32_t kvoff[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) {
        const int tok = (1024 * d) / (HD * 2) + lane / RC;
        kvoff[d] = (uint32_t)tok * (HD * 2) + (uint32_t)((lane % RC) ^ swz(tok)) * 16;
    }
    const uint32_t lk = lds_addr(s_k) + w * (KB / 2), lv = lds_addr(s_v) + w * (KB / 2);
    auto load_k = [&](size_t at, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < ND; d++) dma16s(kvoff[d], a.kp + at, lk + slot * (2 * KB) + d * 1024);
    };
    auto load_v = [&](size_t at, int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int d = 0; d < ND; d++) dma16s(16u * lane + 1024u * d, a.vp + at, lv + slot * (2 * KB) + d * 1024);
    };
    // 4 bits: a thread takes HD / 4 elements of a K position, and HD / 32 elements of a V block of 8 positions.
    constexpr int W4 = HD / 32;
    uint32_t rk_w[W4], rk_s, rv_w[W4];
    v4u rv_d, rv_m;
    const int x4 = threadIdx.x;
    auto base4 = [&](const uint8_t *pool, int pp, int &off) {
        const int pg = max(s_pg[((pp < t1 ? pp : t0) >> psh) - (t0 >> psh)], 0);
        off = pp & (page - 1);
        return pool + ((size_t)pg * n_kv + kvh) * head_bytes;
    };
    auto words4 = [&](const uint32_t *p, uint32_t (&r)[W4]) __attribute__((always_inline)) {
        if constexpr (W4 == 4) {
            const v4u v = *(const v4u *)p;
#pragma unroll
            for (int e = 0; e < 4; e++) r[e] = v[e];
        } else {
            const v2u v = *(const v2u *)p;
            r[0] = v[0];
            r[1] = v[1];
        }
    };
    auto load4 = [&](int pk, int pv) __attribute__((always_inline)) {   // K of pair pk, V of pair pv
        int off;
        const uint8_t *kb = base4(a.kp, t0 + 64 * min(pk, np - 1) + (x4 >> 2), off);
        words4((const uint32_t *)kb + off * (HD / 8) + (x4 & 3) * W4, rk_w);
        rk_s = ((const uint32_t *)(kb + page * HD / 2))[off * (HD / 32) + (x4 & 3) * HD / 128];
        const uint8_t *vb = base4(a.vp, t0 + 64 * min(pv, np - 1) + 8 * (x4 >> 5), off);
        words4((const uint32_t *)vb + (off >> 3) * HD + (x4 & 31) * W4, rv_w);
        const v4u *vs = (const v4u *)(vb + page * HD / 2 + ((off >> 3) * (HD / 32) + (x4 & 31) * W4 / 32) * 32);
        rv_d = vs[0];
        rv_m = vs[1];
    };
    auto store_k4 = [&](int slot) __attribute__((always_inline)) {   // what load4 fetched, as fp16
        uint8_t *dst = s_k[slot] + (x4 >> 2) * (HD * 2);
        const uint32_t d = (rk_s & 0xffffu) * 0x10001u, m = (rk_s >> 16) * 0x10001u;
#pragma unroll
        for (int k = 0; k < W4; k++)
            *(v4u *)(dst + (((x4 & 3) * W4 + k) ^ swz(x4 >> 2)) * 16) = q4_v(rk_w[k], v4u{d, d, d, d}, v4u{m, m, m, m});
    };
    auto store_v4 = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < W4; k++) *(v4u *)(s_v[slot] + (x4 * W4 + k) * 16) = q4_v(rv_w[k], rv_d, rv_m);
    };

    // ---- products --------------------------------------------------------------------------------
    // K operand: row r of the tile's 32 is position 16 (r / 16) + 8 (r / 4 % 2) + 4 (r / 8 % 2) + r % 4, so
    // that lane (c, h) receives positions 16 s + 8 h + 0 .. 7 of row c in registers 8 s .. 8 s + 7.
    const int ktok = 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3);
    uint32_t kad[KS];
#pragma unroll
    for (int j = 0; j < KS; j++) kad[j] = ktok * (HD * 2) + (((2 * j + h) ^ swz(ktok)) * 16);
    const uint32_t vad = h * (HD * 16) + c * 16;

    v16f S[2], O[2][NJ];
    v4u P[2][2], kf[KS], vf[2][NJ];   // weights, operands of K and V
    float m[2] = {NEG_INF, NEG_INF}, msub[2] = {0, 0}, l[2] = {0, 0}, mx[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
#pragma unroll
        for (int j = 0; j < NJ; j++) O[b][j] = v16f{};
        P[b][0] = P[b][1] = v4u{0, 0, 0, 0};
    }
    auto read_k = [&](const uint8_t *k) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < KS; j++) kf[j] = *(const v4u *)(k + kad[j]);
    };
    auto read_v = [&](const uint8_t *v) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < NJ; j++) vf[k][j] = *(const v4u *)(v + vad + k * (2 * HD * 16) + j * 512);
    };
    auto scores = [&](int b) __attribute__((always_inline)) {
        v16f x = v16f{};
#pragma unroll
        for (int j = 0; j < KS; j++) x = mfma32<MT>(kf[j], qf[b][j], x);
        S[b] = x;
    };
    auto products = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < NJ; j++) O[b][j] = mfma32<MT>(vf[k][j], P[b][k], O[b][j]);
    };
    auto maximum = [&](int b) __attribute__((always_inline)) {
        float y = fmaxf(S[b][0], S[b][1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2) y = fmaxf(fmaxf(y, S[b][e]), S[b][e + 1]);
        mx[b] = y * sc2[b];
    };
    // m rises to the tile's maximum, O and l go to the new unit (no weights of block b in flight)
    auto rescale = [&](int b) __attribute__((always_inline)) {
        const float y = fmaxf(mx[b], xor32_f(mx[b]));
        const float mn = y > m[b] ? y : m[b];
        const float f = mn == m[b] ? 1.0f : __builtin_amdgcn_exp2f(m[b] - mn);
        m[b] = mn;
        msub[b] = mn == NEG_INF ? 0.0f : mn;
        l[b] *= f;
#pragma unroll
        for (int j = 0; j < NJ; j++) O[b][j] *= f;
    };
    float lt[2];   // the tile's sum of weights (of the lane's positions)
    auto weights = [&](int b) __attribute__((always_inline)) {
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[b][8 * k + 2 * e], sc2[b], -msub[b]));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[b][8 * k + 2 * e + 1], sc2[b], -msub[b]));
                const uint32_t p = pack2<MT>(p0, p1);
                P[b][k][e] = p;
                y = add2<MT>(p, y);
            }
        lt[b] = y;
    };
    // After a half: its weights are good as long as their sum is below 2^14, which fp16 holds and with which
    // sums over bf16 V up to 2^100 stay finite (a row that has no maximum yet: not good).  Else m follows.
    auto settle = [&](int b) __attribute__((always_inline)) {
        if (__any(!(lt[b] < 16384.0f) || m[b] == NEG_INF)) {
            maximum(b);
            rescale(b);
            weights(b);
        }
        l[b] += lt[b];
    };
    // The half's weights are made in it (the compiler would move them to where they are used).
    auto here = [&](int b) __attribute__((always_inline)) {
        asm volatile("" ::"v"(P[b][0]), "v"(P[b][1]), "v"(lt[b]));
    };
    // Order of a half: after each matrix instruction the vector instructions that fit beside it; in the
    // first half the next operands' reads behind the last use of each.
    auto interleave = [&](bool reads) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < KS; g++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, 4, 0);
        }
#pragma unroll
        for (int g = 0; g < 2 * NJ; g++) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            if (reads) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, 4, 0);
        }
    };
    // Validity of the tile's two groups of 16 positions (their pages).
    auto ok16 = [&](int i, int k) {
        const int t = t0 + 32 * i + 16 * k;
        return t < t1 && s_pg[(t >> psh) - (t0 >> psh)] >= 0;
    };
    auto mask = [&](int i, int b) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const bool ok = ok16(i, k);
            const int p = t0 + 32 * i + 16 * k + 8 * h;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (!(ok && p + e <= pos[b])) S[b][8 * k + e] = NEG_INF;
        }
    };
    // V of a tile that not every row sees whole, before its products: the positions that no row has as
    // zeros, and elements that are not finite taken out, because 0 times such an element would reach the
    // rows that do not see it.  Rows see a prefix of the positions, so the first place of each element
    // where it is +inf, and where it is -inf (a NaN: both), says at the end which rows take it.
    auto clean = [&](int i) __attribute__((always_inline)) {
        constexpr uint32_t EXP = MT == X100_T_F16 ? 0x7c00u : 0x7f80u;
        for (int x = threadIdx.x; x < KB / 16; x += 256) {
            const int blk = x / HD, el = x % HD, p = t0 + 32 * i + 8 * blk;
            const int left = ok16(i, blk >> 1) ? q.kv_len - p : 0;
            uint16_t *v = (uint16_t *)(s_v[(i >> 1) & 1] + (i & 1) * KB + x * 16);
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

    // One tile: see the head of this file.  kn: K of tile i + 1, v: V of tile i.
    auto step = [&](int i, const uint8_t *kn, const uint8_t *v) __attribute__((always_inline)) {
        if (i >= nw) {
            clean(i);
            mask(i, 0);
        }
        scores(1);
        weights(0);
        read_k(kn);
        products(1);
        read_v(v);
        interleave(true);
        here(0);
        settle(0);

        if (i >= nw) mask(i, 1);
        if (i == 0) {
            maximum(1);
            rescale(1);
        }
        scores(0);
        weights(1);
        products(0);
        interleave(false);
        here(1);
        settle(1);
    };

    if (n > 0) {
        size_t at = 0;   // where the wave's positions of the next V pair are
        int pg = 0;      // page of the next K pair
        if constexpr (!Q4) {
            const size_t a0 = place(0, page_at(0));
            load_k(a0, 0);
            load_v(a0, 0);
            at = place(min(1, np - 1), page_at(min(1, np - 1)));
            load_k(at, 1);
            pg = page_at(min(2, np - 1));
        } else {
            load4(0, 0);
            store_k4(0);
            store_v4(0);
            load4(1, 1);
            store_k4(1);
            load4(2, 1);
        }
        for (int x = threadIdx.x; x < 2 * HD; x += 256) s_inf[x / HD][x % HD] = INT_MAX;
        if (threadIdx.x == 0) s_odd = 0;
        if constexpr (!Q4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_sync();
        read_k(s_k[0]);
#pragma unroll
        for (int j = 0; j < NJ; j++) vf[0][j] = vf[1][j] = v4u{0, 0, 0, 0};
        scores(0);
        if (nw == 0) mask(0, 0);
        maximum(0);
        rescale(0);
        // Pair pp: K of pairs pp and pp + 1 and V of pair pp are in LDS for every wave, the places of K pair pp - 1
        // and V pair pp - 1 free.
        int ks = 0;   // pp % 3
        for (int pp = 0; pp < np; pp++) {
            const int ks1 = ks == 2 ? 0 : ks + 1, ks2 = ks1 == 2 ? 0 : ks1 + 1;
            if constexpr (!Q4) {
                asm volatile("s_waitcnt vmcnt(0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                load_v(at, (pp + 1) & 1);
                at = place(min(pp + 2, np - 1), pg);
                load_k(at, ks2);
                pg = page_at(min(pp + 3, np - 1));
            } else {
                lds_sync();
                store_k4(ks2);
                store_v4((pp + 1) & 1);
                load4(pp + 3, pp + 2);
            }
            step(2 * pp, s_k[ks] + KB, s_v[pp & 1]);
            if (2 * pp + 1 < n) step(2 * pp + 1, s_k[ks1], s_v[pp & 1] + KB);
            ks = ks1;
        }
        products(1);
        if constexpr (!Q4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // every copy into this block's LDS
        if (s_odd) {
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const int el = 32 * j + 8 * (e >> 2) + 4 * h + (e & 3);
                        if (pos[b] >= s_inf[0][el]) O[b][j][e] += __builtin_inff();
                        if (pos[b] >= s_inf[1][el]) O[b][j][e] -= __builtin_inff();
                    }
        }
    }

    // ---- results -----------------------------------------------------------------------------------
#pragma unroll
    for (int b = 0; b < 2; b++) {
        l[b] += xor32_f(l[b]);
        const int i = i0 + 64 * w + 32 * b + c;
        if (i >= n_rows) continue;
        const int tok = i / G, head = kvh * G + i % G;
        const size_t row = q.q0 + tok;
        if (ns == 1) {
            const float f = l[b] == 0.0f ? 0.0f : 1.0f / l[b];
            uint16_t *o = a.out + row * a.ldo + (size_t)head * HD + 4 * h;
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    v2u y = {0, 0};
                    if (l[b] != 0.0f)
                        y = v2u{pack2<AT>(O[b][j][4 * e] * f, O[b][j][4 * e + 1] * f), pack2<AT>(O[b][j][4 * e + 2] * f, O[b][j][4 * e + 3] * f)};
                    *(v2u *)(o + 32 * j + 8 * e) = y;
                }
        } else {
            const size_t at = part_prompt(a, q.q0, kvh, i) + sp;
            float *o = a.o_p + at * HD + 4 * h;
#pragma unroll
            for (int j = 0; j < NJ; j++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    *(float4 *)(o + 32 * j + 8 * e) = make_float4(O[b][j][4 * e], O[b][j][4 * e + 1], O[b][j][4 * e + 2], O[b][j][4 * e + 3]);
            if (h == 0) a.ml_p[at] = make_float2(m[b], l[b]);
        }
    }
}

template <int HD, int AT> hipError_t prompt_as(const PagedAttnArgs &a, int tiles, hipStream_t s)
{
    const dim3 grid((unsigned)(tiles * a.n_split_p * a.c.n_head_kv), a.b.n_seq);
    if (a.c.kv_type == X100_KV_Q4) k_attn_prompt<HD, AT, true><<<grid, 256, 0, s>>>(a);
    else k_attn_prompt<HD, AT, false><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t x100_attn_prompt_launch(const PagedAttnArgs &a, int tiles, hipStream_t s)
{
    if (a.c.head_dim == 64)
        return a.c.act_type == X100_T_F16 ? prompt_as<64, X100_T_F16>(a, tiles, s) : prompt_as<64, X100_T_BF16>(a, tiles, s);
    return a.c.act_type == X100_T_F16 ? prompt_as<128, X100_T_F16>(a, tiles, s) : prompt_as<128, X100_T_BF16>(a, tiles, s);
}
