// Attention over the paged KV cache for many rows (x100_paged.h): prompts and pieces of prompts.
//
// One block: 256 rows (token, head) of a sequence and KV head, eight waves of 32 rows, and one split of
// the positions in tiles of 32.  As in attn_paged.hip the scores come transposed, S^T = K Q^T
// (v_mfma 32x32x16), and go as the operand P^T into O^T += V^T P^T in the registers they were made in.
//
// A wave makes the scores of tile i + 1 beside the weights of tile i (which do not depend on them), then
// the products of tile i; two waves share a SIMD, so that one's products run beside the other's
// weights.  K and V tiles come by asynchronous copies from the cache into rings of four tiles in LDS (4-bit
// pages: through registers, where they become fp16), read by all waves.
//
// The running maximum m may lag far behind (LAG), so that O and l are rescaled seldom.
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

template <int HD, int AT, bool Q4> __global__ __launch_bounds__(512, 2) void k_attn_prompt(const PagedAttnArgs a)
{
    constexpr int MT = Q4 ? X100_T_F16 : AT;
    constexpr int NT = 512;
    constexpr int KS = HD / 16, NJ = HD / 32;
    constexpr int KB = 32 * HD * 2;       // bytes of a K (or V) tile
    constexpr int NDW = KB / 4096;        // copies of 1 KiB per wave and step: K and V each (HD 128), or one of them (64)
    __shared__ __attribute__((aligned(1024))) uint8_t s_k[4][KB], s_v[4][KB];
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
    for (int i = threadIdx.x; i < n_pg; i += NT) {
        const int g = tab[i];
        const bool ok = g >= 0 && g < a.c.n_pages;
        s_pg[i] = ok ? g : -1;
        bad |= !ok;
    }
    bad = __syncthreads_or(bad);
    // Tiles that every row of the block sees whole; of the wave's rows: that they see whole, and see at all
    // (a wave without rows: none).
    const int iw = i0 + 32 * w;
    const int nw = bad ? 0 : max(0, min(n, (pos0 + i0 / G + 1 - t0) >> 5));
    const int ww = bad ? 0 : max(0, min(n, (pos0 + min(iw, n_rows - 1) / G + 1 - t0) >> 5));
    const int wn = iw >= n_rows ? 0 : max(0, min(n, (pos0 + min(iw + 31, n_rows - 1) / G + 1 - t0 + 31) >> 5));

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

    // ---- tiles into LDS --------------------------------------------------------------------------
    // K: [32 positions][HD], the 16-byte pieces of a row exchanged by an XOR with the position, so that
    // 16 lanes that read one piece of 16 positions meet different banks.  V: [4][HD][8] as in the cache.
    constexpr int RC = HD / 8;   // pieces of a row
    auto swz = [](int tok) { return HD == 128 ? tok & 15 : (tok >> 1) & 7; };
    const size_t head_bytes = page_head_bytes<HD, Q4>(page);
    // Copies: KiB `wd` of the tile; head_dim 128: every wave one of K and one of V; 64: waves 0 .. 3 of K, 4 .. 7 of V.
    const int wd = NDW == 2 ? w : w & 3, grp = (wd * (32 / (4 * NDW))) >> 4;   // its 16 positions
    const int wtok = wd * (1024 / (HD * 2));                                  // its first K position
    const uint32_t kvoff = (uint32_t)((wtok + lane / RC) & 15) * (HD * 2) + (uint32_t)((lane % RC) ^ swz(wtok + lane / RC)) * 16;
    const uint32_t lk = lds_addr(s_k) + wd * 1024, lv = lds_addr(s_v) + wd * 1024;
    auto head_of = [&](const uint8_t *pool, int t) __attribute__((always_inline)) {   // the head's part of position t's page
        const int pg = __builtin_amdgcn_readfirstlane(max(s_pg[((t < t1 ? t : t0) >> psh) - (t0 >> psh)], 0));
        return pool + (size_t)(pg * n_kv + kvh) * head_bytes;
    };
    auto load_k = [&](int i) __attribute__((always_inline)) {
        const int t = t0 + 32 * min(i, n - 1) + 16 * grp;
        dma16s(kvoff, head_of(a.kp, t) + (t & (page - 1)) * (HD * 2), lk + (i & 3) * KB);
    };
    auto load_v = [&](int i) __attribute__((always_inline)) {
        const int t = t0 + 32 * min(i, n - 1) + 16 * grp;
        // KiB wd of a tile whose block of 8 positions is HD * 16 bytes, from the group's first block on
        const uint32_t in = (t & (page - 1)) * (HD * 2) + (wd * 1024 - 16 * grp * (HD * 2));
        dma16s(16u * lane, head_of(a.vp, t) + in, lv + (i & 3) * KB);
    };
    // 4 bits: waves 0 .. 3 take K (a thread: HD / 8 elements of a position), 4 .. 7 V (HD / 64 elements of 8
    // positions); one tile waits in registers.
    constexpr int W4 = HD / 64;
    uint32_t r_w[W4];
    v4u r_d, r_m;
    const int x4 = threadIdx.x & 255;
    const bool isk = w < 4;
    auto load4 = [&](int i) __attribute__((always_inline)) {   // K of tile i, or V of tile i - 1
        const int ti = isk ? min(i, n - 1) : min(max(i - 1, 0), n - 1);
        const int pp = t0 + 32 * ti + (isk ? x4 >> 3 : 8 * (x4 >> 6));
        const int pg = max(s_pg[((pp < t1 ? pp : t0) >> psh) - (t0 >> psh)], 0);
        const uint8_t *base = (isk ? a.kp : a.vp) + ((size_t)pg * n_kv + kvh) * head_bytes;
        const int off = pp & (page - 1);
        const uint32_t *cw = (const uint32_t *)base + (isk ? off * (HD / 8) + (x4 & 7) * W4 : (off >> 3) * HD + (x4 & 63) * W4);
        if constexpr (W4 == 2) {
            const v2u v = *(const v2u *)cw;
            r_w[0] = v[0];
            r_w[1] = v[1];
        } else {
            r_w[0] = cw[0];
        }
        const uint8_t *sb = base + page * HD / 2;
        if (isk) {
            r_d[0] = ((const uint32_t *)sb)[off * (HD / 32) + (x4 & 7) * HD / 256];
        } else {
            const v4u *vs = (const v4u *)(sb + ((off >> 3) * (HD / 32) + (x4 & 63) * W4 / 32) * 32);
            r_d = vs[0];
            r_m = vs[1];
        }
    };
    auto store4 = [&](int i) __attribute__((always_inline)) {   // what load4(i) fetched
        uint8_t *dst;
        int tok = 0;
        if (isk) {
            tok = x4 >> 3;
            dst = s_k[i & 3] + tok * (HD * 2);
            const uint32_t d = (r_d[0] & 0xffffu) * 0x10001u, m = (r_d[0] >> 16) * 0x10001u;
            r_d = v4u{d, d, d, d};
            r_m = v4u{m, m, m, m};
        } else {
            dst = s_v[(i - 1) & 3] + x4 * (W4 * 16);
        }
#pragma unroll
        for (int k = 0; k < W4; k++)
            *(v4u *)(dst + (isk ? (((x4 & 7) * W4 + k) ^ swz(tok)) * 16 : k * 16)) = q4_v(r_w[k], r_d, r_m);
    };
    // Step i: K(i + 1) and V(i) are in LDS for every wave, the slots of K(i) and V(i - 1) free.
    auto next_tiles = [&](int i) __attribute__((always_inline)) {
        if constexpr (!Q4) {
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_waitcnt lgkmcnt(0)\n\ts_barrier" ::"n"(NDW) : "memory");
            if (NDW == 2 || w < 4) load_k(i + 3);
            if (NDW == 2 || w >= 4) load_v(i + 2);
        } else {
            lds_sync();
            store4(i + 2);
            load4(i + 3);
        }
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
    v4u P[2];
    float m = NEG_INF, msub = 0.0f, l = 0.0f, mx = NEG_INF;
#pragma unroll
    for (int j = 0; j < NJ; j++) O[j] = v16f{};
    auto scores = [&](int i, v16f &X) __attribute__((always_inline)) {
        const uint8_t *k = s_k[i & 3];
        X = v16f{};
#pragma unroll
        for (int j = 0; j < KS; j++) X = mfma32<MT>(*(const v4u *)(k + kad[j]), qf[j], X);
    };
    auto products = [&](int i) __attribute__((always_inline)) {
        const uint8_t *v = s_v[i & 3] + vad;
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int j = 0; j < NJ; j++) O[j] = mfma32<MT>(*(const v4u *)(v + k * (2 * HD * 16) + j * 512), P[k], O[j]);
    };
    auto maximum = [&](const v16f &X) __attribute__((always_inline)) {
        float y = fmaxf(X[0], X[1]);
#pragma unroll
        for (int e = 2; e < 16; e += 2) y = fmaxf(fmaxf(y, X[e]), X[e + 1]);
        mx = y * sc2;
    };
    // Weights may be up to 2^LAG: fp16 holds them, and sums of bf16 V up to 2^100 stay finite.
    constexpr float LAG = MT == X100_T_F16 ? 14.0f : 16.0f;
    // m rises to the maximum so far, O and l go to the new unit
    auto rescale = [&]() __attribute__((always_inline)) {
        if (!__any(mx > m + LAG)) return;
        const float y = fmaxf(mx, xor32_f(mx));
        const float mn = y > m + LAG ? y : m;
        const float f = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        msub = mn == NEG_INF ? 0.0f : mn;
        l *= f;
#pragma unroll
        for (int j = 0; j < NJ; j++) O[j] *= f;
    };
    auto weights = [&](const v16f &X) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < 2; k++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(X[8 * k + 2 * e], sc2, -msub));
                const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(X[8 * k + 2 * e + 1], sc2, -msub));
                const uint32_t p = pack2<MT>(p0, p1);
                P[k][e] = p;
                l = add2<MT>(p, l);
            }
    };
    // Validity of the tile's two groups of 16 positions (their pages).
    auto ok16 = [&](int i, int k) {
        const int t = t0 + 32 * i + 16 * k;
        return t < t1 && s_pg[(t >> psh) - (t0 >> psh)] >= 0;
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
        maximum(X);
    };
    // V of a tile that not every row sees whole, before its products: the positions that no row has as
    // zeros, and elements that are not finite taken out, because 0 times such an element would reach the
    // rows that do not see it.  Rows see a prefix of the positions, so the first place of each element
    // where it is +inf, and where it is -inf (a NaN: both), says at the end which rows take it.
    auto clean = [&](int i) __attribute__((always_inline)) {
        constexpr uint32_t EXP = MT == X100_T_F16 ? 0x7c00u : 0x7f80u;
        for (int x = threadIdx.x; x < KB / 16; x += NT) {
            const int blk = x / HD, el = x % HD, p = t0 + 32 * i + 8 * blk;
            const int left = ok16(i, blk >> 1) ? q.kv_len - p : 0;
            uint16_t *v = (uint16_t *)(s_v[i & 3] + x * 16);
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
    auto step = [&](int i, v16f &X, v16f &Y) __attribute__((always_inline)) {
        next_tiles(i);
        if (i >= nw) clean(i);
        if (i < wn) {
            if (i >= ww) mask(i, X);
            rescale();
            scores(i + 1, Y);
            weights(X);
            products(i);
            maximum(Y);
            // order: K's operands on their way, weights beside the scores' matrix instructions with V's
            // operands on their way, products
            __builtin_amdgcn_sched_group_barrier(0x100, KS, 0);
            __builtin_amdgcn_sched_group_barrier(0x402, 12, 0);
#pragma unroll
            for (int g = 0; g < KS; g++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 4, 0);
            }
#pragma unroll
            for (int g = 0; g < 2 * NJ; g++) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x402, 1, 0);
            }
        }
    };

    if (n > 0) {
        if constexpr (!Q4) {
            if (NDW == 2 || w < 4) {
                load_k(0);
                load_k(1);
                load_k(2);
            }
            if (NDW == 2 || w >= 4) {
                load_v(0);
                load_v(1);
            }
        } else {
            // K(0), K(1), V(0) (V slot 3 gets tile 0 on the way)
            load4(0);
            store4(0);
            load4(1);
            store4(1);
            load4(2);
        }
        for (int x = threadIdx.x; x < 2 * HD; x += NT) s_inf[x / HD][x % HD] = INT_MAX;
        if (threadIdx.x == 0) s_odd = 0;
        if constexpr (!Q4) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        lds_sync();
        scores(0, S);
        maximum(S);
        for (int i = 0;;) {
            step(i, S, T);
            if (++i >= n) break;
            step(i, T, S);
            if (++i >= n) break;
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
    l += xor32_f(l);
    const int i = iw + c;
    if (i >= n_rows) return;
    const int tok = i / G, head = kvh * G + i % G;
    const size_t row = q.q0 + tok;
    if (ns == 1) {
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        uint16_t *o = a.out + row * a.ldo + (size_t)head * HD + 4 * h;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                v2u y = {0, 0};
                if (l != 0.0f)
                    y = v2u{pack2<AT>(O[j][4 * e] * f, O[j][4 * e + 1] * f), pack2<AT>(O[j][4 * e + 2] * f, O[j][4 * e + 3] * f)};
                *(v2u *)(o + 32 * j + 8 * e) = y;
            }
    } else {
        const size_t at = part_prompt(a, q.q0, kvh, i) + sp;
        float *o = a.o_p + at * HD + 4 * h;
#pragma unroll
        for (int j = 0; j < NJ; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                *(float4 *)(o + 32 * j + 8 * e) = make_float4(O[j][4 * e], O[j][4 * e + 1], O[j][4 * e + 2], O[j][4 * e + 3]);
        if (h == 0) a.ml_p[at] = make_float2(m, l);
    }
}

template <int HD, int AT> hipError_t prompt_as(const PagedAttnArgs &a, int tiles, hipStream_t s)
{
    const dim3 grid((unsigned)(tiles * a.n_split_p * a.c.n_head_kv), a.b.n_seq);
    if (a.c.kv_type == X100_KV_Q4) k_attn_prompt<HD, AT, true><<<grid, 512, 0, s>>>(a);
    else k_attn_prompt<HD, AT, false><<<grid, 512, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t x100_attn_prompt_launch(const PagedAttnArgs &a, int tiles, hipStream_t s)
{
    if (a.c.head_dim == 64)
        return a.c.act_type == X100_T_F16 ? prompt_as<64, X100_T_F16>(a, tiles, s) : prompt_as<64, X100_T_BF16>(a, tiles, s);
    return a.c.act_type == X100_T_F16 ? prompt_as<128, X100_T_F16>(a, tiles, s) : prompt_as<128, X100_T_BF16>(a, tiles, s);
}
