// Paged KV cache (x100_paged.h): new rows into the pages (head norms, rotation, 16 or 4 bits), cached
// rows back out, and the rotation table.
//
// Bound by HBM for prompts (a row is read once, its queries, keys and values written once): 6400 rows of 40 heads
// of 128, int32 to f16 and 4 bits, 44 us, 4.2 TB/s (a copy of 2 GiB: 5.0).  For single tokens bound by the launch and
// dependent loads (q_start -> kv_len -> block_table): 64 rows 4.4 us.
#include <algorithm>

#include "paged.h"
#include "x100_internal.h"

namespace {

// ---- rotation table ------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_rope_table(int half, int n_pos, double base, float2 *__restrict__ t)
{
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (size_t)n_pos * half) return;
    const int p = (int)(i / half), k = (int)(i % half);
    double sn, cs;
    sincos((double)p * pow(base, -(double)k / half), &sn, &cs);
    t[i] = make_float2((float)cs, (float)sn);
}

// Exchanges among the 16 lanes of an item: xor 1, 2 within a quad, half-row mirror (the other quad
// of 8 lanes), rotation by 8 (the other 8 lanes).
X100_DEV float sum16(float v)
{
    v += dpp_f<0xB1>(0.0f, v);
    v += dpp_f<0x4E>(0.0f, v);
    v += dpp_f<0x141>(0.0f, v);
    v += dpp_f<0x128>(0.0f, v);
    return v;
}
// min / max over the lanes of a group of 32 elements: 4 lanes of 8 (head_dim 128), 8 of 4 (64)
template <int HD> X100_DEV float gmin(float v)
{
    v = fminf(v, dpp_f<0xB1>(v, v));
    v = fminf(v, dpp_f<0x4E>(v, v));
    if constexpr (HD == 64) v = fminf(v, dpp_f<0x141>(v, v));
    return v;
}

// Smallest (SGN = 1; -1: minus the largest) of 8 positions each over the 32 lanes of a group: halves of the positions
// are exchanged for halves of the lanes twice, so that lane c % 4 ends with positions c % 4 and 4 + c % 4.
template <int SGN> X100_DEV void gmin8(const float (&v)[8], float (&m)[2])
{
    const bool b0 = threadIdx.x & 1, b1 = threadIdx.x & 2;
    float a[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float x = SGN * v[2 * j], y = SGN * v[2 * j + 1];
        a[j] = fminf(b0 ? y : x, dpp_f<0xB1>(0.0f, b0 ? x : y));
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float r = fminf(b1 ? a[2 * i + 1] : a[2 * i], dpp_f<0x4E>(0.0f, b1 ? a[2 * i] : a[2 * i + 1]));
        r = fminf(r, dpp_f<0x124>(0.0f, r));
        r = fminf(r, dpp_f<0x128>(0.0f, r));
        m[i] = fminf(r, xor16_f(r));
    }
}
// lane C of each four
template <int C> X100_DEV float quad(float v) { return dpp_f<0x55 * C>(0.0f, v); }

// Where row r of a wave's four (lane / 16) lies: the sequence s, the position (pos < 0: before the first),
// mine: the row is one of a sequence that is not refused.
struct RowPlace {
    int s, pos;
    bool mine;
};
X100_DEV RowPlace row_place(const x100_kv_batch &b, int rbase, int sub)
{
    RowPlace p = {0, -1, false};
    const int r = rbase + sub, f0 = paged_find(b, rbase), l = threadIdx.x & 15;
    if (f0 >= b.n_seq) return p;
    // mostly the row is one of the next 16 sequences' (a search for each of four single tokens of 512: 14.8 us, so
    // 11.5)
    const bool le = f0 + l < b.n_seq && b.q_start[f0 + l + 1] <= r;
    const int n = __popc((uint32_t)(__ballot(le) >> (16 * sub)) & 0xffffu);
    int f = f0 + n;
    for (uint64_t far = __ballot(n == 16); far;) {
        const int i = __builtin_ctzll(far) >> 4, g = paged_find(b, rbase + i);
        if (i == sub) f = g;
        far &= ~(0xffffull << (16 * i));
    }
    if (r < b.n_rows && f < b.n_seq) {
        const PagedSeq q = paged_seq(b, f);
        if (q.holds(r)) p = {f, q.position(r), true};
    }
    return p;
}

struct AppendArgs {
    x100_kv_cfg c;
    x100_kv_batch b;
    x100_kv_rows r;
    uint8_t *kp, *vp;
    uint16_t *q_out;
    int heads;     // query and key heads of a wave, one after the other
    int xq, nq;    // blocks of one group of heads (16 rows each), of all query and key heads; behind them: values
    int xv;        // blocks of one KV head's values
    int vrows;     // rows of a value block's unit: 2, or 8
};

// Queries and keys: a wave has four consecutive rows, 16 lanes each with 8 or 4 elements of a head (the
// pair (i, i + HD/2) of the rotation is 8 lanes away), and takes `heads` heads one after the other, the next
// one's elements on their way; a row's place and rotation are looked up once.
template <int HD, int ST, int AT, bool Q4> X100_DEV void append_qk(const AppendArgs &a)
{
    constexpr int E = HD / 16;
    const int lane = threadIdx.x & 63, w = wave_id(), l = lane & 15, sub = lane >> 4;
    const int n_h = a.c.n_head, n_kv = a.c.n_head_kv, page = a.c.page;
    const int rbase = blockIdx.x % a.xq * 16 + 4 * w;
    int head = blockIdx.x / a.xq * a.heads;
    const int end = min(head + a.heads, n_h + n_kv);
    if (!a.q_out) head = max(head, n_h);   // keys only
    if (head >= end || rbase >= a.b.n_rows) return;
    const int row = min(rbase + sub, a.b.n_rows - 1);
    // What a head needs goes out one head ahead, without a branch around it: behind a branch, or with the column scales
    // loaded at their use, the wait for them was one for the next head's elements (62 us, so 57).
    RowBits<ST, E> raw;
    float cl[E];   // column scales
    auto fetch = [&](int hd) __attribute__((always_inline)) {
        const x100_rows &src = hd < n_h ? a.r.q : a.r.k;
        const int col = (hd < n_h ? hd : hd - n_h) * HD + E * l;
        if constexpr (ST == X100_T_I32)
#pragma unroll
            for (int e = 0; e < E; e++) cl[e] = src.col_scale[col + e];
        raw.load(src.p, (size_t)row * src.ld + col);
    };
    fetch(head);
    const RowPlace at = row_place(a.b, rbase, sub);
    float2 cs[E];
    if (a.r.rope) {
        const float2 *t = (const float2 *)a.r.rope + (size_t)max(at.pos, 0) * (HD / 2) + E * (l & 7);
#pragma unroll
        for (int e = 0; e < E; e++) {
            cs[e] = t[e];
            if (l < 8) cs[e].y = -cs[e].y;
        }
    }
    const int pg = at.mine && at.pos >= 0 ? paged_page(a.c, a.b, at.s, at.pos) : -1;
    const int off = at.pos & (page - 1);
    // norm weights and the row's scale, of queries or keys
    float nw[E], rs = 1.0f;
    auto weights = [&](const x100_rows &src, const float *w) __attribute__((always_inline)) {
        if constexpr (ST == X100_T_I32) rs = src.row_scale[row];
        if (w)
#pragma unroll
            for (int e = 0; e < E; e++) nw[e] = w[E * l + e];
    };
    // the head's values, normalised and rotated; the next head's on their way
    auto values = [&](float (&v)[E], bool norm) __attribute__((always_inline)) {
        raw.values(v);
        if constexpr (ST == X100_T_I32)
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = v[e] * rs * cl[e];
        fetch(min(head + 1, end - 1));
        // The formula's own products and sums, each rounded, the squares added by fours and then as a tree over
        // neighbours: a 4-bit code of a key that lies between two steps is then the one that a tensor library's fp32
        // gets.  Weights and rotation multiplied beforehand, a fused sum and an estimated root were no faster and turned
        // some codes of 10^5 groups.
        if (norm) {
            float sq[E];
#pragma unroll
            for (int e = 0; e < E; e++) sq[e] = v[e] * v[e];
#pragma unroll
            for (int e = 0; e < E; e += 4) sq[e] = ((sq[e] + sq[e + 1]) + sq[e + 2]) + sq[e + 3];
            if constexpr (E == 8) sq[0] += sq[4];
            const float sc = 1.0f / sqrtf(sum16(sq[0]) / (float)HD + a.r.eps);
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = v[e] * sc * nw[e];
        }
        if (a.r.rope) {
#pragma unroll
            for (int e = 0; e < E; e++) {
                const float o = dpp_f<0x128>(0.0f, v[e]);   // the pair's other element
                v[e] = v[e] * cs[e].x + o * cs[e].y;
            }
        }
    };
    if (head < min(end, n_h)) weights(a.r.q, a.r.q_norm);
    for (; head < min(end, n_h); head++) {
        float v[E];
        values(v, a.r.q_norm);
        if (at.pos < 0) {   // a row before position 0: zeros
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = 0.0f;
        }
        if (at.mine) {
            uint32_t u[E / 2];
#pragma unroll
            for (int e = 0; e < E / 2; e++) u[e] = f2act<AT>(v[2 * e]) | f2act<AT>(v[2 * e + 1]) << 16;
            uint16_t *o = a.q_out + ((size_t)row * n_h + head) * HD + E * l;
            if constexpr (E == 8) *(v4u *)o = v4u{u[0], u[1], u[2], u[3]};
            else *(v2u *)o = v2u{u[0], u[1]};
        }
    }
    if (head < end) weights(a.r.k, a.r.k_norm);
    for (; head < end; head++) {
        float v[E];
        values(v, a.r.k_norm);
        uint8_t *base = a.kp + ((size_t)max(pg, 0) * n_kv + head - n_h) * page_head_bytes<HD, Q4>(page);
        if constexpr (!Q4) {
            if (pg >= 0) {
                uint32_t u[E / 2];
#pragma unroll
                for (int e = 0; e < E / 2; e++) u[e] = f2act<AT>(v[2 * e]) | f2act<AT>(v[2 * e + 1]) << 16;
                uint16_t *o = (uint16_t *)base + (size_t)off * HD + E * l;
                if constexpr (E == 8) *(v4u *)o = v4u{u[0], u[1], u[2], u[3]};
                else *(v2u *)o = v2u{u[0], u[1]};
            }
        } else {
            float lo = v[0], hi = v[0], fin = 1.0f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                lo = fminf(lo, v[e]);
                hi = fmaxf(hi, v[e]);
                if (!(fabsf(v[e]) <= 3.402823466e38f)) fin = 0.0f;
            }
            const Q4Scale sc = q4_scale(gmin<HD>(lo), -gmin<HD>(-hi), gmin<HD>(fin) == 0.0f);
            uint32_t word = 0;
#pragma unroll
            for (int e = 0; e < E; e++) word |= q4_code(sc, v[e]) << q4_shift(e);
            uint32_t *cw = (uint32_t *)base + (size_t)off * (HD / 8);
            if constexpr (E == 4) {   // two lanes of 4 elements share a word: elements 4 .. 7 sit 8 bits higher
                if (l & 1) word <<= 8;
                word |= (uint32_t)dpp_i<0xB1>(0, (int)word);
            }
            if (pg >= 0) {
                if (E == 8) cw[l] = word;
                else if (!(l & 1)) cw[l >> 1] = word;
                constexpr int LG = 32 / E;   // lanes of a group
                if (l % LG == 0)
                    ((uint32_t *)(base + page * HD / 2))[(size_t)off * (HD / 32) + l / LG] = sc.d | (uint32_t)sc.m << 16;
            }
        }
    }
}

// Values: HD / 64 waves per unit of `vrows` rows, a thread per element of the head.  The rows of one sequence in
// one block of 8 positions are stored together (a 16-byte store of 8 positions, or the word that holds their
// codes), by the unit that holds the first of them.
template <int HD, int ST, int AT, bool Q4> X100_DEV void append_v(const AppendArgs &a)
{
    constexpr int WH = HD / 64;
    const int lane = threadIdx.x & 63, w = wave_id(), n_kv = a.c.n_head_kv, page = a.c.page;
    const int bv = blockIdx.x - a.nq, kvh = bv / a.xv, el = (w % WH) * 64 + lane;
    const x100_rows &src = a.r.v;
    const int col = kvh * HD + el;
    const int first = (bv % a.xv * (4 / WH) + w / WH) * a.vrows, last = min(first + a.vrows, a.b.n_rows);
    paged_blocks(
        first, last, a.b.n_seq, [&](int row) __attribute__((always_inline)) { return paged_find(a.b, row); },
        [&](int s) __attribute__((always_inline)) { return paged_seq(a.b, s); },
        [&](int s, int row, int pos, int n) __attribute__((always_inline)) {
            const int o0 = pos & 7, pg = paged_page(a.c, a.b, s, pos), blk = (pos & (page - 1)) >> 3;
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; k++) v[k] = row_elem<ST>(src.p, (size_t)(row + min(k, n - 1)) * src.ld + col);
            if constexpr (ST == X100_T_I32) {
                const float cl = src.col_scale[col];
#pragma unroll
                for (int k = 0; k < 8; k++) v[k] = v[k] * src.row_scale[row + min(k, n - 1)] * cl;
            }
            if (pg < 0) return;
            uint8_t *base = a.vp + ((size_t)pg * n_kv + kvh) * page_head_bytes<HD, Q4>(page);
            if constexpr (!Q4) {
                uint16_t *o = (uint16_t *)base + ((size_t)blk * HD + el) * 8;
                if (n == 8) {
                    uint32_t u[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) u[k] = f2act<AT>(v[2 * k]) | f2act<AT>(v[2 * k + 1]) << 16;
                    *(v4u *)o = v4u{u[0], u[1], u[2], u[3]};
                } else {
#pragma unroll
                    for (int k = 0; k < 8; k++)
                        if (k < n) o[o0 + k] = (uint16_t)f2act<AT>(v[k]);
                }
            } else {
                uint32_t *cw = (uint32_t *)base + (size_t)blk * HD + el;
                uint16_t *sc16 = (uint16_t *)(base + page * HD / 2) + ((size_t)blk * (HD / 32) + el / 32) * 16;
                float z = 0.0f;   // NaN where a value is not finite
#pragma unroll
                for (int k = 0; k < 8; k++) z = __builtin_fmaf(v[k], 0.0f, z);
                if (n == 8 && !__any(z != 0.0f)) {
                    // A whole block: each scale is worked out by one lane of four (position by position, below, 1100
                    // instructions instead of 230).
                    float lo[2], hi[2];
                    gmin8<1>(v, lo);
                    gmin8<-1>(v, hi);
                    Q4Scale sc[2];
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        sc[i] = q4_scale(lo[i], -hi[i], false);
                        if ((lane & 28) == 0) {
                            sc16[4 * i + (lane & 3)] = sc[i].d;
                            sc16[8 + 4 * i + (lane & 3)] = sc[i].m;
                        }
                        if (sc[i].bad) sc[i].mf = 0.0f;   // codes 0
                    }
                    uint32_t word = 0;
                    auto code = [&](int e, float mf, float inv) __attribute__((always_inline)) {
                        const float n = __builtin_amdgcn_fmed3f(rintf((v[e] - mf) * inv), 0.0f, 15.0f);
                        word |= (uint32_t)n << q4_shift(e);
                    };
                    code(0, quad<0>(sc[0].mf), quad<0>(sc[0].inv));
                    code(1, quad<1>(sc[0].mf), quad<1>(sc[0].inv));
                    code(2, quad<2>(sc[0].mf), quad<2>(sc[0].inv));
                    code(3, quad<3>(sc[0].mf), quad<3>(sc[0].inv));
                    code(4, quad<0>(sc[1].mf), quad<0>(sc[1].inv));
                    code(5, quad<1>(sc[1].mf), quad<1>(sc[1].inv));
                    code(6, quad<2>(sc[1].mf), quad<2>(sc[1].inv));
                    code(7, quad<3>(sc[1].mf), quad<3>(sc[1].inv));
                    *cw = word;
                    return;
                }
                uint32_t word = n == 8 ? 0u : *cw;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    if (k >= n) break;
                    float lo = gmin<64>(v[k]), hi = -gmin<64>(-v[k]);
                    float fin = gmin<64>(fabsf(v[k]) <= 3.402823466e38f ? 1.0f : 0.0f);
                    lo = fminf(lo, dpp_f<0x128>(lo, lo));
                    hi = fmaxf(hi, dpp_f<0x128>(hi, hi));
                    fin = fminf(fin, dpp_f<0x128>(fin, fin));
                    lo = fminf(lo, xor16_f(lo));
                    hi = fmaxf(hi, xor16_f(hi));
                    fin = fminf(fin, xor16_f(fin));
                    const Q4Scale sc = q4_scale(lo, hi, fin == 0.0f);
                    const int e = o0 + k, sh = 16 * (e & 1) + 4 * (e >> 1);
                    word = (word & ~(15u << sh)) | q4_code(sc, v[k]) << sh;
                    if ((lane & 31) == 0) {
                        sc16[e] = sc.d;
                        sc16[8 + e] = sc.m;
                    }
                }
                *cw = word;
            }
        });
}

template <int HD, int ST, int AT, bool Q4> __global__ __launch_bounds__(256) void k_append(const AppendArgs a)
{
    if ((int)blockIdx.x < a.nq) append_qk<HD, ST, AT, Q4>(a);
    else append_v<HD, ST, AT, Q4>(a);
}

// ---- cached rows back out ------------------------------------------------------------------------
struct ReadArgs {
    x100_kv_cfg c;
    x100_kv_batch b;
    const uint8_t *kp, *vp;
    uint16_t *k_out, *v_out;
};

// 16 lanes per (row, KV head), HD / 16 elements each.
template <int HD, int AT, bool Q4> __global__ __launch_bounds__(256) void k_read(const ReadArgs a)
{
    constexpr int E = HD / 16;
    const int lane = threadIdx.x & 63, w = wave_id(), l = lane & 15, sub = lane >> 4;
    const int kvh = blockIdx.y, n_kv = a.c.n_head_kv, page = a.c.page;
    const int rbase = blockIdx.x * 16 + 4 * w;
    if (rbase >= a.b.n_rows) return;
    const RowPlace place = row_place(a.b, rbase, sub);
    if (!place.mine) return;
    const int pos = place.pos, pg = pos >= 0 ? paged_page(a.c, a.b, place.s, pos) : -1;
    const int row = rbase + sub, off = pos & (page - 1);
    uint32_t k[E], v[E];   // act_type bits
#pragma unroll
    for (int e = 0; e < E; e++) k[e] = v[e] = 0;
    if (pg >= 0) {
        const size_t at = ((size_t)pg * n_kv + kvh) * page_head_bytes<HD, Q4>(page);
        if constexpr (!Q4) {
            const uint16_t *kr = (const uint16_t *)(a.kp + at) + (size_t)off * HD + E * l;
            const uint16_t *vr = (const uint16_t *)(a.vp + at) + ((size_t)(off >> 3) * HD + E * l) * 8 + (off & 7);
#pragma unroll
            for (int e = 0; e < E; e++) {
                k[e] = kr[e];
                v[e] = vr[8 * e];
            }
        } else {
            const int g = E * l / 32;
            const uint32_t kw = ((const uint32_t *)(a.kp + at))[(size_t)off * (HD / 8) + E * l / 8];
            const uint32_t ks = ((const uint32_t *)(a.kp + at + page * HD / 2))[(size_t)off * (HD / 32) + g];
            const uint32_t *vw = (const uint32_t *)(a.vp + at) + (size_t)(off >> 3) * HD + E * l;
            const uint16_t *vs = (const uint16_t *)(a.vp + at + page * HD / 2) + ((size_t)(off >> 3) * (HD / 32) + g) * 16;
            const _Float16 kd = __builtin_bit_cast(_Float16, (uint16_t)ks), km = __builtin_bit_cast(_Float16, (uint16_t)(ks >> 16));
            const _Float16 vd = __builtin_bit_cast(_Float16, vs[off & 7]), vm = __builtin_bit_cast(_Float16, vs[8 + (off & 7)]);
            const int vsh = 16 * (off & 1) + 4 * ((off & 7) >> 1);
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int ke = E == 8 ? e : (l & 1) * 4 + e;
                const _Float16 nk = (_Float16)(int)((kw >> (16 * (ke & 1) + 4 * (ke >> 1))) & 15);
                const _Float16 nv = (_Float16)(int)((vw[e] >> vsh) & 15);
                k[e] = f2act<AT>((float)__builtin_fmaf16(nk, kd, km));
                v[e] = f2act<AT>((float)__builtin_fmaf16(nv, vd, vm));
            }
        }
    }
    const size_t o = ((size_t)row * n_kv + kvh) * HD + E * l;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        *(uint32_t *)(a.k_out + o + e) = k[e] | k[e + 1] << 16;
        *(uint32_t *)(a.v_out + o + e) = v[e] | v[e + 1] << 16;
    }
}

template <int HD, int ST> hipError_t append_as(AppendArgs a, hipStream_t s)
{
    // Heads per wave: as many as leave 2048 waves, so that few rows are spread over the chip and many look their places
    // up once for several heads, but 12 at most, which leaves more loads on their way (us for 512 tokens / 6400 rows
    // of 36 heads, int32 to 4 bits and read back: one head 11.5 / -, 4096 waves 11.5 / 56, 2048 9.4 / 58-62, with the
    // bound 9.4 / 56; a bound of 9 or 18: 62).
    // Values: a unit of 8 rows holds whole blocks of prompts; of single tokens each row is looked up and stored by
    // itself, and shorter units do that beside each other (512 tokens 17.6 us in eights, 14.9 in twos, 14.8 alone;
    // 2048 rows of a prompt 13.0 / 13.2 / 16.2).
    const int n_rows = a.b.n_rows, all = a.c.n_head + a.c.n_head_kv, quads = (n_rows + 3) / 4;
    const int most = std::max(1, (int)std::min<int64_t>(std::min(all, 12), (int64_t)quads * all / 2048)), groups = (all + most - 1) / most;
    a.heads = (all + groups - 1) / groups;
    a.xq = (n_rows + 15) / 16;
    a.nq = a.xq * ((all + a.heads - 1) / a.heads);
    a.vrows = n_rows < 4 * (int64_t)a.b.n_seq ? 2 : 8;
    const int per = 4 / (HD / 64) * a.vrows;   // rows of a value block
    a.xv = (n_rows + per - 1) / per;
    const int64_t blocks = (int64_t)a.nq + (int64_t)a.xv * a.c.n_head_kv;
    if (blocks >= 1 << 24) return hipErrorInvalidValue;   // past one launch
    const unsigned grid = (unsigned)blocks;
    const bool q4 = a.c.kv_type == X100_KV_Q4;
    if (a.c.act_type == X100_T_F16) {
        if (q4) k_append<HD, ST, X100_T_F16, true><<<grid, 256, 0, s>>>(a);
        else k_append<HD, ST, X100_T_F16, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (q4) k_append<HD, ST, X100_T_BF16, true><<<grid, 256, 0, s>>>(a);
        else k_append<HD, ST, X100_T_BF16, false><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}
template <int HD> hipError_t append_from(const AppendArgs &a, hipStream_t s)
{
    switch (a.r.k.type) {
    case X100_T_F32: return append_as<HD, X100_T_F32>(a, s);
    case X100_T_F16: return append_as<HD, X100_T_F16>(a, s);
    case X100_T_BF16: return append_as<HD, X100_T_BF16>(a, s);
    case X100_T_I32: return append_as<HD, X100_T_I32>(a, s);
    }
    return hipErrorInvalidValue;
}
template <int HD> hipError_t read_as(const ReadArgs &a, hipStream_t s)
{
    const dim3 grid((a.b.n_rows + 15) / 16, a.c.n_head_kv);
    const bool q4 = a.c.kv_type == X100_KV_Q4;
    if (a.c.act_type == X100_T_F16) {
        if (q4) k_read<HD, X100_T_F16, true><<<grid, 256, 0, s>>>(a);
        else k_read<HD, X100_T_F16, false><<<grid, 256, 0, s>>>(a);
    } else {
        if (q4) k_read<HD, X100_T_BF16, true><<<grid, 256, 0, s>>>(a);
        else k_read<HD, X100_T_BF16, false><<<grid, 256, 0, s>>>(a);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t x100_rope_table_launch(int head_dim, int n_pos, float base, float *table, hipStream_t s)
{
    const size_t n = (size_t)n_pos * (head_dim / 2);
    k_rope_table<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(head_dim / 2, n_pos, (double)base, (float2 *)table);
    return hipGetLastError();
}

hipError_t x100_kv_append_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const x100_kv_rows &r, void *kp,
                                 void *vp, void *q_out, hipStream_t s)
{
    const AppendArgs a = {c, b, r, (uint8_t *)kp, (uint8_t *)vp, (uint16_t *)q_out, 0, 0, 0, 0, 0};
    return c.head_dim == 64 ? append_from<64>(a, s) : append_from<128>(a, s);
}

hipError_t x100_kv_read_launch(const x100_kv_cfg &c, const x100_kv_batch &b, const void *kp, const void *vp,
                               void *k_out, void *v_out, hipStream_t s)
{
    const ReadArgs a = {c, b, (const uint8_t *)kp, (const uint8_t *)vp, (uint16_t *)k_out, (uint16_t *)v_out};
    return c.head_dim == 64 ? read_as<64>(a, s) : read_as<128>(a, s);
}
