// What the kernels of attention over the paged cache share (attn_paged.hip, attn_prompt.hip).
#pragma once
#include "paged.h"

constexpr float X100_NEG_INF = -__builtin_inff();

// Weights are powers of two relative to m, the running maximum less a lift.  fp16 has no numbers below 2^-24: without
// the lift the weights of a long tail, each below 2^-25 of the largest one, were all zero (60000 positions at 2^-25
// beside a peak: 0.18% of the sum).  What is lifted is lost above: m lags by up to 2^8 in the tile kernel, and in the
// prompt kernel until 16 weights sum to prompt_most, where following it stops all waves of a block.
template <int MT> constexpr float tile_lift() { return MT == X100_T_F16 ? 7.0f : 0.0f; }
template <int MT> constexpr float prompt_lift() { return MT == X100_T_F16 ? 4.0f : 0.0f; }
template <int MT> constexpr float prompt_most() { return MT == X100_T_F16 ? 60000.0f : 16384.0f; }

// How a kernel splits the positions: a sequence's in n equal parts, so that the blocks of a batch of unequal
// sequences are as equal as its lengths let them be; a multiple of 128, `least` or more.
struct PagedSplit {
    int n, least;
    X100_DEV int positions(int kv_len) const { return max(least, ((kv_len + n - 1) / n + 127) & ~127); }
};

struct PagedAttnArgs {
    x100_kv_cfg c;
    x100_kv_batch b;
    const uint16_t *q;
    int64_t ldq;
    const uint8_t *kp, *vp;
    float scale2;        // scale * log2(e): weights are powers of two
    uint16_t *out;
    int64_t ldo;
    float *part_o;       // split results: O, HD floats each, not divided by l,
    float2 *part_ml;     // and (m, l)
    int few;             // sequences of up to this many rows (token, head) are the tile kernel's, the rest the prompt kernel's
    PagedSplit tile, prompt;
    size_t tile_at;      // the tile kernel's first split result
    int tile_rows, tiles;   // rows of a sequence there, and their tiles
    int run;             // units of a run of blocks there
    const int *sel;      // sparse: lists of blocks [row][KV head][n_sel]
    int n_sel;
};

template <int T> struct Mfma16;
template <> struct Mfma16<X100_T_F16> {
    static X100_DEV v4f mul(v4u a, v4u b, v4f c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    }
};
template <> struct Mfma16<X100_T_BF16> {
    static X100_DEV v4f mul(v4u a, v4u b, v4f c)
    {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
    }
};

// The row's power of two 2^-e that brings its largest element (in size) to 1 .. 2: bf16 queries become fp16 that way
// whatever their size.  Exact for elements down to 2^-17 of the largest; below, fp16's numbers are multiples of 2^-24,
// so that an element is off by 2^-25 of the largest at most, far less than a rounding of the largest to bf16.
X100_DEV int row_exponent(float amax)
{
    const int e = (int)(__float_as_uint(amax) >> 23) - 127;
    return amax > 0.0f && e < 128 ? e : 0;
}

typedef float v16f __attribute__((ext_vector_type(16)));

template <int T> X100_DEV v16f mfma32(v4u a, v4u b, v16f c)
{
    if constexpr (T == X100_T_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}
// c + the two 16-bit numbers of w
template <int T> X100_DEV float add2(uint32_t w, float c)
{
    if constexpr (T == X100_T_F16)
        return __builtin_amdgcn_fdot2(as_h2(w), v2h{(_Float16)1.0f, (_Float16)1.0f}, c, false);
    else {
        const uint32_t one = 0x3f803f80u;
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, w), __builtin_bit_cast(v2b, one), c, false);
    }
}

// Number of row i's (token, head) first split result: by rows of the batch (q0: the sequence's first), and by
// sequences.
X100_DEV size_t prompt_part(const PagedAttnArgs &a, int q0, int kvh, int i)
{
    const int G = a.c.n_head / a.c.n_head_kv;
    return (((size_t)q0 * G + i) * a.c.n_head_kv + kvh) * a.prompt.n;
}
X100_DEV size_t tile_part(const PagedAttnArgs &a, int s, int kvh, int i)
{
    return a.tile_at + (((size_t)s * a.tile_rows + i) * a.c.n_head_kv + kvh) * a.tile.n;
}

// The same of a row with a list (sparse): by rows.
X100_DEV size_t sparse_part(const PagedAttnArgs &a, int row, int kvh, int i)
{
    const int G = a.c.n_head / a.c.n_head_kv;
    return (((size_t)row * G + i) * a.c.n_head_kv + kvh) * a.tile.n;
}

constexpr int PROMPT_ROWS = 256;      // rows (token, head) of a block of the prompt kernel
constexpr int PROMPT_PAGES = 8192;    // most pages of a split there (their list is in LDS)
int64_t x100_attn_prompt_blocks(const x100_kv_cfg &c, const x100_kv_batch &b, int splits);
hipError_t x100_attn_prompt_launch(const PagedAttnArgs &a, hipStream_t s);
