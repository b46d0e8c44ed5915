// int8 rows with one scale per row (x100_rows.h): the residual's addition with RMSNorm, and plain rows.
//
// t_i = h_i w_i (or x_i), amax = max |t_i|, code_i = rint(t_i 127 (1 / amax)).  The norm's factor
// r = 1/sqrt(mean h^2 + eps) multiplies every t_i alike and cancels in the code, so the maximum and the
// sum of squares come from the same single read of the row, and only the scale depends on the sum.
// Bound by HBM: every input is read once into registers, every output written once.  16381 rows of 2048, bf16 with
// an int32 delta: 59 us, 5.1 TB/s; 16384 rows of 4096, f16 without the norm: 39 us, 5.2 TB/s (a copy of 2 GiB: 5.0).
// 64 rows: 3.7 us, a launch and two trips to memory.
#include "rows_load.h"
#include "x100_internal.h"

namespace {

template <int CTRL, int ROWM = 0xf> X100_DEV double dpp_d(double v)
{
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = dpp_i<CTRL, ROWM>(0, (int)(uint32_t)u), hi = dpp_i<CTRL, ROWM>(0, (int)(uint32_t)(u >> 32));
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// sum over the wave, in its last lane
X100_DEV double wave_sum_last(double v)
{
    v += dpp_d<0x111>(v);
    v += dpp_d<0x112>(v);
    v += dpp_d<0x114>(v);
    v += dpp_d<0x118>(v);
    v += dpp_d<0x142, 0xa>(v);
    v += dpp_d<0x143, 0xc>(v);
    return v;
}
// mx / (127 sqrt(m)) for m > 0, in fp32: m is brought to 1 .. 4 first, the root's power of two goes into the result
X100_DEV float norm_scale(float mx, double m)
{
    const int e = ((int)(__builtin_bit_cast(uint64_t, m) >> 52) - 1023) & ~1;
    return ldexpf(mx * (1.0f / sqrtf((float)ldexp(m, -e))) / 127.0f, -e / 2);
}

struct RowArgs {
    int n_rows, d;
    x100_rows x, delta;
    const float *weight;
    float eps;
    void *h;
    int64_t ldh;
    int8_t *q;
    float *scale;
};

// NT threads of a block of max(NT, 256) take a row each time; thread t of a row has the chunks of 8
// elements t, t + NT, ...  (CH of them).  VEC: every chunk is whole and aligned; else element by
// element.  XT / DT: types of x and delta (DT < 0: none); NORM: with weight and the norm's factor.
template <int NT, int CH, bool VEC, int XT, int DT, bool NORM>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void k_rows_i8(const RowArgs a)
{
    constexpr int BT = NT < 256 ? 256 : NT, RPB = BT / NT, NW = NT / 64;
    __shared__ float s_mx[BT / 64];
    __shared__ double s_ss[BT / 64];
    const int t = threadIdx.x % NT, row = blockIdx.x * RPB + threadIdx.x / NT, w = threadIdx.x >> 6;
    const bool live = row < a.n_rows;
    const int d = a.d;
    float v[CH][8];
    // Squares are summed in fp64, where those of every fp32 number are normal: in fp32 they left its range at 1e18 and
    // below 1e-22 (a row of 1e-24 got the scale inf for eps = 0).
    double ss = 0.0;
    float mx = 0.0f;
    bool bad = false;
    if (live) {
        const float drs = DT == X100_T_I32 ? a.delta.row_scale[row] : 1.0f;
        const float xrs = XT == X100_T_I32 ? a.x.row_scale[row] : 1.0f;
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const int e0 = 8 * (t + NT * c);
            const size_t xo = (size_t)row * a.x.ld + e0;
            float dv[8];
            if constexpr (VEC) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[c][e] = 0.0f;
                if (e0 >= d) continue;
                row_elems<XT>(a.x.p, xo, v[c]);
                if constexpr (DT >= 0) row_elems<DT>(a.delta.p, (size_t)row * a.delta.ld + e0, dv);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    v[c][e] = e0 + e < d ? row_elem<XT>(a.x.p, xo + e) : 0.0f;
                    if constexpr (DT >= 0)
                        dv[e] = e0 + e < d ? row_elem<DT>(a.delta.p, (size_t)row * a.delta.ld + e0 + e) : 0.0f;
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (!VEC && e0 + e >= d) continue;
                if constexpr (XT == X100_T_I32) v[c][e] = v[c][e] * xrs * a.x.col_scale[e0 + e];
                if constexpr (DT >= 0) {
                    if constexpr (DT == X100_T_I32) dv[e] = dv[e] * drs * a.delta.col_scale[e0 + e];
                    v[c][e] += dv[e];
                    if constexpr (XT != X100_T_F32) v[c][e] = act2f<XT == X100_T_I32 ? X100_T_F16 : XT>(f2act<XT == X100_T_I32 ? X100_T_F16 : XT>(v[c][e]));
                }
            }
            if constexpr (DT >= 0) {   // h, in its type
                const size_t ho = (size_t)row * a.ldh + e0;
                if constexpr (VEC) {
                    if constexpr (XT == X100_T_F32) {
                        *(float4 *)((float *)a.h + ho) = make_float4(v[c][0], v[c][1], v[c][2], v[c][3]);
                        *(float4 *)((float *)a.h + ho + 4) = make_float4(v[c][4], v[c][5], v[c][6], v[c][7]);
                    } else {
                        v4u u;
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            u[e] = f2act<XT>(v[c][2 * e]) | f2act<XT>(v[c][2 * e + 1]) << 16;
                        *(v4u *)((uint16_t *)a.h + ho) = u;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (e0 + e < d) {
                            if constexpr (XT == X100_T_F32) ((float *)a.h)[ho + e] = v[c][e];
                            else ((uint16_t *)a.h)[ho + e] = (uint16_t)f2act<XT>(v[c][e]);
                        }
                }
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if constexpr (NORM) {
                    ss = __builtin_fma((double)v[c][e], (double)v[c][e], ss);
                    if (VEC || e0 + e < d) v[c][e] *= a.weight[e0 + e];
                }
                mx = fmaxf(mx, fabsf(v[c][e]));
                bad |= !(fabsf(v[c][e]) <= 3.402823466e38f);   // an infinity or a NaN
            }
        }
    }
    // over the row's threads; a value that is not finite makes mx an infinity
    if (bad) mx = __builtin_inff();
    mx = wave_max_u(mx);
    if constexpr (NORM) ss = wave_sum_last(ss);
    if constexpr (NW > 1) {
        if ((threadIdx.x & 63) == 63) {
            s_mx[w] = mx;
            s_ss[w] = ss;
        }
        __syncthreads();
        mx = s_mx[w / NW * NW];
        ss = s_ss[w / NW * NW];
#pragma unroll
        for (int i = 1; i < NW; i++) {
            mx = fmaxf(mx, s_mx[w / NW * NW + i]);
            ss += s_ss[w / NW * NW + i];
        }
    }
    if (!live) return;
    const bool fin = mx <= 3.402823466e38f, some = fin && mx >= 0x1p-100f;
    const float inv = some ? 127.0f * (1.0f / mx) : 0.0f;
    if (t == NT - 1) {   // NT = 64: the lane that has the sum
        float sc = fin ? 0.0f : __builtin_nanf("");
        if (some) sc = NORM ? norm_scale(mx, ss / d + (double)a.eps) : mx / 127.0f;
        a.scale[row] = sc;
    }
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const int e0 = 8 * (t + NT * c);
        if (e0 >= d) continue;
        uint32_t u[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int n = some ? (int)rintf(v[c][e] * inv) : 0;
            u[e >> 2] |= (uint32_t)(n & 255) << (8 * (e & 3));
        }
        int8_t *q = a.q + (size_t)row * d + e0;
        if constexpr (VEC) {
            *(v2u *)q = v2u{u[0], u[1]};
        } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (e0 + e < d) q[e] = (int8_t)(u[e >> 2] >> (8 * (e & 3)));
        }
    }
}

template <int NT, int CH, bool VEC, int XT, int DT, bool NORM> hipError_t launch(const RowArgs &a, hipStream_t s)
{
    constexpr int BT = NT < 256 ? 256 : NT, RPB = BT / NT;
    k_rows_i8<NT, CH, VEC, XT, DT, NORM><<<(a.n_rows + RPB - 1) / RPB, BT, 0, s>>>(a);
    return hipGetLastError();
}

// Threads and chunks per thread by the row's length: a wave up to 512 elements, 256 threads up to 4096 (one or
// two chunks), then 1024 threads: a row stays in 16 registers per thread.
template <bool VEC, int XT, int DT, bool NORM> hipError_t by_length(const RowArgs &a, hipStream_t s)
{
    if (a.d <= 512) return launch<64, 1, VEC, XT, DT, NORM>(a, s);
    if (a.d <= 2048) return launch<256, 1, VEC, XT, DT, NORM>(a, s);
    if (a.d <= 4096) return launch<256, 2, VEC, XT, DT, NORM>(a, s);
    return launch<1024, 2, VEC, XT, DT, NORM>(a, s);
}

bool rows_vec(const x100_rows &r)
{
    const int e = r.type == X100_T_F32 || r.type == X100_T_I32 ? 4 : 2;
    return !((uintptr_t)r.p & 15) && (r.ld * e) % 16 == 0;
}

template <int XT, int DT, bool NORM> hipError_t by_align(const RowArgs &a, hipStream_t s)
{
    bool vec = a.d % 8 == 0 && rows_vec(a.x) && !((uintptr_t)a.q & 7);
    if (DT >= 0)
        vec = vec && rows_vec(a.delta) && !((uintptr_t)a.h & 15) && (a.ldh * row_elem_bytes<XT>()) % 16 == 0;
    return vec ? by_length<true, XT, DT, NORM>(a, s) : by_length<false, XT, DT, NORM>(a, s);
}

template <int XT> hipError_t norm_by_delta(const RowArgs &a, hipStream_t s)
{
    if (!a.delta.p) return by_align<XT, -1, true>(a, s);
    switch (a.delta.type) {
    case X100_T_F32: return by_align<XT, X100_T_F32, true>(a, s);
    case X100_T_F16: return by_align<XT, X100_T_F16, true>(a, s);
    case X100_T_BF16: return by_align<XT, X100_T_BF16, true>(a, s);
    case X100_T_I32: return by_align<XT, X100_T_I32, true>(a, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t x100_quant_i8_launch(int n_rows, int d, const x100_rows *x, int8_t *q, float *scale, hipStream_t s)
{
    const RowArgs a = {n_rows, d, *x, {}, nullptr, 0.0f, nullptr, 0, q, scale};
    switch (x->type) {
    case X100_T_F32: return by_align<X100_T_F32, -1, false>(a, s);
    case X100_T_F16: return by_align<X100_T_F16, -1, false>(a, s);
    case X100_T_BF16: return by_align<X100_T_BF16, -1, false>(a, s);
    case X100_T_I32: return by_align<X100_T_I32, -1, false>(a, s);
    }
    return hipErrorInvalidValue;
}

hipError_t x100_add_rmsnorm_i8_launch(int n_rows, int d, const x100_rows *x, const x100_rows *delta,
                                      const float *weight, float eps, void *h, int64_t ldh, int8_t *q, float *scale,
                                      hipStream_t s)
{
    RowArgs a = {n_rows, d, *x, {}, weight, eps, h, ldh, q, scale};
    if (delta) a.delta = *delta;
    switch (x->type) {
    case X100_T_F32: return norm_by_delta<X100_T_F32>(a, s);
    case X100_T_F16: return norm_by_delta<X100_T_F16>(a, s);
    case X100_T_BF16: return norm_by_delta<X100_T_BF16>(a, s);
    }
    return hipErrorInvalidValue;
}
