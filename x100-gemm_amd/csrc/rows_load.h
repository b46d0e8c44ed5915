// Rows of the four element types of x100_rows.h as fp32 values, shared by rows.hip and paged.hip.
#pragma once
#include "x100_common.h"
#include "x100_rows.h"

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));

// by value: __builtin_bit_cast of a vector's element reads element 0
X100_DEV v2h as_h2(uint32_t u) { return __builtin_bit_cast(v2h, u); }
X100_DEV float bf2f(uint32_t b) { return __uint_as_float(b << 16); }
// fp32 -> fp16, nearest even, of the fp32 number: with a product or a sum in front the compiler would take an
// instruction that rounds once, from more than fp32 (a group of 4-bit codes in 30000 got another scale).
X100_DEV _Float16 f2h_rne(float f)
{
    asm("" : "+v"(f));
    return (_Float16)f;
}
// fp32 -> 16 bits, nearest even (NaN stays NaN)
template <int T> X100_DEV uint32_t f2act(float f)
{
    if constexpr (T == X100_T_F16) return __builtin_bit_cast(uint16_t, f2h_rne(f));
    return __builtin_bit_cast(uint16_t, (__bf16)f);
}
template <int T> X100_DEV float act2f(uint32_t b)
{
    if constexpr (T == X100_T_F16) return h2f((uint16_t)b);
    return bf2f(b);
}
template <int T> constexpr int row_elem_bytes() { return T == X100_T_F32 || T == X100_T_I32 ? 4 : 2; }

// One element of a row as it is stored, as a float (X100_T_I32: unscaled).
template <int T> X100_DEV float row_elem(const void *p, size_t i)
{
    if constexpr (T == X100_T_F32) return ((const float *)p)[i];
    if constexpr (T == X100_T_I32) return (float)((const int32_t *)p)[i];
    return act2f<T>(((const uint16_t *)p)[i]);
}
// N consecutive elements (4 or 8) from an address aligned to min(16, N * element) bytes: as they are stored (a load
// that can stay on its way), and as floats.
template <int T, int N> struct RowBits {
    static constexpr int W = N * row_elem_bytes<T>() / 4;
    uint32_t w[W];
    X100_DEV void load(const void *p, size_t i)
    {
        const uint8_t *at = (const uint8_t *)p + i * row_elem_bytes<T>();
        if constexpr (W == 2) {
            const v2u u = *(const v2u *)at;
            w[0] = u[0];
            w[1] = u[1];
        } else {
#pragma unroll
            for (int k = 0; k < W / 4; k++) {
                const v4u u = *(const v4u *)(at + 16 * k);
#pragma unroll
                for (int e = 0; e < 4; e++) w[4 * k + e] = u[e];
            }
        }
    }
    X100_DEV void values(float (&v)[N]) const
    {
#pragma unroll
        for (int e = 0; e < W; e++) {
            if constexpr (T == X100_T_F32) v[e] = __uint_as_float(w[e]);
            else if constexpr (T == X100_T_I32) v[e] = (float)(int)w[e];
            else {
                v[2 * e] = act2f<T>(w[e] & 0xffffu);
                v[2 * e + 1] = T == X100_T_F16 ? h2f((uint16_t)(w[e] >> 16)) : __uint_as_float(w[e] & 0xffff0000u);
            }
        }
    }
};
template <int T, int N> X100_DEV void row_elems(const void *p, size_t i, float (&v)[N])
{
    RowBits<T, N> b;
    b.load(p, i);
    b.values(v);
}
