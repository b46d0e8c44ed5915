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
// fp32 -> 16 bits, nearest even (NaN stays NaN)
template <int T> X100_DEV uint32_t f2act(float f)
{
    if constexpr (T == X100_T_F16) return __builtin_bit_cast(uint16_t, (_Float16)f);
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
// N consecutive elements (4 or 8) from an address aligned to min(16, N * element) bytes.
template <int T, int N> X100_DEV void row_elems(const void *p, size_t i, float (&v)[N])
{
    if constexpr (row_elem_bytes<T>() == 4) {
#pragma unroll
        for (int k = 0; k < N / 4; k++) {
            const v4u u = *(const v4u *)((const uint32_t *)p + i + 4 * k);
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 * k + e] = T == X100_T_F32 ? __uint_as_float(u[e]) : (float)(int)u[e];
        }
    } else {
        uint32_t u[N / 2];
        if constexpr (N == 8) {
            const v4u w = *(const v4u *)((const uint16_t *)p + i);
#pragma unroll
            for (int e = 0; e < 4; e++) u[e] = w[e];
        } else {
            const v2u w = *(const v2u *)((const uint16_t *)p + i);
            u[0] = w[0];
            u[1] = w[1];
        }
#pragma unroll
        for (int e = 0; e < N / 2; e++) {
            v[2 * e] = act2f<T>(u[e] & 0xffffu);
            v[2 * e + 1] = T == X100_T_F16 ? h2f((uint16_t)(u[e] >> 16)) : __uint_as_float(u[e] & 0xffff0000u);
        }
    }
}
