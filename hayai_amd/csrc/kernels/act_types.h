// Activation element types of the 8-bit operators (i8_rows.hip, i8_gemm.hip, sample.hip): f32, f16
// or bf16 in memory, f32 in registers.  Vectors are 16 bytes and need only their elements'
// alignment (gfx950 loads and stores unaligned dwords whole), so rows of any stride take them.
#ifndef HH_KERNELS_ACT_TYPES_H
#define HH_KERNELS_ACT_TYPES_H

#include "common.h"

struct hh_af32 {
    typedef float E;
    static constexpr int VEC = 4;
    HH_DEV static float get(E v) { return v; }
    HH_DEV static E put(float v) { return v; }
};
struct hh_af16 {
    typedef _Float16 E;
    static constexpr int VEC = 8;
    HH_DEV static float get(E v) { return (float)v; }
    HH_DEV static E put(float v) { return (E)v; }
};
struct hh_abf16 {
    typedef __bf16 E;
    static constexpr int VEC = 8;
    HH_DEV static float get(E v) { return (float)v; }
    HH_DEV static E put(float v) { return (E)v; }
};

// N elements at p, aligned as one element is.
template <class T, int N>
struct hh_unaligned {
    T v[N];
};
template <class T, int N>
HH_DEV void hh_load_n(const T* p, T (&v)[N]) {
    hh_unaligned<T, N> t;
    __builtin_memcpy(&t, p, sizeof t);
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = t.v[i];
}
template <class T, int N>
HH_DEV void hh_store_n(T* p, const T (&v)[N]) {
    hh_unaligned<T, N> t;
#pragma unroll
    for (int i = 0; i < N; i++) t.v[i] = v[i];
    __builtin_memcpy(p, &t, sizeof t);
}

#endif
