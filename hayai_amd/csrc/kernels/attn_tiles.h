// What the attention kernels share: 16-byte operands of the matrix cores, weights of a softmax that is
// summed while its largest score may still rise, and pages as sources of operands.
//
// Scores are computed turned, S^T = K Q^T: a lane then holds one query's scores of several keys, and
// the second product O^T = V^T P^T takes its weights from that very lane.  The rows of K may stand in any
// order, so they are given the one in which a lane's scores are of the EF neighbouring keys that its
// 16-byte operand of V^T holds (EF elements of the cache's type): no value moves between lanes but a
// query's largest score.
#ifndef HH_KERNELS_ATTN_TILES_H
#define HH_KERNELS_ATTN_TILES_H

#include "kv_pages.h"
#include "wave64.h"

typedef float hh_f32x4 __attribute__((ext_vector_type(4)));
typedef float hh_f32x16 __attribute__((ext_vector_type(16)));

// Operands and products.  frag: EF elements of the summed axis; products sum over 2 EF (32 rows and columns)
// or 4 EF (16), lane l's being the (l / 32)th or (l / 16)th EF of them.
template <class C>
struct hh_mat;
template <>
struct hh_mat<hh_af16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    HH_DEV static hh_f32x16 mul32(frag a, frag b, hh_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
    HH_DEV static hh_f32x4 mul16(frag a, frag b, hh_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct hh_mat<hh_abf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    HH_DEV static hh_f32x16 mul32(frag a, frag b, hh_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    HH_DEV static hh_f32x4 mul16(frag a, frag b, hh_f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct hh_mat<hh_af32> {
    typedef hh_f32x4 frag;
    HH_DEV static hh_f32x16 mul32(frag a, frag b, hh_f32x16 c) {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    HH_DEV static hh_f32x4 mul16(frag a, frag b, hh_f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// EF elements of a query at element d, rounded to the cache's type (a no-op but for f32 queries over a 16-bit
// cache, whose products are 16-bit operands with f32 sums), zeros from dim on.
template <class A, class C, bool FULL>
HH_DEV typename hh_mat<C>::frag hh_query(const typename A::E* q, uint32_t d, uint32_t dim, bool ok) {
    constexpr int EF = C::VEC;
    typename hh_mat<C>::frag f;
    typename A::E e[EF];
    const bool in = ok && (FULL || d < dim);  // (dim is a multiple of 8)
    hh_load_n(q + (in ? d : 0), e);
#pragma unroll
    for (int i = 0; i < EF; i++) f[i] = in ? C::put(A::get(e[i])) : C::put(0.f);
    return f;
}

// The frag's first n elements, zeros for the others.
template <class C>
HH_DEV typename hh_mat<C>::frag hh_first(typename hh_mat<C>::frag f, int n) {
    constexpr int PER = 4 / sizeof(typename C::E);
    hh_u4 u = __builtin_bit_cast(hh_u4, f);
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = n >= (i + 1) * PER ? u[i] : PER == 2 && n == 2 * i + 1 ? u[i] & 0xffffu : 0u;
    return __builtin_bit_cast(typename hh_mat<C>::frag, u);
}
// The frag with zeros for its infinities and NaNs (exponents of ones: one more carries into the sign's place);
// odd gets bits where there are any.
template <class C>
HH_DEV typename hh_mat<C>::frag hh_finite(typename hh_mat<C>::frag f, uint32_t& odd) {
    hh_u4 u = __builtin_bit_cast(hh_u4, f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t bad;
        if (sizeof(typename C::E) == 4) {
            bad = (uint32_t)((int)((u[i] & 0x7f800000u) + 0x00800000u) >> 31);
        } else {
            const bool half = __is_same(C, hh_af16);
            bad = ((u[i] & (half ? 0x7c007c00u : 0x7f807f80u)) + (half ? 0x04000400u : 0x00800080u)) >> 15 & 0x00010001u;
            bad = (bad << 16) - bad;
        }
        odd |= bad;
        u[i] &= ~bad;
    }
    return __builtin_bit_cast(typename hh_mat<C>::frag, u);
}

// Scores are in units of log2: weight = exp2(score * c - base), c = scale * log2(e).  base follows the
// largest score, but only once it falls more than HH_ATTN_SLACK behind: weights of up to 2^8 are as good as
// those of up to 1, and sums need no rescaling meanwhile.  In f16 it stays 2^7 below, so that weights are up to 2^15 and
// what is lost under f16's smallest number is 2^-32 of the largest: at 2^-25 of it the many small weights of a long context
// would be lost together.  It starts at the lowest f32, where exp2(-inf - base) is 0 as well.
#define HH_ATTN_SLACK 8.f
#define HH_ATTN_LOWEST (-3.402823466e38f)
template <class C>
HH_DEV constexpr float hh_attn_lift() {
    return __is_same(C, hh_af16) ? 7.f : 0.f;
}
HH_DEV float hh_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// A 16-byte source for what a page number outside the cache stands for: zeros.
__device__ const hh_u4 hh_kv_zeros = {0, 0, 0, 0};

// Workgroups of four waves that registers are made for: two a CU where a tile fits half its LDS and half its
// registers.
#define HH_ATTN_PER_CU(C, D) ((D) == 256 || (sizeof(C::E) == 4 && (D) == 128) ? 1 : 2)

template <class Op>
HH_DEV uint32_t hh_wave32(uint32_t v) {
    v = Op::of(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));
    v = Op::of(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));
    v = Op::of(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x124, 0xf, 0xf, true));
    v = Op::of(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x128, 0xf, 0xf, true));
    v = Op::of(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xa, 0xf, true));
    v = Op::of(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xc, 0xf, true));
    return __builtin_amdgcn_readlane(v, 63);
}
struct hh_add32 {
    HH_DEV static uint32_t of(uint32_t a, uint32_t b) { return a + b; }
};
struct hh_max32 {
    HH_DEV static uint32_t of(uint32_t a, uint32_t b) { return a > b ? a : b; }
};
HH_DEV uint32_t hh_wave_sum32(uint32_t v) { return hh_wave32<hh_add32>(v); }
HH_DEV uint32_t hh_wave_max32(uint32_t v) { return hh_wave32<hh_max32>(v); }

// A kernel for each width of heads: whole 64, 128 and 256 elements, and those within 64, 96, 128 and 256.
#define HH_ATTN_DIMS(KERNEL, N, A, C)                                                                          \
    KERNEL(N, A, C, 64, 0, 64) KERNEL(N, A, C, 64, 64, 64_any) KERNEL(N, A, C, 128, 96, 96_any) KERNEL(N, A, C, 128, 0, 128) \
    KERNEL(N, A, C, 128, 128, 128_any) KERNEL(N, A, C, 256, 0, 256) KERNEL(N, A, C, 256, 256, 256_any)

constexpr int hh_attn_wait(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | 0x70 | (lgkm << 8); }
// This wave's copies into LDS landed and its LDS reads done, then the workgroup meets.
HH_DEV void hh_attn_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(hh_attn_wait(0, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
template <int ID, int BYTES>
HH_DEV uint8_t* hh_attn_lds() {
    __shared__ __attribute__((aligned(128))) uint8_t buf[BYTES];
    return buf;
}
HH_DEV void hh_copy16(const uint8_t* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// The entry of sequence s's table that token t is in, as an unsigned page number (negative ones pass any cache).
HH_DEV uint32_t hh_page(const int32_t* table, uint32_t t, uint32_t shift, uint32_t entries) {
    return (uint32_t)table[min(t >> shift, entries - 1)];
}

#endif
