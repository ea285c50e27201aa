// The product of int8 codes with a scale per token and per weight row:
//   y[t][r] = (sum_k x[t][k] w[r][k]) * xs[t] * ws[r] (+ res[t][r])
// Both matrices hold k contiguously, which is how v_mfma_i32_16x16x64_i8 takes its operands: lane
// l holds 16 consecutive k (16 (l / 16) onwards) of A's row l % 16 and of B's column l % 16.  A is
// the weights and B the tokens, so lane l's four sums are rows 4 (l / 16) .. + 3 of token l % 16:
// neighbours in y.  Sums are 32-bit integers, exact for n <= 131071 (2^31 / 128^2).
#include "act_types.h"

typedef int hh_i4 __attribute__((ext_vector_type(4)));

// 16 codes of a row from k on, zeros from n on (the row's stride is a multiple of 16, so the
// load stays inside the row wherever k < n).
HH_DEV hh_i4 hh_i8_ld(const int8_t* row, uint32_t k, uint32_t n) {
    if (k >= n) return hh_i4{0, 0, 0, 0};
    hh_i4 v = *reinterpret_cast<const hh_i4*>(row + k);
    if (k + 16 > n) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int left = (int)(n - k) - 4 * i;  // bytes of dword i inside the row
            v[i] = left >= 4 ? v[i] : left <= 0 ? 0 : (int)((uint32_t)v[i] & ((1u << (8 * left)) - 1u));
        }
    }
    return v;
}

// y of four consecutive rows r.. of token t
template <class F>
HH_DEV void hh_i8_out(const hh_i8_gemm_args& a, uint32_t t, uint32_t r, hh_i4 sum) {
    if (t >= a.t || r >= a.m) return;
    const float xs = a.xs[t];
    const typename F::E* res = a.res ? (const typename F::E*)a.res + t * a.res_stride : nullptr;
    typename F::E* y = (typename F::E*)a.y + t * a.y_stride;
    for (uint32_t i = 0; i < 4 && r + i < a.m; i++) {
        float v = (float)sum[i] * xs * a.ws[r + i];
        if (res) v += F::get(res[r + i]);
        y[r + i] = F::put(v);
    }
}

// 64 rows x 64 tokens a workgroup, wave w taking rows 16 w .. + 15.
template <class F>
HH_DEV void hh_i8_gemm_simple(const hh_i8_gemm_args& a) {
    const uint32_t lane = threadIdx.x % HH_WAVE, wave = threadIdx.x / HH_WAVE;
    const uint32_t r0 = blockIdx.x * 64 + wave * 16, t0 = blockIdx.y * 64;
    const uint32_t row = min(r0 + lane % 16, a.m - 1);
    const int8_t* w = a.w + row * a.w_stride;
    const int8_t* x[4];
    hh_i4 acc[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        x[j] = a.x + min(t0 + 16 * j + lane % 16, a.t - 1) * a.x_stride;
        acc[j] = hh_i4{0, 0, 0, 0};
    }
    for (uint32_t k0 = 0; k0 < a.n; k0 += 64) {
        const uint32_t k = k0 + lane / 16 * 16;
        const hh_i4 wf = hh_i8_ld(w, k, a.n);
#pragma unroll
        for (int j = 0; j < 4; j++)
            acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf, hh_i8_ld(x[j], k, a.n), acc[j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; j++) hh_i8_out<F>(a, t0 + 16 * j + lane % 16, r0 + lane / 16 * 4, acc[j]);
}

#define HH_I8_GEMM(T, F)                                                                              \
    extern "C" __global__ void __launch_bounds__(256) hh_i8_gemm_simple_##T(const hh_i8_gemm_args a) { \
        hh_i8_gemm_simple<F>(a);                                                                      \
    }
HH_I8_GEMM(f32, hh_af32)
HH_I8_GEMM(f16, hh_af16)
HH_I8_GEMM(bf16, hh_abf16)
