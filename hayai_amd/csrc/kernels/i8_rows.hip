// Rows of activations (or weights) into int8 codes with one scale per row:
//   hh_i8_rows_<type>_plain   u = x
//   hh_i8_rows_<type>_act     u = act(x) * up
//   hh_i8_rows_<type>_norm    v = x (+ res, v stored), u = v * norm
// With a = max|u| over the row: code = rint(127 u / a), scale = a / 127 * (norm: 1 / rms(v)).  The
// factor 1 / rms(v) is common to the row, so it cancels out of the codes and only enters the
// scale.
//
// Which of two codes is nearest is decided at borders 1 / 254 of the row's largest value apart,
// and a different decision is a whole step of error; every element is therefore carried in 64
// bits from its load to its code: v and u, the sum of squares, and t = u * (127 / a), whose error is
// a few 2^-53 of t; within 1e-9 of a border the quotient 127 u / a itself decides.  The 64-bit
// vector rate equals the 32-bit one on this chip.
//
// One workgroup per row, the row in registers between the two phases (CH chunks of 16 bytes a
// thread); rows past 1024 threads * 4 chunks are read twice (hh_i8_rows_<...>_loop).
#include "act_types.h"

struct hh_i8_red {
    uint64_t top[16];
    double ss[16];
};

// |u| of the row's largest element as bits (NaN sorts above infinity above every number) and the
// sum of squares, over the workgroup.
HH_DEV void hh_i8_reduce(uint64_t& top, double& ss, hh_i8_red& red) {
#pragma unroll
    for (int off = 32; off; off >>= 1) {
        const uint64_t o = __shfl_xor(top, off, HH_WAVE);
        top = o > top ? o : top;
        ss += __shfl_xor(ss, off, HH_WAVE);
    }
    const uint32_t waves = blockDim.x / HH_WAVE;
    if (waves == 1) return;
    if (threadIdx.x % HH_WAVE == 0) {
        red.top[threadIdx.x / HH_WAVE] = top;
        red.ss[threadIdx.x / HH_WAVE] = ss;
    }
    __syncthreads();
    top = red.top[0];
    ss = red.ss[0];
    for (uint32_t w = 1; w < waves; w++) {
        top = red.top[w] > top ? red.top[w] : top;
        ss += red.ss[w];
    }
}

enum { HH_I8_PLAIN, HH_I8_ACT, HH_I8_NORM };

// SiLU(g) * u or tanh-GELU(g) * u; 1 + tanh(y) as 2 / (1 + exp(-2 y)).
HH_DEV double hh_i8_act(double g, double u, int act) {
    if (act == HH_ACT_GELU_TANH) {
        const double y = 0.79788456080286535588 * (g + 0.044715 * g * g * g);
        return g / (1.0 + exp(-2.0 * y)) * u;
    }
    return g / (1.0 + exp(-g)) * u;
}

template <class F, int KIND>
struct hh_i8_row {
    typedef typename F::E E;
    static constexpr int VEC = F::VEC;
    const E* x;
    const E* b;
    E* sum;
    const float* norm;
    int8_t* q;
    float* values;
    uint32_t cols;
    int act;

    HH_DEV hh_i8_row(const hh_i8_rows_args& a, uint64_t row) {
        x = (const E*)a.x + row * a.x_stride;
        b = a.b ? (const E*)a.b + row * a.b_stride : nullptr;
        sum = a.sum ? (E*)a.sum + row * a.sum_stride : nullptr;
        norm = a.norm;
        q = a.q + row * a.q_stride;
        values = a.values ? a.values + row * a.cols : nullptr;
        cols = a.cols;
        act = a.act;
    }
    // u of the elements e..e+VEC (zeros past the row), v where the norm needs it
    HH_DEV void load(uint32_t e, double (&u)[VEC], double (&v)[VEC], uint32_t count) const {
        E xe[VEC], be[VEC];
        float ne[VEC];
        const bool two = KIND == HH_I8_ACT || (KIND == HH_I8_NORM && b);
        if (count == VEC) {
            hh_load_n(x + e, xe);
            if (two) hh_load_n(b + e, be);
            if (KIND == HH_I8_NORM) hh_load_n(norm + e, ne);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                const bool in = (uint32_t)i < count;
                xe[i] = in ? x[e + i] : F::put(0.f);
                if (two) be[i] = in ? b[e + i] : F::put(0.f);
                if (KIND == HH_I8_NORM) ne[i] = in ? norm[e + i] : 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            v[i] = (double)F::get(xe[i]);
            if (KIND == HH_I8_NORM) {
                if (two) v[i] += (double)F::get(be[i]);
                u[i] = v[i] * (double)ne[i];
            } else {
                u[i] = KIND == HH_I8_ACT ? hh_i8_act(v[i], (double)F::get(be[i]), act) : v[i];
            }
        }
    }
    HH_DEV void store_sum(uint32_t e, const double (&v)[VEC], uint32_t count) const {
        E s[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) s[i] = F::put((float)v[i]);
        if (count == VEC) {
            hh_store_n(sum + e, s);
        } else {
            for (uint32_t i = 0; i < count; i++) sum[e + i] = s[i];
        }
    }
    HH_DEV void store(uint32_t e, const double (&u)[VEC], uint32_t count, double top, double inv, float scale) const {
        int8_t c[VEC];
        float val[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const double t = u[i] * inv;
            double k = rint(t);
            if (fabs(t - k) > 0.5 - 1e-9) k = rint(127.0 * u[i] / top);
            const int code = (int)k;
            c[i] = (int8_t)code;
            val[i] = (float)code * scale;
        }
        if (count == VEC) {
            hh_store_n(q + e, c);
            if (values) hh_store_n(values + e, val);
        } else {
            for (uint32_t i = 0; i < count; i++) {
                q[e + i] = c[i];
                if (values) values[e + i] = val[i];
            }
        }
    }
};

// The row's factors from its reduced statistics: inv turns u into codes.  A row with a NaN or an
// infinity, and one whose scale is 0, has codes 0.
template <int KIND>
HH_DEV float hh_i8_factors(const hh_i8_rows_args& a, uint64_t bits, double ss, double& top, double& inv) {
    top = __longlong_as_double((long long)bits);
    const bool bad = bits >= 0x7ff0000000000000ull;
    double s = top;
    if (KIND == HH_I8_NORM && bits) s *= 1.0 / sqrt(ss / (double)a.cols + (double)a.eps);
    const float scale = bad ? __builtin_nanf("") : (float)(s / 127.0);
    inv = scale > 0.f ? 127.0 / top : 0.0;
    if (!(scale > 0.f)) top = 1.0;
    return scale;
}

template <class F, int KIND, int CH>
HH_DEV void hh_i8_rows_regs(const hh_i8_rows_args& a) {
    constexpr int VEC = F::VEC;
    __shared__ hh_i8_red red;
    const hh_i8_row<F, KIND> row(a, blockIdx.x);
    double u[CH][VEC], ss = 0.0;
    uint64_t bits = 0;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const uint32_t e = (c * blockDim.x + threadIdx.x) * VEC;
        const uint32_t count = e >= a.cols ? 0u : min((uint32_t)VEC, a.cols - e);
        double v[VEC];
        row.load(e, u[c], v, count);
        if (KIND == HH_I8_NORM && row.sum && count) row.store_sum(e, v, count);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const uint64_t m = (uint64_t)__double_as_longlong(u[c][i]) & 0x7fffffffffffffffull;
            bits = m > bits ? m : bits;
            if (KIND == HH_I8_NORM) ss += v[i] * v[i];
        }
    }
    hh_i8_reduce(bits, ss, red);
    double top, inv;
    const float scale = hh_i8_factors<KIND>(a, bits, ss, top, inv);
    const bool zero = !(scale > 0.f);
    if (threadIdx.x == 0) a.scale[blockIdx.x] = scale;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const uint32_t e = (c * blockDim.x + threadIdx.x) * VEC;
        const uint32_t count = e >= a.cols ? 0u : min((uint32_t)VEC, a.cols - e);
        if (!count) break;
        if (zero) {
#pragma unroll
            for (int i = 0; i < VEC; i++) u[c][i] = 0.0;
        }
        row.store(e, u[c], count, top, inv, scale);
    }
}

template <class F, int KIND>
HH_DEV void hh_i8_rows_loop(const hh_i8_rows_args& a) {
    constexpr int VEC = F::VEC;
    __shared__ hh_i8_red red;
    const hh_i8_row<F, KIND> row(a, blockIdx.x);
    double u[VEC], v[VEC], ss = 0.0;
    uint64_t bits = 0;
    const uint32_t step = blockDim.x * VEC;
    for (uint64_t e = threadIdx.x * VEC; e < a.cols; e += step) {
        row.load((uint32_t)e, u, v, (uint32_t)min((uint64_t)VEC, a.cols - e));
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const uint64_t m = (uint64_t)__double_as_longlong(u[i]) & 0x7fffffffffffffffull;
            bits = m > bits ? m : bits;
            if (KIND == HH_I8_NORM) ss += v[i] * v[i];
        }
    }
    hh_i8_reduce(bits, ss, red);
    double top, inv;
    const float scale = hh_i8_factors<KIND>(a, bits, ss, top, inv);
    const bool zero = !(scale > 0.f);
    if (threadIdx.x == 0) a.scale[blockIdx.x] = scale;
    for (uint64_t e = threadIdx.x * VEC; e < a.cols; e += step) {
        const uint32_t count = (uint32_t)min((uint64_t)VEC, a.cols - e);
        row.load((uint32_t)e, u, v, count);
        if (KIND == HH_I8_NORM && row.sum) row.store_sum((uint32_t)e, v, count);
        if (zero) {
#pragma unroll
            for (int i = 0; i < VEC; i++) u[i] = 0.0;
        }
        row.store((uint32_t)e, u, count, top, inv, scale);
    }
}

#define HH_I8_ROWS_CH(T, F, NAME, KIND, CH)                                                                         \
    extern "C" __global__ void __launch_bounds__(1024) hh_i8_rows_##T##_##NAME##_c##CH(const hh_i8_rows_args a) {  \
        hh_i8_rows_regs<F, KIND, CH>(a);                                                                            \
    }
#define HH_I8_ROWS_KIND(T, F, NAME, KIND)                                                                           \
    HH_I8_ROWS_CH(T, F, NAME, KIND, 1)                                                                              \
    HH_I8_ROWS_CH(T, F, NAME, KIND, 2)                                                                              \
    extern "C" __global__ void __launch_bounds__(1024) hh_i8_rows_##T##_##NAME##_loop(const hh_i8_rows_args a) {   \
        hh_i8_rows_loop<F, KIND>(a);                                                                                \
    }
#define HH_I8_ROWS(T, F)                                                                                            \
    HH_I8_ROWS_KIND(T, F, plain, HH_I8_PLAIN)                                                                       \
    HH_I8_ROWS_KIND(T, F, act, HH_I8_ACT)                                                                           \
    HH_I8_ROWS_KIND(T, F, norm, HH_I8_NORM)
HH_I8_ROWS(f32, hh_af32)
HH_I8_ROWS(f16, hh_af16)
HH_I8_ROWS(bf16, hh_abf16)
