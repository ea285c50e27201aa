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
// One workgroup per row (many short rows: four, a wave each), the row in registers between the two phases
// (CH chunks of 16 bytes a thread); rows of more than 4096 chunks are read twice (hh_i8_rows_<...>_loop).
// Bound by HBM where there are many rows: 14336 x 4096 f32 with values 92.7 us = 5.7 TB/s; 2048 x 4096 f32 with
// residual, sum and values 32.9 us = 4.3 TB/s (without values 27.9 = 3.9); 509 x 14336 bf16 gated 22.6 us = 2.9
// TB/s, 19.5 over three sets of tensors in turn, which the memory-side cache holds in part (with 64-bit act 27;
// without values 19.7 and 17.5).  By latency where there are few: 64 x 8192 bf16 with residual 7.2 us, 5.9 over
// three sets, 576 f32 4.0 to 4.6 us.
#include "act_types.h"
#include "wave64.h"

// Op over the workgroup of up to 16 waves; red: 16 words of LDS not read since the last meeting.
template <class Op>
HH_DEV uint64_t hh_i8_block64(uint64_t v, uint64_t* red) {
    v = hh_wave64<Op>(v);
    const uint32_t waves = blockDim.x / HH_WAVE, lane = threadIdx.x % HH_WAVE;
    if (waves == 1) return v;
    if (lane == 0) red[threadIdx.x / HH_WAVE] = v;
    __syncthreads();
    return hh_lane64(hh_row16<Op>(lane < waves ? red[lane] : 0), 0);
}
struct hh_i8_red {
    uint64_t top[16], ss[16];
};

// |u| of the row's largest element as bits (NaN sorts above infinity above every number) and the
// sum of squares, over the workgroup.
template <bool SUM>
HH_DEV void hh_i8_reduce(uint64_t& top, double& ss, hh_i8_red& red) {
    if (SUM) {
        const uint64_t s = hh_wave64<hh_addf64>((uint64_t)__double_as_longlong(ss));
        if (threadIdx.x % HH_WAVE == 0 && blockDim.x > HH_WAVE) red.ss[threadIdx.x / HH_WAVE] = s;
        ss = __longlong_as_double((long long)s);
    }
    top = hh_i8_block64<hh_max64>(top, red.top);  // meets
    const uint32_t waves = blockDim.x / HH_WAVE, lane = threadIdx.x % HH_WAVE;
    if (SUM && waves > 1)
        ss = __longlong_as_double((long long)hh_lane64(hh_row16<hh_addf64>(lane < waves ? red.ss[lane] : 0), 0));
}

enum { HH_I8_PLAIN, HH_I8_ACT, HH_I8_NORM };

// How many of the elements e..e+VEC lie in the row (e + VEC stays under 2^32).  Neither difference can
// wrap.  With e >= cols ? 0 : min(VEC, cols - e) the compiler computed cols - e in every lane as a
// subtraction that does not wrap, concluded e <= cols, and dropped the tests that guard the stores.
template <int VEC>
HH_DEV uint32_t hh_i8_count(uint32_t e, uint32_t cols) {
    return min(cols, e + VEC) - min(cols, e);
}

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
    // v to f32, then to the type: for a v that is the sum of two values of the type this is the one rounding
    // (checked over all pairs of bf16 and of f16; f32 of a 64-bit sum is innocuous, 53 >= 2 * 24 + 2).
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

// The row of this wave: a workgroup has blockDim.y rows where one wave holds a row, else one.
HH_DEV bool hh_i8_my_row(const hh_i8_rows_args& a, uint32_t& r) {
    r = blockIdx.x * blockDim.y + __builtin_amdgcn_readfirstlane(threadIdx.y);
    return r < a.rows;
}

template <class F, int KIND, int CH>
HH_DEV void hh_i8_rows_regs(const hh_i8_rows_args& a) {
    uint32_t r;
    if (!hh_i8_my_row(a, r)) return;
    constexpr int VEC = F::VEC;
    __shared__ hh_i8_red red;
    const hh_i8_row<F, KIND> row(a, r);
    double u[CH][VEC], ss = 0.0;
    uint64_t bits = 0;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const uint32_t e = (c * blockDim.x + threadIdx.x) * VEC;
        const uint32_t count = hh_i8_count<VEC>(e, a.cols);
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
    hh_i8_reduce<KIND == HH_I8_NORM>(bits, ss, red);
    double top, inv;
    const float scale = hh_i8_factors<KIND>(a, bits, ss, top, inv);
    const bool zero = !(scale > 0.f);
    if (threadIdx.x == 0) a.scale[r] = scale;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const uint32_t e = (c * blockDim.x + threadIdx.x) * VEC;
        const uint32_t count = hh_i8_count<VEC>(e, a.cols);
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
    hh_i8_reduce<KIND == HH_I8_NORM>(bits, ss, red);
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

// The gated intermediate in 32 bits, decided in 64: act costs ~60 64-bit operations an element, which
// is twice the memory's time (509 x 14336 bf16: 27 us).  h = act(g) u is computed in f32 with a bound e
// on its relative error: the exponent y is within 8 2^-24 |y| (GELU's polynomial, log2 e; it counts
// where y < 0, as exp(-y) / (1 + exp(-y)) of it reaches h), v_exp_f32 and v_rcp_f32 are within 2^-23,
// and the products, the sum and 127 / a add at most 2^-24 each.  The product g u comes first: the factor
// 1 / (1 + exp(-y)) is at most 1, so a product that leaves f32's normal range below is of an h under 2^-126,
// whose code is 0 beside a largest of 1e-25 or more however it is rounded, and one that leaves it above
// makes the row's largest infinite or NaN.  (act(g) first: the half of a subnormal g is off by up to itself,
// and a large u makes an ordinary h of it.)  A code whose t lies within e |t| of
// a border, every element that may be the row's largest, and all with y < -80, are recomputed in 64
// bits from memory, one by one (about one element in 4000).  Rows whose largest element is outside
// 1e-25..1e25 (or NaN) are recomputed whole.
HH_DEV float hh_i8_act32(float g, float u, int act, float& y) {
    y = act == HH_ACT_GELU_TANH ? 1.5957691216f * (g + 0.044715f * g * g * g) : g;
    return g * u * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y * -1.4426950409f));
}
HH_DEV float hh_i8_act32_error(float y) { return (8.f * fmaxf(-y, 0.f) + 36.f) * 0x1p-24f; }

template <class F, int CH>
HH_DEV void hh_i8_act_rows(const hh_i8_rows_args& a) {
    uint32_t r;
    if (!hh_i8_my_row(a, r)) return;
    typedef typename F::E E;
    constexpr int VEC = F::VEC;
    static_assert(CH * VEC <= 32, "a bit for each element of a thread");
    constexpr float FAR = (8.f * 89.f + 36.f) * 0x1p-24f;  // the error bound at y = -89, past which h is 0
    __shared__ uint64_t red[2][16];
    const hh_i8_row<F, HH_I8_ACT> row(a, r);
    auto count = [&](int c) {
        return hh_i8_count<VEC>((c * blockDim.x + threadIdx.x) * VEC, a.cols);
    };
    E g[CH][VEC];
    float h[CH][VEC];
    uint32_t seen = 0, far = 0, here = 0;  // largest |h| as bits: NaN and infinities sort above every number
    {
        E p[CH][VEC];
#pragma unroll
        for (int c = 0; c < CH; c++) {
            const uint32_t e = (c * blockDim.x + threadIdx.x) * VEC, n = count(c);
            if (n == VEC) {
                hh_load_n(row.x + e, g[c]);
                hh_load_n(row.b + e, p[c]);
            } else {
#pragma unroll
                for (int i = 0; i < VEC; i++) {
                    const bool in = (uint32_t)i < n;
                    g[c][i] = in ? row.x[e + i] : F::put(0.f);
                    p[c][i] = in ? row.b[e + i] : F::put(0.f);
                }
            }
            here |= ((1u << n) - 1u) << (c * VEC);
        }
#pragma unroll
        for (int c = 0; c < CH; c++)
#pragma unroll
            for (int i = 0; i < VEC; i++) {
                float y;
                h[c][i] = hh_i8_act32(F::get(g[c][i]), F::get(p[c][i]), a.act, y);
                seen = max(seen, __float_as_uint(fabsf(h[c][i])));
                far |= (y < -80.f ? 1u : 0u) << (c * VEC + i);
            }
    }
    auto exact = [&](uint32_t bit, uint32_t& e) {  // element `bit` of this thread in 64 bits
        e = (bit / VEC * blockDim.x + threadIdx.x) * VEC + bit % VEC;
        return hh_i8_act((double)F::get(row.x[e]), (double)F::get(row.b[e]), a.act);
    };
    // the 64-bit magnitude of whatever may be the largest: |h| (1 +- FAR) holds it
    const float top32 = __uint_as_float((uint32_t)hh_i8_block64<hh_max64>(seen, red[0]));
    const bool wide = !(top32 >= 1e-25f && top32 <= 1e25f);
    const float least = top32 * (1.f - 2.f * FAR);
    uint32_t todo = far;
#pragma unroll
    for (int c = 0; c < CH; c++)
#pragma unroll
        for (int i = 0; i < VEC; i++) todo |= (fabsf(h[c][i]) >= least ? 1u : 0u) << (c * VEC + i);
    todo = (wide ? ~0u : todo) & here;
    uint64_t bits = 0;
    for (; todo; todo &= todo - 1) {
        uint32_t e;
        const double v = exact((uint32_t)__builtin_ctz(todo), e);
        const uint64_t m = (uint64_t)__double_as_longlong(v) & 0x7fffffffffffffffull;
        bits = m > bits ? m : bits;
    }
    bits = hh_i8_block64<hh_max64>(bits, red[1]);
    double top, inv;
    const float scale = hh_i8_factors<HH_I8_ACT>(a, bits, 0.0, top, inv);
    const float inv32 = scale > 0.f && !wide ? (float)inv : 0.f;  // 0: codes 0 until recomputed
    if (threadIdx.x == 0) a.scale[r] = scale;
    todo = far;
#pragma unroll
    for (int c = 0; c < CH; c++) {
        const uint32_t at = (c * blockDim.x + threadIdx.x) * VEC, n = count(c);
        int8_t code[VEC];
        float val[VEC];
#pragma unroll
        for (int i = 0; i < VEC; i++) {
            const float t = inv32 > 0.f ? h[c][i] * inv32 : 0.f;
            const float k = rintf(t), gi = F::get(g[c][i]);
            const float y = a.act == HH_ACT_GELU_TANH ? 1.5957691216f * (gi + 0.044715f * gi * gi * gi) : gi;
            // |t - k| is exact; the border is at one half
            todo |= (0.5f - fabsf(t - k) > fabsf(t) * hh_i8_act32_error(y) ? 0u : 1u) << (c * VEC + i);
            code[i] = (int8_t)(int)k;
            val[i] = k * scale;
        }
        if (n == VEC) {
            hh_store_n(row.q + at, code);
            if (row.values) hh_store_n(row.values + at, val);
        } else {
            for (uint32_t i = 0; i < n; i++) {
                row.q[at + i] = code[i];
                if (row.values) row.values[at + i] = val[i];
            }
        }
    }
    if (!(scale > 0.f)) return;
    for (todo = (wide ? ~0u : todo) & here; todo; todo &= todo - 1) {
        uint32_t e;
        const float k = (float)rint(127.0 * exact((uint32_t)__builtin_ctz(todo), e) / top);
        row.q[e] = (int8_t)(int)k;
        if (row.values) row.values[e] = k * scale;
    }
}

#define HH_I8_ROWS_KIND(T, F, NAME, KIND)                                                                           \
    HH_I8_ROWS_CH(T, F, NAME, KIND, 1)                                                                              \
    HH_I8_ROWS_CH(T, F, NAME, KIND, 2)                                                                              \
    HH_I8_ROWS_CH(T, F, NAME, KIND, 4)                                                                              \
    extern "C" __global__ void __launch_bounds__(1024) hh_i8_rows_##T##_##NAME##_loop(const hh_i8_rows_args a) {   \
        hh_i8_rows_loop<F, KIND>(a);                                                                                \
    }
#define HH_I8_ROWS_CH(T, F, NAME, KIND, CH)                                                                         \
    extern "C" __global__ void __launch_bounds__(1024) hh_i8_rows_##T##_##NAME##_c##CH(const hh_i8_rows_args a) {   \
        if constexpr (KIND == HH_I8_ACT)                                                                            \
            hh_i8_act_rows<F, CH>(a);                                                                               \
        else                                                                                                        \
            hh_i8_rows_regs<F, KIND, CH>(a);                                                                        \
    }
#define HH_I8_ROWS(T, F)                                                                                            \
    HH_I8_ROWS_KIND(T, F, plain, HH_I8_PLAIN)                                                                       \
    HH_I8_ROWS_KIND(T, F, act, HH_I8_ACT)                                                                           \
    HH_I8_ROWS_KIND(T, F, norm, HH_I8_NORM)
HH_I8_ROWS(f32, hh_af32)
HH_I8_ROWS(f16, hh_af16)
HH_I8_ROWS(bf16, hh_abf16)
