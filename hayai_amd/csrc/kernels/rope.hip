// Rotary positions and the cache's new entries: for each token, queries and keys turned by the
// token's position, keys and values put into the token's slot of the cache.
//   angle_i = position * base^(-2i / rot) / factors[i],   i < rot / 2
//   (a, b) -> mscale * (a cos - b sin, b cos + a sin)
// over the pairs (x[i], x[i + rot/2]) (halves) or (x[2i], x[2i + 1]) (pairs) of a head's first rot
// elements; the others go through.  Angles are taken in 64 bits, in whole turns whose fraction alone
// is kept: in 32 bits a position of 100000 would leave 2^-7 of a radian.  cos and sin are rounded to
// f32 once, products and sums are f32, each output is rounded once.
//
// Bound by launch latency for few tokens (9 + 6 heads of 64 f32, one token: the kernel 3.5 us), by memory for a prompt (2048
// tokens, 32/4 heads of 128 f16: 11.8 us a call among others, 3.5 TB/s; a token a workgroup 15.2).  A workgroup takes a token, or
// eight neighbouring ones of a prompt; its threads ask for their first 16 bytes of either half of a head, make the tokens' cosines and sines (64-bit functions,
// once for all heads), then turn.  Both of a pair are read and written by one thread, so q may be turned in
// place.  Values go to [dim][tokens]: eight tokens in neighbouring slots as 16 bytes, others an element at a time.
#include "kv_pages.h"

#define HH_ROPE_MAX_PAIRS 128

template <class A, class C, bool PAIRS, int TB>
HH_DEV void hh_rope(const hh_rope_args& a) {
    typedef typename A::E E;
    typedef typename C::E CE;
    constexpr uint32_t V = A::VEC, THREADS = TB == 1 ? 256 : 1024;
    __shared__ float cs[TB][HH_ROPE_MAX_PAIRS], sn[TB][HH_ROPE_MAX_PAIRS];
    const size_t t0 = (size_t)blockIdx.x * TB;
    const uint32_t tid = threadIdx.x, half = a.rot / 2, dim = a.kv.dim, nt = TB == 1 ? 1 : min(a.tokens - (uint32_t)t0, TB);
    const uint32_t first = blockIdx.y * THREADS + tid, step = gridDim.y * THREADS;

    // a head's items: its turned part, then the rest
    const uint32_t turned = ((PAIRS ? a.rot : half) + V - 1) / V, each = turned + (dim - a.rot + V - 1) / V;
    const uint32_t qk = (a.heads + a.kv.heads) * each, all = nt * qk;
    struct Item {
        float u[V], w[V];  // elements d.. and, of halves, half + d..
        uint32_t t, h, d, n;
        bool turn, key;
    };
    auto take = [&](const E* x, uint32_t n, float (&v)[V]) {
        E e[V];
        if (n == V) {
            hh_load_n(x, e);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < V; i++) e[i] = x[min(i, n - 1)];
        }
#pragma unroll
        for (uint32_t i = 0; i < V; i++) v[i] = A::get(e[i]);
    };
    auto load = [&](uint32_t i, Item& it) {
        it.t = TB == 1 ? 0 : i / qk;
        const uint32_t j = i - it.t * qk, h = j / each, r = j - h * each;
        it.key = h >= a.heads;
        it.h = it.key ? h - a.heads : h;
        it.turn = r < turned;
        it.d = it.turn ? r * V : a.rot + (r - turned) * V;
        it.n = min(V, (it.turn ? (PAIRS ? a.rot : half) : dim) - it.d);
        const E* x = (it.key ? (const E*)a.k + (t0 + it.t) * a.k_stride : (const E*)a.q + (t0 + it.t) * a.q_stride) + it.h * dim;
        take(x + it.d, it.n, it.u);
        if (!PAIRS && it.turn) take(x + half + it.d, it.n, it.w);
    };
    Item it;
    if (first < all) load(first, it);

    for (uint32_t i = tid; i < nt * half; i += THREADS) {
        const uint32_t t = TB == 1 ? 0 : i / half, p = i - t * half;
        double turns = (double)a.positions[t0 + t] * exp2(-(2.0 * p / a.rot) * a.log2_base) * 0.15915494309189533577;
        if (a.factors) turns /= (double)a.factors[p];
        double s, c;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        cs[t][p] = (float)(c * (double)a.mscale);
        sn[t][p] = (float)(s * (double)a.mscale);
    }
    __syncthreads();
    auto stored = [&](int slot) { return slot >= 0 && (uint32_t)slot >> a.kv.shift < a.kv.pages; };
    auto page = [&](int slot) { return a.kv.base + (uint64_t)((uint32_t)slot >> a.kv.shift) * a.kv.stride; };
    const uint32_t mask = (1u << a.kv.shift) - 1;

    // values: all heads' elements, or of one token V at a time
    if (TB > 1) {
        const int slot = a.slots[t0];
        bool run = nt == TB && stored(slot) && (slot & (TB - 1)) == 0;
#pragma unroll
        for (int t = 1; t < TB; t++) run = run && a.slots[t0 + min((uint32_t)t, nt - 1)] == slot + t;
        for (uint32_t i = first; i < a.kv.heads * dim; i += step) {
            E e[TB];
#pragma unroll
            for (uint32_t t = 0; t < TB; t++) e[t] = ((const E*)a.v)[(t0 + min(t, nt - 1)) * a.v_stride + i];
            const uint32_t h = i / dim, at = hh_kv_value<C>(a.kv, h, i - h * dim);
            if (run) {
                CE o[TB];
#pragma unroll
                for (int t = 0; t < TB; t++) o[t] = C::put(A::get(e[t]));
                hh_store_n((CE*)(page(slot) + at) + (slot & mask), o);
            } else {
                for (uint32_t t = 0; t < nt; t++) {
                    const int s = a.slots[t0 + t];
                    E v = e[0];
#pragma unroll
                    for (uint32_t k = 1; k < TB; k++) v = t == k ? e[k] : v;
                    if (stored(s)) ((CE*)(page(s) + at))[s & mask] = C::put(A::get(v));
                }
            }
        }
    } else {
        const int slot = a.slots[t0];
        const uint32_t vitems = (dim + V - 1) / V;
        // (they follow the other items, so that few tokens' threads have one each)
        for (uint32_t i = first >= all ? first : first + (all - first + step - 1) / step * step; i < all + a.kv.heads * vitems; i += step) {
            if (!stored(slot)) break;
            const uint32_t h = (i - all) / vitems, d = (i - all) % vitems * V, n = min(V, dim - d);
            const E* x = (const E*)a.v + t0 * a.v_stride + h * dim + d;
            CE* y = (CE*)(page(slot) + hh_kv_value<C>(a.kv, h, d)) + (slot & mask);
            float v[V];
            take(x, n, v);
#pragma unroll
            for (uint32_t k = 0; k < V; k++)
                if (k < n) y[(size_t)k << a.kv.shift] = C::put(v[k]);
        }
    }

    for (uint32_t i = first; i < all; i += step) {
        if (i != first) load(i, it);
        const int slot = it.key ? a.slots[t0 + it.t] : 0;
        if (it.key && !stored(slot)) continue;
        E* const out = (E*)a.out + (t0 + it.t) * a.out_stride + it.h * dim;  // (unused by keys)
        CE* const kout = it.key ? (CE*)(page(slot) + hh_kv_key<C>(a.kv, it.h, slot & mask)) : nullptr;
        auto put = [&](uint32_t d, const float (&v)[V]) {
            if (it.key) {
                CE o[V];
#pragma unroll
                for (uint32_t k = 0; k < V; k++) o[k] = C::put(v[k]);
                if (it.n == V)
                    hh_store_n(kout + d, o);
                else
                    for (uint32_t k = 0; k < it.n; k++) kout[d + k] = o[k];
            } else {
                E o[V];
#pragma unroll
                for (uint32_t k = 0; k < V; k++) o[k] = A::put(v[k]);
                if (it.n == V)
                    hh_store_n(out + d, o);
                else
                    for (uint32_t k = 0; k < it.n; k++) out[d + k] = o[k];
            }
        };
        const float *const c = cs[it.t], *const s = sn[it.t];
        if (!it.turn) {
            put(it.d, it.u);
        } else if (PAIRS) {
            float o[V];
#pragma unroll
            for (uint32_t k = 0; k < V; k += 2) {
                const uint32_t p = min(it.d / 2 + k / 2, half - 1);
                o[k] = fmaf(it.u[k], c[p], -(it.u[k + 1] * s[p]));
                o[k + 1] = fmaf(it.u[k + 1], c[p], it.u[k] * s[p]);
            }
            put(it.d, o);
        } else {
            float o[V], q[V];
#pragma unroll
            for (uint32_t k = 0; k < V; k++) {
                const uint32_t p = min(it.d + k, half - 1);
                o[k] = fmaf(it.u[k], c[p], -(it.w[k] * s[p]));
                q[k] = fmaf(it.w[k], c[p], it.u[k] * s[p]);
            }
            put(it.d, o);
            put(half + it.d, q);
        }
    }
}

#define HH_ROPE_FORM(N, A, C, L, PAIRS)                                                                                                         \
    extern "C" __global__ void __launch_bounds__(256) hh_rope_##L##_##N(const hh_rope_args a) { hh_rope<A, C, PAIRS, 1>(a); }    \
    extern "C" __global__ void __launch_bounds__(1024) hh_rope_##L##8_##N(const hh_rope_args a) { hh_rope<A, C, PAIRS, 8>(a); }
#define HH_ROPE(N, A, C) HH_ROPE_FORM(N, A, C, halves, false) HH_ROPE_FORM(N, A, C, pairs, true)
HH_ROPE(f32, hh_af32, hh_af32)
HH_ROPE(f16, hh_af16, hh_af16)
HH_ROPE(bf16, hh_abf16, hh_abf16)
HH_ROPE(f32_f16, hh_af32, hh_af16)
HH_ROPE(f32_bf16, hh_af32, hh_abf16)
