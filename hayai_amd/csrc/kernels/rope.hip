// Rotary positions and the cache's new entries: for each token, queries and keys turned by the
// token's position, keys and values put into the token's slot of the cache.
//   angle_i = position * base^(-2i / rot) / factors[i],   i < rot / 2
//   (a, b) -> mscale * (a cos - b sin, b cos + a sin)
// over the pairs (x[i], x[i + rot/2]) (halves) or (x[2i], x[2i + 1]) (pairs) of a head's first rot
// elements; the others go through.  Angles are taken in 64 bits, in whole turns whose fraction alone
// is kept: in 32 bits a position of 100000 would leave 2^-7 of a radian.  cos and sin are rounded to
// f32 once, products and sums are f32, each output is rounded once.
//
// Bound by launch latency for few tokens (9 + 6 heads of 64, one token), by memory for a prompt: a
// workgroup takes a token, the first rot / 2 threads make its cosines and sines (64-bit functions:
// 100 instructions for two waves, once for all heads), then a thread turns 16 bytes of either half of
// a head at a time.  Both of a pair are read and written by one thread, so q may be turned in place.
#include "kv_pages.h"

#define HH_ROPE_MAX_PAIRS 128

template <class A, class C, bool PAIRS>
HH_DEV void hh_rope(const hh_rope_args& a) {
    typedef typename A::E E;
    constexpr int V = A::VEC;
    __shared__ float cs[HH_ROPE_MAX_PAIRS], sn[HH_ROPE_MAX_PAIRS];
    const size_t t = blockIdx.x;
    const uint32_t tid = threadIdx.x, half = a.rot / 2, dim = a.kv.dim;
    if (tid < half) {
        double turns = (double)a.positions[t] * exp2(-(2.0 * tid / a.rot) * a.log2_base) * 0.15915494309189533577;
        if (a.factors) turns /= (double)a.factors[tid];
        double s, c;
        sincospi(2.0 * (turns - rint(turns)), &s, &c);
        cs[tid] = (float)(c * (double)a.mscale);
        sn[tid] = (float)(s * (double)a.mscale);
    }
    __syncthreads();
    const int64_t slot = a.slots[t];
    const bool stored = slot >= 0 && slot >> a.kv.shift < a.kv.pages;
    uint8_t* const page = a.kv.base + (stored ? (uint64_t)(slot >> a.kv.shift) * a.kv.stride : 0);
    const uint32_t at = (uint32_t)slot & ((1u << a.kv.shift) - 1);
    // a head's items: its turned part, then the rest
    const uint32_t turned = ((PAIRS ? a.rot : half) + V - 1) / V, each = turned + (dim - a.rot + V - 1) / V;
    const uint32_t vitems = (dim + V - 1) / V, qk = (a.heads + a.kv.heads) * each, all = qk + a.kv.heads * vitems;
    for (uint32_t item = blockIdx.y * 256 + tid; item < all; item += gridDim.y * 256) {
        if (item >= qk) {  // a value, turned to [dim][tokens]
            if (!stored) continue;
            const uint32_t h = (item - qk) / vitems, d = (item - qk) % vitems * V, n = min((uint32_t)V, dim - d);
            const E* x = (const E*)a.v + t * a.v_stride + h * dim + d;
            typename C::E* y = (typename C::E*)(page + hh_kv_value<C>(a.kv, h, d)) + at;
            E v[V];
            if (n == V)
                hh_load_n(x, v);
            else
                for (uint32_t i = 0; i < n; i++) v[i] = x[i];
#pragma unroll
            for (uint32_t i = 0; i < V; i++)
                if (i < n) y[(size_t)i << a.kv.shift] = C::put(A::get(v[i]));
            continue;
        }
        const uint32_t h = item / each, r = item % each;
        const bool key = h >= a.heads;
        if (key && !stored) continue;
        const E* x = key ? (const E*)a.k + t * a.k_stride + (h - a.heads) * dim : (const E*)a.q + t * a.q_stride + h * dim;
        E* const out = (E*)a.out + t * a.out_stride + h * dim;  // (unused by keys)
        typename C::E* const kout = (typename C::E*)(page + hh_kv_key<C>(a.kv, key ? h - a.heads : 0, at));
        auto put = [&](uint32_t d, const float (&v)[V], uint32_t n) {
            if (key) {
                typename C::E o[V];
#pragma unroll
                for (int i = 0; i < V; i++) o[i] = C::put(v[i]);
                if (n == V)
                    hh_store_n(kout + d, o);
                else
                    for (uint32_t i = 0; i < n; i++) kout[d + i] = o[i];
            } else {
                E o[V];
#pragma unroll
                for (int i = 0; i < V; i++) o[i] = A::put(v[i]);
                if (n == V)
                    hh_store_n(out + d, o);
                else
                    for (uint32_t i = 0; i < n; i++) out[d + i] = o[i];
            }
        };
        auto get = [&](uint32_t d, float (&v)[V], uint32_t n) {
            E e[V];
            if (n == V) {
                hh_load_n(x + d, e);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < V; i++) e[i] = x[d + min(i, n - 1)];
            }
#pragma unroll
            for (int i = 0; i < V; i++) v[i] = A::get(e[i]);
        };
        float u[V], w[V], o[V];
        if (r >= turned) {
            const uint32_t d = a.rot + (r - turned) * V, n = min((uint32_t)V, dim - d);
            get(d, u, n);
            put(d, u, n);
        } else if (PAIRS) {
            const uint32_t d = r * V, n = min((uint32_t)V, a.rot - d);  // even
            get(d, u, n);
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const uint32_t p = min(d / 2 + i / 2, half - 1);
                o[i] = fmaf(u[i], cs[p], -(u[i + 1] * sn[p]));
                o[i + 1] = fmaf(u[i + 1], cs[p], u[i] * sn[p]);
            }
            put(d, o, n);
        } else {
            const uint32_t d = r * V, n = min((uint32_t)V, half - d);
            get(d, u, n);
            get(half + d, w, n);
#pragma unroll
            for (int i = 0; i < V; i++) {
                const uint32_t p = min(d + i, half - 1);
                o[i] = fmaf(u[i], cs[p], -(w[i] * sn[p]));
                w[i] = fmaf(w[i], cs[p], u[i] * sn[p]);
            }
            put(d, o, n);
            put(half + d, w, n);
        }
    }
}

#define HH_ROPE(N, A, C)                                                                                    \
    extern "C" __global__ void __launch_bounds__(256) hh_rope_halves_##N(const hh_rope_args a) { hh_rope<A, C, false>(a); } \
    extern "C" __global__ void __launch_bounds__(256) hh_rope_pairs_##N(const hh_rope_args a) { hh_rope<A, C, true>(a); }
HH_ROPE(f32, hh_af32, hh_af32)
HH_ROPE(f16, hh_af16, hh_af16)
HH_ROPE(bf16, hh_abf16, hh_abf16)
HH_ROPE(f32_f16, hh_af32, hh_af16)
HH_ROPE(f32_bf16, hh_af32, hh_abf16)
