// The next token of each row of logits: temperature, top-k, top-p and min-p, then the draw by a
// given random number u (include/hayai_hip.h has the definition).
//
// No sort: each filter keeps a prefix of the row's order (logit descending, index ascending), so it
// is described by the key of its last token and how many of that key's tokens are in, found by a
// radix select over the 32-bit ordered keys (8 bits at a time, counts or weights per digit).
// Weights are exp((logit - max) / T) in 64 bits, held as whole multiples of 2^-42: sums of whole
// numbers do not depend on their order, so atomics leave the answer fixed, and 2^21 tokens of weight 1
// stay below 2^63.  One workgroup per row.
#include "act_types.h"

struct hh_sample_row_params {
    float temperature;
    int32_t top_k;
    float top_p;
    float min_p;
};

#define HH_SMP_BLOCK 1024u
#define HH_SMP_ONE 4398046511104.0  // 2^42

// Order of logits as unsigned integers; NaN below everything, -0 as +0.
HH_DEV uint32_t hh_smp_key(float v) {
    if (v != v) return 0u;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
#define HH_SMP_KEY_NINF 0x007fffffu  // of -inf
#define HH_SMP_KEY_INF 0xff800000u   // of +inf
HH_DEV float hh_smp_value(uint32_t key) { return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu)); }

// Weight of the token with this key in a row whose largest key is top.
HH_DEV double hh_smp_weight(uint32_t key, uint32_t top, float temperature) {
    if (key <= HH_SMP_KEY_NINF) return 0.0;
    if (key == top) return 1.0;
    if (top == HH_SMP_KEY_INF) return 0.0;
    return exp(((double)hh_smp_value(key) - (double)hh_smp_value(top)) / (double)temperature);
}
HH_DEV uint64_t hh_smp_mass(double w) { return (uint64_t)(w * HH_SMP_ONE); }

struct hh_smp_lds {
    unsigned long long hist[256];
    uint64_t wave[16];
    uint64_t before, found;
    uint32_t digit, top;
};

// Inclusive sums over the workgroup's threads in thread order.
HH_DEV uint64_t hh_smp_scan(uint64_t v, hh_smp_lds& s) {
    const uint32_t lane = threadIdx.x % HH_WAVE, w = threadIdx.x / HH_WAVE;
#pragma unroll
    for (int off = 1; off < HH_WAVE; off <<= 1) {
        const uint64_t o = __shfl_up(v, off, HH_WAVE);
        if (lane >= (uint32_t)off) v += o;
    }
    __syncthreads();
    if (lane == HH_WAVE - 1) s.wave[w] = v;
    __syncthreads();
    for (uint32_t i = 0; i < w; i++) v += s.wave[i];
    return v;
}

// The key at which the running amount, from the largest key down over keys > floor, first reaches
// want: amount(key) a token.  before: the amount of the keys above it.  Returns 0 where the whole
// row has less.
template <class F, class A>
HH_DEV uint32_t hh_smp_select(const typename F::E* x, uint32_t n, uint32_t floor, double want, A amount, hh_smp_lds& s,
                              uint64_t& before) {
    uint32_t prefix = 0;
    uint64_t above = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        if (threadIdx.x < 256) s.hist[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += HH_SMP_BLOCK) {
            const uint32_t key = hh_smp_key(F::get(x[i]));
            if (key > floor && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))))
                atomicAdd(&s.hist[(key >> shift) & 255u], (unsigned long long)amount(key));
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            uint64_t run = above;
            int d = 255;
            for (; d >= 0; d--) {
                if (s.hist[d] && (double)(run + s.hist[d]) >= want) break;
                run += s.hist[d];
            }
            s.digit = (uint32_t)d;
            s.before = run;
        }
        __syncthreads();
        if ((int)s.digit < 0) {
            before = s.before;
            return 0u;
        }
        prefix |= s.digit << shift;
        above = s.before;
    }
    before = above;
    return prefix;
}

template <class F>
HH_DEV void hh_sample_simple(const hh_sample_args& a) {
    __shared__ hh_smp_lds s;
    const uint32_t row = blockIdx.x, n = a.vocab, tid = threadIdx.x;
    const typename F::E* x = (const typename F::E*)a.x + row * a.stride;
    const hh_sample_row_params p = ((const hh_sample_row_params*)a.params)[row];
    const bool greedy = !(p.temperature > 0.f);

    // the largest key
    uint32_t top = 0;
    for (uint32_t i = tid; i < n; i += HH_SMP_BLOCK) top = max(top, hh_smp_key(F::get(x[i])));
    if (tid == 0) s.top = 0;
    __syncthreads();
    atomicMax(&s.top, top);
    __syncthreads();
    top = s.top;
    if (top <= HH_SMP_KEY_NINF) {
        if (tid == 0) {
            a.ids[row] = -1;
            if (a.probs) a.probs[row] = 0.f;
        }
        return;
    }
    const float T = p.temperature;
    auto mass = [&](uint32_t key) { return hh_smp_mass(hh_smp_weight(key, top, T)); };

    // cut: tokens with larger keys are in, of those with this key the first `ties` by index
    uint32_t cut = HH_SMP_KEY_NINF;
    uint64_t ties = 0;
    if (greedy) {
        cut = top;
        ties = 1;
    } else {
        uint64_t before;
        if (p.top_k > 0 && (uint32_t)p.top_k < n) {
            const uint32_t key =
                hh_smp_select<F>(x, n, HH_SMP_KEY_NINF, (double)p.top_k, [](uint32_t) { return 1ull; }, s, before);
            if (key) {
                cut = key;
                ties = (uint64_t)p.top_k - before;
            }
        }
        if (p.top_p < 1.f) {
            // the weight top-k left, then the key at which the share is reached
            const uint64_t at_cut = ties ? ties * mass(cut) : 0;
            uint64_t sum = 0;
            for (uint32_t i = tid; i < n; i += HH_SMP_BLOCK) {
                const uint32_t key = hh_smp_key(F::get(x[i]));
                if (key > cut) sum += mass(key);
            }
            sum = hh_smp_scan(sum, s);
            __syncthreads();
            if (tid == HH_SMP_BLOCK - 1) s.found = sum;
            __syncthreads();
            const double want = (double)p.top_p * (double)(s.found + at_cut);
            const uint32_t key = hh_smp_select<F>(x, n, cut, want, mass, s, before);
            // a tie is in while the weight before it is below what is wanted
            const uint32_t at = key ? key : cut;
            if (key || ties) {
                const double left = (want - (double)before) / (double)mass(at);
                uint64_t c = left > 0.0 ? (uint64_t)ceil(left < 4e9 ? left : 4e9) : 0;
                if (at == top && c == 0) c = 1;
                if (!key && c > ties) c = ties;
                cut = at;
                ties = c;
            }
        }
        if (p.min_p > 1.f) {  // heavier than any token: the first alone
            cut = top;
            ties = 1;
        }
    }
    const double floor_w = !greedy && p.min_p > 0.f ? (double)p.min_p : 0.0;
    auto heavy = [&](uint32_t key) { return key == top || hh_smp_weight(key, top, T) >= floor_w; };
    const bool only_top = greedy || cut == top;
    if (only_top && ties == 0) ties = 1;

    // each thread takes a run of indices: how many ties precede it, then the kept weight
    const uint32_t per = (n + HH_SMP_BLOCK - 1) / HH_SMP_BLOCK;
    const uint32_t lo = min(n, tid * per), hi = min(n, lo + per);
    uint64_t mine = 0;
    for (uint32_t i = lo; i < hi; i++) mine += hh_smp_key(F::get(x[i])) == cut;
    const uint64_t rank0 = hh_smp_scan(mine, s) - mine;
    auto kept_mass = [&](uint32_t key, uint64_t& rank) -> uint64_t {
        if (key < cut || key <= HH_SMP_KEY_NINF) return 0;
        if (key == cut && rank++ >= ties) return 0;
        if (greedy) return 1;
        return heavy(key) ? mass(key) : 0;
    };
    uint64_t rank = rank0, sum = 0;
    for (uint32_t i = lo; i < hi; i++) sum += kept_mass(hh_smp_key(F::get(x[i])), rank);
    const uint64_t after = hh_smp_scan(sum, s);
    __syncthreads();
    if (tid == HH_SMP_BLOCK - 1) s.found = after;
    __syncthreads();
    const uint64_t total = s.found;
    double u = (double)a.u[row];
    if (!(u > 0.0)) u = 0.0;
    uint64_t want = (uint64_t)(u * (double)total);
    if (want >= total) want = total - 1;
    // the token at which the running weight first exceeds `want`
    if (after > want && after - sum <= want) {
        uint64_t run = after - sum;
        rank = rank0;
        for (uint32_t i = lo; i < hi; i++) {
            const uint32_t key = hh_smp_key(F::get(x[i]));
            const uint64_t m = kept_mass(key, rank);
            run += m;
            if (run > want) {
                a.ids[row] = (int32_t)i;
                if (a.probs)
                    a.probs[row] = greedy ? 1.f : (float)(hh_smp_weight(key, top, T) * HH_SMP_ONE / (double)total);
                break;
            }
        }
    }
}

#define HH_SAMPLE(T, F)                                                                               \
    extern "C" __global__ void __launch_bounds__(1024) hh_sample_simple_##T(const hh_sample_args a) { \
        hh_sample_simple<F>(a);                                                                       \
    }
HH_SAMPLE(f32, hh_af32)
HH_SAMPLE(f16, hh_af16)
HH_SAMPLE(bf16, hh_abf16)
