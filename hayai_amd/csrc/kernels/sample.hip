// The next token of each row of logits: temperature, top-k, top-p and min-p, then the draw by a
// given random number u (include/hayai_hip.h has the definition).
//
// No sort: each filter keeps a prefix of the row's order (logit descending, index ascending), which is
// described by its last token's key and index.  Weights are exp((logit - max) / T) in 64 bits, held
// as whole multiples of 2^-42: sums of whole numbers do not depend on their order, so atomics leave the
// answer fixed, and 2^21 tokens of weight 1 stay below 2^63.
//
// Four launches, the row cut into parts (workgroups) of whole 512-token chunks:
//   hh_sample_max     the part's largest key and its first index
//   hh_sample_hist    counts and weights of the row's tokens by distance from the largest logit, in
//                     1023 bins of T / 32 and one for what weighs nothing
//   hh_sample_gather  the bins in which top-k and top-p end; the weight that each chunk surely keeps,
//                     and the tokens of those bins into a list
//   hh_sample_pick    one workgroup a row: where in the list the prefix ends (radix select), the
//                     chunk at which the running weight passes u, the token in it
// 128256 f32 logits, a row: 20 us, near all of it the chain of four launches (3, 5, 6 and 7 us); 64 rows: 57 us,
// of which max 7.5 (at the memory's rate), hist 15 and gather 20 (both the weights, about 45 operations a token) and
// pick 15 (sorts and scans one after the other).
// A row whose list passes 8192 tokens, whose largest logit is infinite or whose T is past 1e30 is done by one
// workgroup from the logits (hh_sample_row): about a dozen reads of the row with atomics on few bins.  A list
// passes where a filter ends among more than 8192 tokens within T / 32 of each other: 128256 logits of deviation 2
// from T = 11 on at a top-p of 0.5, from 35 to 40 on at 0.95; equal logits at any T.  128256 f32 logits: 450 us a
// row at an infinite T, 640 to 705 where all are equal; 64 such rows 580 and 1290 to 1400.
#include "act_types.h"
#include "wave64.h"

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

// A row's weights, in units of 2^-42: 2^42 e^((logit - max) / T) is 2^(n + 42) 2^f, |f| <= 1/2, with 2^f
// as the Taylor polynomial of e^(f ln 2), whose 12 terms leave 0.35^12 / 12! = 6e-15.  (T enters as
// log2 e / T: a quotient an element would cost as much again.)
struct hh_smp_weights {
    uint32_t top;
    double value, scale;
    HH_DEV hh_smp_weights(uint32_t top_, float temperature) : top(top_) {
        value = (double)hh_smp_value(top_);
        scale = 1.4426950408889634074 / (double)temperature;
    }
    HH_DEV static double pow2(double y) {  // 2^(y + 42)
        constexpr double L = 0.69314718055994530942, L2 = L * L, L4 = L2 * L2, L8 = L4 * L4;
        constexpr double c[11] = {1.0, L, L2 / 2, L2 * L / 6, L4 / 24, L4 * L / 120, L4 * L2 / 720, L4 * L2 * L / 5040,
                                  L8 / 40320, L8 * L / 362880, L8 * L2 / 3628800};
        const double n = rint(y), f = y - n;
        double p = L8 * L2 * L / 39916800;
#pragma unroll
        for (int i = 10; i >= 0; i--) p = fma(p, f, c[i]);
        return ldexp(p, (int)n + 42);
    }
    // of a logit within a few hundred temperatures of a finite largest
    HH_DEV double near(float v) const { return pow2(((double)v - value) * scale); }
    HH_DEV double of(uint32_t key) const {
        if (key <= HH_SMP_KEY_NINF || (top == HH_SMP_KEY_INF && key != top)) return 0.0;
        if (key == top) return HH_SMP_ONE;
        return pow2(fmax(((double)hh_smp_value(key) - value) * scale, -1100.0));
    }
};
// The nearest whole number of a weight (below 2^43): the low bits of 2^52 + w.
HH_DEV uint64_t hh_smp_mass(double w) {
    return (uint64_t)__double_as_longlong(w + 4503599627370496.0) & 0xfffffffffffffull;
}

struct hh_smp_lds {
    unsigned long long hist[256];
    uint64_t wave[16];
    uint64_t before, found;
    unsigned long long any, all;
    uint64_t sort[HH_SMP_BLOCK];
    uint32_t digit;
};

HH_DEV uint64_t hh_smp_scan(uint64_t v, hh_smp_lds& s) { return hh_block_scan64(v, s.wave); }

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

// A whole row by one workgroup of 1024: its largest key is `top`, above -inf's, and its temperature above 0.
template <class F>
HH_DEV void hh_sample_row(const hh_sample_args& a, uint32_t top, hh_smp_lds& s) {
    const uint32_t row = blockIdx.x, n = a.vocab, tid = threadIdx.x;
    const typename F::E* x = (const typename F::E*)a.x + row * a.stride;
    const hh_sample_row_params p = ((const hh_sample_row_params*)a.params)[row];
    const hh_smp_weights weights(top, p.temperature);
    auto mass = [&](uint32_t key) { return hh_smp_mass(weights.of(key)); };

    // cut: tokens with larger keys are in, of those with this key the first `ties` by index
    uint32_t cut = HH_SMP_KEY_NINF;
    uint64_t ties = 0, before;
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
    const double floor_w = p.min_p > 0.f ? (double)p.min_p * HH_SMP_ONE : 0.0;
    auto heavy = [&](uint32_t key) { return key == top || weights.of(key) >= floor_w; };

    // each thread takes a run of indices: how many ties precede it, then the kept weight
    const uint32_t per = (n + HH_SMP_BLOCK - 1) / HH_SMP_BLOCK;
    const uint32_t lo = min(n, tid * per), hi = min(n, lo + per);
    uint64_t mine = 0;
    for (uint32_t i = lo; i < hi; i++) mine += hh_smp_key(F::get(x[i])) == cut;
    const uint64_t rank0 = hh_smp_scan(mine, s) - mine;
    auto kept_mass = [&](uint32_t key, uint64_t& rank) -> uint64_t {
        if (key < cut || key <= HH_SMP_KEY_NINF) return 0;
        if (key == cut && rank++ >= ties) return 0;
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
    uint64_t want = u < 1.0 ? (uint64_t)(u * (double)total) : total - 1;
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
                if (a.probs) a.probs[row] = (float)(weights.of(key) / (double)total);
                break;
            }
        }
    }
}

// ------------------------------------------------------------------ the four launches
#define HH_SMP_CHUNK 512u    // tokens whose kept weight is one sum (4096 of them at most)
#define HH_SMP_BINS 1024u
#define HH_SMP_LIST 8192u    // tokens of a row's list, and of a part's before they join it
#define HH_SMP_STAGE 2048u
#define HH_SMP_THREADS 512u  // of the first three

// What hh_sample_gather finds about a row, for hh_sample_pick.
struct hh_smp_cut {
    uint32_t kbin, plo, phi;  // top-k ends in kbin, top-p in plo..phi (HH_SMP_BINS: no such end)
    uint32_t kneed;           // tokens of kbin that top-k keeps
    uint64_t kmass, pmass;    // weight of the bins before kbin (all: no such end), before plo
};

// A row's distance bins: 32 to a temperature; the last one's tokens are 31 temperatures below the
// largest or more, which weighs less than 2^-43, and -inf and NaN are among them.  For a finite largest logit
// and T <= 1e30 (other rows are left to hh_sample_row).
struct hh_smp_bins {
    float value, scale;
    HH_DEV hh_smp_bins(uint32_t top, float temperature) {
        value = hh_smp_value(top);
        scale = 32.f / temperature;
    }
    HH_DEV static bool hold(uint32_t top, float temperature) { return top < HH_SMP_KEY_INF && temperature <= 1e30f; }
    // rounding keeps the order: a lower logit never has a lower bin; fminf drops a NaN
    HH_DEV uint32_t of(float v) const { return v == value ? 0u : (uint32_t)fminf((value - v) * scale, 1023.f); }
};

// A token as one number: the row's order is that of falling numbers.
#define HH_SMP_INDEX_BITS 21
HH_DEV uint64_t hh_smp_entry(uint32_t key, uint32_t i) {
    return (uint64_t)key << HH_SMP_INDEX_BITS | ((1u << HH_SMP_INDEX_BITS) - 1u - i);
}
HH_DEV uint32_t hh_smp_entry_key(uint64_t e) { return (uint32_t)(e >> HH_SMP_INDEX_BITS); }
HH_DEV uint32_t hh_smp_entry_index(uint64_t e) {
    const uint32_t mask = (1u << HH_SMP_INDEX_BITS) - 1u;
    return mask - ((uint32_t)e & mask);
}

// The row's first token, from the parts'.
HH_DEV uint64_t hh_smp_top(const hh_sample_args& a, uint32_t row) {
    uint64_t v = 0;
    for (uint32_t i = threadIdx.x % HH_WAVE; i < a.parts; i += HH_WAVE) {
        const uint64_t o = a.top[(size_t)row * a.parts + i];
        v = o > v ? o : v;
    }
    return hh_wave64<hh_max64>(v);
}
// The tokens [lo, hi) of this workgroup's part.
HH_DEV void hh_smp_part(const hh_sample_args& a, uint32_t& lo, uint32_t& hi) {
    const uint32_t chunks = (a.vocab + HH_SMP_CHUNK - 1) / HH_SMP_CHUNK, per = (chunks + a.parts - 1) / a.parts;
    lo = min(a.vocab, blockIdx.x * per * HH_SMP_CHUNK);
    hi = min(a.vocab, lo + per * HH_SMP_CHUNK);
}
// f(eight logits, their indices) over the tokens of [lo, hi) by `threads` threads, of which this is one, the
// next eight's loads ahead of them.  (-inf past hi.)
template <class F, class Fn>
HH_DEV void hh_smp_each(const typename F::E* x, uint32_t lo, uint32_t hi, uint32_t threads, uint32_t thread, Fn f) {
    constexpr uint32_t VEC = F::VEC, NV = 8 / VEC;
    typename F::E now[NV][VEC], next[NV][VEC];
    auto load = [&](uint32_t base, typename F::E (&v)[NV][VEC]) {
#pragma unroll
        for (uint32_t j = 0; j < NV; j++) {
            const uint32_t i = base + (j * threads + thread) * VEC;
            if (i + VEC <= hi) {
                hh_load_n(x + i, v[j]);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < VEC; e++) v[j][e] = i + e < hi ? x[i + e] : F::put(-__builtin_inff());
            }
        }
    };
    if (lo < hi) load(lo, next);
    for (uint32_t base = lo; base < hi; base += threads * 8) {
#pragma unroll
        for (uint32_t j = 0; j < NV; j++)
#pragma unroll
            for (uint32_t e = 0; e < VEC; e++) now[j][e] = next[j][e];
        if (base + threads * 8 < hi) load(base + threads * 8, next);
        float v[8];
        uint32_t at[8];
#pragma unroll
        for (uint32_t j = 0; j < NV; j++)
#pragma unroll
            for (uint32_t e = 0; e < VEC; e++) {
                v[j * VEC + e] = F::get(now[j][e]);
                at[j * VEC + e] = base + (j * threads + thread) * VEC + e;
            }
        f(v, at);
    }
}

template <class F>
HH_DEV void hh_sample_max(const hh_sample_args& a) {
    __shared__ uint64_t red[HH_SMP_THREADS / HH_WAVE];
    const uint32_t row = blockIdx.y, tid = threadIdx.x;
    const typename F::E* x = (const typename F::E*)a.x + row * a.stride;
    uint32_t lo, hi;
    hh_smp_part(a, lo, hi);
    // the thread's first eight with its largest logit, then which of them it is
    float most = -__builtin_inff(), eight[8];
    uint32_t where[8];
#pragma unroll
    for (int e = 0; e < 8; e++) eight[e] = most, where[e] = 0;
    hh_smp_each<F>(x, lo, hi, HH_SMP_THREADS, tid, [&](const float (&l)[8], const uint32_t (&at)[8]) {
        float m = l[0];
#pragma unroll
        for (int e = 1; e < 8; e++) m = fmaxf(m, l[e]);  // (drops NaN)
        if (m > most) {
            most = m;
#pragma unroll
            for (int e = 0; e < 8; e++) eight[e] = l[e], where[e] = at[e];
        }
    });
    uint64_t v = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const uint64_t o = hh_smp_entry(hh_smp_key(eight[e]), where[e]);
        v = o > v ? o : v;
    }
    v = hh_wave64<hh_max64>(v);
    if (tid % HH_WAVE == 0) red[tid / HH_WAVE] = v;
    __syncthreads();
    // this part's share of the row's bins and the list's length to zero, for the next launches
    uint64_t* mass = a.mass + (size_t)row * HH_SMP_BINS;
    uint32_t* count = a.count + (size_t)row * HH_SMP_BINS;
    for (uint32_t i = blockIdx.x * HH_SMP_THREADS + tid; i < HH_SMP_BINS; i += a.parts * HH_SMP_THREADS) {
        mass[i] = 0;
        count[i] = 0;
    }
    if (tid == 0) {
        for (uint32_t w = 1; w < HH_SMP_THREADS / HH_WAVE; w++) v = red[w] > v ? red[w] : v;
        a.top[(size_t)row * a.parts + blockIdx.x] = v;
        if (blockIdx.x == 0) a.listed[row] = 0;
    }
}

HH_DEV bool hh_smp_filters(const hh_sample_row_params& p, uint32_t vocab) {
    return (p.top_k > 0 && (uint32_t)p.top_k < vocab) || p.top_p < 1.f;
}

template <class F>
HH_DEV void hh_sample_hist(const hh_sample_args& a) {
    __shared__ unsigned long long mass[HH_SMP_BINS];
    __shared__ uint32_t count[HH_SMP_BINS];
    const uint32_t row = blockIdx.y, tid = threadIdx.x;
    const hh_sample_row_params p = ((const hh_sample_row_params*)a.params)[row];
    if (!(p.temperature > 0.f) || !hh_smp_filters(p, a.vocab)) return;
    const uint32_t top = hh_smp_entry_key(hh_smp_top(a, row));
    if (top <= HH_SMP_KEY_NINF || !hh_smp_bins::hold(top, p.temperature)) return;
    for (uint32_t i = tid; i < HH_SMP_BINS; i += HH_SMP_THREADS) {
        mass[i] = 0;
        count[i] = 0;
    }
    __syncthreads();
    const hh_smp_bins bins(top, p.temperature);
    const hh_smp_weights weights(top, p.temperature);
    uint32_t lo, hi;
    hh_smp_part(a, lo, hi);
    const bool counts = p.top_k > 0 && (uint32_t)p.top_k < a.vocab, weigh = p.top_p < 1.f;
    hh_smp_each<F>((const typename F::E*)a.x + row * a.stride, lo, hi, HH_SMP_THREADS, tid,
                   [&](const float (&l)[8], const uint32_t (&)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t b = bins.of(l[e]);
            if (b == HH_SMP_BINS - 1) continue;
            if (counts) atomicAdd(&count[b], 1u);
            if (weigh) atomicAdd(&mass[b], (unsigned long long)hh_smp_mass(weights.near(l[e])));
        }
    });
    __syncthreads();
    for (uint32_t i = tid; i < HH_SMP_BINS; i += HH_SMP_THREADS)
        if (count[i] || mass[i]) {
            if (counts) atomicAdd(&a.count[(size_t)row * HH_SMP_BINS + i], count[i]);
            if (weigh) atomicAdd((unsigned long long*)&a.mass[(size_t)row * HH_SMP_BINS + i], mass[i]);
        }
}

// The bins in which the filters end, from the row's sums: the same in every workgroup of the row.
HH_DEV void hh_smp_find_cut(const hh_sample_args& a, uint32_t row, const hh_sample_row_params& p, hh_smp_cut& cut,
                            uint64_t* red) {
    static_assert(HH_SMP_BINS == 2 * HH_SMP_THREADS, "two bins a thread");
    const uint32_t tid = threadIdx.x;
    if (tid == 0) cut = hh_smp_cut{HH_SMP_BINS, HH_SMP_BINS, HH_SMP_BINS, 0, 0, 0};
    const size_t at = (size_t)row * HH_SMP_BINS + 2 * tid;
    const uint64_t c0 = a.count[at], c1 = a.count[at + 1], m0 = a.mass[at], m1 = a.mass[at + 1];
    const uint64_t cs = hh_block_scan64(c0 + c1, red), cb = cs - c0 - c1;  // (meets: cut is set)
    const uint64_t ms = hh_block_scan64(m0 + m1, red), mb = ms - m0 - m1;
    const bool topk = p.top_k > 0 && (uint32_t)p.top_k < a.vocab;
    if (topk) {
        const uint64_t k = (uint32_t)p.top_k;
        if (cb < k && cb + c0 >= k) {
            cut.kbin = 2 * tid;
            cut.kneed = (uint32_t)(k - cb);
            cut.kmass = mb;
        } else if (cb + c0 < k && cs >= k) {
            cut.kbin = 2 * tid + 1;
            cut.kneed = (uint32_t)(k - cb - c0);
            cut.kmass = mb + m0;
        }
    }
    __syncthreads();
    if (tid == HH_SMP_THREADS - 1 && cut.kbin == HH_SMP_BINS) cut.kmass = ms;
    if (p.top_p < 1.f) {
        // between what top-k keeps at least and at most: less than the weight through kbin, so plo and phi are
        // kbin at most
        __shared__ double want[2];
        const uint32_t kbin = cut.kbin;
        if (tid == HH_SMP_THREADS - 1 && kbin == HH_SMP_BINS) want[0] = want[1] = (double)p.top_p * (double)ms;
        if (kbin < HH_SMP_BINS && tid == kbin / 2) {
            want[0] = (double)p.top_p * (double)cut.kmass;
            want[1] = (double)p.top_p * (double)(cut.kmass + (kbin % 2 ? m1 : m0));
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 2; q++) {
            // the bin at which the running weight reaches want (0 and less: the first)
            const uint64_t before = q ? mb + m0 : mb, here = q ? m1 : m0;
            if (here && (before == 0 || (double)before < want[0]) && (double)(before + here) >= want[0]) {
                cut.plo = 2 * tid + q;
                cut.pmass = before;
            }
            if (here && (before == 0 || (double)before < want[1]) && (double)(before + here) >= want[1])
                cut.phi = 2 * tid + q;
        }
    } else if (tid == 0) {
        cut.plo = cut.phi = cut.kbin;
        cut.pmass = cut.kmass;
    }
    __syncthreads();
}

template <class F>
HH_DEV void hh_sample_gather(const hh_sample_args& a) {
    __shared__ hh_smp_cut cut;
    __shared__ uint64_t red[16], stage[HH_SMP_STAGE];
    __shared__ uint32_t found, base;
    const uint32_t row = blockIdx.y, tid = threadIdx.x;
    const hh_sample_row_params p = ((const hh_sample_row_params*)a.params)[row];
    if (!(p.temperature > 0.f)) return;
    const uint32_t top = hh_smp_entry_key(hh_smp_top(a, row));
    if (top <= HH_SMP_KEY_NINF) return;
    if (!hh_smp_bins::hold(top, p.temperature)) {
        if (blockIdx.x == 0 && tid == 0) a.listed[row] = HH_SMP_LIST + 1;
        return;
    }
    if (hh_smp_filters(p, a.vocab)) {
        hh_smp_find_cut(a, row, p, cut, red);
    } else {
        if (tid == 0) cut = hh_smp_cut{HH_SMP_BINS, HH_SMP_BINS, HH_SMP_BINS, 0, 0, 0};
        __syncthreads();
    }
    if (blockIdx.x == 0 && tid == 0) ((hh_smp_cut*)a.cut)[row] = cut;
    const uint32_t kbin = cut.kbin, plo = min(cut.plo, HH_SMP_BINS - 1), phi = cut.phi;
    const hh_smp_bins bins(top, p.temperature);
    const hh_smp_weights weights(top, p.temperature);
    const double heavy = p.min_p > 0.f ? (double)p.min_p * HH_SMP_ONE : 0.0;
    uint64_t* list = a.list + (size_t)row * HH_SMP_LIST;
    if (tid == 0) found = 0;
    __syncthreads();
    uint32_t lo, hi;
    hh_smp_part(a, lo, hi);
    // a wave takes a run of chunks, one chunk (eight tokens a lane) at a time
    const uint32_t chunks = (hi - lo + HH_SMP_CHUNK - 1) / HH_SMP_CHUNK, waves = HH_SMP_THREADS / HH_WAVE;
    const uint32_t per = (chunks + waves - 1) / waves * HH_SMP_CHUNK;
    const uint32_t wlo = min(hi, lo + tid / HH_WAVE * per), whi = min(hi, wlo + per);
    static_assert(HH_SMP_CHUNK == 8 * HH_WAVE, "a chunk is a wave's eight tokens a lane");
    hh_smp_each<F>((const typename F::E*)a.x + row * a.stride, wlo, whi, HH_WAVE, tid % HH_WAVE,
                   [&](const float (&l)[8], const uint32_t (&at)[8]) {
        uint64_t mine = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const uint32_t b = bins.of(l[e]);
            if (b < plo) {
                const double w = weights.near(l[e]);
                if (w >= heavy) mine += hh_smp_mass(w);
            } else if ((b <= phi && phi < HH_SMP_BINS) || b == kbin) {
                // into LDS first: a count on a device word takes microseconds
                const uint32_t to = atomicAdd(&found, 1u);
                const uint64_t entry = hh_smp_entry(hh_smp_key(l[e]), at[e]);
                if (to < HH_SMP_STAGE) {
                    stage[to] = entry;
                } else {
                    const uint32_t past = atomicAdd(&a.listed[row], 1u);
                    if (past < HH_SMP_LIST) list[past] = entry;
                }
            }
        }
        mine = hh_wave64<hh_addu64>(mine);
        if (tid % HH_WAVE == 0) a.sure[(size_t)row * a.chunks + at[0] / HH_SMP_CHUNK] = mine;
    });
    __syncthreads();
    const uint32_t n = min(found, HH_SMP_STAGE);
    if (n == 0) return;
    if (tid == 0) base = atomicAdd(&a.listed[row], n);
    __syncthreads();
    for (uint32_t i = tid; i < n; i += HH_SMP_THREADS)
        if (base + i < HH_SMP_LIST) list[base + i] = stage[i];
}

// The list's entries of a thread, 0: none.
#define HH_SMP_EACH (HH_SMP_LIST / HH_SMP_BLOCK)

// The entry at which the running amount, from the largest down over the entries that `take` takes, first
// reaches want; before: the amount of the entries above it.  (want is within their sum.)
template <class Take, class Amount>
HH_DEV uint64_t hh_smp_list_cut(const uint64_t (&v)[HH_SMP_EACH], double want, Take take, Amount amount, hh_smp_lds& s,
                                uint64_t& before) {
    // the bits in which the entries differ
    uint64_t any = 0, all = ~0ull;
#pragma unroll
    for (uint32_t i = 0; i < HH_SMP_EACH; i++)
        if (take(v[i])) {
            any |= v[i];
            all &= v[i];
        }
#pragma unroll
    for (int off = 32; off; off >>= 1) {
        any |= __shfl_xor(any, off, HH_WAVE);
        all &= __shfl_xor(all, off, HH_WAVE);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        s.any = 0;
        s.all = ~0ull;
    }
    __syncthreads();
    if (threadIdx.x % HH_WAVE == 0) {
        atomicOr(&s.any, (unsigned long long)any);
        atomicAnd(&s.all, (unsigned long long)all);
    }
    __syncthreads();
    const uint64_t differ = s.any & ~s.all;
    uint64_t prefix = s.all, above = 0;  // bits above the first that differs are common
    int shift = differ ? 64 - __builtin_clzll(differ) : 0;
    if (shift < 64) prefix = shift ? prefix >> shift << shift : prefix;
    else prefix = 0;
    while (shift > 0) {
        const int width = shift < 8 ? shift : 8;
        shift -= width;
        __syncthreads();
        if (threadIdx.x < 256) s.hist[threadIdx.x] = 0;
        if (threadIdx.x == 0) {  // the lowest, should rounding let none reach want
            s.digit = 0;
            s.before = above;
        }
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < HH_SMP_EACH; i++)
            if (take(v[i]) && (shift + width >= 64 || (v[i] >> (shift + width)) == (prefix >> (shift + width))))
                atomicAdd(&s.hist[(v[i] >> shift) & ((1u << width) - 1u)], (unsigned long long)amount(v[i]));
        __syncthreads();
        if (threadIdx.x < HH_WAVE) {
            // lane l has digits 255 - 4 l down to 252 - 4 l
            const uint32_t d0 = 255 - 4 * threadIdx.x;
            uint64_t h[4], sum = 0;
#pragma unroll
            for (int q = 0; q < 4; q++) sum += h[q] = s.hist[d0 - q];
            uint64_t run = hh_scan64(sum) + above - sum;
#pragma unroll
            for (int q = 0; q < 4; q++) {
                if (h[q] && (run == 0 || (double)run < want) && (double)(run + h[q]) >= want) {
                    s.digit = d0 - q;
                    s.before = run;
                }
                run += h[q];
            }
        }
        __syncthreads();
        prefix |= (uint64_t)s.digit << shift;
        above = s.before;
    }
    before = above;
    return prefix;
}

// The last token of the row that the filters keep, from a list of more than HH_SMP_BLOCK.
template <class Weigh>
HH_DEV uint64_t hh_smp_end_select(const uint64_t* list, uint32_t n, const hh_sample_row_params& p, const hh_smp_cut& cut,
                                  const hh_smp_bins& bins, Weigh weigh, hh_smp_lds& s) {
    uint64_t v[HH_SMP_EACH], last = 0, before;
#pragma unroll
    for (uint32_t i = 0; i < HH_SMP_EACH; i++) {
        const uint32_t at = i * HH_SMP_BLOCK + threadIdx.x;
        v[i] = at < n ? list[at] : 0;
    }
    if (cut.kbin < HH_SMP_BINS) {
        auto in_k = [&](uint64_t e) { return e && bins.of(hh_smp_value(hh_smp_entry_key(e))) == cut.kbin; };
        last = hh_smp_list_cut(v, (double)cut.kneed, in_k, [](uint64_t) { return 1ull; }, s, before);
    }
    if (!(p.top_p < 1.f)) return last;
    uint64_t kept = 0;  // of top-k's last bin
    if (cut.kbin < HH_SMP_BINS) {
#pragma unroll
        for (uint32_t i = 0; i < HH_SMP_EACH; i++)
            if (v[i] && v[i] >= last && bins.of(hh_smp_value(hh_smp_entry_key(v[i]))) == cut.kbin) kept += weigh(v[i]);
        kept = hh_smp_scan(kept, s);
        __syncthreads();
        if (threadIdx.x == HH_SMP_BLOCK - 1) s.found = kept;
        __syncthreads();
        kept = s.found;
    }
    const double want = (double)p.top_p * (double)(cut.kmass + kept);
    const uint64_t klast = last;
    auto in_p = [&](uint64_t e) { return e && e >= klast && bins.of(hh_smp_value(hh_smp_entry_key(e))) <= cut.phi; };
    return hh_smp_list_cut(v, want - (double)cut.pmass, in_p, weigh, s, before);
}

// The same from a list that has a thread for each entry: sorted (a bitonic network over the power of two
// that holds it, in shuffles where partners share a wave), its weights summed up once.
template <class Weigh>
HH_DEV uint64_t hh_smp_end_sorted(const uint64_t* list, uint32_t n, const hh_sample_row_params& p, const hh_smp_cut& cut,
                                  const hh_smp_bins& bins, Weigh weigh, hh_smp_lds& s) {
    const uint32_t tid = threadIdx.x;
    uint64_t e = tid < n ? list[tid] : 0;
    uint32_t size = 2;
    while (size < n) size *= 2;
    for (uint32_t k = 2; k <= size; k *= 2)
        for (uint32_t j = k / 2; j > 0; j /= 2) {
            uint64_t o;
            if (j >= HH_WAVE) {
                __syncthreads();
                s.sort[tid] = e;
                __syncthreads();
                o = s.sort[tid ^ j];
            } else {
                o = __shfl_xor(e, (int)j, HH_WAVE);
            }
            const bool keep_large = ((tid & j) == 0) == ((tid & k) == 0);
            e = (o > e) == keep_large ? o : e;
        }
    const uint64_t m = e ? weigh(e) : 0, run = hh_smp_scan(m, s);
    const uint32_t bin = e ? bins.of(hh_smp_value(hh_smp_entry_key(e))) : HH_SMP_BINS;
    // entries of kbin follow those of lower bins: its first entry, then the last that top-k keeps
    __syncthreads();
    s.sort[tid] = (uint64_t)bin;
    if (tid == 0) {
        s.digit = 0;
        s.any = 0;
        s.before = 0;
        s.found = 0;
    }
    __syncthreads();
    const bool topk = cut.kbin < HH_SMP_BINS;
    if (topk && bin == cut.kbin && (tid == 0 || s.sort[tid - 1] != bin)) {
        s.digit = tid;
        s.before = run - m;
    }
    __syncthreads();
    const uint32_t kend = topk ? s.digit + cut.kneed - 1 : HH_SMP_BLOCK;
    if (topk && tid == kend) {
        s.any = e;
        s.found = run - s.before;  // kbin's weight that top-k keeps
    }
    __syncthreads();
    uint64_t last = s.any;
    if (p.top_p < 1.f) {
        const double want = (double)p.top_p * (double)(cut.kmass + s.found);
        const uint64_t before = cut.pmass + run - m;
        __syncthreads();
        if (e && bin <= cut.phi && tid <= kend && (before == 0 || (double)before < want) && (double)(before + m) >= want && m)
            s.any = e;
        __syncthreads();
        last = s.any;
    }
    return last;
}

template <class F>
HH_DEV void hh_sample_pick(const hh_sample_args& a) {
    __shared__ hh_smp_lds s;
    __shared__ unsigned long long mass[2097152 / HH_SMP_CHUNK];
    const uint32_t row = blockIdx.x, tid = threadIdx.x;
    const typename F::E* x = (const typename F::E*)a.x + row * a.stride;
    const hh_sample_row_params p = ((const hh_sample_row_params*)a.params)[row];
    const uint64_t best = hh_smp_top(a, row);
    const uint32_t top = hh_smp_entry_key(best), n = a.listed[row];
    if (top <= HH_SMP_KEY_NINF || !(p.temperature > 0.f)) {
        const bool none = top <= HH_SMP_KEY_NINF;
        if (tid == 0) {
            a.ids[row] = none ? -1 : (int32_t)hh_smp_entry_index(best);
            if (a.probs) a.probs[row] = none ? 0.f : 1.f;
        }
        return;
    }
    if (n > HH_SMP_LIST) return hh_sample_row<F>(a, top, s);
    const hh_smp_cut cut = ((const hh_smp_cut*)a.cut)[row];
    const hh_smp_bins bins(top, p.temperature);
    const hh_smp_weights weights(top, p.temperature);
    auto weigh = [&](uint64_t e) { return hh_smp_mass(weights.of(hh_smp_entry_key(e))); };
    const uint64_t* list = a.list + (size_t)row * HH_SMP_LIST;
    // tokens from `last` on are in
    uint64_t last = 0;
    if (n) last = n <= HH_SMP_BLOCK ? hh_smp_end_sorted(list, n, p, cut, bins, weigh, s) : hh_smp_end_select(list, n, p, cut, bins, weigh, s);
    if (p.min_p > 1.f) last = best;  // heavier than any token: the first alone
    const double heavy = p.min_p > 0.f ? (double)p.min_p * HH_SMP_ONE : 0.0;
    auto kept_mass = [&](uint64_t e) -> uint64_t {
        const uint32_t key = hh_smp_entry_key(e);
        if (e < last || key <= HH_SMP_KEY_NINF) return 0;
        const double w = weights.of(key);
        return key == top || w >= heavy ? hh_smp_mass(w) : 0;
    };
    // the chunks' kept weight, four a thread: what is sure and the list's
    constexpr uint32_t EACH = sizeof mass / sizeof mass[0] / HH_SMP_BLOCK;
#pragma unroll
    for (uint32_t q = 0; q < EACH; q++) {
        const uint32_t c = EACH * tid + q;
        mass[c] = c < a.chunks && !(p.min_p > 1.f) ? a.sure[(size_t)row * a.chunks + c] : 0;
    }
    __syncthreads();
    if (p.min_p > 1.f) {
        if (tid == 0) mass[hh_smp_entry_index(best) / HH_SMP_CHUNK] = (unsigned long long)HH_SMP_ONE;
    } else {
        for (uint32_t i = tid; i < n; i += HH_SMP_BLOCK) {
            const uint64_t e = list[i], m = kept_mass(e);
            if (m) atomicAdd(&mass[hh_smp_entry_index(e) / HH_SMP_CHUNK], (unsigned long long)m);
        }
    }
    __syncthreads();
    uint64_t mine = 0;
#pragma unroll
    for (uint32_t q = 0; q < EACH; q++) mine += mass[EACH * tid + q];
    uint64_t after = hh_smp_scan(mine, s);
    __syncthreads();
    if (tid == HH_SMP_BLOCK - 1) s.found = after;
    __syncthreads();
    const uint64_t total = s.found;
    double u = (double)a.u[row];
    if (!(u > 0.0)) u = 0.0;
    uint64_t want = u < 1.0 ? (uint64_t)(u * (double)total) : total - 1;
    if (want >= total) want = total - 1;
    // the chunk at which the running weight first exceeds `want`
    if (after > want && after - mine <= want) {
        uint64_t run = after - mine;
        for (uint32_t q = 0; q < EACH; q++) {
            const uint64_t m = mass[EACH * tid + q];
            if (run + m > want) {
                s.digit = EACH * tid + q;
                s.before = want - run;
                break;
            }
            run += m;
        }
    }
    __syncthreads();
    want = s.before;
    // and the token in it
    const uint32_t i = s.digit * HH_SMP_CHUNK + tid;
    uint64_t m = 0;
    uint32_t key = 0;
    if (tid < HH_SMP_CHUNK && i < a.vocab) {
        key = hh_smp_key(F::get(x[i]));
        m = kept_mass(hh_smp_entry(key, i));
    }
    after = hh_smp_scan(m, s);
    if (after > want && after - m <= want) {
        a.ids[row] = (int32_t)i;
        if (a.probs) a.probs[row] = (float)(weights.of(key) / (double)total);
    }
}

#define HH_SAMPLE(T, F)                                                                                      \
    extern "C" __global__ void __launch_bounds__(512) hh_sample_max_##T(const hh_sample_args a) {            \
        hh_sample_max<F>(a);                                                                                 \
    }                                                                                                        \
    extern "C" __global__ void __launch_bounds__(512) hh_sample_hist_##T(const hh_sample_args a) {           \
        hh_sample_hist<F>(a);                                                                                \
    }                                                                                                        \
    extern "C" __global__ void __launch_bounds__(512) hh_sample_gather_##T(const hh_sample_args a) {         \
        hh_sample_gather<F>(a);                                                                              \
    }                                                                                                        \
    extern "C" __global__ void __launch_bounds__(1024) hh_sample_pick_##T(const hh_sample_args a) {          \
        hh_sample_pick<F>(a);                                                                                \
    }
HH_SAMPLE(f32, hh_af32)
HH_SAMPLE(f16, hh_af16)
HH_SAMPLE(bf16, hh_abf16)
