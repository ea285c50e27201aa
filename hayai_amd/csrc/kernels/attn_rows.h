// A tile of 128 rows against the keys of a page table: the core of a prompt's attention (attn_prompt.hip) and of
// a batch's with the tokens that it shares (attn_decode.hip).
#ifndef HH_KERNELS_ATTN_ROWS_H
#define HH_KERNELS_ATTN_ROWS_H

#include "attn_tiles.h"

// rows of an LDS tile: 16-byte chunk c of row r lies at chunk c ^ swizzle(r), so that the 16 rows that are read
// at once lie in all banks
template <int BYTES>
HH_DEV constexpr uint32_t hh_attn_swizzle(uint32_t row) {
    return BYTES == 128 ? row / 2 % 8 : row % 16;
}

// The tile's rows: heads kvh * group .. of tokens first .. of a run of `tokens`, whose rows of q and out begin at
// `start`; the run's last token sees `len` keys.
struct hh_attn_tile {
    uint32_t seq, start, first, tokens, len;
};

// Keys that the run's token t sees where each earlier token sees a key less.
HH_DEV uint32_t hh_attn_seen(const hh_attn_tile& tile, uint32_t t) {
    return (uint32_t)max(0, min((int)tile.len, (int)tile.len - (int)tile.tokens + (int)t + 1));
}

// Bytes of a tile of keys and values in LDS.
template <class C, int DP, int DU>
constexpr int hh_attn_bytes() {
    return 128 * DP + 128 * (DU ? DU : DP);
}

// DP: a head's elements, or those that they lie within; DU: 0 where the head has all of them, else how many are computed
// (a head of 72 to 96 takes three quarters of 128's products).  CAUSAL: each earlier token sees a key less; else all of
// them see len, and the sums always go to `part`.  at: the tile's number in `part`, where each has a.splits parts; split:
// which of the `splits` parts that it takes.
template <class A, class C, int DP, int DU, bool CAUSAL>
HH_DEV void hh_attn_rows(const hh_attn_args& a, const hh_attn_tile& tile, const int32_t* table, uint32_t entries, uint32_t kvh,
                         uint32_t at, uint32_t split, uint32_t splits) {
    typedef typename A::E E;
    typedef typename C::E CE;
    typedef hh_mat<C> M;
    typedef typename M::frag F;
    constexpr int EF = C::VEC, SZ = sizeof(CE), BN = 128 / SZ, NT = BN / 32, D = DU ? DU : DP, NC = D / (2 * EF), DT = D / 32;
    constexpr bool FULL = DU == 0;
    constexpr float LIFT = hh_attn_lift<C>();
    constexpr int NG = BN / 16;  // a page's end may lie after any 16 keys
    constexpr int KB = DP * SZ, VB = BN * SZ, KBYTES = BN * KB, BYTES = hh_attn_bytes<C, DP, DU>();
    constexpr int KP = KBYTES / 1024 / 4, VP = D * VB / 1024 / 4;  // 1 KB pieces a wave copies
    static_assert(BYTES == KBYTES + D * VB && (!FULL || VP % 2 == 0), "a whole head's waves begin at even pieces of V");
    const uint32_t lane = threadIdx.x % HH_WAVE, ln = lane % 32, hf = lane / 32;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / HH_WAVE);
    const uint32_t dim = FULL ? DP : a.kv.dim, group = a.group, shift = a.kv.shift;

    const uint32_t rows = min(a.tile_tokens, tile.tokens - tile.first) * group;
    const uint32_t r = wave * 32 + ln, tok = tile.first + min(r, rows - 1) / group, head = kvh * group + min(r, rows - 1) % group;
    // keys that the lane's row sees, and the tile's first and last row
    auto seen = [&](uint32_t t) { return CAUSAL ? hh_attn_seen(tile, t) : tile.len; };
    const uint32_t limit = seen(tok), least = seen(tile.first), most = seen(tile.first + (rows - 1) / group);
    const uint32_t tiles = (most + BN - 1) / BN;
    const uint32_t t0 = (uint32_t)((uint64_t)tiles * split / splits);
    const uint32_t t1 = (uint32_t)((uint64_t)tiles * (split + 1) / splits);

    F q[NC];
    const E* qrow = (const E*)a.q + (size_t)(tile.start + tok) * a.q_stride + head * dim;
#pragma unroll
    for (int c = 0; c < NC; c++) q[c] = hh_query<A, C, FULL>(qrow, (2 * c + hf) * EF, dim, true);

    // copies: a piece's rows and chunks by lane
    constexpr int KC = KB / 16, KR = 64 / KC;  // chunks of a row of K, rows a piece
    const uint32_t krow = lane / KC, vrow = lane / 8, pmask = (1u << shift) - 1;
    uint32_t id_k = 0, id_v[2] = {0, 0};  // page numbers: lane g's of granule g; the lane's values' granules
    auto vchunk = [&](int odd) { return lane % 8 ^ hh_attn_swizzle<128>(vrow + 8 * odd); };
    auto ask_k = [&](uint32_t t) { id_k = hh_page(table, t * BN + lane % NG * 16, shift, entries); };
    auto ask_v = [&](uint32_t t) {
#pragma unroll
        for (int o = 0; o < 2; o++) id_v[o] = hh_page(table, t * BN + vchunk(o) * EF, shift, entries);
    };
    // row 8j + 4h + i of 32 holds key 16 (j / 2) + 8 h + 4 (j % 2) + i of 16-bit types: hf's EF keys are neighbours in
    // its registers
    auto key_of = [&](uint32_t row) {
        return SZ == 4 ? row : (row & ~31u) | (row & 16) | (row & 4) << 1 | (row & 8) >> 1 | (row & 3);
    };
    const uint8_t* const zeros = (const uint8_t*)&hh_kv_zeros;
    const uint32_t p0k = wave * KP, p0v = wave * VP;
    uint32_t koff[KP];  // from the piece's 16 keys on
#pragma unroll
    for (int i = 0; i < KP; i++) {
        const uint32_t row = (p0k + i) * KR + krow;
        koff[i] = key_of(row) % 16 * dim * SZ + (lane % KC ^ hh_attn_swizzle<KB>(row)) * 16;
    }
    auto copy_k = [&](uint8_t* buf, uint32_t t) {
#pragma unroll
        for (int i = 0; i < KP; i++) {
            const uint32_t g = __builtin_amdgcn_readfirstlane((p0k + i) * KR / 16);
            const uint32_t id = __builtin_amdgcn_readlane(id_k, g);
            const uint8_t* from = a.kv.base + id * a.kv.stride + hh_kv_key<C>(a.kv, kvh, (t * BN + g * 16) & pmask);
            uint8_t* const to = buf + (p0k + i) * 1024;
            if (FULL && __builtin_expect(id < a.kv.pages, 1))
                hh_copy16(from + koff[i], to);
            else
                hh_copy16(id < a.kv.pages && (lane % KC ^ hh_attn_swizzle<KB>((p0k + i) * KR + krow)) * EF < dim ? from + koff[i] : zeros, to);
        }
    };
    auto copy_v = [&](uint8_t* buf, uint32_t t) {
        const uint8_t* from[2];
        const bool in[2] = {id_v[0] < a.kv.pages, id_v[1] < a.kv.pages};
#pragma unroll
        for (int o = 0; o < 2; o++)
            from[o] = a.kv.base + id_v[o] * a.kv.stride + ((t * BN + vchunk(o) * EF) & pmask) * SZ + (vrow << shift) * SZ;
        const uint32_t first = hh_kv_value<C>(a.kv, kvh, 0);
        if (FULL && __builtin_expect(__all(in[0] && in[1]), 1)) {
#pragma unroll
            for (int i = 0; i < VP; i++)
                hh_copy16(from[i & 1] + (first + ((p0v + i) * 8 << shift) * SZ), buf + (p0v + i) * 1024);
        } else {
#pragma unroll
            for (int i = 0; i < VP; i++) {
                const uint32_t o = (p0v + i) & 1, d = (p0v + i) * 8;  // (rows past dim: the last one's place)
                const uint8_t* src = (o ? from[1] : from[0]) + (first + ((min(d + vrow, dim - 1) - vrow) << shift) * SZ);
                hh_copy16((o ? in[1] : in[0]) ? src : zeros, buf + (p0v + i) * 1024);
            }
        }
    };

    hh_f32x16 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = hh_f32x16{};
    float base = HH_ATTN_LOWEST, sum = 0;
    uint32_t odd = 0;  // not 0: a value of a crossed tile is no finite number
    const uint32_t kswz = hh_attn_swizzle<KB>(ln) ^ hf, vswz = hh_attn_swizzle<128>(ln) ^ hf;

    const bool idle = wave * 32 >= rows;
    auto compute = [&](uint8_t* buf, uint32_t t) {
        const uint32_t k0 = t * BN;
        uint8_t* const vbuf = buf + KBYTES;
        const bool crossed = k0 + BN > least;
        if (crossed) {  // values past the sequence's end and those that are no finite numbers as zeros
            for (uint32_t i = threadIdx.x; i < D * 8; i += 256) {
                F* const at = (F*)(vbuf + i / 8 * VB + (i % 8 ^ hh_attn_swizzle<128>(i / 8)) * 16);
                *at = hh_finite<C>(hh_first<C>(*at, (int)tile.len - (int)(k0 + i % 8 * EF)), odd);
            }
            __syncthreads();
        }
        if (idle) return;
        float s[NT * 16];
        hh_f32x16 acc[NT];
#pragma unroll
        for (int j = 0; j < NT; j++) acc[j] = hh_f32x16{};
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                acc[j] = M::mul32(*(const F*)(buf + (j * 32 + ln) * KB + ((2 * c) ^ kswz) * 16), q[c], acc[j]);
#pragma unroll
        for (int x = 0; x < NT * 16; x++) s[x] = acc[x / 16][x % 16];
        if (crossed) {
#pragma unroll
            for (int x = 0; x < NT * 16; x++)
                s[x] = k0 + (2 * (x / EF) + hf) * EF + x % EF < limit ? s[x] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int x = 1; x < NT * 16; x++) top = fmaxf(top, s[x]);
        top *= a.c;
        if (__any(top > base + (HH_ATTN_SLACK + LIFT))) {
            top = fmaxf(top, __shfl_xor(top, 32));
            const float next = top > base + (HH_ATTN_SLACK + LIFT) ? top - LIFT : base, f = hh_exp2(base - next);
            base = next;
            sum *= f;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int x = 0; x < 16; x++) o[i][x] *= f;
        }
        F p[NT * 16 / EF];
        float sums[4] = {0, 0, 0, 0};
#pragma unroll
        for (int x = 0; x < NT * 16; x++) {
            const float w = hh_exp2(fmaf(s[x], a.c, -base));
            p[x / EF][x % EF] = C::put(w);
            sums[x % 4] += w;
        }
        sum += (sums[0] + sums[1]) + (sums[2] + sums[3]);
        auto value = [&](int i, int f) { return *(const F*)(vbuf + (i * 32 + ln) * VB + ((2 * f) ^ vswz) * 16); };
#pragma unroll
        for (int f = 0; f < NT * 16 / EF; f++)
#pragma unroll
            for (int i = 0; i < DT; i++) o[i] = M::mul32(value(i, f), p[f], o[i]);
    };

    uint8_t* const buf0 = hh_attn_lds<0, BYTES>();
    uint8_t* const buf1 = hh_attn_lds<1, BYTES>();
    if (t0 < t1) {
        ask_k(t0);
        ask_v(t0);
        copy_k(buf0, t0);
        copy_v(buf0 + KBYTES, t0);
        ask_k(t0 + 1);
        ask_v(t0 + 1);
    }
    for (uint32_t t = t0; t < t1; t += 2) {
        hh_attn_meet();
        if (t + 1 < t1) {
            copy_k(buf1, t + 1);
            copy_v(buf1 + KBYTES, t + 1);
        }
        ask_k(t + 2);
        ask_v(t + 2);
        compute(buf0, t);
        if (t + 1 >= t1) break;
        hh_attn_meet();
        if (t + 2 < t1) {
            copy_k(buf0, t + 2);
            copy_v(buf0 + KBYTES, t + 2);
        }
        ask_k(t + 3);
        ask_v(t + 3);
        compute(buf1, t + 1);
    }

    sum += __shfl_xor(sum, 32);
    odd = __syncthreads_or(odd != 0);
    if (r >= rows) return;
    // what the crossed tiles left out, added for the row's own keys: to element d of this half's
    auto left_out = [&](auto add) {
        for (uint32_t key = max(least / BN, t0) * BN; key < min(limit, t1 * BN); key++) {
            const uint32_t id = hh_page(table, key, shift, entries);
            if (id >= a.kv.pages) continue;
            const uint8_t* page = a.kv.base + id * a.kv.stride;
            for (uint32_t d = hf * 4; d < dim; d += 8)
                for (uint32_t x = d; x < d + 4; x++) {
                    const float v = C::get(((const CE*)(page + hh_kv_value<C>(a.kv, kvh, x)))[key & ((1u << shift) - 1)]);
                    if (!__builtin_isfinite(v)) add(x, v);
                }
        }
    };
    if (!CAUSAL || splits > 1) {
        const size_t part = (size_t)at * a.splits + split;
        float* const po = a.part + (part * 128 + r) * DP;
#pragma unroll
        for (int i = 0; i < DT; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                *(hh_f32x4*)(po + i * 32 + j * 8 + hf * 4) = hh_f32x4{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
        if (odd) left_out([&](uint32_t d, float v) { po[d] += v; });
        if (hf == 0) {
            a.part_sum[2 * (part * 128 + r)] = base;
            a.part_sum[2 * (part * 128 + r) + 1] = sum;
        }
        return;
    }
    const float by = 1.f / sum;  // (weights of 0 alone: 0 * inf, NaN)
    E* const out = (E*)a.out + (size_t)(tile.start + tok) * a.out_stride + head * dim;
#pragma unroll
    for (int i = 0; i < DT; i++)
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            E v[2][4];
#pragma unroll
            for (int x = 0; x < 8; x++) v[x / 4][x % 4] = A::put(limit == 0 ? 0.f : o[i][4 * j + x] * by);
            if (sizeof(E) == 4) {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t d = i * 32 + (j + k) * 8 + hf * 4;
                    if (FULL || d < dim) hh_store_n(out + d, v[k]);
                }
            } else {  // 8 bytes of j and j + 1 here and in the row's other half: 16 of one of them in each
                uint32_t u[2][2];
                __builtin_memcpy(u, v, 16);
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const auto both = __builtin_amdgcn_permlane32_swap(u[0][k], u[1][k], false, false);
                    u[0][k] = both[0];
                    u[1][k] = both[1];
                }
                E w[8];
                __builtin_memcpy(w, u, 16);
                const uint32_t d = i * 32 + (j + hf) * 8;
                if (FULL || d < dim) hh_store_n(out + d, w);
            }
        }
    if (odd) {
        __threadfence();  // (some of these elements were stored by the row's other half)
        left_out([&](uint32_t d, float v) { out[d] = A::put(A::get(out[d]) + v); });
    }
}

// Two runs of a row's parts, joined: sum_i f_i o_i / sum_i f_i s_i, f_i = exp2(base_i - max base), by `teams` (a power of
// two) of the workgroup's teams of DP / 4 threads, which hold 4 elements each and take every teams-th part; all threads
// call it, and the first team's store the row.  A part that saw no key, or none with a weight, has sum 0 and is left out (its o
// may hold 0 * NaN).  any_key: the row saw one; if none had a weight it is 0 / 0, NaN, as it would be in one part.
struct hh_attn_parts {
    const float *o, *s;  // the first part's elements, base and sum
    uint32_t n;
    size_t step;  // rows from a part to the next
};
template <class A, int DP>
HH_DEV void hh_attn_join_row(const hh_attn_parts& x, const hh_attn_parts& y, uint32_t teams, bool any_key, bool store, typename A::E* out) {
    typedef typename A::E E;
    constexpr uint32_t L = DP / 4, N = 256 / L;
    const uint32_t team = threadIdx.x / L, d = threadIdx.x % L * 4;
    float top = HH_ATTN_LOWEST, sum = 0;
    hh_f32x4 o = {0, 0, 0, 0};
#pragma unroll 4
    for (uint32_t i = team % teams; i < x.n + y.n; i += teams) {
        const bool late = i >= x.n;
        const size_t at = late ? (i - x.n) * y.step : i * x.step;
        const float* sums = (late ? y.s : x.s) + 2 * at;
        const hh_f32x4 v = *(const hh_f32x4*)((late ? y.o : x.o) + at * DP + d);
        const float b = sums[0], w = sums[1];
        const bool any = w != 0;
        const float next = any ? fmaxf(top, b) : top, f = hh_exp2(top - next), g = hh_exp2(b - next);
        top = next;
        sum = any ? fmaf(w, g, sum * f) : sum;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = any ? fmaf(v[e], g, o[e] * f) : o[e];
    }
    __shared__ float tops[N], weights[N];
    __shared__ hh_f32x4 red[256];
    red[threadIdx.x] = o;
    if (d == 0) {
        tops[team] = top;
        weights[team] = sum;
    }
    __syncthreads();
    if (team % teams || !store) return;
    for (uint32_t i = 1; i < teams; i++) top = fmaxf(top, tops[team + i]);
    o = hh_f32x4{0, 0, 0, 0};
    sum = 0;
    for (uint32_t i = 0; i < teams; i++) {
        const float f = hh_exp2(tops[team + i] - top);
        sum = fmaf(weights[team + i], f, sum);
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = fmaf(red[i * L + threadIdx.x][e], f, o[e]);
    }
    const float by = any_key ? 1.f / sum : 0.f;
    E v[4];
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] = A::put(o[e] * by);
    hh_store_n(out + d, v);
}

#endif
