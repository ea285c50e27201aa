// Attention of one token a sequence over its pages, for a batch whose sequences begin with the same `prefix`
// tokens: out[s][h] = sum_j p_j v_j / sum_j p_j over all tokens j of sequence s.
//
// The shared tokens are taken once for all: tiles of 128 rows (32 sequences' 4 heads) against the prefix's
// pages, as a prompt's are (attn_rows.h), their keys in parts.  A sequence's own tokens are read by workgroups
// of one kv head's up to 16 heads, memory bound: keys and values go from the pages straight into operands of
// the 16-column matrix products (attn_tiles.h), 16 KB in flight a wave, each of the four waves every fourth
// step of 32 keys (16 of f32), joined through LDS at the end.  Lengths are known on the device alone, so every workgroup sums them up
// and finds the piece of work that falls to it: pieces are of equal length whatever the sequences' are.  A second kernel joins the parts of a row.
//
// Weights are rounded to the cache's type for the second product (by up to 2^-8 of each for bf16, 2^-11 for f16); sums and
// the parts are f32.
#include "attn_rows.h"

#define HH_ATTN_UNIT 128u  // keys a piece is a multiple of
#define HH_ATTN_MOST 64u   // pieces of a sequence

// Tokens of sequence s that are not taken with the shared ones, and the first of them.  A sequence shorter than the caller's
// prefix has none of its tokens in those pages, also where it reaches the whole tiles of it that are taken apart.
HH_DEV uint32_t hh_attn_own(const hh_attn_decode_args& p, uint32_t s, uint32_t& from) {
    const uint32_t len = (uint32_t)min((int64_t)max(0, p.a.lens[s]), (int64_t)p.a.entries << p.a.kv.shift);
    from = len >= p.sharing ? p.prefix : 0;
    return len - from;
}

struct hh_attn_piece {
    uint32_t seq, at, count, units;  // the at-th of the sequence's `count` pieces of `units` units
};
// Piece number `piece`; the first workgroup leaves the plan for the join.  (32-bit sums: the host bounds what the tables
// have room for.)
HH_DEV bool hh_attn_plan(const hh_attn_decode_args& p, uint32_t piece, bool first, hh_attn_piece& out) {
    __shared__ uint32_t red[8], sums[4];
    __shared__ hh_attn_piece found;
    const uint32_t tid = threadIdx.x, lane = tid % HH_WAVE, wave = tid / HH_WAVE;
    // a sequence's units, and how many of them count: one that is shorter than the prefix has longer pieces
    auto units = [&](uint32_t s) {
        uint32_t from;
        return s < p.a.seqs ? (hh_attn_own(p, s, from) + HH_ATTN_UNIT - 1) / HH_ATTN_UNIT : 0;
    };
    uint32_t all = 0;
    for (uint32_t s = tid; s < p.a.seqs; s += 256) all += min(units(s), p.room);
    all = (uint32_t)hh_wave64<hh_addu64>(all);
    if (lane == 0) sums[wave] = all;
    if (tid == 0) found.count = 0;
    __syncthreads();
    all = sums[0] + sums[1] + sums[2] + sums[3];
    // Units a piece: four (one sequence of 4000: 7.7 us, with two 9.2), fewer where that would leave CUs without one, more
    // where pieces would be too many in all or, for the join, in one sequence.
    const uint32_t each = max((all + p.pieces - 1) / p.pieces, min(4u, max(1u, all / p.least)));
    uint32_t before = 0;
    for (uint32_t s0 = 0; s0 < p.a.seqs; s0 += 256) {
        const uint32_t s = s0 + tid, own = units(s), most = min(HH_ATTN_MOST, (p.room + each - 1) / each);
        const uint32_t size = max(each, (own + max(1u, most) - 1) / max(1u, most));
        const uint32_t n = s < p.a.seqs ? max(1u, (own + size - 1) / size) : 0, scan = (uint32_t)hh_scan64(n);
        uint32_t* const part = red + (s0 / 256 & 1) * 4;
        if (lane == HH_WAVE - 1) part[wave] = scan;
        __syncthreads();
        uint32_t at = before + scan - n;
        for (uint32_t w = 0; w < 4; w++) {
            if (w < wave) at += part[w];
            before += part[w];
        }
        if (piece - at < n) found = hh_attn_piece{s, piece - at, n, size};
        if (first && s < p.a.seqs) {
            p.plan[2 * s] = at;
            p.plan[2 * s + 1] = n;
        }
    }
    __syncthreads();
    out = found;
    return out.count != 0;
}

template <class A, class C, int DP, int DU>
HH_DEV void hh_attn_single(const hh_attn_decode_args& p, uint32_t block) {
    typedef typename A::E E;
    typedef typename C::E CE;
    typedef hh_mat<C> M;
    typedef typename M::frag F;
    constexpr float LIFT = hh_attn_lift<C>();
    constexpr int EF = C::VEC, SZ = sizeof(CE), STEP = 4 * EF, KT = STEP / 16, D = DU ? DU : DP, NC = D / (4 * EF), DT = D / 16;
    constexpr bool FULL = DU == 0;
    const hh_attn_args& a = p.a;
    const uint32_t lane = threadIdx.x % HH_WAVE, ln = lane % 16, g = lane / 16;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / HH_WAVE);
    const uint32_t kvh = block % a.kv.heads, rt = block / a.kv.heads % p.row_tiles, number = block / a.kv.heads / p.row_tiles;
    const uint32_t dim = FULL ? DP : a.kv.dim, shift = a.kv.shift, mask = (1u << shift) - 1;
    hh_attn_piece piece;
    if (!hh_attn_plan(p, number, block == 0, piece)) return;
    uint32_t from;
    const uint32_t own = hh_attn_own(p, piece.seq, from);
    const uint32_t k0 = min(own, piece.at * piece.units * HH_ATTN_UNIT) + from;
    const uint32_t k1 = min((uint64_t)own, (uint64_t)(piece.at + 1) * piece.units * HH_ATTN_UNIT) + from;
    const bool alone = piece.count == 1 && (p.prefix == 0 || from == 0);
    const int32_t* const table = a.tables + (size_t)piece.seq * a.entries;

    const uint32_t head = kvh * a.group + min(rt * 16 + ln, a.group - 1);
    F q[NC];
    const E* qrow = (const E*)a.q + (size_t)piece.seq * a.q_stride + head * dim;
#pragma unroll
    for (int c = 0; c < NC; c++) q[c] = hh_query<A, C, FULL>(qrow, (4 * c + g) * EF, dim, true);

    // row ln of K's t-th tile is key 8 (ln / 4) + 4 t + ln % 4 of 16-bit types, so that a lane's scores are of keys EF g ..
    const uint32_t krow = SZ == 4 ? ln : 8 * (ln / 4) + ln % 4;
    uint32_t id_k = 0, id_v = 0;
    auto ask = [&](uint32_t k) {
        id_k = hh_page(table, k + krow, shift, a.entries);
        id_v = hh_page(table, k + EF * g, shift, a.entries);
    };
    F kf[KT][NC], vf[DT];
    auto load_k = [&](uint32_t k, uint32_t id) {
        const uint8_t* page = a.kv.base + (id < a.kv.pages ? id : 0) * a.kv.stride + g * 16;
#pragma unroll
        for (int t = 0; t < KT; t++) {
            const uint8_t* row = page + hh_kv_key<C>(a.kv, kvh, (k + krow + 4 * t) & mask);
#pragma unroll
            for (int c = 0; c < NC; c++) {
                const bool in = FULL || (4 * c + g) * EF < dim;
                kf[t][c] = *(const F*)(in ? row + c * 64 : row - g * 16);
            }
        }
    };
    auto load_v = [&](uint32_t k, uint32_t id) {
        const uint8_t* page = a.kv.base + (id < a.kv.pages ? id : 0) * a.kv.stride + ((k + EF * g) & mask) * SZ;
#pragma unroll
        for (int i = 0; i < DT; i++)
            vf[i] = *(const F*)(page + hh_kv_value<C>(a.kv, kvh, FULL ? i * 16 + ln : min(i * 16 + ln, dim - 1)));
    };

    hh_f32x4 o[DT];
#pragma unroll
    for (int i = 0; i < DT; i++) o[i] = hh_f32x4{0, 0, 0, 0};
    float base = HH_ATTN_LOWEST, sum = 0;
    uint32_t k = k0 + wave * STEP;
    bool zero_k = false, zero_v = false;
    if (k < k1) {
        ask(k);
        load_k(k, id_k);
        zero_k = id_k >= a.kv.pages;
    }
    for (; k < k1; k += 4 * STEP) {
        load_v(k, id_v);
        zero_v = id_v >= a.kv.pages;
        const bool more = k + 4 * STEP < k1;
        if (more) ask(k + 4 * STEP);
        if (!FULL || __any(zero_k)) {
#pragma unroll
            for (int t = 0; t < KT; t++)
#pragma unroll
                for (int c = 0; c < NC; c++)
                    if (zero_k || (!FULL && (4 * c + g) * EF >= dim)) kf[t][c] = F{};
        }
        float s[EF];
#pragma unroll
        for (int t = 0; t < KT; t++) {
            hh_f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < NC; c++) acc = M::mul16(kf[t][c], q[c], acc);
#pragma unroll
            for (int x = 0; x < 4; x++) s[4 * t + x] = acc[x];
        }
        if (more) {
            load_k(k + 4 * STEP, id_k);
            zero_k = id_k >= a.kv.pages;
        }
        const bool last = k + STEP > k1;
        if (last) {
#pragma unroll
            for (int x = 0; x < EF; x++) s[x] = k + EF * g + x < k1 ? s[x] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int x = 1; x < EF; x++) top = fmaxf(top, s[x]);
        top *= a.c;
        if (__any(top > base + (HH_ATTN_SLACK + LIFT))) {
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            const float next = top > base + (HH_ATTN_SLACK + LIFT) ? top - LIFT : base, f = hh_exp2(base - next);
            base = next;
            sum *= f;
#pragma unroll
            for (int i = 0; i < DT; i++)
#pragma unroll
                for (int x = 0; x < 4; x++) o[i][x] *= f;
        }
        F w;
#pragma unroll
        for (int x = 0; x < EF; x++) {
            s[x] = hh_exp2(fmaf(s[x], a.c, -base));
            w[x] = C::put(s[x]);
        }
#pragma unroll
        for (int n = EF / 2; n > 0; n /= 2)
#pragma unroll
            for (int x = 0; x < n; x++) s[x] += s[x + n];
        sum += s[0];
        if (last || __any(zero_v)) {
#pragma unroll
            for (int i = 0; i < DT; i++) vf[i] = hh_first<C>(vf[i], zero_v ? 0 : (int)(k1 - k) - (int)(EF * g));
        }
#pragma unroll
        for (int i = 0; i < DT; i++) o[i] = M::mul16(vf[i], w, o[i]);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);

    // the waves' sums, joined: 4-element chunk c of row r lies at chunk c ^ r % 8
    __shared__ float bases[4][16], weights[4][16];
    hh_f32x4* const red = (hh_f32x4*)hh_attn_lds<0, hh_attn_bytes<C, DP, DU>()>();
    static_assert(64 * D * 4 <= hh_attn_bytes<C, DP, DU>(), "the sums fit the tile's buffer");
    if (lane < 16) {
        bases[wave][lane] = base;
        weights[wave][lane] = sum;
    }
    __syncthreads();
    const float top = fmaxf(fmaxf(bases[0][ln], bases[1][ln]), fmaxf(bases[2][ln], bases[3][ln])), f = hh_exp2(base - top);
#pragma unroll
    for (int i = 0; i < DT; i++)
        red[(wave * 16 + ln) * (D / 4) + ((i * 4 + g) ^ ln % 8)] = o[i] * f;
    __syncthreads();
    const size_t rows = ((size_t)number * p.row_tiles + rt) * a.kv.heads + kvh;
#pragma unroll
    for (uint32_t at = threadIdx.x; at < 4 * D; at += 256) {
        const uint32_t r = at / (D / 4), c = at % (D / 4), d = c * 4;
        if (rt * 16 + r >= a.group || d >= dim) continue;
        const float t = fmaxf(fmaxf(bases[0][r], bases[1][r]), fmaxf(bases[2][r], bases[3][r]));
        float total = 0;
        hh_f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            total = fmaf(weights[w][r], hh_exp2(bases[w][r] - t), total);
            v += red[(w * 16 + r) * (D / 4) + (c ^ r % 8)];
        }
        if (alone) {
            const float by = own ? 1.f / total : 0.f;  // (weights of 0 alone: 0 * inf, NaN)
            E e[4];
#pragma unroll
            for (int x = 0; x < 4; x++) e[x] = A::put(v[x] * by);
            hh_store_n((E*)a.out + (size_t)piece.seq * a.out_stride + (kvh * a.group + rt * 16 + r) * dim + d, e);
        } else {
            *(hh_f32x4*)(p.piece + (rows * 16 + r) * DP + d) = v;
            if (d == 0) {
                p.piece_sum[2 * (rows * 16 + r)] = t;
                p.piece_sum[2 * (rows * 16 + r) + 1] = total;
            }
        }
    }
}

// The shared tokens' tiles first, then the sequences' own pieces.
template <class A, class C, int DP, int DU>
HH_DEV void hh_attn_shared(const hh_attn_decode_args& p) {
    const hh_attn_args& a = p.a;
    const uint32_t ahead = p.tiles * a.kv.heads * a.splits;
    if (blockIdx.x >= ahead) {
        hh_attn_single<A, C, DP, DU>(p, blockIdx.x - ahead);
        return;
    }
    const uint32_t kvh = blockIdx.x % a.kv.heads, tile = blockIdx.x / a.kv.heads % p.tiles, split = blockIdx.x / a.kv.heads / p.tiles;
    hh_attn_rows<A, C, DP, DU, false>(a, hh_attn_tile{0, 0, tile * a.tile_tokens, a.seqs, p.prefix}, p.shared,
                                        p.shared_entries, kvh, tile * a.kv.heads + kvh, split, a.splits);
}

// A row's parts, joined: one head of a sequence a workgroup.
template <class A, int DP>
HH_DEV void hh_attn_join(const hh_attn_decode_args& p) {
    const hh_attn_args& a = p.a;
    const uint32_t heads = a.kv.heads * a.group, s = blockIdx.x / heads, head = blockIdx.x % heads;
    const uint32_t kvh = head / a.group, r = head % a.group;
    const uint32_t first = p.plan[2 * s], count = p.plan[2 * s + 1];
    uint32_t from;
    const uint32_t own = hh_attn_own(p, s, from);
    const uint32_t splits = p.prefix && from ? a.splits : 0;
    if (splits == 0 && count == 1) return;
    const size_t row0 = ((size_t)(s / a.tile_tokens) * a.kv.heads + kvh) * a.splits * 128 + s % a.tile_tokens * a.group + r;
    const size_t row1 = (((size_t)first * p.row_tiles + r / 16) * a.kv.heads + kvh) * 16 + r % 16;
    hh_attn_join_row<A, DP>(hh_attn_parts{a.part + row0 * DP, a.part_sum + row0 * 2, splits, 128},
                            hh_attn_parts{p.piece + row1 * DP, p.piece_sum + row1 * 2, count, (size_t)p.row_tiles * a.kv.heads * 16},
                            1024 / DP, from + own != 0, threadIdx.x % (DP / 4) * 4 < a.kv.dim,
                            (typename A::E*)a.out + (size_t)s * a.out_stride + head * a.kv.dim);
}

#define HH_ATTN_DECODE(N, A, C, D, DU, NAME)                                                                                    \
    extern "C" __global__ void __launch_bounds__(256, HH_ATTN_PER_CU(C, (DU) ? (DU) : (D))) hh_attn_decode_##NAME##_##N(const hh_attn_decode_args p) { \
        hh_attn_single<A, C, D, DU>(p, blockIdx.x);                                                                             \
    }                                                                                                                           \
    extern "C" __global__ void __launch_bounds__(256, HH_ATTN_PER_CU(C, (DU) ? (DU) : (D))) hh_attn_shared_##NAME##_##N(const hh_attn_decode_args p) { \
        hh_attn_shared<A, C, D, DU>(p);                                                                                         \
    }
#define HH_ATTN_DECODES(N, A, C) HH_ATTN_DIMS(HH_ATTN_DECODE, N, A, C)
HH_ATTN_DECODES(f32, hh_af32, hh_af32)
HH_ATTN_DECODES(f16, hh_af16, hh_af16)
HH_ATTN_DECODES(bf16, hh_abf16, hh_abf16)
HH_ATTN_DECODES(f32_f16, hh_af32, hh_af16)
HH_ATTN_DECODES(f32_bf16, hh_af32, hh_abf16)
#define HH_ATTN_JOIN(N, A, D) \
    extern "C" __global__ void __launch_bounds__(256) hh_attn_join_##D##_##N(const hh_attn_decode_args p) { hh_attn_join<A, D>(p); }
#define HH_ATTN_JOINS(N, A) HH_ATTN_JOIN(N, A, 64) HH_ATTN_JOIN(N, A, 128) HH_ATTN_JOIN(N, A, 256)
HH_ATTN_JOINS(f32, hh_af32)
HH_ATTN_JOINS(f16, hh_af16)
HH_ATTN_JOINS(bf16, hh_abf16)
