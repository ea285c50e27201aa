// Causal attention of a prompt's tokens over their sequences' pages.
//   out[t][h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t][h] . k_j),  j <= position of t
// A workgroup takes 128 rows: the heads that share a kv head, of as many neighbouring tokens as fit (32
// tokens of 4 heads).  Its four waves hold 32 rows each, as queries Q^T and sums O^T in registers, and go
// through the keys in tiles that all of them read from LDS; the next tile is copied there meanwhile.  Weights go
// from the first product's result to the second's operand inside a lane (attn_tiles.h).
//
// Weights are rounded to the cache's type for the second product (by up to 2^-8 of each for bf16, 2^-11 for f16;
// f32 keeps them): the matrix cores take both operands in one type.  Sums of weights and outputs are f32.
//
// Tiles in which some row sees fewer keys than another are masked by comparison.  There values that are no
// finite numbers are left out of the product (0 * inf would be NaN in rows that do not see the key) and
// added afterwards to the rows that see them, whose result they alone decide.
#include "attn_rows.h"

// Which tile is number `slot`.  Up to 64 sequences: the one that sees the slot-th most keys, so that the longest tiles go
// first and share their CU with short ones (7 sequences of 82 to 490 tokens,
// 32/8 heads of 128 bf16: 22.8 us, in their own order 27.3).  More: sequence s
// has the slots from starts[s] / tile_tokens + s on, as many as it can have tiles, and its later tiles go first.
HH_DEV bool hh_attn_find(const hh_attn_prompt_args& p, uint32_t slot, uint32_t lane, hh_attn_tile& t) {
    const hh_attn_args& a = p.a;
    auto start = [&](uint32_t s) { return (uint32_t)max(0, min((int)p.tokens, p.starts[s])); };
    uint32_t lo = 0, hi = a.seqs, from, to;
    int len;
    if (a.seqs > 1 && a.seqs <= HH_WAVE) {
        // A sequence a lane.  Its last tile weighs e (as many tiles of keys), the one before e - 1, ...: find the weight x
        // of tile number `slot` in descending order and which of the sequences that have a tile of it.
        const bool real = lane < a.seqs;
        const uint32_t s = min(lane, a.seqs - 1);
        from = start(s);
        to = start(s + 1);
        len = min((int64_t)max(0, a.lens[s]), (int64_t)a.entries << a.kv.shift);
        const uint32_t n = real && to > from ? (to - from + a.tile_tokens - 1) / a.tile_tokens : 0;
        const uint32_t e = n ? max(n, (len + a.tile_tokens - 1) / a.tile_tokens) : 0;
        auto above = [&](uint32_t x) { return hh_wave_sum32(e >= x ? min(e - x + 1, n) : 0); };  // tiles of x or more, x > 0
        if (slot >= above(1)) return false;
        uint32_t x = 1, y = hh_wave_max32(e) + 1;  // above(x) > slot >= above(y)
        while (y - x > 1) {
            const uint32_t m = x + (y - x) / 2;
            if (above(m) > slot)
                x = m;
            else
                y = m;
        }
        const uint64_t with = __ballot(x <= e && x + n > e);
        const uint32_t nth = slot - above(x + 1);
        const uint32_t at = __builtin_ctzll(__ballot((with >> lane & 1) && __popcll(with & ((1ull << lane) - 1)) == nth));
        t.seq = at;
        t.start = __builtin_amdgcn_readlane(from, at);
        t.tokens = __builtin_amdgcn_readlane(to, at) - t.start;
        t.first = (__builtin_amdgcn_readlane(n, at) - 1 - (__builtin_amdgcn_readlane(e, at) - x)) * a.tile_tokens;
        t.len = __builtin_amdgcn_readlane(len, at);
        return true;
    }
    for (;;) {  // 64 sequences at a time, one a lane
        const uint32_t step = (hi - lo + 63) / 64, s = lo + lane * step, here = min(s, a.seqs - 1);
        const uint32_t f = start(here), e = start(here + 1);  // (asked for at once: one latency)
        const int n = a.lens[here];
        const bool before = s < hi && f / a.tile_tokens + s <= slot;
        const uint32_t at = max(1, __popcll(__ballot(before))) - 1;
        from = __builtin_amdgcn_readlane(f, at);
        to = __builtin_amdgcn_readlane(e, at);
        len = __builtin_amdgcn_readlane(n, at);
        lo += at * step;
        if (step == 1) break;
        hi = min(lo + step, hi);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    const uint32_t at = from / a.tile_tokens + lo;
    t.seq = lo;
    t.start = from;
    t.tokens = to > from ? to - from : 0;
    if (slot < at || (uint64_t)(slot - at) * a.tile_tokens >= t.tokens) return false;
    t.first = (slot - at) * a.tile_tokens;
    t.len = (uint32_t)min((int64_t)max(0, len), (int64_t)a.entries << a.kv.shift);
    return true;
}

// The workgroup's tile and part: a tile's parts and kv heads next to each other (kv heads go round the XCDs), the tiles with the
// most keys first.  From p.turn on the least come first, where the chip holds all: the second workgroup of a CU that has one of
// the longest is one of the shortest (us, so and all in descending order: 1000 tokens, 32/8 heads of 80 f32: 79.0, 96.7; 1500
// of 64 f32: 119, 140; 1500 of 128 bf16: 43.4, 45.4).
struct hh_attn_place {
    uint32_t kvh, slot, split;
};
HH_DEV hh_attn_place hh_attn_place_of(const hh_attn_prompt_args& p, uint32_t block, uint32_t blocks) {
    uint32_t i = block / p.a.kv.heads;
    if (i >= p.turn) i = blocks / p.a.kv.heads - 1 - (i - p.turn);
    const uint32_t tile = i / p.a.splits;
    return {block % p.a.kv.heads, p.a.seqs > 1 && p.a.seqs <= HH_WAVE ? tile : p.slots - 1 - tile, i % p.a.splits};
}

// In how many parts a tile takes its keys: what the host found best for a full table, but none without a tile of
// keys, and one for few: it needs no join (us, with empty parts in brackets: 100 tokens in a table for 32000, 32/8 heads of
// 128 bf16: 13.4 [22.0]; 300: 24.0 [28.5]; 30 behind 1000: 13.8 [14.8]; 1000 behind 1000 in their own: 56.4 [54.7]).
HH_DEV uint32_t hh_attn_splits(const hh_attn_prompt_args& p, const hh_attn_tile& t) {
    const uint32_t to = min(t.first + p.a.tile_tokens, t.tokens);
    const uint32_t keys = hh_attn_seen(t, to - 1);
    const uint32_t tiles = (keys + (1u << p.step) - 1) >> p.step;
    return keys > p.whole ? min(p.a.splits, tiles) : 1;
}

template <class A, class C, int DP, int DU>
HH_DEV void hh_attn_prompt(const hh_attn_prompt_args& p) {
    const hh_attn_place at = hh_attn_place_of(p, blockIdx.x, gridDim.x);
    hh_attn_tile tile;
    if (!hh_attn_find(p, at.slot, threadIdx.x % HH_WAVE, tile)) return;
    const uint32_t splits = hh_attn_splits(p, tile);
    if (at.split >= splits) return;
    hh_attn_rows<A, C, DP, DU, true>(p.a, tile, p.a.tables + (size_t)tile.seq * p.a.entries, p.a.entries, at.kvh,
                                     at.slot * p.a.kv.heads + at.kvh, at.split, splits);
}

// The parts of rows whose keys were split, joined.
template <class A, int DP>
HH_DEV void hh_attn_prompt_join(const hh_attn_prompt_args& p) {
    const hh_attn_args& a = p.a;
    const uint32_t kvh = blockIdx.x % a.kv.heads, slot = blockIdx.x / a.kv.heads;
    hh_attn_tile tile;
    if (!hh_attn_find(p, slot, threadIdx.x % HH_WAVE, tile)) return;
    const uint32_t rows = min(a.tile_tokens, tile.tokens - tile.first) * a.group, splits = hh_attn_splits(p, tile);
    if (splits == 1) return;
    constexpr uint32_t N = 1024 / DP;
    uint32_t teams = 1;  // a row
    while (teams < N && teams < a.splits) teams *= 2;
    const uint32_t r = blockIdx.y * (N / teams) + threadIdx.x / (DP / 4) / teams, at = min(r, rows - 1);
    if (blockIdx.y * (N / teams) >= rows) return;
    const size_t row = ((size_t)slot * a.kv.heads + kvh) * a.splits * 128 + at;
    const hh_attn_parts parts = {a.part + row * DP, a.part_sum + row * 2, splits, 128};
    typename A::E* const out = (typename A::E*)a.out + (size_t)(tile.start + tile.first + at / a.group) * a.out_stride +
                               (kvh * a.group + at % a.group) * a.kv.dim;
    hh_attn_join_row<A, DP>(parts, hh_attn_parts{}, teams, hh_attn_seen(tile, tile.first + at / a.group) != 0,
                            r < rows && threadIdx.x % (DP / 4) * 4 < a.kv.dim, out);
}

#define HH_ATTN_PROMPT(N, A, C, D, DU, NAME)                                                                                    \
    extern "C" __global__ void __launch_bounds__(256, HH_ATTN_PER_CU(C, (DU) ? (DU) : (D))) hh_attn_prompt_##NAME##_##N(const hh_attn_prompt_args a) { \
        hh_attn_prompt<A, C, D, DU>(a);                                                                                         \
    }
#define HH_ATTN_PROMPTS(N, A, C) HH_ATTN_DIMS(HH_ATTN_PROMPT, N, A, C)
HH_ATTN_PROMPTS(f32, hh_af32, hh_af32)
HH_ATTN_PROMPTS(f16, hh_af16, hh_af16)
HH_ATTN_PROMPTS(bf16, hh_abf16, hh_abf16)
HH_ATTN_PROMPTS(f32_f16, hh_af32, hh_af16)
HH_ATTN_PROMPTS(f32_bf16, hh_af32, hh_abf16)
#define HH_ATTN_PROMPT_JOIN(N, A, D) \
    extern "C" __global__ void __launch_bounds__(256) hh_attn_prompt_join_##D##_##N(const hh_attn_prompt_args a) { hh_attn_prompt_join<A, D>(a); }
#define HH_ATTN_PROMPT_JOINS(N, A) HH_ATTN_PROMPT_JOIN(N, A, 64) HH_ATTN_PROMPT_JOIN(N, A, 128) HH_ATTN_PROMPT_JOIN(N, A, 256)
HH_ATTN_PROMPT_JOINS(f32, hh_af32)
HH_ATTN_PROMPT_JOINS(f16, hh_af16)
HH_ATTN_PROMPT_JOINS(bf16, hh_abf16)
