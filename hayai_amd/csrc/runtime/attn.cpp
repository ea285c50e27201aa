// Dispatch of the attention operators: rotary positions into the cache (rope.hip), copies of its
// pages (kv_pages.hip), attention of prompts (attn_prompt.hip) and of decode batches (attn_decode.hip).
#include <algorithm>

#include "engine.h"

namespace hh {

std::string attn_types(int type, int kv_type) {
    std::string s = act_type(type)->name;
    return kv_type == type ? s : s + "_" + act_type(kv_type)->name;
}

static const int kAttnTypes[][2] = {{HH_TYPE_F32, HH_TYPE_F32}, {HH_TYPE_F16, HH_TYPE_F16}, {HH_TYPE_BF16, HH_TYPE_BF16},
                                    {HH_TYPE_F32, HH_TYPE_F16}, {HH_TYPE_F32, HH_TYPE_BF16}};

void attn_kernels(std::vector<std::string>& k) {
    for (auto& t : kAttnTypes) {
        const std::string ty = attn_types(t[0], t[1]);
        for (const char* v : {"halves_", "pairs_", "halves8_", "pairs8_"}) k.push_back(std::string("hh_rope_") + v + ty);
        for (const char* v : {"64_", "64_any_", "96_any_", "128_", "128_any_", "256_", "256_any_"})
            for (const char* kind : {"hh_attn_prompt_", "hh_attn_decode_", "hh_attn_shared_"})
                k.push_back(std::string(kind) + v + ty);
        for (const char* v : {"64_", "128_", "256_"})
            for (const char* kind : {"hh_attn_prompt_join_", "hh_attn_join_"})
                if (t[0] == t[1]) k.push_back(std::string(kind) + v + ty);
    }
    k.push_back("hh_kv_copy");
}

bool attn_kernel(const std::string& name) {
    for (const char* stem : {"hh_rope_", "hh_kv_", "hh_attn_"})
        if (name.rfind(stem, 0) == 0) return true;
    return false;
}

}  // namespace hh

using namespace hh;

hh_status hh_engine::enqueue_rope(int type, int kv_type, int layout, size_t tokens, const hh_rope_args& a) {
    hipFunction_t f;
    const size_t el = act_type(type)->bytes, cus = (size_t)props.multiProcessorCount;
    // Eight tokens a workgroup of 1024 threads from three tokens a CU on (32/8 heads of 128 bf16, us, eight and one: 512 tokens
    // 9.1, 8.4; 1024 tokens 10.1, 12.6; 4096 tokens 30, 51), else one a workgroup of 256, and of few tokens each is given to
    // several.
    const size_t each = tokens >= 3 * cus ? 8 : 1;
    HH_TRY(kernel(std::string("hh_rope_") + (layout == HH_ROPE_PAIRS ? "pairs" : "halves") + (each == 8 ? "8_" : "_") +
                      attn_types(type, kv_type), &f));
    const size_t pieces = (a.heads + 2 * (size_t)a.kv.heads) * ((a.kv.dim * el + 15) / 16);
    const size_t parts = each == 8 ? 1 : std::max<size_t>(1, std::min((pieces + 255) / 256, 2 * cus / tokens));
    // a grid has fewer than 2^32 threads: 2^20 tokens at a time (parts are 1 there)
    for (size_t t = 0; t < tokens; t += (size_t)1 << 20) {
        const size_t n = std::min(tokens - t, (size_t)1 << 20);
        hh_rope_args p = a;
        p.tokens = (uint32_t)n;
        p.q = (const char*)a.q + t * a.q_stride * el;
        p.k = (const char*)a.k + t * a.k_stride * el;
        p.v = (const char*)a.v + t * a.v_stride * el;
        p.out = (char*)a.out + t * a.out_stride * el;
        p.positions = a.positions + t;
        p.slots = a.slots + t;
        void* params[] = {&p};
        HH_TRY_HIP(hipModuleLaunchKernel(f, (uint32_t)((n + each - 1) / each), (uint32_t)parts, 1, each == 8 ? 1024 : 256, 1, 1, 0,
                                         stream, params, nullptr),
                   "hipModuleLaunchKernel(rope)");
    }
    return HH_OK;
}

hh_status hh_engine::enqueue_kv_copy(size_t layers, const hh_kv_copy_args& a) {
    hipFunction_t f;
    HH_TRY(kernel("hh_kv_copy", &f));
    const size_t cus = (size_t)props.multiProcessorCount, blocks = (a.chunks + 255) / 256;
    // Moves are also split where the pages' pieces give fewer than eight workgroups a CU, and a bit for each page
    // fits 32 KB of LDS.
    size_t parts = 1, lds = 0;
    if (a.kv.pages <= (1u << 18) && blocks * layers < 8 * cus) {
        parts = std::min<size_t>((a.n + 7) / 8, 8 * cus / (blocks * layers));
        if (parts > 1) lds = (a.kv.pages + 31) / 32 * 4;
    }
    hh_kv_copy_args p = a;
    void* params[] = {&p};
    HH_TRY_HIP(hipModuleLaunchKernel(f, (uint32_t)blocks, (uint32_t)layers, (uint32_t)std::max<size_t>(parts, 1), 256, 1, 1,
                                     (unsigned)lds, stream, params, nullptr),
               "hipModuleLaunchKernel(kv_copy)");
    return HH_OK;
}

// Kernels are made for heads of 64, 128 and 256 elements, whole or with the rest as zeros, and for those of up to 96 laid
// out as 128 (us, computed as 96 and as 128: 3000 tokens, 32/8 heads of 80 bf16: 86.7, 96.5; 64 sequences of 2000: 74.3, 77.9).
static size_t padded_dim(size_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
static std::string dim_name(size_t dim) {
    if (dim > 64 && dim <= 96) return "96_any_";
    return std::to_string(padded_dim(dim)) + (dim == padded_dim(dim) ? "_" : "_any_");
}

// In how many parts the keys of a prompt's tiles are best taken, by an estimate in the time that a workgroup alone on its CU
// takes for one key (of 128 elements in 16 bits: 22 ns).  A part has keys / splits.  Two on a CU take 1.5 times as long (f32,
// bound by its products: twice) for the mean of the keys that tiles see, and no less than 1.25 times the longest.  Joining
// costs a launch (160) and writing and reading the parts' sums (2.3 a row and CU); a key of f32 takes about six times as long.
// Measured (us; 32/8 heads of 128 bf16, by splits, the one taken in brackets): 256 tokens behind 1000: 1: 34.9, 2: 28.3,
// 3: 27.9, [4: 26.3], 6: 31.4; behind 16000: 2: 186, 4: 110, [8: 97]; 512 behind 1000: 1: 40.7, [2: 34.9], 3: 39.5, 4: 37.0;
// 1024: [1: 30.0], 2: 36.2; behind 4000: 1: 115, [2: 104]; 1024 of 8/2 heads of 256: 1: 55.5, 2: 44.0, [4: 39.4], 6: 45.8;
// 100 f32 behind 1000: 4: 54.4, [8: 41.2], 12: 51.1, 16: 54.0.
static uint32_t prompt_splits(size_t tiles, size_t keys, size_t mean, size_t rows, size_t cus, size_t dp, bool f32) {
    const float unit = f32 ? 1 / 6.0f : 1.0f, both = f32 ? 2.0f : 1.5f;
    float least = 0;
    uint32_t best = 1;
    for (uint32_t s = 1; s == 1 || (s <= 64 && s * tiles <= 2 * cus && s * 16 <= keys); s++) {
        const float per_cu = (float)(s * tiles) / (float)cus;
        float cost = (float)keys / (float)s;
        if (per_cu > 1) cost = std::max(1.25f * cost, both * (float)mean / (float)s);
        if (s > 1) cost += unit * (160.0f * 128 / (float)dp + 2.3f * (float)(s * rows) / (float)cus);
        if (s == 1 || cost < least) least = cost, best = s;
    }
    return best;
}

hh_status hh_engine::enqueue_attn_prompt(int type, int kv_type, hh_attn_prompt_args p) {
    hh_attn_args& a = p.a;
    hipFunction_t f, join;
    const size_t dp = padded_dim(a.kv.dim), cus = (size_t)props.multiProcessorCount;
    const std::string name = "hh_attn_prompt_" + dim_name(a.kv.dim) + attn_types(type, kv_type);
    HH_TRY(kernel(name, &f));
    HH_TRY(kernel("hh_attn_prompt_join_" + std::to_string(dp) + "_" + act_type(type)->name, &join));
    a.tile_tokens = 128 / a.group;
    // as many tiles as the sequences can have: ranked by keys or, of more than a wave's lanes, each from its own slot on
    const size_t slots = a.seqs <= 64 ? (p.tokens + (size_t)a.seqs * (a.tile_tokens - 1)) / a.tile_tokens
                                      : (size_t)p.tokens / a.tile_tokens + a.seqs;
    const size_t tiles = slots * a.kv.heads;
    if (tiles >= 1u << 24) return fail(HH_ERR_INVALID, "attn_prompt: %u tokens of %u sequences are too many", p.tokens, a.seqs);
    p.slots = (uint32_t)slots;
    // Few tiles: their keys are split, for at most two workgroups a CU.
    const size_t keys = (size_t)a.entries << a.kv.shift;
    const size_t all_rows = (size_t)p.tokens * a.group * a.kv.heads;
    const bool f32 = act_type(kv_type)->bytes == 4;
    a.splits = prompt_splits(tiles, keys, keys - std::min<size_t>(keys, p.tokens / a.seqs / 2), all_rows, cus, dp, f32);
    p.step = f32 ? 5 : 6;
    p.whole = f32 ? 32 : 128;
    if (a.splits > 1) {
        const size_t rows = tiles * a.splits * 128;
        HH_TRY(grow(&ws_attn, &ws_attn_cap, rows * (dp + 2) * sizeof(float)));
        a.part = (float*)ws_attn;
        a.part_sum = a.part + rows * dp;
    }
    // Between one and two workgroups a CU, all there at once: the second ones in ascending order.
    const size_t blocks = tiles * a.splits;  // (2 cus at most where splits > 1)
    const bool pairs = blocks > cus && blocks <= 2 * cus && occupancy(name, 256) >= 2;
    p.turn = pairs ? (uint32_t)(cus / a.kv.heads) : UINT32_MAX;
    void* params[] = {&p};
    HH_TRY_HIP(hipModuleLaunchKernel(f, (uint32_t)blocks, 1, 1, 256, 1, 1, 0, stream, params, nullptr),
               "hipModuleLaunchKernel(attn_prompt)");
    size_t teams = 1;  // of dp / 4 threads a row
    while (teams < 1024 / dp && teams < a.splits) teams *= 2;
    if (a.splits > 1)
        HH_TRY_HIP(hipModuleLaunchKernel(join, (uint32_t)tiles, (uint32_t)(128 * teams * dp / 1024), 1, 256, 1, 1, 0, stream, params, nullptr),
                   "hipModuleLaunchKernel(attn_prompt_join)");
    return HH_OK;
}

hh_status hh_engine::enqueue_attn_decode(int type, int kv_type, hh_attn_decode_args p) {
    hh_attn_args& a = p.a;
    hipFunction_t f, join;
    const size_t dp = padded_dim(a.kv.dim), cus = (size_t)props.multiProcessorCount, heads = a.kv.heads;
    const size_t part_keys = act_type(kv_type)->bytes == 4 ? 64 : 256;  // (f32 products take eight times as long)
    // Shared tokens are taken apart, in whole tiles of keys, where that saves attn_share_min bytes of reading: more kernels' time
    // than it costs (us, apart and not; 8/2 heads of 128 bf16 unless said: 8 x 1024, 7 MB: 12.2, 9.6; 4 x 4096, 13 MB: 12.9,
    // 13.5; 30 x 1024, 30 MB: 14.4, 14.7; 60 x 600 of 9/3 heads of 64 f32, 54 MB: 14.3, 20.1; 2 x 8192 of 32/8, 34 MB: 15.9,
    // 23.1; 16 x 2048 of 32/8, 126 MB: 15.0, 29.1).
    const size_t token = 2 * heads * a.kv.dim * act_type(kv_type)->bytes;
    const bool apart = a.seqs > 1 && (double)(a.seqs - 1) * p.prefix * (double)token >= (double)attn_share_min;
    p.sharing = p.prefix;
    p.prefix = apart ? p.prefix / 64 * 64 : 0;
    const std::string name = (p.prefix ? "hh_attn_shared_" : "hh_attn_decode_") + dim_name(a.kv.dim) + attn_types(type, kv_type);
    HH_TRY(kernel(name, &f));
    HH_TRY(kernel("hh_attn_join_" + std::to_string(dp) + "_" + act_type(type)->name, &join));
    size_t ahead = 0, part_rows = 0;
    a.tile_tokens = 128 / a.group;  // (the join divides by it also where no tokens are taken apart)
    if (p.prefix) {
        p.tiles = (a.seqs + a.tile_tokens - 1) / a.tile_tokens;
        // parts for half the CUs, more where not all four waves have rows (2 sequences of 8192, 32/8 heads of 128 bf16: 32 parts
        // 15.8 us, 16 parts 18.9; 64: 8 parts 49, 16 parts 54)
        const size_t tiles = p.tiles * heads, waves = std::min<size_t>(4, ((size_t)a.seqs * a.group + 31) / 32);
        a.splits = (uint32_t)std::max<size_t>(1, std::min<size_t>(2 * cus / waves / tiles, p.prefix / part_keys));
        ahead = tiles * a.splits;
        part_rows = ahead * 128;
    }
    // The sequences' own tokens: the kernel makes pieces by the lengths (hh_attn_plan).  Each workgroup that is not
    // needed costs its look at the lengths, so that their number follows what the tables have room for: eight a CU for
    // long ones (64 sequences of 2000: 109 us, four 117), else four, in half the room (64 of 8192 + 500: 50 us either way).
    p.row_tiles = (a.group + 15) / 16;
    const size_t keys = (size_t)a.entries << a.kv.shift, room = ((keys > p.prefix ? keys - p.prefix : 0) + 127) / 128;
    const size_t least = std::max<size_t>(1, cus / (heads * p.row_tiles));
    if (a.seqs * heads * a.group >= 1u << 24 || std::max<size_t>(room, 1) * a.seqs >= 1u << 31)
        return fail(HH_ERR_INVALID, "attn_decode: %u sequences are too many", a.seqs);
    p.room = (uint32_t)room;
    p.least = (uint32_t)least;
    p.pieces = (uint32_t)std::min(std::max(room * a.seqs / 8, 4 * least), 8 * least);
    // (with fewer than four units a piece there are fewer than twice `least` of them)
    const size_t numbers = std::min(room * a.seqs, std::max(2 * least, std::min<size_t>(p.pieces, room * a.seqs / 4))) + a.seqs;
    const size_t blocks = numbers * p.row_tiles * heads, piece_rows = blocks * 16;
    if (ahead + blocks >= 1u << 24) return fail(HH_ERR_INVALID, "attn_decode: %u sequences are too many", a.seqs);
    HH_TRY(grow(&ws_attn, &ws_attn_cap, (part_rows + piece_rows) * (dp + 2) * sizeof(float) + a.seqs * 8));
    a.part = (float*)ws_attn;
    p.piece = a.part + part_rows * dp;
    a.part_sum = p.piece + piece_rows * dp;
    p.piece_sum = a.part_sum + part_rows * 2;
    p.plan = (uint32_t*)(p.piece_sum + piece_rows * 2);
    void* params[] = {&p};
    HH_TRY_HIP(hipModuleLaunchKernel(f, (uint32_t)(ahead + blocks), 1, 1, 256, 1, 1, 0, stream, params, nullptr),
               "hipModuleLaunchKernel(attn_decode)");
    // (no table has room for a second piece: every row is whole)
    if (p.prefix || room > 1)
        HH_TRY_HIP(hipModuleLaunchKernel(join, (uint32_t)(a.seqs * heads * a.group), 1, 1, 256, 1, 1, 0, stream, params, nullptr),
                   "hipModuleLaunchKernel(attn_join)");
    return HH_OK;
}
