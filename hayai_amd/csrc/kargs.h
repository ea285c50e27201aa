// Kernel argument blocks shared by the host runtime and the gfx950 kernels.
//
// Every kernel takes exactly one of these structs by value; the host passes its address
// as the single entry of hipModuleLaunchKernel's kernelParams.  Plain C layout only.
#ifndef HH_KARGS_H
#define HH_KARGS_H

#include <stdint.h>

#define HH_TYPE_F32 0
#define HH_TYPE_F16 1
#define HH_TYPE_Q4_0 2
#define HH_TYPE_Q8_0 8
#define HH_TYPE_Q4_K 12
#define HH_TYPE_Q6_K 14
#define HH_TYPE_IQ2_XXS 16
#define HH_TYPE_IQ3_XXS 18
#define HH_TYPE_BF16 30

#define HH_ACT_SILU 0
#define HH_ACT_GELU_TANH 1

// y[m] = W[m x n] . x[n]   (one GEMV; W row-major GGUF blocks along n)
struct hh_gemv_args {
    const uint8_t* w;  // first byte of row 0
    const float* x;    // n floats
    float* y;          // m floats
    uint32_t m;
    uint32_t n;
    uint64_t row_bytes;
};

// h[m] = act(Wg . x) * (Wu . x)   (fused gate/up GEMV + SwiGLU/GELU)
struct hh_gateup_args {
    const uint8_t* wg;
    const uint8_t* wu;
    const float* x;
    float* h;
    uint32_t m;  // d_ff
    uint32_t n;  // d_model
    uint64_t row_bytes;
    int32_t act;
    int32_t pad;
};

// h[i] = act(g[i]) * u[i]
struct hh_act_args {
    const float* g;
    const float* u;
    float* h;
    uint32_t n;
    int32_t act;
};

// y = RMSNorm(x) * w over n elements (one workgroup)
struct hh_norm_args {
    const float* x;
    const float* w;
    float* y;
    uint32_t n;
    float eps;
};

// x (n f32) -> q1[n] | q2[n] int8 | scale[n/8] f32, the ring down kernels' digit form
struct hh_xd_args {
    const float* x;
    uint8_t* hx;
    uint32_t n;
    uint32_t pad;
};

// y = a + b over n elements (the residual add)
struct hh_add_args {
    const float* a;
    const float* b;
    float* y;
    uint32_t n;
    uint32_t pad;
};

// out[n] = dequant(w[...]) for n elements (the dequant probe)
struct hh_dequant_args {
    const uint8_t* w;
    float* out;
    uint64_t n;
};

// Rows into int8 codes (i8_rows.hip).  b: up, or the residual (null: none); strides in elements.
struct hh_i8_rows_args {
    const void* x;
    const void* b;
    const float* norm;
    void* sum;
    int8_t* q;
    float* scale;
    float* values;
    uint64_t x_stride, b_stride, sum_stride, q_stride;
    uint32_t rows, cols;
    int32_t act;
    float eps;
};

// y[t][r] = sum_k x[t][k] w[r][k] * xs[t] * ws[r] (+ res[t][r]) over codes (i8_gemm.hip);
// w and x strides in bytes, y and res strides in elements.
struct hh_i8_gemm_args {
    const int8_t* w;
    const int8_t* x;
    const float* ws;
    const float* xs;
    const void* res;
    void* y;
    uint64_t w_stride, x_stride, res_stride, y_stride;
    uint32_t m, n, t;
    uint32_t mtiles, ttiles, pad;
    int* cut;         // sums of tiles cut between workgroups, two tiles a workgroup
    uint32_t* count;  // arrivals at each tile: zero between launches
};

// The next token of each row of logits (sample.hip); stride in elements.  The workspaces hold, per row:
struct hh_sample_args {
    const void* x;
    const void* params;  // hh_sample_params
    const float* u;
    int32_t* ids;
    float* probs;
    uint64_t* top;     // `parts`: a part's first token
    uint64_t* mass;    // 1024: weight by distance from the largest logit
    uint64_t* sure;    // `chunks`: weight surely kept
    uint64_t* list;    // 8192: tokens at the filters' ends
    uint32_t* count;   // 1024: tokens by distance
    uint32_t* listed;  // the list's length
    void* cut;         // hh_smp_cut
    uint64_t stride;
    uint32_t vocab, parts, chunks, pad;
};

// Pages of keys and values (kv_pages.h): page p at base + p * stride bytes, its keys [heads][1 << shift][dim],
// then its values [heads][dim][1 << shift].
struct hh_kv_args {
    uint8_t* base;
    uint64_t stride;
    uint32_t pages, shift, heads, dim;
};

// Rotated queries and keys, and the tokens' places in the cache (rope.hip); strides in elements.
struct hh_rope_args {
    hh_kv_args kv;
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* positions;
    const int32_t* slots;
    const float* factors;  // null: all 1
    uint64_t q_stride, k_stride, v_stride, out_stride;
    double log2_base;
    float mscale;
    uint32_t tokens, heads, rot;
};

// Pages moves[i][0] -> moves[i][1] in each layer (kv_pages.hip); strides and sizes in bytes.
struct hh_kv_copy_args {
    hh_kv_args kv;
    const int32_t* moves;
    uint64_t layer_stride;
    uint32_t n, chunks;  // moves, 16-byte chunks of a page
};

// What attention of a prompt and of a decode batch have in common (attn_rows.h); strides in elements.  A tile is
// `tile_tokens` tokens' `group` heads of one kv head.
struct hh_attn_args {
    hh_kv_args kv;
    const void* q;
    void* out;
    const int32_t* lens;    // of each sequence
    const int32_t* tables;  // rows of `entries`
    float* part;            // tiles whose keys are in `splits` parts: 128 rows of sums a part
    float* part_sum;        // their bases and sums of weights
    uint64_t q_stride, out_stride;
    uint32_t seqs, entries, group, tile_tokens, splits;
    float c;  // scale * log2(e)
};

// Causal attention of packed prompts (attn_prompt.hip).  `slots` bounds the tiles of a kv head.
struct hh_attn_prompt_args {
    hh_attn_args a;
    const int32_t* starts;  // seqs + 1
    uint32_t tokens, slots;
    uint32_t turn;  // tiles' parts from which on the shortest come first
    uint32_t step, whole;  // log2 of the keys in a tile; as many as are taken in one part
};

// Attention of one token a sequence (attn_decode.hip): the first `prefix` tokens of the sequences of `sharing` or more from the
// pages of `shared` (tiles of `a`), the others in pieces, each with row_tiles * heads * 16 rows of sums.
struct hh_attn_decode_args {
    hh_attn_args a;
    const int32_t* shared;
    float* piece;
    float* piece_sum;
    uint32_t* plan;  // each sequence's first piece and how many it has
    uint32_t prefix, sharing, shared_entries, tiles, row_tiles;
    uint32_t room;           // units of own tokens that a table has room for
    uint32_t pieces, least;  // at most (but for one a sequence more); for a workgroup a CU
};

// Synthetic GGUF bytes: splitmix64 stream, then f16 scale fields drawn U(lo, hi).
struct hh_synth_args {
    uint8_t* dst;
    uint64_t nbytes;     // bytes of the random stream (whole blocks)
    uint64_t seed;
    uint64_t nblocks;    // blocks whose scale fields are patched
    int32_t type;
    float lo;
    float hi;
    int32_t pad;
};

#endif
