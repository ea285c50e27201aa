// Products of int8 codes with a scale per token and per weight row:
//   y[t][r] = (sum_k x[t][k] w[r][k]) * xs[t] * ws[r] (+ res[t][r])
// Sums are 32-bit integers, exact for n <= 131071 (2^31 / 128^2), so they may be split over k and
// added in any order: every form below gives the same bits.  The sum is rounded to f32 once, then
// the scales and the residual in f32, then the output type.
//
// Three forms (enqueue_i8_gemm chooses and has the measured sides):
//   hh_i8_rowdot_t<T>   up to 8 tokens: v_dot4 over rows read end to end, tokens in LDS
//   hh_i8_tile_<shape>  small tiles on the matrix cores, the tiles' k cut into equal runs for all
//                       workgroups
//   hh_i8_big_<shape>   large tiles, whole, with a scheduled inner loop
#include "act_types.h"

typedef int hh_i4 __attribute__((ext_vector_type(4)));

// The bytes of 16 codes at k that lie inside a row of n (k may pass it).
HH_DEV hh_i4 hh_i8_mask(hh_i4 v, uint32_t k, uint32_t n) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int left = (int)n - (int)k - 4 * i;
        v[i] = left >= 4 ? v[i] : left <= 0 ? 0 : (int)((uint32_t)v[i] & ((1u << (8 * left)) - 1u));
    }
    return v;
}

HH_DEV float hh_i8_value(int sum, float xs, float ws) { return (float)sum * xs * ws; }

// ------------------------------------------------------------------ few tokens
// A wave reads R = 2 rows at a time, 1 KB of each in one load (16 codes a lane), D steps ahead, and
// multiplies them with the tokens' same columns from LDS; v_dot4_i32_i8 sums stay in the lane until
// the rows' end, then one DPP sum a row and token.  Rows go round over the grid's waves, so at any
// moment the requests lie next to each other.  Bound by HBM: 28672 x 4096, one token, 22 us = 5.3
// TB/s (v_mfma_i32_16x16x64_i8 straight from memory, 16 rows x 64 bytes a load: 28 us).
#define HH_I8_RD_R 2
#define HH_I8_RD_D 4

template <int CTRL, int ROWS>
HH_DEV int hh_i8_dpp(int v) {
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
HH_DEV int hh_i8_wave_sum(int v) {
    v += hh_i8_dpp<0xB1, 0xf>(v);   // quad_perm [1,0,3,2]
    v += hh_i8_dpp<0x4E, 0xf>(v);   // quad_perm [2,3,0,1]
    v += hh_i8_dpp<0x124, 0xf>(v);  // row_ror:4
    v += hh_i8_dpp<0x128, 0xf>(v);  // row_ror:8
    v += hh_i8_dpp<0x142, 0xa>(v);  // row_bcast:15
    v += hh_i8_dpp<0x143, 0xc>(v);  // row_bcast:31: lane 63 has the total
    return __builtin_amdgcn_readlane(v, 63);
}

extern __shared__ __attribute__((aligned(16))) int8_t hh_i8_smem[];

template <class F, int T>
HH_DEV void hh_i8_rowdot(const hh_i8_gemm_args& a) {
    constexpr int R = HH_I8_RD_R, D = HH_I8_RD_D;
    typedef typename F::E E;
    const uint32_t lane = threadIdx.x % HH_WAVE;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / HH_WAVE);
    const uint32_t chunks = (a.n + 1023) / 1024, n16 = (a.n + 15) & ~15u;
    const uint32_t first = wave * gridDim.x + blockIdx.x, step = gridDim.x * (blockDim.x / HH_WAVE);
    const uint32_t groups = (a.m + R - 1) / R;
    const uint32_t total = first < groups ? (groups - first + step - 1) / step * chunks : 0;
    hh_i4 wr[D][R];
    uint32_t lg = first, lc = 0;  // the next load's rows and chunk (past the end: the last ones again)
    auto load = [&](int slot) {
        const uint32_t k = min(lc * 1024 + lane * 16, n16 - 16);
#pragma unroll
        for (int i = 0; i < R; i++)
            wr[slot][i] = *reinterpret_cast<const hh_i4*>(a.w + (size_t)min(lg * R + i, a.m - 1) * a.w_stride + k);
        if (++lc == chunks) {
            lc = 0;
            lg = min(lg + step, groups - 1);
        }
    };
    if (total) {
#pragma unroll
        for (int p = 0; p < D; p++) load(p);
    }
    // the tokens, codes past n and tokens past t as zeros
    for (uint32_t i = threadIdx.x; i < T * chunks * 64; i += blockDim.x) {
        const uint32_t t = i / (chunks * 64), k = i % (chunks * 64) * 16;
        hh_i4 v{0, 0, 0, 0};
        if (t < a.t && k < a.n)
            v = hh_i8_mask(*reinterpret_cast<const hh_i4*>(a.x + t * a.x_stride + k), k, a.n);
        *reinterpret_cast<hh_i4*>(hh_i8_smem + i * 16) = v;
    }
    __syncthreads();
    int acc[R][T];
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int t = 0; t < T; t++) acc[i][t] = 0;
    uint32_t g = first, c = 0;
    for (uint32_t it = 0; it < total; it += D) {
#pragma unroll
        for (int p = 0; p < D; p++) {
            if (it + p >= total) break;
#pragma unroll
            for (int t = 0; t < T; t++) {
                const hh_i4 x = *reinterpret_cast<const hh_i4*>(hh_i8_smem + (t * chunks + c) * 1024 + lane * 16);
#pragma unroll
                for (int i = 0; i < R; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][t] = __builtin_amdgcn_sdot4(wr[p][i][e], x[e], acc[i][t], false);
            }
            load(p);
            if (++c < chunks) continue;
            int v = 0;  // lane i * T + t: row i, token t
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int t = 0; t < T; t++) {
                    const int s = hh_i8_wave_sum(acc[i][t]);
                    v = lane == (uint32_t)(i * T + t) ? s : v;
                    acc[i][t] = 0;
                }
            const uint32_t r = g * R + lane / T, t = lane % T;
            if (lane < R * T && r < a.m && t < a.t) {
                float f = hh_i8_value(v, a.xs[t], a.ws[r]);
                if (a.res) f += F::get(((const E*)a.res)[t * a.res_stride + r]);
                ((E*)a.y)[t * a.y_stride + r] = F::put(f);
            }
            c = 0;
            g += step;
        }
    }
}

// ------------------------------------------------------------------ tiles
// A tile is TM weight rows x TN tokens, by WM x WN waves, on v_mfma_i32_16x16x64_i8: lane l holds
// 16 consecutive k (16 (l / 16) onwards) of A's row and of B's column l % 16; A is the weights, so a
// lane's four sums are four consecutive rows of one token.  (32x32x32 needs no fewer LDS bytes and
// draws more power: 3.4 POP/s on random codes against 4.0.)
//
// Stages of 128 codes of the tile's rows come into LDS by DMA, three of four buffers ahead.  A row's 128 bytes are
// eight 16-byte chunks, chunk c at position c ^ (row / 2 % 8): the DMA writes lanes in order, so
// the swizzle is in which chunk a lane asks for, and reads of 16 rows' same chunk meet every bank
// once (measured 550 B/ns a CU, 290 with row % 8, 76 without).  A stage buffer is a __shared__ object of
// its own, which is how the compiler knows that a read of one need not wait for a copy into another.
//
// The tiles' stages, tile after tile, are cut into W equal runs, one a workgroup, so all finish
// together whatever the shape.  A tile cut between workgroups is summed by the last of them to
// arrive: the others leave their sums in a workspace (stores and loads at device scope, then a count
// on a device word; the count returns to zero) and nobody waits.  Bound by HBM to 64 tokens: 128256 x
// 4096, 8 tokens, 106 us = 5.0 TB/s; 4096 x 14336, 61 tokens, 23.5 us = 2.6 TB/s, 15.4 where the weights lie in
// the memory-side cache (256 tiles, each cut in two: an exchange at every end).
template <int B, int BYTES>
HH_DEV int8_t* hh_i8_lds() {
    __shared__ __attribute__((aligned(128))) int8_t buf[BYTES];
    return buf;
}
constexpr int hh_i8_wait(int vm, int lgkm) { return (vm & 15) | ((vm >> 4) << 14) | 0x70 | (lgkm << 8); }
// Copies but the newest `vm` landed, this wave's LDS reads done, then the workgroup meets.
template <int VM>
HH_DEV void hh_i8_meet() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(hh_i8_wait(VM, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
template <int N>
struct hh_i8_int {
    static constexpr int value = N;
};

typedef uint32_t hh_u4 __attribute__((ext_vector_type(4)));
// Device-scope (past the XCD's L2) 16-byte accesses of the workspace.
HH_DEV void hh_i8_leave(int* base, uint32_t off, hh_i4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(hh_u4, v),
                                           __builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7fffffff, 0x00027000), off, 0, 17);
}
HH_DEV hh_i4 hh_i8_take(int* base, uint32_t off) {
    return __builtin_bit_cast(hh_i4, __builtin_amdgcn_raw_buffer_load_b128(
                                         __builtin_amdgcn_make_buffer_rsrc(base, 0, 0x7fffffff, 0x00027000), off, 0, 17));
}

template <int TM, int TN, int WM, int WN>
struct hh_i8_shape {
    static constexpr int MT = TM / WM / 16, NT = TN / WN / 16;
    // where this lane's operands lie in a 128-code stage row block, and its outputs in the tile
    uint32_t wrow, xrow, pos[2], row, token;
    uint32_t quarter;
    HH_DEV hh_i8_shape(uint32_t lane, uint32_t wave) {
        const uint32_t wm = wave / WN, wn = wave % WN, r16 = lane % 16, swz = (r16 >> 1) & 7;
        quarter = lane / 16;
        wrow = (wm * (TM / WM) + r16) * 128;
        xrow = (TM + wn * (TN / WN) + r16) * 128;
        pos[0] = (quarter ^ swz) * 16;
        pos[1] = ((4 + quarter) ^ swz) * 16;
        row = wm * (TM / WM) + quarter * 4;
        token = wn * (TN / WN) + r16;
    }
};

// Leaves this workgroup's sums of a cut tile, or adds the others' to them: true in the last of the
// tile's workgroups w0..w1 to arrive.  cut[2 w], cut[2 w + 1]: workgroup w's sums of a tile begun by
// an earlier one, and of one that it begins.
template <int MT, int NT, int TILE>
HH_DEV bool hh_i8_join(const hh_i8_gemm_args& a, hh_i4 (&acc)[MT][NT], uint32_t tile, uint32_t wg, uint32_t w0,
                       uint32_t w1, uint32_t wave, uint32_t lane, uint32_t* last) {
    const uint32_t off = (wave * (MT * NT * 256) + lane * 4) * 4;
    int* mine = a.cut + ((size_t)wg * 2 + (wg == w0)) * TILE;
#pragma unroll
    for (int i = 0; i < MT; i++)
#pragma unroll
        for (int j = 0; j < NT; j++) hh_i8_leave(mine, off + (i * NT + j) * 1024, acc[i][j]);
    __builtin_amdgcn_s_waitcnt(hh_i8_wait(0, 0));
    __syncthreads();
    if (threadIdx.x == 0) {
        const uint32_t k = __hip_atomic_fetch_add(a.count + tile, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = k == w1 - w0;
        if (k == w1 - w0) __hip_atomic_store(a.count + tile, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return false;
    // Q workgroups' sums at a time, as a trip past the L2 is long (64 x 16384, 16 tokens, 64 to a tile: 9.8 us,
    // one after the other 23.7).  This workgroup's own are in registers; its place, and those past w1, count as zeros.
    constexpr uint32_t Q = MT * NT == 1 ? 8 : 4;
    for (uint32_t q = w0; q <= w1; q += Q) {
        hh_i4 part[Q][MT][NT];
#pragma unroll
        for (uint32_t k = 0; k < Q; k++) {
            const uint32_t from = q + k <= w1 ? q + k : wg;
            int* p = a.cut + ((size_t)from * 2 + (from == w0)) * TILE;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) part[k][i][j] = hh_i8_take(p, off + (i * NT + j) * 1024);
        }
#pragma unroll
        for (uint32_t k = 0; k < Q; k++) {
            const int keep = q + k <= w1 && q + k != wg ? -1 : 0;
#pragma unroll
            for (int i = 0; i < MT; i++)
#pragma unroll
                for (int j = 0; j < NT; j++) acc[i][j] += part[k][i][j] & keep;
        }
    }
    return true;
}

// Outputs r..r+3 of token t from their sums (r < m, t < the call's tokens).
template <class F>
HH_DEV void hh_i8_put(const hh_i8_gemm_args& a, typename F::E* y, const typename F::E* res, uint32_t r, hh_i4 sum,
                      float xs, const float (&ws)[4]) {
    typename F::E o[4];
    if (r + 4 <= a.m) {
        if (res) hh_load_n(res + r, o);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float v = hh_i8_value(sum[e], xs, ws[e]);
            o[e] = F::put(res ? v + F::get(o[e]) : v);
        }
        hh_store_n(y + r, o);
    } else {
        for (int e = 0; e < 4; e++)
            if (r + e < a.m) {
                const float v = hh_i8_value(sum[e], xs, ws[e]);
                y[r + e] = F::put(res ? v + F::get(res[r + e]) : v);
            }
    }
}

template <class F, int TM, int TN, int WM, int WN>
HH_DEV void hh_i8_tile(const hh_i8_gemm_args& a) {
    typedef typename F::E E;
    typedef hh_i8_shape<TM, TN, WM, WN> Shape;
    constexpr int WAVES = WM * WN, MT = Shape::MT, NT = Shape::NT;
    constexpr int NB = 4, BYTES = (TM + TN) * 128;
    constexpr int LP = (TM + TN) / 8 / WAVES;  // 8-row pieces of a stage that a wave copies
    static_assert((TM + TN) / 8 % WAVES == 0, "pieces of a stage over the waves");
    const uint32_t lane = threadIdx.x % HH_WAVE;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / HH_WAVE);
    const Shape sh(lane, wave);
    const uint32_t stages = (a.n + 127) / 128, W = gridDim.x, n16 = (a.n + 15) & ~15u;
    const uint64_t units = (uint64_t)a.mtiles * a.ttiles * stages;
    // consecutive workgroups go to the 8 XCDs in turn: each XCD's have neighbouring runs, which share rows
    const uint32_t wg = W % 8 ? blockIdx.x : blockIdx.x % 8 * (W / 8) + blockIdx.x / 8;
    uint64_t u = units * wg / W;
    const uint64_t u1 = units * (wg + 1) / W;
    const uint32_t c0 = ((lane % 8) ^ (lane / 16)) * 16;  // lane / 8 of a piece is the row: row / 2 % 4
    __shared__ uint32_t last;
    while (u < u1) {
        const uint32_t tile = (uint32_t)(u / stages), sa = (uint32_t)(u - (uint64_t)tile * stages);
        const uint32_t sb = (uint32_t)min((uint64_t)stages, sa + (u1 - u));
        const uint32_t m0 = tile / a.ttiles * TM, t0 = tile % a.ttiles * TN;
        const int8_t* src[LP];
#pragma unroll
        for (int i = 0; i < LP; i++) {
            const uint32_t r = (wave * LP + i) * 8 + lane / 8;
            src[i] = r < TM ? a.w + (size_t)min(m0 + r, a.m - 1) * a.w_stride
                            : a.x + (size_t)min(t0 + r - TM, a.t - 1) * a.x_stride;
        }
        auto copy = [&](int8_t* buf, uint32_t s) {  // past n: the row's last 16 codes
#pragma unroll
            for (int i = 0; i < LP; i++) {
                const uint32_t p = wave * LP + i, k = s * 128 + (c0 ^ ((p & 1) * 64));
                __builtin_amdgcn_global_load_lds(
                    (const __attribute__((address_space(1))) void*)(src[i] + min(k, n16 - 16)),
                    (__attribute__((address_space(3))) void*)(buf + p * 1024), 16, 0, 0);
            }
        };
        hh_i4 acc[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = hh_i4{0, 0, 0, 0};
        auto compute = [&](const int8_t* buf, uint32_t s, bool tail) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                hh_i4 w[MT], x[NT];
                const int8_t* st = buf + sh.pos[h];
#pragma unroll
                for (int i = 0; i < MT; i++) w[i] = *reinterpret_cast<const hh_i4*>(st + sh.wrow + i * 2048);
#pragma unroll
                for (int j = 0; j < NT; j++) x[j] = *reinterpret_cast<const hh_i4*>(st + sh.xrow + j * 2048);
                if (tail) {
#pragma unroll
                    for (int i = 0; i < MT; i++) w[i] = hh_i8_mask(w[i], s * 128 + h * 64 + sh.quarter * 16, a.n);
                }
#pragma unroll
                for (int i = 0; i < MT; i++)
#pragma unroll
                    for (int j = 0; j < NT; j++)
                        acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[i], x[j], acc[i][j], 0, 0, 0);
            }
        };
        // stage s from its buffer; s + NB - 1 goes where s - 1 was, which everyone has left
        auto step = [&](auto b, uint32_t s, bool tail) {
            constexpr int me = decltype(b)::value;
            hh_i8_meet<(NB - 2) * LP>();
            copy(hh_i8_lds<(me + NB - 1) % NB, BYTES>(), s + NB - 1);
            compute(hh_i8_lds<me, BYTES>(), s, tail);
        };
        copy(hh_i8_lds<0, BYTES>(), sa);
        copy(hh_i8_lds<1, BYTES>(), sa + 1);
        copy(hh_i8_lds<2, BYTES>(), sa + 2);
        uint32_t s = sa;
        const uint32_t whole = min(sb, a.n / 128);  // stages without codes past n
        for (; s + NB <= whole; s += NB) {
            step(hh_i8_int<0>{}, s, false);
            step(hh_i8_int<1>{}, s + 1, false);
            step(hh_i8_int<2>{}, s + 2, false);
            step(hh_i8_int<3>{}, s + 3, false);
        }
        // up to NB stages left (NB where the last has a tail)
        if (s < sb) step(hh_i8_int<0>{}, s, true);
        if (s + 1 < sb) step(hh_i8_int<1>{}, s + 1, true);
        if (s + 2 < sb) step(hh_i8_int<2>{}, s + 2, true);
        if (s + 3 < sb) step(hh_i8_int<3>{}, s + 3, true);
        hh_i8_meet<0>();  // the copies past the run have landed, every wave has left the buffers
        u += sb - sa;
        if (sb - sa < stages) {
            const uint64_t f = (uint64_t)tile * stages;  // workgroups with the tile's first and last stage
            const uint32_t w0 = (uint32_t)(((f + 1) * W - 1) / units), w1 = (uint32_t)(((f + stages) * W - 1) / units);
            if (!hh_i8_join<MT, NT, TM * TN>(a, acc, tile, wg, w0, w1, wave, lane, &last)) continue;
        }
        float ws[MT][4];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) ws[i][e] = a.ws[min(m0 + sh.row + i * 16 + e, a.m - 1)];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const uint32_t t = t0 + sh.token + j * 16;
            if (t >= a.t) break;
            const float xs = a.xs[t];
            E* y = (E*)a.y + t * a.y_stride;
            const E* res = a.res ? (const E*)a.res + t * a.res_stride : nullptr;
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const uint32_t r = m0 + sh.row + i * 16;
                if (r < a.m) hh_i8_put<F>(a, y, res, r, acc[i][j], xs, ws[i]);
            }
        }
    }
}

// ------------------------------------------------------------------ large tiles
// Whole tiles, W workgroups taking every W-th, stages of 128 codes in two buffers.  A stage's
// second half's operands are read while the first half multiplies, the next stage's first half's
// while the second does (sched_group_barrier: one LDS read to PER products), and the next tile's
// first stages are asked for before this one's outputs are written.  Cut tiles cost more here than
// idle CUs: 28672 x 4096, 512 tokens, 224 tiles of 256 x 256: 67 us, cut into 256 runs 106.  Bound by
// power: 28672 x 4096, 2048 tokens, 242 us = 1.99 POP/s at a clock of 1.65 to 1.95 GHz.
template <class F, int TM, int TN, int WM, int WN>
HH_DEV void hh_i8_big(const hh_i8_gemm_args& a) {
    constexpr int WAVES = WM * WN, HALF = (TM + TN) * 128;
    typedef typename F::E E;
    typedef hh_i8_shape<TM, TN, WM, WN> Shape;
    constexpr int MT = Shape::MT, NT = Shape::NT, LW = TM / 8 / WAVES, LX = TN / 8 / WAVES, PER = MT * NT / (MT + NT);
    int8_t* const buf0 = hh_i8_lds<0, HALF>();
    int8_t* const buf1 = hh_i8_lds<1, HALF>();
    const uint32_t lane = threadIdx.x % HH_WAVE;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / HH_WAVE);
    const Shape sh(lane, wave);
    const uint32_t stages = (a.n + 127) / 128, W = gridDim.x, n16 = (a.n + 15) & ~15u;
    const uint32_t tiles = a.mtiles * a.ttiles;
    // consecutive workgroups go to the 8 XCDs in turn: each XCD's take neighbouring tiles, which share rows
    uint32_t tile = blockIdx.x % 8 * (W / 8) + blockIdx.x / 8;
    if (tile >= tiles) return;

    const uint32_t lrow = lane / 8, c0 = ((lane % 8) ^ (lane / 16)) * 16;
    uint32_t woff[LW], xoff[LX];  // 255 strides of 2^24 and a row of codes stay below 2^32
    const int8_t *wbase, *xbase;
    uint32_t m0, t0;
    auto place = [&]() {
        m0 = tile / a.ttiles * TM;
        t0 = tile % a.ttiles * TN;
        wbase = a.w + (size_t)m0 * a.w_stride;
        xbase = a.x + (size_t)t0 * a.x_stride;
#pragma unroll
        for (int i = 0; i < LW; i++) woff[i] = min((wave * LW + i) * 8 + lrow, a.m - 1 - m0) * (uint32_t)a.w_stride;
#pragma unroll
        for (int i = 0; i < LX; i++) xoff[i] = min((wave * LX + i) * 8 + lrow, a.t - 1 - t0) * (uint32_t)a.x_stride;
    };
    // codes k.. of the tile's rows into a buffer (past n: the row's last 16 codes)
    auto copy = [&](int8_t* buf, uint32_t k) {
#pragma unroll
        for (int i = 0; i < LW; i++) {
            const uint32_t c = c0 ^ (((wave * LW + i) & 1) * 64);
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(wbase + (woff[i] + min(k + c, n16 - 16))),
                (__attribute__((address_space(3))) void*)(buf + (wave * LW + i) * 1024), 16, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < LX; i++) {
            const uint32_t c = c0 ^ (((wave * LX + i) & 1) * 64);
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)(xbase + (xoff[i] + min(k + c, n16 - 16))),
                (__attribute__((address_space(3))) void*)(buf + TM * 128 + (wave * LX + i) * 1024), 16, 0, 0);
        }
    };
    hh_i4 acc[MT][NT];
    struct Frag {
        hh_i4 w[MT], x[NT];
    };
    auto fetch = [&](const int8_t* buf, int h, Frag& f) {
#pragma unroll
        for (int j = 0; j < NT; j++) f.x[j] = *reinterpret_cast<const hh_i4*>(buf + sh.xrow + j * 2048 + sh.pos[h]);
#pragma unroll
        for (int i = 0; i < MT; i++) f.w[i] = *reinterpret_cast<const hh_i4*>(buf + sh.wrow + i * 2048 + sh.pos[h]);
    };
    auto multiply = [&](const Frag& f) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
    };
    Frag f, g;
    // stage s (f holds its first half): s + 1 has landed in `next` by the middle, s + 2 goes where s was
    auto stage = [&](int8_t* here, int8_t* next, uint32_t s) {
        fetch(here, 1, g);
        multiply(f);
#pragma unroll
        for (int q = 0; q < MT + NT; q++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // an LDS read
            __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        hh_i8_meet<0>();
        copy(here, (s + 2) * 128);
        fetch(next, 0, f);
        multiply(g);
#pragma unroll
        for (int q = 0; q < MT + NT; q++) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x008, PER, 0);
            if (q < LW + LX) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);  // a copy
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    place();
    copy(buf0, 0);
    copy(buf1, 128);
    for (;;) {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = hh_i4{0, 0, 0, 0};
        hh_i8_meet<0>();
        fetch(buf0, 0, f);
        uint32_t s = 0;
        for (; s + 2 < stages; s += 2) {
            stage(buf0, buf1, s);
            stage(buf1, buf0, s + 1);
        }
        const int8_t* end = buf0;
        if (s + 1 < stages) {
            stage(buf0, buf1, s);
            end = buf1;
            s++;
        }
        // the last stage, codes past n as zeros
#pragma unroll
        for (int h = 0; h < 2; h++) {
            fetch(end, h, f);
#pragma unroll
            for (int i = 0; i < MT; i++) f.w[i] = hh_i8_mask(f.w[i], s * 128 + h * 64 + sh.quarter * 16, a.n);
            multiply(f);
        }
        const uint32_t r0 = m0 + sh.row, tt0 = t0 + sh.token;
        float ws[MT][4], xs[NT];
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) ws[i][e] = a.ws[min(r0 + i * 16 + e, a.m - 1)];
#pragma unroll
        for (int j = 0; j < NT; j++) xs[j] = a.xs[min(tt0 + j * 16, a.t - 1)];
        hh_i8_meet<0>();  // every wave is done with the last stage
        tile += W;
        const bool more = tile < tiles;
        if (more) {
            place();
            copy(buf0, 0);
            copy(buf1, 128);
        }
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const uint32_t t = tt0 + j * 16;
            if (t >= a.t) break;
            E* y = (E*)a.y + t * a.y_stride;
            const E* res = a.res ? (const E*)a.res + t * a.res_stride : nullptr;
#pragma unroll
            for (int i = 0; i < MT; i++)
                if (r0 + i * 16 < a.m) hh_i8_put<F>(a, y, res, r0 + i * 16, acc[i][j], xs[j], ws[i]);
        }
        if (!more) break;
    }
}

#define HH_I8_ROWDOT(T, F, N)                                                                            \
    extern "C" __global__ void __launch_bounds__(512) hh_i8_rowdot_t##N##_##T(const hh_i8_gemm_args a) { \
        hh_i8_rowdot<F, N>(a);                                                                           \
    }
#define HH_I8_TILE(T, F, TM, TN, WM, WN)                                                                                 \
    extern "C" __global__ void __launch_bounds__((WM) * (WN) * 64) hh_i8_tile_##TM##x##TN##_##T(const hh_i8_gemm_args a) { \
        hh_i8_tile<F, TM, TN, WM, WN>(a);                                                                                \
    }
#define HH_I8_BIG(T, F, TM, TN, WM, WN)                                                                                  \
    extern "C" __global__ void __launch_bounds__((WM) * (WN) * 64) hh_i8_big_##TM##x##TN##_##T(const hh_i8_gemm_args a) { \
        hh_i8_big<F, TM, TN, WM, WN>(a);                                                                                 \
    }
#define HH_I8_GEMM(T, F)                                                                        \
    HH_I8_ROWDOT(T, F, 1)                                                                       \
    HH_I8_ROWDOT(T, F, 2)                                                                       \
    HH_I8_ROWDOT(T, F, 4)                                                                       \
    HH_I8_ROWDOT(T, F, 8)                                                                       \
    HH_I8_TILE(T, F, 32, 32, 2, 2)                                                        \
    HH_I8_TILE(T, F, 64, 64, 2, 2)                                                        \
    HH_I8_BIG(T, F, 256, 256, 4, 2)                                                             \
    HH_I8_BIG(T, F, 192, 256, 2, 4)                                                             \
    HH_I8_BIG(T, F, 128, 256, 2, 4)                                                             \
    HH_I8_BIG(T, F, 128, 128, 2, 2)
HH_I8_GEMM(f32, hh_af32)
HH_I8_GEMM(f16, hh_af16)
HH_I8_GEMM(bf16, hh_abf16)
