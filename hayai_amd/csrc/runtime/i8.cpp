// Dispatch of the 8-bit path: rows into codes (i8_rows.hip), products of codes (i8_gemm.hip) and
// the choice of the next token (sample.hip).
#include <algorithm>

#include "engine.h"

namespace hh {

const ActType* act_type(int t) {
    static const ActType f32{"f32", 4}, f16{"f16", 2}, bf16{"bf16", 2};
    return t == HH_TYPE_F32 ? &f32 : t == HH_TYPE_F16 ? &f16 : t == HH_TYPE_BF16 ? &bf16 : nullptr;
}

void i8_kernels(std::vector<std::string>& k) {
    for (int t : {HH_TYPE_F32, HH_TYPE_F16, HH_TYPE_BF16}) {
        const std::string ty = act_type(t)->name;
        for (const char* kind : {"plain", "act", "norm"})
            for (const char* v : {"c1", "c2", "c4", "loop"}) k.push_back("hh_i8_rows_" + ty + "_" + kind + "_" + v);
        for (const char* v : {"rowdot_t1", "rowdot_t2", "rowdot_t4", "rowdot_t8", "tile_32x32", "tile_64x64", "big_128x128",
                              "big_128x256", "big_192x256", "big_256x256"})
            k.push_back(std::string("hh_i8_") + v + "_" + ty);
        for (const char* v : {"max", "hist", "gather", "pick"}) k.push_back(std::string("hh_sample_") + v + "_" + ty);
    }
}

}  // namespace hh

using namespace hh;

hh_status hh_engine::enqueue_i8_rows(int type, size_t rows, const hh_i8_rows_args& a) {
    const ActType* ty = act_type(type);
    const size_t chunks = (a.cols * ty->bytes + 15) / 16;
    // Few rows: as many threads as chunks, for latency.  More rows than CUs: up to four chunks a thread, so
    // that a CU holds several rows and asks for more of them at once (400 x 4096 f32 normalised: 6.0 us, one
    // chunk a thread 6.9; 300 x 16384 bf16: 12.2, 13.0); and where one wave holds a row, four rows a
    // workgroup (7178 rows of 208 f16: 8.2 us, one a workgroup with four chunks a thread 19.1, eight a
    // workgroup 8.4; 13527 of 1076: 22.0, 32.1, 22.3).
    const bool many = rows > (size_t)props.multiProcessorCount && chunks <= 4096;
    const size_t threads = std::min<size_t>(1024, ((many ? (chunks + 3) / 4 : chunks) + 63) / 64 * 64);
    const char* kind = a.norm ? "norm" : a.b ? "act" : "plain";
    const size_t each = (chunks + threads - 1) / threads;
    const char* v = each <= 1 ? "c1" : each <= 2 ? "c2" : each <= 4 ? "c4" : "loop";
    const size_t per = many && threads == 64 ? 4 : 1;
    hipFunction_t f;
    HH_TRY(kernel(std::string("hh_i8_rows_") + ty->name + "_" + kind + "_" + v, &f));
    // a grid has fewer than 2^32 threads: 2^21 rows at a time
    for (size_t r = 0; r < rows; r += (size_t)1 << 21) {
        const size_t n = std::min(rows - r, (size_t)1 << 21);
        hh_i8_rows_args p = a;
        p.rows = (uint32_t)n;
        p.x = (const char*)a.x + r * a.x_stride * ty->bytes;
        p.b = a.b ? (const char*)a.b + r * a.b_stride * ty->bytes : nullptr;
        p.sum = a.sum ? (char*)a.sum + r * a.sum_stride * ty->bytes : nullptr;
        p.q = a.q + r * a.q_stride;
        p.scale = a.scale + r;
        p.values = a.values ? a.values + r * a.cols : nullptr;
        void* params[] = {&p};
        HH_TRY_HIP(hipModuleLaunchKernel(f, (uint32_t)((n + per - 1) / per), 1, 1, (uint32_t)threads, (uint32_t)per, 1, 0,
                                         stream, params, nullptr),
                   "hipModuleLaunchKernel(i8 rows)");
    }
    return HH_OK;
}

// Which form, by the weights' bytes, the tokens and the tiles.  Measured (us) over three sets of tensors in
// turn / over 1 GB of them: three sets of up to 85 MB stay in the 256 MB memory-side cache.
//   rows by v_dot4: one or two tokens (28672 x 4096: 22.4 / 22.6 and 23.6 / 23.8, small tiles 27.1 / 27.1 and
//     27.2 / 27.4; 4096 x 14336: 11.3 / 13.2 and 12.2 / 14.1, 12.9 / 18.4); up to four where their codes take
//     32 KB of LDS or less (4096 x 4096: 7.0 / 7.8, 7.3 / 8.9; 32000 x 2048: 15.0 / 17.3, 16.2 / 20.6; past it
//     4096 x 14336: 14.5 / 16.8, 12.8 / 18.6); up to eight under 4 MB of weights (576 x 1536: 5.3 / 5.7,
//     6.1 / 6.8; past it 4096 x 4096: 8.9 / 10.0, 7.2 / 9.1)
//   tiles of 32 x 32 to 32 tokens (28672 x 4096, 32 tokens: 31.0 / 31.3, of 64 x 64 31.4 / 32.2), and to 64 where
//     64-row tiles are few (4096 x 14336, 61 tokens: 15.4 / 23.2, 15.9 / 18.5, so the side that the cache favours;
//     28672 x 4096, 64 tokens: 40.5 / 41.5, 33.7 / 34.5), and where 64 x 64 tiles would not give every other CU
//     one (1000 x 2048, 100 tokens: 5.7 / 6.9, 8.7 / 9.4; 512 x 4096, 200: 7.6 / 9.7, 8.7 / 9.6; with 256 of
//     them, 4096 x 4096, 200: 17.3 / 20.9, 9.8 / 13.0)
//   past that the least of the estimates below.
struct I8Big {
    const char* name;
    size_t tm, tn, threads, per_cu;
    double first, round, stage;  // us: once, per round of tiles, per stage of 128 codes and round
};
// Fitted to all forms' times, three sets in turn, at 20 shapes of 128 to 14336 codes, 159 to 49152 rows and 100 to
// 4096 tokens: there the choice is within 1% of the best on average and 6% at most; of nine more shapes it is
// 10% off at one (28672 x 4096, 256 tokens: 128x256 54.6 / 57.1, 128x128 49.8 / 49.4).  As above: 4751 x 467,
// 612 tokens: 128x128 8.7 / 11.1, 64 x 64 15.7 / 17.1; 4096 x 4096, 256: 23.5 / 32.8, 10.2 / 13.7; 14336 x 4096, 200:
// 25.9 / 34.7, 36.7 / 39.6; 28672 x 4096, 2048: 256x256 242, 192x256 250.
static const I8Big kI8Big[] = {
    {"128x128", 128, 128, 256, 2, 2, 6, 1.04},  // one a CU: 3 a round, 0.67 a stage
    {"128x256", 128, 256, 512, 1, 2, 7, 0.92},
    {"192x256", 192, 256, 512, 1, 5, 10, 1.2},
    {"256x256", 256, 256, 512, 1, 5, 13, 1.45},
};

hh_status hh_engine::enqueue_i8_gemm(int type, hh_i8_gemm_args a) {
    const std::string ty = act_type(type)->name;
    const size_t cus = (size_t)props.multiProcessorCount, chunk_bytes = (a.n + 1023) / 1024 * 1024;
    const size_t weights = (size_t)a.m * a.n, stages = (a.n + 127) / 128;
    hipFunction_t f;
    const uint32_t T = a.t <= 2 ? a.t : a.t <= 4 ? 4 : 8;
    const size_t lds = T * chunk_bytes;
    if (lds <= 131072 && (a.t <= 2 || (a.t <= 4 && lds <= 32768) || (a.t <= 8 && weights < (4u << 20)))) {
        HH_TRY(kernel("hh_i8_rowdot_t" + std::to_string(T) + "_" + ty, &f));
        const size_t grid = std::min(cus, ((size_t)a.m + 15) / 16);
        void* params[] = {&a};
        HH_TRY_HIP(hipModuleLaunchKernel(f, (uint32_t)grid, 1, 1, 512, 1, 1, (unsigned)lds, stream, params, nullptr),
                   "hipModuleLaunchKernel(i8_gemm rows)");
        return HH_OK;
    }
    auto tiles = [&](size_t tm, size_t tn) { return (a.m + tm - 1) / tm * ((a.t + tn - 1) / tn); };
    size_t tm = 64;  // the small tiles' side
    if (a.t <= 32 || (a.t <= 64 && a.m < 8192) || 2 * tiles(64, 64) <= cus) tm = 32;
    const size_t n = tiles(tm, tm), whole = n >= 2 * cus ? 2 * cus : cus;  // (workgroups: below)
    // whole tiles hold the offsets of up to 256 rows in 32 bits
    if (tm == 64 && std::max(a.w_stride, a.x_stride) <= (1u << 24)) {
        const I8Big* best = nullptr;
        // small tiles: each one, its stages, and the exchange unless the workgroups get whole ones
        double least = 3 + (1.3 + 0.208 * (double)stages) * (double)n / (double)cus + (n % whole ? 8 : 0);
        for (const I8Big& b : kI8Big) {
            const size_t k = tiles(b.tm, b.tn), slots = cus * b.per_cu;
            const bool one = b.per_cu > 1 && k <= cus;
            const double t = b.first + (double)((k + slots - 1) / slots) *
                                           ((one ? 3 : b.round) + (one ? 0.67 : b.stage) * (double)stages);
            if (t < least) {
                least = t;
                best = &b;
            }
        }
        if (best) {
            a.mtiles = (uint32_t)((a.m + best->tm - 1) / best->tm);
            a.ttiles = (uint32_t)((a.t + best->tn - 1) / best->tn);
            const size_t k = (size_t)a.mtiles * a.ttiles;
            const size_t grid = std::min(std::max<size_t>(cus * best->per_cu / 8, 1) * 8, (k + 7) / 8 * 8);
            if (k > UINT32_MAX / 2) return fail(HH_ERR_INVALID, "gemm_i8: %u x %u outputs are too many", a.t, a.m);
            HH_TRY(kernel(std::string("hh_i8_big_") + best->name + "_" + ty, &f));
            return launch(f, (uint32_t)grid, (uint32_t)best->threads, a);
        }
    }
    a.mtiles = (uint32_t)((a.m + tm - 1) / tm);
    a.ttiles = (uint32_t)((a.t + tm - 1) / tm);
    const size_t units = n * stages;
    if (n > UINT32_MAX / 2) return fail(HH_ERR_INVALID, "gemm_i8: %u x %u outputs are too many", a.t, a.m);
    // workgroups, each a tile or two stages at least: two a CU where that cuts few tiles (28672 x 4096, 32 tokens, 896
    // tiles: 29.4, one a CU 35.6; 4096 x 14336, 32 tokens, 128 tiles: 14.4, 13.2)
    size_t W = n >= (tm == 32 ? 1 : 2) * cus ? 2 * cus : cus;
    W = std::min(W, std::max(n, units / 2));
    W = W >= 8 ? W / 8 * 8 : W;
    HH_TRY(grow(&ws_part, &ws_part_cap, W * 2 * tm * tm * sizeof(int)));
    if (ws_cnt_cap < n * sizeof(uint32_t)) {
        HH_TRY(grow(&ws_cnt, &ws_cnt_cap, n * sizeof(uint32_t)));
        if (hipError_t err = hipMemsetAsync(ws_cnt, 0, ws_cnt_cap, stream); err != hipSuccess) {
            ws_cnt_cap = 0;
            return hip_fail(err, "hipMemsetAsync(counters)");
        }
    }
    a.cut = (int*)ws_part;
    a.count = (uint32_t*)ws_cnt;
    HH_TRY(kernel(std::string("hh_i8_tile_") + (tm == 32 ? "32x32_" : "64x64_") + ty, &f));
    return launch(f, (uint32_t)W, 256, a);
}

// Sizes of sample.hip.
static const size_t kSmpChunk = 512, kSmpBins = 1024, kSmpList = 8192, kSmpCutBytes = 32;
static const size_t kSmpRows = 1024;  // rows a pass: bounds the workspace (80 KB a row and 8 bytes a chunk)

hh_status hh_engine::enqueue_sample(int type, size_t rows, hh_sample_args a) {
    const ActType* ty = act_type(type);
    hipFunction_t f[4];
    const char* names[] = {"max", "hist", "gather", "pick"};
    for (int i = 0; i < 4; i++) HH_TRY(kernel(std::string("hh_sample_") + names[i] + "_" + ty->name, &f[i]));
    const size_t pass = std::min(rows, kSmpRows);
    a.chunks = (uint32_t)((a.vocab + kSmpChunk - 1) / kSmpChunk);
    // parts of 4096 tokens or more (of 8192: 23.6 us a row of 128256, 21.3), two a CU at most: each begins
    // with the row's largest logit and bins (64 x 128256, a normal body and 40 likely tokens a row, eight requests'
    // filters in turn: 56.6 us, four a CU 55.9, one 62.1; 330 x 14006: 48.1, 50.5, 53.6)
    a.parts = (uint32_t)std::max<size_t>(
        1, std::min<size_t>((a.vocab + 4095) / 4096, (2 * (size_t)props.multiProcessorCount + pass - 1) / pass));
    const size_t row_bytes = 8 * (a.parts + kSmpBins + a.chunks + kSmpList) + 4 * kSmpBins + kSmpCutBytes + 4;
    HH_TRY(grow(&ws_smp, &ws_smp_cap, pass * row_bytes));
    a.top = (uint64_t*)ws_smp;
    a.mass = a.top + pass * a.parts;
    a.sure = a.mass + pass * kSmpBins;
    a.list = a.sure + pass * a.chunks;
    a.cut = a.list + pass * kSmpList;
    a.count = (uint32_t*)((char*)a.cut + pass * kSmpCutBytes);
    a.listed = a.count + pass * kSmpBins;
    for (size_t r = 0; r < rows; r += pass) {
        const size_t n = std::min(pass, rows - r);
        hh_sample_args b = a;
        b.x = (const char*)a.x + r * a.stride * ty->bytes;
        b.params = (const char*)a.params + r * sizeof(hh_sample_params);
        b.u = a.u + r;
        b.ids = a.ids + r;
        b.probs = a.probs ? a.probs + r : nullptr;
        void* params[] = {&b};
        for (int i = 0; i < 3; i++)
            HH_TRY_HIP(hipModuleLaunchKernel(f[i], a.parts, (uint32_t)n, 1, 512, 1, 1, 0, stream, params, nullptr),
                       "hipModuleLaunchKernel(sample)");
        HH_TRY(launch(f[3], (uint32_t)n, 1024, b));
    }
    return HH_OK;
}
