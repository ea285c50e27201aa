// Copies of whole pages, as if one after another: a thread owns 16 bytes of a layer's page and takes
// the moves in order, so a page may be a target twice, or a source after it was a target.  Eight moves
// at a time are read before any is written, where none reads what another of them writes.
//
// Moves of which none reads or writes what another writes (forks into free pages, live pages into
// holes) are also split over workgroups: each looks all moves through with a bit a page in LDS.  Where
// the look finds a page twice, the first part takes all of them in order.
#include "kv_pages.h"

#define HH_KV_COPY_AT_ONCE 8

extern __shared__ uint32_t hh_kv_bits[];

extern "C" __global__ void __launch_bounds__(256) hh_kv_copy(const hh_kv_copy_args a) {
    constexpr int U = HH_KV_COPY_AT_ONCE;
    uint32_t first = 0, last = a.n;
    if (gridDim.z > 1) {
        __shared__ uint32_t again;
        const uint32_t words = (a.kv.pages + 31) / 32;
        if (threadIdx.x == 0) again = 0;
        for (uint32_t i = threadIdx.x; i < words; i += 256) hh_kv_bits[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.n; i += 256) {
            const uint32_t s = a.moves[2 * i], d = a.moves[2 * i + 1];
            if (s < a.kv.pages && d < a.kv.pages && atomicOr(&hh_kv_bits[d / 32], 1u << d % 32) >> d % 32 & 1) again = 1;
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < a.n; i += 256) {
            const uint32_t s = a.moves[2 * i], d = a.moves[2 * i + 1];
            if (s < a.kv.pages && d < a.kv.pages && hh_kv_bits[s / 32] >> s % 32 & 1) again = 1;
        }
        __syncthreads();
        if (!again) {
            first = (uint32_t)((uint64_t)a.n * blockIdx.z / gridDim.z);
            last = (uint32_t)((uint64_t)a.n * (blockIdx.z + 1) / gridDim.z);
        } else if (blockIdx.z) {
            return;
        }
    }
    const uint32_t chunk = blockIdx.x * 256 + threadIdx.x;
    if (chunk >= a.chunks) return;
    uint8_t* const mine = a.kv.base + blockIdx.y * a.layer_stride + (size_t)chunk * 16;
    for (uint32_t i = first; i < last; i += U) {
        uint32_t s[U], d[U];
        bool clash = false;
#pragma unroll
        for (int j = 0; j < U; j++) {
            const uint32_t m = min(i + j, last - 1);
            s[j] = a.moves[2 * m];
            d[j] = a.moves[2 * m + 1];
            if (i + j >= last || s[j] >= a.kv.pages || d[j] >= a.kv.pages) d[j] = s[j] = ~0u;
#pragma unroll
            for (int k = 0; k < j; k++) clash |= s[j] == d[k] && s[j] != ~0u;
        }
        if (!clash) {
            hh_u4 v[U];
#pragma unroll
            for (int j = 0; j < U; j++) v[j] = *(const hh_u4*)(mine + (s[j] != ~0u ? s[j] : 0) * a.kv.stride);
#pragma unroll
            for (int j = 0; j < U; j++)
                if (s[j] != ~0u) *(hh_u4*)(mine + d[j] * a.kv.stride) = v[j];
        } else {
#pragma unroll
            for (int j = 0; j < U; j++)
                if (s[j] != ~0u) {
                    const hh_u4 w = *(const hh_u4*)(mine + s[j] * a.kv.stride);
                    *(hh_u4*)(mine + d[j] * a.kv.stride) = w;
                }
        }
    }
}
