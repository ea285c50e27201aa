// Reductions and scans of 64-bit values over a wave by DPP (a shuffle goes through LDS: five times the
// latency).
#ifndef HH_KERNELS_WAVE64_H
#define HH_KERNELS_WAVE64_H

#include "common.h"

template <int CTRL, int ROWS = 0xf>
HH_DEV uint64_t hh_dpp64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, true);
    return (uint64_t)hi << 32 | lo;
}
HH_DEV uint64_t hh_lane64(uint64_t v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
    return (uint64_t)hi << 32 | lo;
}
struct hh_max64 {
    HH_DEV static uint64_t of(uint64_t a, uint64_t b) { return b > a ? b : a; }
};
struct hh_addu64 {
    HH_DEV static uint64_t of(uint64_t a, uint64_t b) { return a + b; }
};
struct hh_addf64 {
    HH_DEV static uint64_t of(uint64_t a, uint64_t b) {
        return (uint64_t)__double_as_longlong(__longlong_as_double((long long)a) + __longlong_as_double((long long)b));
    }
};
// Op over each row of 16 lanes, then over the wave (in lane 63).  Zero is neutral to both.
template <class Op>
HH_DEV uint64_t hh_row16(uint64_t v) {
    v = Op::of(v, hh_dpp64<0xB1>(v));
    v = Op::of(v, hh_dpp64<0x4E>(v));
    v = Op::of(v, hh_dpp64<0x124>(v));
    return Op::of(v, hh_dpp64<0x128>(v));
}
template <class Op>
HH_DEV uint64_t hh_wave64(uint64_t v) {
    v = hh_row16<Op>(v);
    v = Op::of(v, hh_dpp64<0x142, 0xa>(v));
    v = Op::of(v, hh_dpp64<0x143, 0xc>(v));
    return hh_lane64(v, 63);
}
// Inclusive sums over the wave's lanes.
HH_DEV uint64_t hh_scan64(uint64_t v) {
    v += hh_dpp64<0x111>(v);  // row_shr:1, 2, 4, 8: within each 16
    v += hh_dpp64<0x112>(v);
    v += hh_dpp64<0x114>(v);
    v += hh_dpp64<0x118>(v);
    v += hh_dpp64<0x142, 0xa>(v);  // row_bcast:15: rows 1 and 3 add rows 0 and 2
    v += hh_dpp64<0x143, 0xc>(v);  // row_bcast:31: rows 2 and 3 add the first half
    return v;
}
// Inclusive sums over the workgroup's threads (up to 16 waves) in thread order; red: 16 words of LDS.
HH_DEV uint64_t hh_block_scan64(uint64_t v, uint64_t* red) {
    const uint32_t lane = threadIdx.x % HH_WAVE, w = threadIdx.x / HH_WAVE;
    v = hh_scan64(v);
    __syncthreads();
    if (lane == HH_WAVE - 1) red[w] = v;
    __syncthreads();
    return v + hh_lane64(hh_row16<hh_addu64>(lane < w ? red[lane] : 0), 0);
}

#endif
