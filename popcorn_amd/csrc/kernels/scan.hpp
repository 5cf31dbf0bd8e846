// Sums of whole numbers over a wave and over a block, in registers (DPP moves;
// a shuffle through LDS takes about 130 cycles, and a scan six of them).
#pragma once

#include "common.hpp"

namespace pk {

// v of the lane that kCtrl names, 0 where there is none or kRows leaves the row out.
template <int kCtrl, int kRows = 0xf>
__device__ inline uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kCtrl, kRows, 0xf, false);
}
template <int kCtrl, int kRows = 0xf>
__device__ inline uint64_t moved(uint64_t v) {
    return (uint64_t)moved<kCtrl, kRows>((uint32_t)(v >> 32)) << 32 | moved<kCtrl, kRows>((uint32_t)v);
}
__device__ inline uint32_t of_lane(uint32_t v, uint32_t lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)lane); }
__device__ inline uint64_t of_lane(uint64_t v, uint32_t lane) {
    return (uint64_t)of_lane((uint32_t)(v >> 32), lane) << 32 | of_lane((uint32_t)v, lane);
}

// Inclusive sums over a row of 16 lanes, and over the wave.
template <typename U>
__device__ inline U row_scan(U v) {
    v += moved<0x111>(v);  // row_shr:1, 2, 4, 8
    v += moved<0x112>(v);
    v += moved<0x114>(v);
    return v + moved<0x118>(v);
}
template <typename U>
__device__ inline U wave_scan(U v) {
    v = row_scan(v);
    v += moved<0x142, 0xa>(v);        // lane 15 of a row to the odd row behind it
    return v + moved<0x143, 0xc>(v);  // lane 31 to the upper half
}
__device__ inline uint64_t wave_sum64(uint64_t v) { return of_lane(wave_scan(v), 63); }
__device__ inline uint32_t wave_max_u32(uint32_t v) {  // (0 is the least)
    v = max(v, moved<0x111>(v));
    v = max(v, moved<0x112>(v));
    v = max(v, moved<0x114>(v));
    v = max(v, moved<0x118>(v));
    v = max(v, moved<0x142, 0xa>(v));
    return of_lane(max(v, moved<0x143, 0xc>(v)), 63);
}
__device__ inline uint64_t wave_or64(uint64_t v) {
    v |= moved<0x111>(v);
    v |= moved<0x112>(v);
    v |= moved<0x114>(v);
    v |= moved<0x118>(v);
    v |= moved<0x142, 0xa>(v);
    return of_lane(v | moved<0x143, 0xc>(v), 63);
}

template <typename U>
struct Scan {
    U upto, total;
};
// Inclusive sums over a block of kWaves waves (at most 16), and the total;
// `sums` has an entry per wave.
template <uint32_t kWaves, typename U>
__device__ inline Scan<U> block_scan(U v, U *sums) {
    static_assert(kWaves <= 16, "one row of lanes");
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    const U run = row_scan(sums[min(lane & 15, kWaves - 1)]);
    return {(wave ? of_lane(run, wave - 1) : 0) + v, of_lane(run, kWaves - 1)};
}

}  // namespace pk
