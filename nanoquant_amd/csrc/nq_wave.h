// Reductions and scans over a wave without LDS: a ds_bpermute (what __shfl compiles to) takes over a hundred cycles on a
// chain of dependent steps, these a few each.
#pragma once

#include "nq_common.h"

namespace nq {

// Largest over lanes l, l ^ 16, l ^ 32 and l ^ 48; over l and l ^ 32.
__device__ inline float max_xor32(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // {low half twice, high half twice}
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}
__device__ inline float max_xor16(float v) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);  // the even rows of 16 lanes twice, the odd ones twice
    return fmaxf(__builtin_bit_cast(float, static_cast<uint32_t>(r[0])), __builtin_bit_cast(float, static_cast<uint32_t>(r[1])));
}

// Smallest and largest over lanes 0 to kLanes - 1 (16 or 32), the same in the whole wave.
template <int kControl>
__device__ inline int dpp_or_own(int v) {  // of the lane that a DPP control names, the lane's own where there is none
    return __builtin_amdgcn_update_dpp(v, v, kControl, 0xF, 0xF, false);
}
template <int kLanes>
__device__ inline int least_of(int v) {
    v = min(v, dpp_or_own<0x111>(v));  // row_shr:1
    v = min(v, dpp_or_own<0x112>(v));
    v = min(v, dpp_or_own<0x114>(v));
    v = min(v, dpp_or_own<0x118>(v));
    if (kLanes == 32) v = min(v, dpp_or_own<0x142>(v));  // row_bcast:15
    return __builtin_amdgcn_readlane(v, kLanes - 1);
}
template <int kLanes>
__device__ inline int largest_of(int v) { return ~least_of<kLanes>(~v); }

// u of the lane that a DPP control names, 0 where there is none or the row is masked out.
template <int kControl, int kRows>
__device__ inline uint64_t dpp(uint64_t u) {
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u), kControl, kRows, 0xF, false));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), kControl, kRows, 0xF, false));
    return static_cast<uint64_t>(hi) << 32 | lo;
}
template <int kControl, int kRows>
__device__ inline double dpp(double v) {
    return __builtin_bit_cast(double, dpp<kControl, kRows>(__builtin_bit_cast(uint64_t, v)));
}

// Inclusive running sum over the lanes: shifts within rows of 16, then each row's last lane to the rows behind it.
__device__ inline double wave_scan(double v) {
    v += dpp<0x111, 0xF>(v);  // row_shr:1
    v += dpp<0x112, 0xF>(v);
    v += dpp<0x114, 0xF>(v);
    v += dpp<0x118, 0xF>(v);
    v += dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ inline uint64_t read_lane(uint64_t u, int lane) {  // the same lane for the whole wave
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u), lane));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane));
    return static_cast<uint64_t>(hi) << 32 | lo;
}
__device__ inline double read_lane(double v, int lane) {
    return __builtin_bit_cast(double, read_lane(__builtin_bit_cast(uint64_t, v), lane));
}
__device__ inline uint64_t wave_largest(uint64_t v) {
    auto larger = [](uint64_t a, uint64_t b) { return a > b ? a : b; };
    v = larger(v, dpp<0x111, 0xF>(v));
    v = larger(v, dpp<0x112, 0xF>(v));
    v = larger(v, dpp<0x114, 0xF>(v));
    v = larger(v, dpp<0x118, 0xF>(v));
    v = larger(v, dpp<0x142, 0xA>(v));
    v = larger(v, dpp<0x143, 0xC>(v));
    return read_lane(v, 63);
}
__device__ inline double wave_total(double v) { return read_lane(wave_scan(v), 63); }

}  // namespace nq
