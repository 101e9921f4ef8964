// qmag_wavesort.h -- selection keys (a value and its place) and a wave's bitonic
// networks over them: what the sampler and the log probabilities share.
#pragma once

#include "qmag_device.h"

namespace qmag {

// value order as unsigned order: larger key = larger value; NaN lowest of
// the numbers' keys (1), 0 = no element
__device__ __forceinline__ uint32_t samp_key(float v)
{
    if (v != v) return 1u;
    const uint32_t b = __float_as_uint(v + 0.0f);        // -0 folded to +0
    const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return k < 2u ? 2u : k;
}
__device__ __forceinline__ float samp_val(uint32_t k)
{
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// unique selection key: the value half, then the complemented index shifted
// up one bit (ids are below 2^31, so the dropped top bit is 1 for all and the
// order among ids is kept); the low bit is the sign of a zero value, which
// the value half folds into +0 (the reference compares -0 and +0 as equal),
// so it never decides an order and only restores the reported value
__device__ __forceinline__ uint64_t samp_comp(uint32_t key, int id, float v)
{
    const uint32_t neg_zero = __float_as_uint(v) == 0x80000000u ? 1u : 0u;
    return ((uint64_t)key << 32) | ((uint32_t)~(uint32_t)id << 1) | neg_zero;
}
__device__ __forceinline__ int samp_id(uint64_t c) { return (int)~(((uint32_t)c >> 1) | 0x80000000u); }
__device__ __forceinline__ float samp_value(uint64_t c)
{
    return (c & 1u) ? -0.0f : samp_val((uint32_t)(c >> 32));
}

// The value of lane (lane ^ m), m one of 1, 2, 4, 8, 16, 32 (a constant once
// the callers' loops are unrolled), by DPP moves and the gfx950 lane swaps
// instead of the LDS crossbar: xor 4 is a half-row mirror (xor 7) then a
// quad reversal (xor 3), xor 8 a row mirror (xor 15) then a half-row mirror.
constexpr int DPP_XOR3 = 0x1B;          // quad_perm [3,2,1,0]
__device__ __forceinline__ uint32_t xor_lane(uint32_t v, int m)
{
    const int x = (int)v;
    switch (m) {
    case 1: return (uint32_t)dpp_i<DPP_XOR1>(x);
    case 2: return (uint32_t)dpp_i<DPP_XOR2>(x);
    case 4: return (uint32_t)dpp_i<DPP_XOR3>(dpp_i<DPP_HALF_MIRROR>(x));
    case 8: return (uint32_t)dpp_i<DPP_HALF_MIRROR>(dpp_i<DPP_MIRROR>(x));
    case 16: {
        // rows 1, 3 of the first result hold rows 0, 2; rows 0, 2 of the
        // second hold rows 1, 3
        auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        return (lane_id() & 16) ? p[0] : p[1];
    }
    default: {
        auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        return (lane_id() & 32) ? p[0] : p[1];
    }
    }
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m)
{
    const uint32_t lo = xor_lane((uint32_t)v, m), hi = xor_lane((uint32_t)(v >> 32), m);
    return ((uint64_t)hi << 32) | lo;
}
// a uniform lane's value
__device__ __forceinline__ uint64_t readlane64(uint64_t v, int src)
{
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, src);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), src);
    return ((uint64_t)hi << 32) | lo;
}

// One compare-exchange step of a bitonic network over keys one per lane
// (element index i): descending order overall.
__device__ __forceinline__ uint64_t bitonic_step(uint64_t v, int i, int size, int stride)
{
    const uint64_t o = shfl_xor64(v, stride);
    const bool keep_max = ((i & stride) == 0) == ((i & size) == 0);
    return (v > o) == keep_max ? v : o;          // one compare: equal keys are equal values
}

// 64 keys, one per lane, sorted descending
__device__ __forceinline__ uint64_t wave_sort64(uint64_t v)
{
    const int lane = lane_id();
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) v = bitonic_step(v, lane, size, stride);
    return v;
}

// a bitonic sequence of 64 keys sorted descending (the merge half of the
// network)
__device__ __forceinline__ uint64_t wave_clean64(uint64_t v)
{
    const int lane = lane_id();
#pragma unroll
    for (int stride = 32; stride > 0; stride >>= 1) v = bitonic_step(v, lane, 64, stride);
    return v;
}

// 32-bit forms of the networks above, for keys without the index half
__device__ __forceinline__ uint32_t bitonic_step32(uint32_t v, int i, int size, int stride)
{
    const uint32_t o = xor_lane(v, stride);
    const bool keep_max = ((i & stride) == 0) == ((i & size) == 0);
    return (v > o) == keep_max ? v : o;
}
__device__ __forceinline__ uint32_t wave_sort64_u32(uint32_t v)
{
    const int lane = lane_id();
#pragma unroll
    for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) v = bitonic_step32(v, lane, size, stride);
    return v;
}
__device__ __forceinline__ uint32_t wave_clean64_u32(uint32_t v)
{
    const int lane = lane_id();
    v = bitonic_step32(v, lane, 64, 32);
    v = bitonic_step32(v, lane, 64, 16);
    v = bitonic_step32(v, lane, 64, 8);
    v = bitonic_step32(v, lane, 64, 4);
    v = bitonic_step32(v, lane, 64, 2);
    return bitonic_step32(v, lane, 64, 1);
}

}  // namespace qmag
