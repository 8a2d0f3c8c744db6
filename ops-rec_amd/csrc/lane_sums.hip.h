// Sums over 8, 16, 32 or all 64 lanes of a wavefront, the same bits in all of them: DPP moves within 16 lanes, lane swaps beyond.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace hstu {

template <int CTRL>
__device__ __forceinline__ float dpp_of(float v)
{
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// (the elements are taken out first: this compiler casts element 0 for every element of a vector)
typedef uint32_t lane_pair_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ float swapped_sum(lane_pair_t s)
{
    const uint32_t a = s[0], b = s[1];
    return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

template <int G>
__device__ __forceinline__ float wave_sum(float v)
{
    v += dpp_of<0xB1>(v);   // lanes 1, 0, 3, 2 of a quad
    v += dpp_of<0x4E>(v);   // 2, 3, 0, 1
    v += dpp_of<0x141>(v);  // the other quad of 8 lanes
    if constexpr (G >= 16) {
        v += dpp_of<0x140>(v);  // the other 8 of 16 lanes
    }
    if constexpr (G >= 32) {
        v = swapped_sum(__builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false));
    }
    if constexpr (G >= 64) {
        v = swapped_sum(__builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v), __builtin_bit_cast(uint32_t, v), false, false));
    }
    return v;
}

}  // namespace hstu
