// Reductions over groups of lanes: every lane of a group of L gets the same result.  The steps inside 16 lanes are
// data-parallel-primitive moves (xor 1, xor 2, mirror of 8, mirror of 16), the ones above swap rows of 16 and halves
// of 32, so none goes through the LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace fbfc {

template <int CTRL, typename T>
__device__ __forceinline__ T lane_move(T v)
{
    static_assert(sizeof(T) == 4, "32 bits a lane");
    const int moved = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(T, moved);
}

template <int L, typename T, typename F>
__device__ __forceinline__ T lanes_reduce(T v, F f)
{
    static_assert(L == 8 || L == 16 || L == 32 || L == 64, "groups of 8, 16, 32 or 64 lanes");
    v = f(v, lane_move<0xB1>(v));
    v = f(v, lane_move<0x4E>(v));
    v = f(v, lane_move<0x141>(v));
    if constexpr (L >= 16) v = f(v, lane_move<0x140>(v));
    if constexpr (L >= 32) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        const unsigned one = s[0], other = s[1];  // a bit cast of s[1] itself would read s[0]
        v = f(__builtin_bit_cast(T, one), __builtin_bit_cast(T, other));
    }
    if constexpr (L >= 64) {
        const unsigned u = __builtin_bit_cast(unsigned, v);
        const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const unsigned one = s[0], other = s[1];  // a bit cast of s[1] itself would read s[0]
        v = f(__builtin_bit_cast(T, one), __builtin_bit_cast(T, other));
    }
    return v;
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v)
{
    return lanes_reduce<L>(v, [](float a, float b) { return a + b; });
}

}  // namespace fbfc
