// Reductions over groups of lanes: every lane of a group of L gets the same result.  The steps inside 16 lanes are
// data-parallel-primitive moves (xor 1, xor 2, mirror of 8, mirror of 16), the ones above swap rows of 16 and halves
// of 32, so none goes through the LDS.
#pragma once
#include <hip/hip_runtime.h>

namespace fbfc {

template <int CTRL>
__device__ __forceinline__ float lane_move(float v)
{
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, true));
}

template <int L, typename F>
__device__ __forceinline__ float lanes_reduce(float v, F f)
{
    static_assert(L == 8 || L == 16 || L == 32 || L == 64, "groups of 8, 16, 32 or 64 lanes");
    v = f(v, lane_move<0xB1>(v));
    v = f(v, lane_move<0x4E>(v));
    v = f(v, lane_move<0x141>(v));
    if (L >= 16) v = f(v, lane_move<0x140>(v));
    if (L >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    if (L >= 64) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = f(__uint_as_float(s[0]), __uint_as_float(s[1]));
    }
    return v;
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v)
{
    return lanes_reduce<L>(v, [](float a, float b) { return a + b; });
}

}  // namespace fbfc
