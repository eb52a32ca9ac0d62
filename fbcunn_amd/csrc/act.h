// Activations in 32, 16 (bfloat16) or 16 (half) bits: vectors of them in memory, numbers of 32 bits in registers.
// Every conversion to fewer bits rounds to the nearest, ties to even.
#pragma once
#include <hip/hip_runtime.h>

namespace fbfc {

enum ActType { kF32 = 0, kBF16 = 1, kF16 = 2 };  // the values of FBFC_F32, FBFC_BF16, FBFC_F16

using bf16 = __bf16;
using f16 = _Float16;

// N consecutive values.  The alignment is that of one value: rows of odd length and views into a flattened storage
// begin anywhere, and gfx950 reads and writes global memory in vectors of up to 16 bytes at any address, so one
// path serves all of them.
template <typename T, int N>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T))));
};
template <typename T, int N>
using Vec = typename VecOf<T, N>::type;

// Always global memory, which the compiler cannot tell of an address that was itself read from memory.
#define FBFC_GLOBAL __attribute__((address_space(1)))
template <int N, typename T>
__device__ __forceinline__ Vec<T, N> load_vec(const T *p)
{
    return *(const FBFC_GLOBAL Vec<T, N> *)(p);
}
template <int N, typename T>
__device__ __forceinline__ void store_vec(T *p, Vec<T, N> v)
{
    *(FBFC_GLOBAL Vec<T, N> *)(p) = v;
}

// The first `n` of N values, the others zero; what lies behind them is not touched.
template <int N, typename T>
__device__ __forceinline__ Vec<T, N> load_some(const T *p, long n)
{
    if (n >= N) return load_vec<N>(p);
    Vec<T, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < n ? ((const FBFC_GLOBAL T *)p)[i] : (T)0.0f;
    return v;
}
template <int N, typename T>
__device__ __forceinline__ void store_some(T *p, Vec<T, N> v, long n)
{
    if (n >= N) {
        store_vec<N>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (i < n) ((FBFC_GLOBAL T *)p)[i] = v[i];
}

// 16 bytes of a row of `channels` values, from place c on.  A load that would pass the row's end is moved back to end there,
// so that no load has a condition (one would make the wavefront wait for the loads before it); end_of_row() then moves the
// values to their places.
template <typename T>
__device__ __forceinline__ Vec<T, 16 / sizeof(T)> load_in_row(const T *row, int c, int channels)
{
    constexpr int V = 16 / sizeof(T);
    if (channels < V) return load_some<V>(row + c, channels - c);  // the same for all lanes
    return load_vec<V>(row + (c + V <= channels ? c : channels - V));
}
template <typename T>
__device__ __forceinline__ void end_of_row(Vec<T, 16 / sizeof(T)> &v, int c, int channels)
{
    constexpr int V = 16 / sizeof(T);
    if (channels < V) return;
    const int over = c + V - channels, bits = (over < 0 ? 0 : over > V ? V : over) * 8 * (int)sizeof(T);
    unsigned long w[2];
    __builtin_memcpy(w, &v, 16);
    if (bits >= 64) {
        w[0] = bits == 128 ? 0 : w[1] >> (bits & 63);
        w[1] = 0;
    } else if (bits > 0) {
        w[0] = w[0] >> bits | w[1] << (64 - bits);
        w[1] >>= bits;
    }
    __builtin_memcpy(&v, w, 16);
}

// sigmoid(z) and sigmoid(-z) = 1 - sigmoid(z), each to its own precision however close the other is to one.  The
// reciprocal is the hardware's, off by one unit.
__device__ __forceinline__ void sigmoid_pair(float z, float &yes, float &no)
{
    const float e = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.0f + e);
    yes = z < 0.0f ? e * r : r;
    no = z < 0.0f ? r : e * r;
}

}  // namespace fbfc
