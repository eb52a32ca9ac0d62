// Sums over the rows of partial results, always in the same order: a workgroup of 1024 threads takes 16 columns and splits the
// rows over 64 slices, each of which keeps 8 loads in flight (with one at a time, 2048 rows of 1000 columns took 42 us).
#pragma once
#include <hip/hip_runtime.h>

namespace fbfc {

constexpr int kSumColumns = 16, kSumSlices = 64, kSumThreads = kSumColumns * kSumSlices;

// Rows slice, slice + 64, ... of a column.
__device__ __forceinline__ float slice_sum(const float *column, long stride, long rows, int slice)
{
    float sum[8] = {};
    long r = slice;
    for (; r + 7 * kSumSlices < rows; r += 8 * kSumSlices)
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] += column[(r + i * kSumSlices) * stride];
    for (; r < rows; r += kSumSlices) sum[0] += column[r * stride];
    return ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
}

// The sum over the slices, in threads 0 to 15; `part` is LDS for this sum alone.
__device__ __forceinline__ float slices_sum(float v, float (*part)[kSumColumns])
{
    const int i = threadIdx.x % kSumColumns, slice = threadIdx.x / kSumColumns;
    part[slice][i] = v;
    __syncthreads();
#pragma unroll
    for (int n = kSumSlices / 2; n >= 1; n /= 2) {
        if (slice < n) part[slice][i] += part[slice + n][i];
        __syncthreads();
    }
    return part[0][i];
}

}  // namespace fbfc
