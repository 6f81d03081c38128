// Sums over the rows of a (rows, n) fp32 array, the last step of every gradient that the whole batch shares: workgroups leave
// partial sums, this adds them up in a fixed order, so that the result repeats to the bit.
#pragma once
#include "common.h"

namespace wkv {

// element i of the result to out[i]
template <class T> struct ToRow {
    T *out;
    __device__ __forceinline__ void operator()(size_t i, float v) const { out[i] = from_float<T>(v); }
};

// 64 columns per workgroup, its four wavefronts every fourth row
template <class O>
static __global__ __launch_bounds__(256) void sum_rows(int rows, size_t n, const float *__restrict__ in, O out) {
    __shared__ float part[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const size_t i = (size_t)blockIdx.x * 64 + lane;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < n) {
        const float *p = in + i;
        int r = wave;
        for (; r + 12 < rows; r += 16)
#pragma unroll
            for (int u = 0; u < 4; u++) s[u] += p[(size_t)(r + 4 * u) * n];
        for (; r < rows; r += 4) s[0] += p[(size_t)r * n];
    }
    part[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (wave == 0 && i < n) out(i, (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]));
}
template <class O> static void sum_rows_launch(hipStream_t s, int rows, size_t n, const float *in, O out) {
    hipLaunchKernelGGL((sum_rows<O>), dim3((unsigned)((n + 63) / 64)), dim3(256), 0, s, rows, n, in, out);
}

}  // namespace wkv
