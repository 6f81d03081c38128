// Sums over the rows of (rows, n) fp32 arrays, the last step of every gradient that the whole batch shares: workgroups leave
// partial sums, this adds them up in a fixed order, so that the result repeats to the bit.
#pragma once
#include "common.h"

namespace wkv {

// where element i of a result goes
template <class T> struct ToRow {
    void *out;
    bool wide;                     // fp32, else T
    __device__ __forceinline__ void operator()(size_t i, float v) const {
        if (wide) static_cast<float *>(out)[i] = v;
        else static_cast<T *>(out)[i] = from_float<T>(v);
    }
};
constexpr int MAX_SUMS = 5;
template <class O> struct Sums {               // up to five arrays in one launch: a launch costs more than a small one's sum
    struct { const float *in; size_t n; int rows, blocks; O out; } job[MAX_SUMS];
    int count = 0;
    void add(int rows, size_t n, const float *in, O out) { job[count++] = {in, n, rows, (int)((n + 63) / 64), out}; }
};

// 64 columns per workgroup; its wavefronts share the rows
template <class O, int WAVES>
static __global__ __launch_bounds__(64 * WAVES) void sum_rows(Sums<O> sums, int first) {
    __shared__ float part[WAVES][64];
    int block = first + (int)blockIdx.x, j = 0;
    while (j + 1 < sums.count && block >= sums.job[j].blocks) block -= sums.job[j++].blocks;
    const auto &job = sums.job[j];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = job.rows;
    const size_t i = (size_t)block * 64 + lane, n = job.n;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (i < n) {
        const float *p = job.in + i;
        int r = wave;
        for (; r + 3 * WAVES < rows; r += 4 * WAVES)
#pragma unroll
            for (int u = 0; u < 4; u++) s[u] += p[(size_t)(r + u * WAVES) * n];
        for (; r < rows; r += WAVES) s[0] += p[(size_t)r * n];
    }
    part[wave][lane] = (s[0] + s[1]) + (s[2] + s[3]);
    __syncthreads();
    if (wave == 0 && i < n) {
        float all = part[0][lane];
#pragma unroll
        for (int w = 1; w < WAVES; w++) all += part[w][lane];
        job.out(i, all);
    }
}
constexpr long long SUMS_PER_LAUNCH = 1 << 21;          // workgroups: a grid has fewer than 2^32 threads
// 16 wavefronts where there are many rows: 1024 rows of 2560 columns 22 us with four, 8 with sixteen
template <class O> static void sum_rows_launch(hipStream_t s, const Sums<O> &sums) {
    long long blocks = 0;
    int rows = 0;
    for (int j = 0; j < sums.count; j++) {
        blocks += sums.job[j].blocks;
        rows = std::max(rows, sums.job[j].rows);
    }
    for (long long first = 0; first < blocks; first += SUMS_PER_LAUNCH) {
        const dim3 grid((unsigned)std::min(blocks - first, SUMS_PER_LAUNCH));
        if (rows >= 64) hipLaunchKernelGGL((sum_rows<O, 16>), grid, dim3(1024), 0, s, sums, (int)first);
        else hipLaunchKernelGGL((sum_rows<O, 4>), grid, dim3(256), 0, s, sums, (int)first);
    }
}

}  // namespace wkv
