// The residual's addition and the root-mean-square norm of a row:
//
//     r = x + residual,   rstd = (mean(r^2) + eps)^(-1/2),   y = r rstd weight
//
// r goes out in the residual's type; y in x's, or in 8 bits (e4m3) as q with the row's scale: y = q scale, scale = max|y| / 448.
// Backwards, with w = gy weight and xhat = r rstd:   gr = gresidual + rstd (w - xhat mean(w xhat)),   gweight = sum over rows of gy xhat;
// gr is the gradient of x and of the incoming residual alike.
//
// Bound by memory (32768 rows of 2560 bf16, residual fp32: forward 171 us = 5.9 TB/s, backward 262 us = 5.1 TB/s; 4096 rows of 4096 to 8 bits
// 28 us = 6.6 TB/s): a row is read once and stays in registers between its sum of squares (and its largest value) and its output.
// A row belongs to one wavefront or to four; wider rows than those hold are read again, from the cache.  The norm is that of the sum before it is
// rounded to the residual's type, also backwards: there r is the forward's fp32 sum, or added up again.
#include "common.h"
#include "row_sums.h"
#include "vec.h"

namespace wkv {
namespace norm {

struct Call {
    int rows, C, w32;                  // w32: weight is fp32, else in x's type
    long long xs, rs;                  // row strides of x and the residual, in elements
    float eps;
    const void *x, *residual, *weight;
    void *y, *out, *q;                 // out: r, in the residual's type, or NULL
    float *rstd, *scale;
    // backward
    const void *gy, *gout;             // gout: of r, or NULL
    void *gx, *gres;                   // gres NULL: of x's type, gx is both
    float *part;
};

template <int V> __device__ __forceinline__ void store_e4m3(uint8_t *p, const float (&o)[V]) {
    if constexpr (V == 8) {
        uint2 b = {0, 0};
        b.x = __builtin_amdgcn_cvt_pk_fp8_f32(o[0], o[1], b.x, false);
        b.x = __builtin_amdgcn_cvt_pk_fp8_f32(o[2], o[3], b.x, true);
        b.y = __builtin_amdgcn_cvt_pk_fp8_f32(o[4], o[5], b.y, false);
        b.y = __builtin_amdgcn_cvt_pk_fp8_f32(o[6], o[7], b.y, true);
        *reinterpret_cast<uint2 *>(p) = b;
    } else {
        *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(o[0], o[0], 0, false);
    }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        const float o = __shfl_xor(v, m);
        v = o > v || o != o ? o : v;          // (a NaN stays)
    }
    return v;
}
// over the row's wavefronts; slot: of `red`, a different one for every use between two barriers
template <int WAVES, bool MAX> __device__ __forceinline__ float over_row(float v, float (&red)[4]) {
    v = MAX ? wave_max(v) : wave_sum(v);
    if constexpr (WAVES == 1) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < WAVES; i++) s = MAX ? (red[i] > s || red[i] != red[i] ? red[i] : s) : s + red[i];
    return s;
}

// a row's elements in registers, N pieces of V per lane, or (N = 0) read again for every use
template <int V, int N, int LANES> struct Pieces {
    template <class F> static __device__ __forceinline__ void each(int C, int lane, F f) {
        if constexpr (N > 0) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int c = (i * LANES + lane) * V;
                if (c < C) f(i, c);
            }
        } else {
            for (int c = lane * V; c < C; c += LANES * V) f(0, c);
        }
    }
};

// N = 0: rows of any width, V = 1 where a row is not in whole 8-element pieces
template <class T, class R, int V, int N, int WAVES, bool Q>
__global__ __launch_bounds__(64 * WAVES) void forward(const Call k) {
    typedef Pieces<V, N, 64 * WAVES> P;
    __shared__ float red[2][4];
    const size_t row = blockIdx.x;
    const int lane = threadIdx.x;
    const T *x = static_cast<const T *>(k.x) + row * k.xs;
    const R *residual = k.residual ? static_cast<const R *>(k.residual) + row * k.rs : nullptr;
    float r[N ? N : 1][V];
    auto take = [&](int i, int c) {
        float e[V];
        load_vec(x + c, r[i]);
        if (residual) {
            load_vec(residual + c, e);
#pragma unroll
            for (int v = 0; v < V; v++) r[i][v] += e[v];
        }
    };
    auto weighted = [&](int i, int c, float by, float (&o)[V]) {
        float w[V];
        if (k.w32) load_vec(static_cast<const float *>(k.weight) + c, w);
        else load_vec(static_cast<const T *>(k.weight) + c, w);
#pragma unroll
        for (int v = 0; v < V; v++) o[v] = r[i][v] * by * w[v];
    };
    float sum = 0.f;
    P::each(k.C, lane, [&](int i, int c) {
        take(i, c);
#pragma unroll
        for (int v = 0; v < V; v++) sum = fmaf(r[i][v], r[i][v], sum);
        if (k.out) store_vec(static_cast<R *>(k.out) + row * k.C + c, r[i]);
    });
    const float rstd = rsqrtf(over_row<WAVES, false>(sum, red[0]) / (float)k.C + k.eps);
    if (k.rstd && lane == 0) k.rstd[row] = rstd;
    if constexpr (!Q) {
        P::each(k.C, lane, [&](int i, int c) {
            if (N == 0) take(i, c);
            float o[V];
            weighted(i, c, rstd, o);
            store_vec(static_cast<T *>(k.y) + row * k.C + c, o);
        });
    } else {
        float top = 0.f;
        P::each(k.C, lane, [&](int i, int c) {
            if (N == 0) take(i, c);
            float o[V];
            weighted(i, c, rstd, o);
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (N > 0) r[i][v] = o[v];
                const float m = fabsf(o[v]);
                top = m > top || m != m ? m : top;
            }
        });
        top = over_row<WAVES, true>(top, red[1]);
        // (a scale below the smallest normal number would have no reciprocal)
        const float scale = top > 0.f || top != top ? fmaxf(top / 448.f, 1.17549435e-38f) : 1.f, by = 1.f / scale;
        if (lane == 0) k.scale[row] = scale;
        P::each(k.C, lane, [&](int i, int c) {
            float o[V];
            if (N == 0) {
                take(i, c);
                weighted(i, c, rstd, o);
            }
#pragma unroll
            for (int v = 0; v < V; v++) o[v] = (N == 0 ? o[v] : r[i][v]) * by;
            store_e4m3(static_cast<uint8_t *>(k.q) + row * k.C + c, o);
        });
    }
}

// A workgroup takes every gridDim.x'th row, so that the weight's gradient is summed in registers (N = 0: in its row of `part`)
template <class T, class R, int V, int N, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void backward(const Call k) {
    typedef Pieces<V, N, 64 * WAVES> P;
    __shared__ float red[2][4];
    const int lane = threadIdx.x;
    float *part = k.part + (size_t)blockIdx.x * k.C;
    float gw[N ? N : 1][V];
    if constexpr (N > 0) {
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int v = 0; v < V; v++) gw[i][v] = 0.f;
    } else {
        P::each(k.C, lane, [&](int, int c) {
#pragma unroll
            for (int v = 0; v < V; v++) part[c + v] = 0.f;
        });
    }
    int turn = 0;
    for (size_t row = blockIdx.x; row < (size_t)k.rows; row += gridDim.x, turn ^= 1) {
        const float rstd = k.rstd[row];
        float xh[N ? N : 1][V], w[N ? N : 1][V];
        auto take = [&](int i, int c, bool sum_weight) {
            float g[V];
            if (k.w32) load_vec(static_cast<const float *>(k.weight) + c, w[i]);
            else load_vec(static_cast<const T *>(k.weight) + c, w[i]);
            load_vec(static_cast<const T *>(k.gy) + row * k.C + c, g);
            if (k.residual) load_vec(static_cast<const R *>(k.residual) + row * k.rs + c, xh[i]);
            if (k.x) {
                float e[V];
                load_vec(static_cast<const T *>(k.x) + row * k.xs + c, e);
#pragma unroll
                for (int v = 0; v < V; v++) xh[i][v] = k.residual ? xh[i][v] + e[v] : e[v];
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                xh[i][v] *= rstd;
                w[i][v] *= g[v];
                if (sum_weight) {
                    if (N > 0) gw[i][v] = fmaf(g[v], xh[i][v], gw[i][v]);
                    else part[c + v] = fmaf(g[v], xh[i][v], part[c + v]);
                }
            }
        };
        float dot = 0.f;
        P::each(k.C, lane, [&](int i, int c) {
            take(i, c, true);
#pragma unroll
            for (int v = 0; v < V; v++) dot = fmaf(w[i][v], xh[i][v], dot);
        });
        const float mean = over_row<WAVES, false>(dot, red[turn]) / (float)k.C;
        P::each(k.C, lane, [&](int i, int c) {
            if (N == 0) take(i, c, false);
            float o[V], e[V];
            if (k.gout) load_vec(static_cast<const R *>(k.gout) + row * k.C + c, e);
#pragma unroll
            for (int v = 0; v < V; v++) o[v] = fmaf(rstd, fmaf(-mean, xh[i][v], w[i][v]), k.gout ? e[v] : 0.f);
            store_vec(static_cast<T *>(k.gx) + row * k.C + c, o);
            if (k.gres) store_vec(static_cast<R *>(k.gres) + row * k.C + c, o);
        });
    }
    if constexpr (N > 0)
        P::each(k.C, lane, [&](int i, int c) {
#pragma unroll
            for (int v = 0; v < V; v++) part[c + v] = gw[i][v];
        });
}

// Wavefronts per row and pieces per lane: one wavefront up to 1024 elements (no barrier), else four, 8192 elements in registers; rows that are not in
// whole 8-element pieces go element by element, by four wavefronts (in registers too: read again, 5424 rows of 646 fp8 20 us, so 12)
struct Shape { int waves, n; };
static inline Shape shape_of(int C, bool wide) {
    if (!wide) return {4, C <= 1024 ? 4 : C <= 4096 ? 16 : C <= 8192 ? 32 : 0};
    const int v = C / 8;
    if (v <= 64) return {1, 1};
    if (v <= 128) return {1, 2};
    return v <= 256 ? Shape{4, 1} : v <= 512 ? Shape{4, 2} : v <= 1024 ? Shape{4, 4} : Shape{4, 0};
}
static inline int backward_groups(int rows, int C) { return std::max(1, std::min(rows, (C <= 1024 ? 8 : 4) * cu_count())); }

#define WKV_NORM_SHAPES(LAUNCH)                                          \
    do {                                                                 \
        const Shape f = shape_of(k.C, wide);                             \
        if (!wide && f.n == 4) LAUNCH(1, 4, 4);                          \
        else if (!wide && f.n == 16) LAUNCH(1, 16, 4);                   \
        else if (!wide && f.n == 32) LAUNCH(1, 32, 4);                   \
        else if (!wide) LAUNCH(1, 0, 4);                                 \
        else if (f.waves == 1 && f.n == 1) LAUNCH(8, 1, 1);              \
        else if (f.waves == 1) LAUNCH(8, 2, 1);                          \
        else if (f.n == 1) LAUNCH(8, 1, 4);                              \
        else if (f.n == 2) LAUNCH(8, 2, 4);                              \
        else if (f.n == 4) LAUNCH(8, 4, 4);                              \
        else LAUNCH(8, 0, 4);                                            \
    } while (0)

template <class T, class R> static hipError_t forward_t(hipStream_t s, const Call &k, bool wide) {
#define WKV_NORM(V, N, W)                                                                                                      \
    do {                                                                                                                       \
        if (k.q) hipLaunchKernelGGL((forward<T, R, V, N, W, true>), dim3(k.rows), dim3(64 * W), 0, s, k);                      \
        else hipLaunchKernelGGL((forward<T, R, V, N, W, false>), dim3(k.rows), dim3(64 * W), 0, s, k);                         \
    } while (0)
    WKV_NORM_SHAPES(WKV_NORM);
#undef WKV_NORM
    return hipGetLastError();
}
template <class T, class R> static hipError_t backward_t(hipStream_t s, const Call &k, bool wide, void *gweight) {
    const int groups = backward_groups(k.rows, k.C);
#define WKV_NORM(V, N, W) hipLaunchKernelGGL((backward<T, R, V, N, W>), dim3(groups), dim3(64 * W), 0, s, k)
    WKV_NORM_SHAPES(WKV_NORM);
#undef WKV_NORM
    Sums<ToRow<T>> sums;
    sums.add(groups, (size_t)k.C, k.part, {gweight, k.w32 != 0});
    sum_rows_launch(s, sums);
    return hipGetLastError();
}

}  // namespace norm
}  // namespace wkv
