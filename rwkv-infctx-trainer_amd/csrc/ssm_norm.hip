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
// A row belongs to a part of a wavefront, to one or to four; wider rows than those hold are read again, from the cache (2^20 rows of 128 bf16, as of
// single heads: forward 92 us = 5.8 TB/s, backward 157 us = 5.1 TB/s).  The norm is that of the sum before it is
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
    } else if constexpr (V == 2) {
        *reinterpret_cast<uint16_t *>(p) = (uint16_t)__builtin_amdgcn_cvt_pk_fp8_f32(o[0], o[1], 0, false);
    } else {
        *p = (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(o[0], o[0], 0, false);
    }
}

// The sum or the largest value (a NaN stays) over a row's lanes: part of a wavefront, or several through `red`, which is another one for every use
// between two barriers
template <bool MAX> __device__ __forceinline__ float both(float v, float o) { return MAX ? (o > v || o != o ? o : v) : v + o; }
template <int LANES, bool MAX> __device__ __forceinline__ float over_row(float v, float (&red)[4]) {
#pragma unroll
    for (int m = (LANES < 64 ? LANES : 64) / 2; m > 0; m >>= 1) v = both<MAX>(v, __shfl_xor(v, m));
    if constexpr (LANES <= 64) return v;
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < LANES / 64; i++) s = both<MAX>(s, red[i]);
    return s;
}
// threads of a workgroup: rows of up to one wavefront share it
template <int LANES> constexpr int forward_threads() { return LANES < 64 ? 256 : LANES; }
template <int LANES> constexpr int backward_threads() { return LANES <= 64 ? 512 : LANES; }
// which of the workgroup's rows a lane is at: a scalar unless a wavefront has several
template <int LANES, int THREADS> __device__ __forceinline__ int row_of() {
    if constexpr (LANES == THREADS) return 0;
    else if constexpr (LANES == 64) return __builtin_amdgcn_readfirstlane((int)threadIdx.x / 64);
    else return (int)threadIdx.x / LANES;
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

// N = 0: rows of any width; V = 2 or 1 where a row is not in whole 8-element pieces
template <class T, class R, int V, int N, int LANES, bool Q>
__global__ __launch_bounds__(forward_threads<LANES>()) void forward(const Call k) {
    typedef Pieces<V, N, LANES> P;
    __shared__ float red[2][4];
    const size_t row = (size_t)blockIdx.x * (forward_threads<LANES>() / LANES) + row_of<LANES, forward_threads<LANES>()>();
    const int lane = LANES == forward_threads<LANES>() ? threadIdx.x : threadIdx.x % LANES;
    if (LANES < 64 && row >= (size_t)k.rows) return;
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
    const float rstd = rsqrtf(over_row<LANES, false>(sum, red[0]) / (float)k.C + k.eps);
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
        top = over_row<LANES, true>(top, red[1]);
        // (a scale below the smallest normal number would have no reciprocal.)  The quotient by the reciprocal and what that leaves is the rounded quotient
        // (Markstein); without the second step it is rounded twice, which moves elements in the middle of two 8-bit values.  A division's own
        // instructions took up to 7 % longer (5424 rows of 646 10.3 us against 9.8, 2000 of 9000 43.5 against 40.3).  What is left is that another order of the
        // row's sum moves y by a step of fp32, and with it up to three in 100000 elements that lie that close to such a middle, by one of their steps.
        // per: an infinite scale leaves nothing.
        const float scale = top != top ? top : top > 0.f ? fmaxf(top / 448.f, 1.17549435e-38f) : 1.f, by = 1.f / scale, per = scale < INFINITY ? scale : 0.f;
        if (lane == 0) k.scale[row] = scale;
        P::each(k.C, lane, [&](int i, int c) {
            float o[V];
            if (N == 0) {
                take(i, c);
                weighted(i, c, rstd, o);
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float e = N == 0 ? o[v] : r[i][v], q = e * by;
                o[v] = fmaf(fmaf(-q, per, e), by, q);
            }
            store_e4m3(static_cast<uint8_t *>(k.q) + row * k.C + c, o);
        });
    }
}

// A workgroup takes rows at the grid's distance, so that the weight's gradient is summed in registers (N = 0: in its row of `part`), at the end
// over the workgroup's rows: a row of `part` each, few enough that their sum is short also for few columns
template <class T, class R, int V, int N, int LANES>
__global__ __launch_bounds__(backward_threads<LANES>()) void backward(const Call k) {
    typedef Pieces<V, N, LANES> P;
    constexpr int THREADS = backward_threads<LANES>(), ROWS = THREADS / LANES, WIDTH = V * N * LANES;
    __shared__ float red[2][4];
    __shared__ float sums[ROWS > 1 ? THREADS / 64 : 1][ROWS > 1 ? WIDTH : 1];
    const int lane = LANES == THREADS ? threadIdx.x : threadIdx.x % LANES;          // (masked for nothing, a row's pieces have an address each: 114 -> 156 registers)
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
    for (size_t row = (size_t)blockIdx.x * ROWS + row_of<LANES, THREADS>(); row < (size_t)k.rows; row += (size_t)gridDim.x * ROWS, turn ^= 1) {
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
        const float mean = over_row<LANES, false>(dot, red[turn]) / (float)k.C;
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
    if constexpr (ROWS > 1) {
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int v = 0; v < V; v++) {
#pragma unroll
                for (int m = LANES; m < 64; m <<= 1) gw[i][v] += __shfl_xor(gw[i][v], m);
                if (threadIdx.x % 64 < LANES) sums[threadIdx.x / 64][(i * LANES + lane) * V + v] = gw[i][v];
            }
        __syncthreads();
        for (int c = threadIdx.x; c < k.C; c += THREADS) {
            float s = sums[0][c];
#pragma unroll
            for (int i = 1; i < THREADS / 64; i++) s += sums[i][c];
            part[c] = s;
        }
    } else if constexpr (N > 0) {
        P::each(k.C, lane, [&](int i, int c) {
#pragma unroll
            for (int v = 0; v < V; v++) part[c + v] = gw[i][v];
        });
    }
}

// Elements per piece (8, or 2 or 1 where width, strides or addresses allow no more), lanes per row and pieces per lane: 8-element pieces by as few
// lanes of a wavefront as hold them once up to 512 elements (2^20 rows of 64 bf16 by 8 lanes 41 us, by a wavefront 237), by one wavefront up to 1024
// (no barrier), else by four, 8192 elements in registers
struct Shape { int v, n, lanes; };
static inline Shape shape_of(int C, int v) {
    if (v == 2 && C <= 8192) return C <= 256 ? Shape{2, 2, 64} : C <= 4096 ? Shape{2, 8, C <= 1024 ? 64 : 256} : Shape{2, 16, 256};
    if (v < 8) return C <= 256 ? Shape{1, 4, 64} : Shape{1, C <= 1024 ? 4 : C <= 4096 ? 16 : C <= 8192 ? 32 : 0, 256};
    const int p = C / 8;
    if (p <= 64) return {8, 1, p <= 8 ? 8 : p <= 16 ? 16 : p <= 32 ? 32 : 64};
    if (p <= 128) return {8, 2, 64};
    return {8, p <= 256 ? 1 : p <= 512 ? 2 : p <= 1024 ? 4 : 0, 256};
}
// an upper bound where a workgroup has several rows
static inline int backward_groups(int rows, int C) { return std::max(1, std::min(rows, (C <= 1024 ? 8 : 4) * cu_count())); }

#define WKV_NORM_SHAPES(LAUNCH)                                                           \
    do {                                                                                  \
        const Shape f = shape_of(k.C, v);                                                 \
        auto is = [&](int v_, int n, int l) { return f.v == v_ && f.n == n && f.lanes == l; }; \
        if (is(1, 4, 64)) LAUNCH(1, 4, 64);                                               \
        else if (is(1, 4, 256)) LAUNCH(1, 4, 256);                                        \
        else if (is(1, 16, 256)) LAUNCH(1, 16, 256);                                      \
        else if (is(1, 32, 256)) LAUNCH(1, 32, 256);                                      \
        else if (f.v == 1) LAUNCH(1, 0, 256);                                             \
        else if (is(2, 2, 64)) LAUNCH(2, 2, 64);                                          \
        else if (is(2, 8, 64)) LAUNCH(2, 8, 64);                                          \
        else if (is(2, 8, 256)) LAUNCH(2, 8, 256);                                        \
        else if (f.v == 2) LAUNCH(2, 16, 256);                                            \
        else if (f.lanes == 8) LAUNCH(8, 1, 8);                                           \
        else if (f.lanes == 16) LAUNCH(8, 1, 16);                                         \
        else if (f.lanes == 32) LAUNCH(8, 1, 32);                                         \
        else if (is(8, 1, 64)) LAUNCH(8, 1, 64);                                          \
        else if (is(8, 2, 64)) LAUNCH(8, 2, 64);                                          \
        else if (f.n == 1) LAUNCH(8, 1, 256);                                             \
        else if (f.n == 2) LAUNCH(8, 2, 256);                                             \
        else if (f.n == 4) LAUNCH(8, 4, 256);                                             \
        else LAUNCH(8, 0, 256);                                                           \
    } while (0)

constexpr int ROWS_PER_LAUNCH = 1 << 23;          // (a grid has fewer than 2^32 threads)
template <class T, class R> static hipError_t forward_t(hipStream_t s, const Call &all, int v) {
    for (int done = 0; done < all.rows; done += std::min(all.rows - done, ROWS_PER_LAUNCH)) {
        Call k = all;
        auto on = [&](auto *p, long long step, size_t bytes) {          // the operand from row `done` on
            return p ? (decltype(p))((uintptr_t)p + (size_t)(done * step) * bytes) : p;
        };
        k.rows = std::min(all.rows - done, ROWS_PER_LAUNCH);
        k.x = on(all.x, all.xs, sizeof(T)); k.residual = on(all.residual, all.rs, sizeof(R));
        k.y = on(all.y, all.C, sizeof(T)); k.out = on(all.out, all.C, sizeof(R)); k.q = on(all.q, all.C, 1);
        k.rstd = on(all.rstd, 1, 4); k.scale = on(all.scale, 1, 4);
#define WKV_NORM(V, N, L)                                                                                                                       \
    do {                                                                                                                                        \
        const dim3 grid((unsigned)((k.rows + (long long)forward_threads<L>() / L - 1) / (forward_threads<L>() / L))), block(forward_threads<L>()); \
        if (k.q) hipLaunchKernelGGL((forward<T, R, V, N, L, true>), grid, block, 0, s, k);                                                       \
        else hipLaunchKernelGGL((forward<T, R, V, N, L, false>), grid, block, 0, s, k);                                                          \
    } while (0)
        WKV_NORM_SHAPES(WKV_NORM);
#undef WKV_NORM
    }
    return hipGetLastError();
}
template <class T, class R> static hipError_t backward_t(hipStream_t s, const Call &k, int v, void *gweight) {
    int groups = backward_groups(k.rows, k.C);
#define WKV_NORM(V, N, L)                                                                                                       \
    do {                                                                                                                        \
        constexpr int each = backward_threads<L>() / L;                                                                         \
        if (each > 1) groups = std::min(2 * cu_count(), (int)(((long long)k.rows + each - 1) / each));                          \
        hipLaunchKernelGGL((backward<T, R, V, N, L>), dim3(groups), dim3(backward_threads<L>()), 0, s, k);                      \
    } while (0)
    WKV_NORM_SHAPES(WKV_NORM);
#undef WKV_NORM
    Sums<ToRow<T>> sums;
    sums.add(groups, (size_t)k.C, k.part, {gweight, k.w32 != 0});
    sum_rows_launch(s, sums);
    return hipGetLastError();
}

}  // namespace norm
}  // namespace wkv
