// The short causal convolution over the tokens in front of the selective scan, a filter of W taps per channel:
//
//     pre[t] = bias + sum over k of w[k] xx[t - (W-1) + k],    y[t] = silu(pre[t]) or pre[t]
//
// where xx continues x to the left by the state, the W-1 inputs before it; the last W-1 of xx are the new state.  Backwards, with
// gp[t] = gy[t] silu'(pre[t]):   gx[s] = sum over k of w[k] gp[s + W-1 - k],   gw[k] = sum over t of gp[t] xx[t - (W-1) + k].
//
// Bound by memory: each input is to be read once and each output written once.  A lane holds four channels and walks
// a run of tokens with the window in registers; the W-1 inputs (backwards also the W-1 gp) on a run's edge are read again, from
// the cache.  The filter's gradient is summed along the run in registers, over the workgroup's four runs in LDS, and over
// the workgroups by sum_rows.
#include "common.h"
#include "row_sums.h"
#include "vec.h"

namespace wkv {
namespace conv {

constexpr int MIN_TAPS = 2, MAX_TAPS = 4, RUNS = 4, WIDE = 4;         // runs per workgroup: one per wavefront

struct Call {
    int B, T, D, run;                         // run: tokens per lane
    long long batch, token;                   // strides of x in elements
    int silu, w32;                            // w32: weight and bias are fp32, else in the streams' type
    const void *x, *weight, *bias, *state_in;
    const int *lengths;
    void *y, *state_out;
    const void *gy, *gstate_out;
    void *gx, *gstate_in;
    float *part;                              // (workgroups per channel, W + 1, D)
};

template <class T, int V> __device__ __forceinline__ void zero(float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = 0.f;
}

// one lane's channels of one sequence
template <class T, int W, int V> struct Lane {
    const Call &k;
    int b, d, run0, len;           // run0: the run's first token
    bool live;
    float w[W][V], bias[V];

    __device__ __forceinline__ Lane(const Call &k_, int run_index) : k(k_) {
        b = blockIdx.z;
        d = (blockIdx.x * 64 + (threadIdx.x & 63)) * V;
        live = d < k.D && (long long)run_index * k.run < k.T;
        run0 = run_index * k.run;
        len = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
        if (!live) return;
#pragma unroll
        for (int v = 0; v < V; v++) {
#pragma unroll
            for (int i = 0; i < W; i++) w[i][v] = parameter(k.weight, (d + v) * W + i);
            bias[v] = k.bias ? parameter(k.bias, d + v) : 0.f;
        }
    }
    __device__ __forceinline__ float parameter(const void *p, int i) const {
        return k.w32 ? static_cast<const float *>(p)[i] : to_float(static_cast<const T *>(p)[i]);
    }
    // xx[t]: the state's tokens are -(W-1) .. -1; nothing from the length on
    __device__ __forceinline__ void input(int t, float (&o)[V]) const {
        if (t >= len) zero<T>(o);
        else if (t >= 0) load_vec(static_cast<const T *>(k.x) + b * k.batch + t * k.token + d, o);
        else if (k.state_in) load_vec(static_cast<const T *>(k.state_in) + ((size_t)b * (W - 1) + t + W - 1) * k.D + d, o);
        else zero<T>(o);
    }
    __device__ __forceinline__ float before(const float (&win)[W][V], int v) const {
        float p = bias[v];
#pragma unroll
        for (int i = 0; i < W; i++) p = fmaf(w[i][v], win[i][v], p);
        return p;
    }
};
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }

template <int W, int V> __device__ __forceinline__ void push(float (&win)[W][V], const float (&x)[V]) {
#pragma unroll
    for (int v = 0; v < V; v++) {
#pragma unroll
        for (int i = 0; i + 1 < W; i++) win[i][v] = win[i + 1][v];
        win[W - 1][v] = x[v];
    }
}

constexpr int AHEAD = 4;                      // tokens asked for together
template <class T, int W, int V>
__global__ __launch_bounds__(64 * RUNS) void forward(const Call k) {
    const int run_index = blockIdx.y * RUNS + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);          // (the same for a wavefront: its tokens are scalars)
    Lane<T, W, V> l(k, run_index);
    if (!l.live) return;
    float win[W][V];
    zero<T>(win[0]);
#pragma unroll
    for (int i = 0; i + 1 < W; i++) l.input(l.run0 - (W - 1) + i, win[i + 1]);
    const int end = min(l.run0 + k.run, k.T);
    T *y = static_cast<T *>(k.y) + ((size_t)l.b * k.T) * k.D + l.d;
    for (int t0 = l.run0; t0 < end; t0 += AHEAD) {
        float x[AHEAD][V];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) l.input(t0 + i, x[i]);
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int t = t0 + i;
            push(win, x[i]);
            float o[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float p = l.before(win, v);
                o[v] = t >= l.len ? 0.f : k.silu ? p * sigmoid(p) : p;
            }
            if (t < end) store_vec(y + (size_t)t * k.D, o);
        }
    }
    // the run that the sequence ends in (its first one if there is nothing) leaves the new state
    const int last = l.len > 0 ? (l.len - 1) / k.run : 0;
    if (run_index != last) return;
    float row[W][V];
#pragma unroll
    for (int i = 0; i + 1 < W; i++) l.input(l.len - (W - 1) + i, row[i]);
#pragma unroll
    for (int i = 0; i + 1 < W; i++) store_vec(static_cast<T *>(k.state_out) + ((size_t)l.b * (W - 1) + i) * k.D + l.d, row[i]);
}

template <class T, int W, int V>
__global__ __launch_bounds__(64 * RUNS) void backward(const Call k) {
    __shared__ float sums[RUNS][64 * V];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, run_index = blockIdx.y * RUNS + wave;
    Lane<T, W, V> l(k, run_index);
    float gw[W][V], gb[V];
#pragma unroll
    for (int i = 0; i < W; i++) zero<T>(gw[i]);
    zero<T>(gb);
    if (l.live) {
        float win[W][V], gp[W][V];          // gp[i]: of token t - (W-1) + i
        zero<T>(win[0]);
#pragma unroll
        for (int i = 0; i < W; i++) zero<T>(gp[i]);
#pragma unroll
        for (int i = 0; i + 1 < W; i++) l.input(l.run0 - (W - 1) + i, win[i + 1]);
        const int end = min(l.run0 + k.run, k.T), begin = l.run0 == 0 ? -(W - 1) : l.run0;
        const T *gy = static_cast<const T *>(k.gy) + (size_t)l.b * k.T * k.D + l.d;
        T *gx = static_cast<T *>(k.gx) + (size_t)l.b * k.T * k.D + l.d;
        for (int t0 = l.run0; t0 < end + W - 1; t0 += AHEAD) {
            float x[AHEAD][V], g[AHEAD][V];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                l.input(t0 + i, x[i]);
                if (t0 + i < l.len) load_vec(gy + (size_t)(t0 + i) * k.D, g[i]);
                else zero<T>(g[i]);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int t = t0 + i, s = t - (W - 1);          // gx[s] is complete with gp[t]
                push(win, x[i]);
                float d[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float p = l.before(win, v), sig = sigmoid(p);
                    d[v] = k.silu ? g[i][v] * fmaf(p * sig, 1.f - sig, sig) : g[i][v];
                    if (t >= l.len) d[v] = 0.f;
                }
                push(gp, d);
                if (t < end)
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        gb[v] += d[v];
#pragma unroll
                        for (int j = 0; j < W; j++) gw[j][v] = fmaf(d[v], win[j][v], gw[j][v]);
                    }
                if (s < begin || s >= end) continue;
                float o[V];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    o[v] = 0.f;
#pragma unroll
                    for (int j = 0; j < W; j++) o[v] = fmaf(l.w[j][v], gp[W - 1 - j][v], o[v]);
                }
                const int kept = s - (l.len - (W - 1));           // the new state's row that token s went into
                if (k.gstate_out && kept >= 0 && s < l.len) {
                    float e[V];
                    load_vec(static_cast<const T *>(k.gstate_out) + ((size_t)l.b * (W - 1) + kept) * k.D + l.d, e);
#pragma unroll
                    for (int v = 0; v < V; v++) o[v] += e[v];
                }
                if (s >= 0) store_vec(gx + (size_t)s * k.D, o);
                else if (k.gstate_in) store_vec(static_cast<T *>(k.gstate_in) + ((size_t)l.b * (W - 1) + s + W - 1) * k.D + l.d, o);
            }
        }
    }
    // over the workgroup's runs
    float *to = k.part + ((size_t)blockIdx.z * gridDim.y + blockIdx.y) * (W + 1) * k.D;
    for (int i = 0; i <= W; i++) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            float s = gb[v];
#pragma unroll
            for (int j = 0; j < W; j++) s = i == j ? gw[j][v] : s;
            sums[wave][lane * V + v] = s;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 64 * V; c += 64 * RUNS) {
            const int d = blockIdx.x * 64 * V + c;
            if (d < k.D) to[(size_t)i * k.D + d] = (sums[0][c] + sums[1][c]) + (sums[2][c] + sums[3][c]);
        }
        __syncthreads();
    }
}

// gradients (W + 1, D) to the weight's (D, W) and the bias
template <class P> struct ToFilter {
    P *weight, *bias;
    int W, D;
    __device__ __forceinline__ void operator()(size_t i, float v) const {
        const int tap = (int)(i / D), d = (int)(i % D);
        if (tap < W) weight[(size_t)d * W + tap] = from_float<P>(v);
        else if (bias) bias[d] = from_float<P>(v);
    }
};

// Tokens per lane: enough lanes to fill the compute units, and as long a run as that leaves, since a run reads W-1 tokens twice
static inline int run_for(int B, int T, int D, int V) {
    int run = 64;
    while (run > 8 && (long long)B * ((T + run - 1) / run) * ((D + 64 * V - 1) / (64 * V)) < 8ll * cu_count()) run /= 2;
    return run;
}
static inline int run_groups(int T, int run) { return (T + RUNS * run - 1) / (RUNS * run); }
static inline int vector_of(int D) { return D % WIDE == 0 ? WIDE : 1; }
// (the largest of what the two widths of a lane need: which one a call takes depends on its pointers)
static inline size_t backward_scratch(int B, int T, int D, int W) {
    size_t n = 0;
    for (int V : {1, vector_of(D)}) n = std::max(n, (size_t)B * run_groups(T, run_for(B, T, D, V)));
    return n * (W + 1) * D * 4;
}

template <class T, int V, bool BACK> static hipError_t launch(hipStream_t s, int W, Call k) {
    k.run = run_for(k.B, k.T, k.D, V);
    const dim3 grid((k.D + 64 * V - 1) / (64 * V), run_groups(k.T, k.run), k.B);
#define WKV_CONV(N)                                                                                      \
    case N:                                                                                              \
        if constexpr (BACK) hipLaunchKernelGGL((backward<T, N, V>), grid, dim3(64 * RUNS), 0, s, k);     \
        else hipLaunchKernelGGL((forward<T, N, V>), grid, dim3(64 * RUNS), 0, s, k);                     \
        break;
    switch (W) { WKV_CONV(2) WKV_CONV(3) WKV_CONV(4) }
#undef WKV_CONV
    return hipGetLastError();
}
template <class T> static hipError_t forward_t(hipStream_t s, int W, const Call &k, bool wide) {
    return wide ? launch<T, WIDE, false>(s, W, k) : launch<T, 1, false>(s, W, k);
}
template <class T> static hipError_t backward_t(hipStream_t s, int W, const Call &k, bool wide, void *gweight, void *gbias) {
    const hipError_t e = wide ? launch<T, WIDE, true>(s, W, k) : launch<T, 1, true>(s, W, k);
    if (e != hipSuccess) return e;
    const int rows = k.B * run_groups(k.T, run_for(k.B, k.T, k.D, wide ? WIDE : 1));
    const size_t n = (size_t)(W + 1) * k.D;
    if (k.w32) sum_rows_launch(s, rows, n, k.part, ToFilter<float>{static_cast<float *>(gweight), static_cast<float *>(gbias), W, k.D});
    else sum_rows_launch(s, rows, n, k.part, ToFilter<T>{static_cast<T *>(gweight), static_cast<T *>(gbias), W, k.D});
    return hipGetLastError();
}

}  // namespace conv
}  // namespace wkv
