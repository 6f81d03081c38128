// The short causal convolution over the tokens in front of the selective scan, a filter of W taps per channel:
//
//     pre[t] = bias + sum over k of w[k] xx[t - (W-1) + k],    y[t] = silu(pre[t]) or pre[t]
//
// where xx continues x to the left by the state, the W-1 inputs before it; the last W-1 of xx are the new state.  Backwards, with
// gp[t] = gy[t] silu'(pre[t]):   gx[s] = sum over k of w[k] gp[s + W-1 - k],   gw[k] = sum over t of gp[t] xx[t - (W-1) + k].
//
// Bound by memory (B8 T4096 D4096 bf16: forward 103 us = 5.2 TB/s, backward 187 us = 4.3 TB/s; single tokens of 64 sequences, the same kernel, 4.4 us): each input is to be read once and each output written once.  A lane holds four channels
// (two or one where four are not aligned) and walks a run of tokens with the window in registers; the W-1 inputs (backwards also the W-1 gp) on a run's edge are read again, from
// the cache.  The filter's gradient is summed along the run in registers, over the workgroup's four runs in LDS, and over
// the workgroups by sum_rows.
#include "common.h"
#include "row_access.h"
#include "row_sums.h"
#include "vec.h"

namespace wkv {
namespace conv {

constexpr int MIN_TAPS = 2, MAX_TAPS = 4, RUNS = 4;         // runs per workgroup: one per wavefront

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

template <int V> __device__ __forceinline__ void zero(float (&o)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) o[i] = 0.f;
}

// one lane's channels of one sequence
template <class T, int W, int V> struct Lane {
    typedef Row<T, V> R;
    typedef typename R::Raw Raw;
    const Call &k;
    int b, d, at, run0, len;           // at: d in bytes; run0: the run's first token
    bool live;
    float w[W][V], bias[V];

    __device__ __forceinline__ Lane(const Call &k_, int run_index) : k(k_) {
        b = blockIdx.z;
        d = (blockIdx.x * 64 + (threadIdx.x & 63)) * V;
        at = d * (int)sizeof(T);
        live = d < k.D && (long long)run_index * k.run < k.T;
        run0 = run_index * k.run;
        len = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
        if (!live) return;
        if (k.w32) parameters(static_cast<const float *>(k.weight), static_cast<const float *>(k.bias));
        else parameters(static_cast<const T *>(k.weight), static_cast<const T *>(k.bias));
    }
    // (V taps' worth of a channel at a time: whole 8 or 16 bytes)
    template <class P> __device__ __forceinline__ void parameters(const P *pw, const P *pb) {
        float flat[W][V];
#pragma unroll
        for (int i = 0; i < W; i++) load_vec(pw + (size_t)d * W + i * V, flat[i]);
#pragma unroll
        for (int v = 0; v < V; v++)
#pragma unroll
            for (int i = 0; i < W; i++) w[i][v] = flat[(v * W + i) / V][(v * W + i) % V];
        if (pb) load_vec(pb + d, bias);
        else zero(bias);
    }
    // xx[t]: the state's tokens are -(W-1) .. -1; nothing from the length on
    __device__ __forceinline__ Raw input(int t) const {
        const T *x = static_cast<const T *>(k.x) + b * k.batch + t * k.token;
        const T *state = static_cast<const T *>(k.state_in) + ((long long)b * (W - 1) + t + W - 1) * k.D;
        return R::load(t >= 0 ? x : state, t < len && (t >= 0 || k.state_in), at);
    }
    __device__ __forceinline__ void input(int t, float (&o)[V]) const { R::floats(input(t), o); }
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

constexpr int AHEAD = 4;                      // tokens asked for together, a group before they are used
template <class T, int W, int V>
__global__ __launch_bounds__(64 * RUNS) void forward(const Call k) {
    typedef Row<T, V> R;
    const int run_index = blockIdx.y * RUNS + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);          // (the same for a wavefront: its tokens are scalars)
    Lane<T, W, V> l(k, run_index);
    if (!l.live) return;
    float win[W][V];
    typename R::Raw next[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) next[i] = l.input(l.run0 + i);
    zero(win[0]);
#pragma unroll
    for (int i = 0; i + 1 < W; i++) l.input(l.run0 - (W - 1) + i, win[i + 1]);
    // the run that the sequence ends in (its first one if there is nothing) leaves the new state
    const bool ends = run_index == (l.len > 0 ? (l.len - 1) / k.run : 0);
    typename R::Raw state[W - 1];
#pragma unroll
    for (int i = 0; i + 1 < W; i++) state[i] = l.input(ends ? l.len - (W - 1) + i : l.len);
    const int end = min(l.run0 + k.run, k.T);
    T *y = static_cast<T *>(k.y) + (size_t)l.b * k.T * k.D;
    for (int t0 = l.run0; t0 < end; t0 += AHEAD) {
        typename R::Raw now[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            now[i] = next[i];
            next[i] = l.input(t0 + AHEAD + i);
        }
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int t = t0 + i;
            float x[V], o[V];
            R::floats(now[i], x);
            push(win, x);
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float p = l.before(win, v);
                o[v] = t >= l.len ? 0.f : k.silu ? p * sigmoid(p) : p;
            }
            R::store(y + (size_t)t * k.D, t < end, l.at, o);
        }
    }
#pragma unroll
    for (int i = 0; i + 1 < W; i++) {
        float row[V];
        R::floats(state[i], row);
        R::store(static_cast<T *>(k.state_out) + ((size_t)l.b * (W - 1) + i) * k.D, ends, l.at, row);
    }
}

template <class T, int W, int V>
__global__ __launch_bounds__(64 * RUNS) void backward(const Call k) {
    typedef Row<T, V> R;
    __shared__ float sums[RUNS][64 * V];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, run_index = blockIdx.y * RUNS + wave;
    Lane<T, W, V> l(k, run_index);
    float gw[W][V], gb[V];
#pragma unroll
    for (int i = 0; i < W; i++) zero(gw[i]);
    zero(gb);
    if (l.live) {
        float win[W][V], gp[W][V];          // gp[i]: of token t - (W-1) + i
        const T *gy = static_cast<const T *>(k.gy) + (size_t)l.b * k.T * k.D;
        T *gx = static_cast<T *>(k.gx) + (size_t)l.b * k.T * k.D;
        typename R::Raw next_x[AHEAD], next_g[AHEAD];
        auto ask = [&](int t0) {
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                next_x[i] = l.input(t0 + i);
                next_g[i] = R::load(gy + (long long)(t0 + i) * k.D, t0 + i < l.len, l.at);
            }
        };
        ask(l.run0);
        zero(win[0]);
#pragma unroll
        for (int i = 0; i < W; i++) zero(gp[i]);
#pragma unroll
        for (int i = 0; i + 1 < W; i++) l.input(l.run0 - (W - 1) + i, win[i + 1]);
        const int end = min(l.run0 + k.run, k.T), begin = l.run0 == 0 ? -(W - 1) : l.run0;
        for (int t0 = l.run0; t0 < end + W - 1; t0 += AHEAD) {
            typename R::Raw now_x[AHEAD], now_g[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                now_x[i] = next_x[i];
                now_g[i] = next_g[i];
            }
            ask(t0 + AHEAD);
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int t = t0 + i, s = t - (W - 1);          // gx[s] is complete with gp[t]
                float x[V], d[V], o[V];
                R::floats(now_x[i], x);
                R::floats(now_g[i], d);                         // (zero from the length on)
                push(win, x);
                if (k.silu)
#pragma unroll
                    for (int v = 0; v < V; v++) {
                        const float p = l.before(win, v), sig = sigmoid(p);
                        d[v] = t < l.len ? d[v] * fmaf(p * sig, 1.f - sig, sig) : 0.f;
                    }
                push(gp, d);
#pragma unroll
                for (int v = 0; v < V; v++) {
                    const float e = t < end ? d[v] : 0.f;          // (the next run's tokens are counted there)
                    gb[v] += e;
#pragma unroll
                    for (int j = 0; j < W; j++) gw[j][v] = fmaf(e, win[j][v], gw[j][v]);
                }
#pragma unroll
                for (int v = 0; v < V; v++) {
                    o[v] = 0.f;
#pragma unroll
                    for (int j = 0; j < W; j++) o[v] = fmaf(l.w[j][v], gp[W - 1 - j][v], o[v]);
                }
                const int kept = s - (l.len - (W - 1));           // the new state's row that token s went into
                if (k.gstate_out && kept >= 0 && s < l.len && s >= begin && s < end) {
                    float e[V];
                    R::floats(R::load(static_cast<const T *>(k.gstate_out) + ((long long)l.b * (W - 1) + kept) * k.D, true, l.at), e);
#pragma unroll
                    for (int v = 0; v < V; v++) o[v] += e[v];
                }
                if (s < 0 && k.gstate_in && s >= begin) R::store(static_cast<T *>(k.gstate_in) + ((long long)l.b * (W - 1) + s + W - 1) * k.D, true, l.at, o);
                R::store(gx + (long long)s * k.D, s >= 0 && s >= begin && s < end, l.at, o);
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
template <class T> struct ToFilter {
    ToRow<T> weight, bias;
    int W, D;
    __device__ __forceinline__ void operator()(size_t i, float v) const {
        const int tap = (int)(i / D), d = (int)(i % D);
        if (tap < W) weight((size_t)d * W + tap, v);
        else if (bias.out) bias(d, v);
    }
};

// Tokens per lane: enough lanes to fill the compute units, and as long a run as that leaves, since a run reads W-1 tokens twice
static inline int run_for(int B, int T, int D, int V) {
    int run = 64;
    while (run > 8 && (long long)B * ((T + run - 1) / run) * ((D + 64 * V - 1) / (64 * V)) < 8ll * cu_count()) run /= 2;
    return run;
}
static inline int run_groups(int T, int run) { return (T + RUNS * run - 1) / (RUNS * run); }
// (the largest of what a lane's possible channels need: how many a call takes depends on its pointers)
static inline size_t backward_scratch(int B, int T, int D, int W) {
    size_t n = 0;
    for (int V : {1, 2, 4}) n = std::max(n, (size_t)B * run_groups(T, run_for(B, T, D, V)));
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
// v: channels per lane, 4, or 2 or 1 where widths, strides or addresses allow no more (B8 T4096 bf16, forward and backward: D 4096 103 and 187 us by four,
// D 4094 158 and 282 by two, D 4095 186 and 345 by one)
template <class T> static hipError_t forward_t(hipStream_t s, int W, const Call &k, int v) {
    return v == 4 ? launch<T, 4, false>(s, W, k) : v == 2 ? launch<T, 2, false>(s, W, k) : launch<T, 1, false>(s, W, k);
}
template <class T> static hipError_t backward_t(hipStream_t s, int W, const Call &k, int v, void *gweight, void *gbias) {
    const hipError_t e = v == 4 ? launch<T, 4, true>(s, W, k) : v == 2 ? launch<T, 2, true>(s, W, k) : launch<T, 1, true>(s, W, k);
    if (e != hipSuccess) return e;
    Sums<ToFilter<T>> sums;
    sums.add(k.B * run_groups(k.T, run_for(k.B, k.T, k.D, v)), (size_t)(W + 1) * k.D, k.part,
             {{gweight, k.w32 != 0}, {gbias, k.w32 != 0}, W, k.D});
    sum_rows_launch(s, sums);
    return hipGetLastError();
}

}  // namespace conv
}  // namespace wkv
