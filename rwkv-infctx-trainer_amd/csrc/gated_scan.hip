// The gated linear recurrence over the tokens, one state per channel:
//
//     a[t] = exp(-scale softplus(decay) sigmoid(r[t])),   h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) sigmoid(i[t]) x[t],   y[t] = h[t] silu(z[t]) or h[t]
//
// Backwards, with go = gy silu(z), b = sqrt(1 - a^2) and log a's slope l:
//
//     g[t] = go[t] + a[t+1] g[t+1],   gx = g b sigmoid(i),   gi = g b x sigmoid'(i),   l = g (a h[t-1] - a^2 / b sigmoid(i) x),
//     gr = l log a (1 - sigmoid(r)),   gdecay = -scale sigmoid(decay) sum of l sigmoid(r),   gz = gy h silu'(z)
//
// Bound by memory: every stream is read once and every result written once.  The recurrence is linear, so a run of tokens is the pair (product of a, its
// end from nothing), and pairs join.  A workgroup walks a sequence for 64 V channels, a step at a time: each of its wavefronts takes K tokens of the step for
// all of the channels, makes its run's pair and leaves it in LDS; behind one barrier every wavefront joins the pairs before its own and finishes
// its tokens from the state that gives, still in registers.  Where that makes too few workgroups the sequences are cut in time, and a pass over the decays
// and inputs alone leaves every segment's pair first.  Backwards a step runs both ways at once: the states again, from one kept
// before every CHECK tokens, and their gradients.
//
// 1 - a^2 loses its digits where a is near one, the very channels that remember long: below 2 log a = -1/4 it is formed from the series of exp(2 log a) - 1.
#include "common.h"
#include "row_access.h"
#include "row_sums.h"

namespace wkv {
namespace gated {

struct Rows { const void *p; long long batch, token; };
struct Call {
    int B, T, D;
    float scale;
    Rows x, r, i, z;                          // z.p NULL: no gate
    const float *decay, *state_in;
    const int *lengths;
    void *y;
    float *state_out, *checkpoints;           // (B, tokens / CHECK, D): the state before every CHECK tokens
    const void *gy;
    const float *gstate_out;
    void *gx, *gr, *gi, *gz;
    float *gstate_in, *part;                  // part (B segments, D)
    // segments of `span` tokens, and their pairs (B, segments, 2, D)
    int segments, span;
    float *pairs;
};

constexpr int WAVES = 16, CHECK = 64, STEP = 128;         // STEP: tokens of a forward step, and what a segment is a multiple of
constexpr int OUTSIDE = (int)0x80000000u;                 // a lane's offset that is in no row's range

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }

// 1 - a^2 of a = 2^l
__device__ __forceinline__ float one_less_square(float l, float a) {
    const float s = -2.f * LN2 * l;
    float p = fmaf(s, -1.f / 6, 1.f);
    p = fmaf(p * s, -1.f / 5, 1.f);
    p = fmaf(p * s, -1.f / 4, 1.f);
    p = fmaf(p * s, -1.f / 3, 1.f);
    p = fmaf(p * s, -1.f / 2, 1.f);
    return s < 0.25f ? s * p : fmaf(-a, a, 1.f);
}
// log2 of a at an open gate; finite, so that a shut gate keeps the state whatever the decay is
__device__ __forceinline__ float rate_of(float decay, float scale) {
    const float soft = decay > 20.f ? decay : log1pf(expf(decay));
    const float rate = -scale * soft * LOG2E;
    return rate < -3e38f ? -3e38f : rate;
}

// one lane's channels of one sequence
template <class T, int V> struct Lane {
    typedef Row<T, V> R;
    typedef typename R::Raw Raw;
    const Call &k;
    int b, d, at, at32, len;           // at, at32: d in bytes of a stream's row and of an fp32 one
    float rate[V];
    __device__ __forceinline__ Lane(const Call &k_) : k(k_) {
        b = blockIdx.y;
        d = (blockIdx.x * 64 + (threadIdx.x & 63)) * V;
        at = d < k.D ? d * (int)sizeof(T) : OUTSIDE;
        at32 = d < k.D ? d * 4 : OUTSIDE;
        len = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
#pragma unroll
        for (int v = 0; v < V; v++) rate[v] = d < k.D ? rate_of(k.decay[d + v], k.scale) : 0.f;
    }
    __device__ __forceinline__ Raw load(const Rows &s, int t) const { return R::load(static_cast<const T *>(s.p) + b * s.batch + t * s.token, t < len, at); }
    __device__ __forceinline__ Raw load(const void *p, int t) const { return R::load(static_cast<const T *>(p) + ((size_t)b * k.T + t) * k.D, t < len, at); }
    __device__ __forceinline__ void store(void *p, int t, const float (&v)[V]) const {
        R::store(static_cast<T *>(p) + ((size_t)b * k.T + t) * k.D, t < k.T, at, v);
    }
    // V floats of a row of D, zeros where there is none
    __device__ __forceinline__ void floats(const float *row, float (&o)[V]) const { Row<float, V>::floats(Row<float, V>::load(row, row != nullptr, at32), o); }
    __device__ __forceinline__ void put(float *row, const float (&o)[V]) const { Row<float, V>::store(row, true, at32, o); }
    __device__ __forceinline__ const float *state_row(const float *p) const { return p ? p + (size_t)b * k.D : nullptr; }
    __device__ __forceinline__ float *pair(int segment) const { return k.pairs + ((size_t)b * k.segments + segment) * 2 * k.D; }
};

// FORWARD the outputs; PAIRS only the segments' pairs
enum { FORWARD, PAIRS };
template <class T, int V, bool GATE, int MODE>
__global__ __launch_bounds__(64 * WAVES) void forward(const Call k) {
    constexpr int K = STEP / WAVES;
    typedef Row<T, V> R;
    typedef typename R::Raw Raw;
    struct Pair { float a[V], h[V]; };
    __shared__ Pair pairs[2][WAVES][64];
    const Lane<T, V> l(k);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), segment = blockIdx.z;
    const int begin = segment * k.span, end = min(begin + k.span, k.T);
    Raw x[K], r[K], i[K], z[K];
    auto ask = [&](int t0) {
#pragma unroll
        for (int j = 0; j < K; j++) {
            const int t = t0 + wave * K + j;
            x[j] = l.load(k.x, t);
            r[j] = l.load(k.r, t);
            i[j] = l.load(k.i, t);
            if (GATE && MODE == FORWARD) z[j] = l.load(k.z, t);
        }
    };
    ask(begin);
    float h[V], all[V];                       // the state before the step; PAIRS: from nothing, with the product of all a
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = 0.f, all[v] = 1.f;
    if (MODE == FORWARD) {
        l.floats(l.state_row(k.state_in), h);
        for (int s = 0; s < segment; s++) {
            float a[V], e[V];
            l.floats(l.pair(s), a);
            l.floats(l.pair(s) + k.D, e);
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = fmaf(a[v], h[v], e[v]);
        }
    }
    int which = 0;
    for (int t0 = begin; t0 < end; t0 += STEP, which ^= 1) {
        float a[K][V], u[K][V];
        Pair mine;
#pragma unroll
        for (int v = 0; v < V; v++) mine.a[v] = 1.f, mine.h[v] = 0.f;
#pragma unroll
        for (int j = 0; j < K; j++) {
            const bool there = t0 + wave * K + j < l.len;
            float xf[V], rf[V], jf[V];
            R::floats(x[j], xf);
            R::floats(r[j], rf);
            R::floats(i[j], jf);
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float lg = l.rate[v] * sigmoid(rf[v]), e = exp2_fast(lg);
                a[j][v] = there ? e : 1.f;
                u[j][v] = there ? __builtin_amdgcn_sqrtf(one_less_square(lg, e)) * sigmoid(jf[v]) * xf[v] : 0.f;
                mine.a[v] *= a[j][v];
                mine.h[v] = fmaf(a[j][v], mine.h[v], u[j][v]);
            }
        }
        float gate[K][V];
        if (GATE && MODE == FORWARD)
#pragma unroll
            for (int j = 0; j < K; j++) R::floats(z[j], gate[j]);
        ask(t0 + STEP);
        pairs[which][wave][lane] = mine;
        lds_barrier();
        float before[V];
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const Pair p = pairs[which][w][lane];
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (w == wave) before[v] = h[v];
                h[v] = fmaf(p.a[v], h[v], p.h[v]);
                if (MODE == PAIRS) all[v] *= p.a[v];
            }
        }
        if (MODE == PAIRS) continue;
        if (k.checkpoints && wave * K % CHECK == 0 && t0 + wave * K < k.T)
            l.put(k.checkpoints + ((size_t)l.b * ((k.T + CHECK - 1) / CHECK) + (t0 + wave * K) / CHECK) * k.D, before);
#pragma unroll
        for (int j = 0; j < K; j++) {
            const int t = t0 + wave * K + j;
            float o[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                before[v] = fmaf(a[j][v], before[v], u[j][v]);
                o[v] = GATE ? before[v] * gate[j][v] * sigmoid(gate[j][v]) : before[v];
                o[v] = t < l.len ? o[v] : 0.f;
            }
            l.store(k.y, t, o);
        }
    }
    if (wave != 0) return;
    if (MODE == PAIRS) {
        l.put(l.pair(segment), all);
        l.put(l.pair(segment) + k.D, h);
    } else if (segment == k.segments - 1) {
        l.put(k.state_out + (size_t)l.b * k.D, h);
    }
}

template <class T, int V, bool GATE, int MODE>
__global__ __launch_bounds__(64 * WAVES) void backward(const Call k) {
    constexpr int K = CHECK / WAVES;
    typedef Row<T, V> R;
    typedef typename R::Raw Raw;
    struct Pair { float a[V], h[V], g[V]; };          // a run's product of a, its state from nothing, what it hands to the token before it from nothing
    __shared__ Pair pairs[2][WAVES][64];
    const Lane<T, V> l(k);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), segment = blockIdx.z;
    const int begin = segment * k.span, end = min(begin + k.span, k.T), checks = (k.T + CHECK - 1) / CHECK;
    Raw x[K], r[K], i[K], z[K], gy[K];
    float start[V];
    auto ask = [&](int t0) {
        t0 = max(t0, begin);
#pragma unroll
        for (int j = 0; j < K; j++) {
            const int t = t0 + wave * K + j;
            r[j] = l.load(k.r, t);
            gy[j] = l.load(k.gy, t);
            if (GATE) z[j] = l.load(k.z, t);
            if (MODE == PAIRS) continue;
            x[j] = l.load(k.x, t);
            i[j] = l.load(k.i, t);
        }
        if (MODE != PAIRS) l.floats(k.checkpoints + ((size_t)l.b * checks + t0 / CHECK) * k.D, start);
    };
    const int last = begin + (end - begin - 1) / CHECK * CHECK;
    ask(last);
    float c[V], all[V], sum[V];               // c: what the tokens behind the step hand to its last one
#pragma unroll
    for (int v = 0; v < V; v++) c[v] = sum[v] = 0.f, all[v] = 1.f;
    if (MODE == FORWARD) {
        l.floats(l.state_row(k.gstate_out), c);
        for (int s = k.segments - 1; s > segment; s--) {
            float a[V], e[V];
            l.floats(l.pair(s), a);
            l.floats(l.pair(s) + k.D, e);
#pragma unroll
            for (int v = 0; v < V; v++) c[v] = fmaf(a[v], c[v], e[v]);
        }
    }
    int which = 0;
    for (int t0 = last; t0 >= begin; t0 -= CHECK, which ^= 1) {
        float a[K][V], lg[K][V], rs[K][V], is[K][V], ix[K][V], b[K][V], go[K][V], gv[K][V], zf[K][V], zs[K][V], h[V];
        Pair mine;
#pragma unroll
        for (int v = 0; v < V; v++) mine.a[v] = 1.f, mine.h[v] = mine.g[v] = 0.f, h[v] = start[v];
#pragma unroll
        for (int j = 0; j < K; j++) {
            const bool there = t0 + wave * K + j < l.len;
            float xf[V], rf[V], jf[V];
            R::floats(r[j], rf);
            R::floats(gy[j], gv[j]);
            if (GATE) R::floats(z[j], zf[j]);
            if (MODE == FORWARD) {
                R::floats(x[j], xf);
                R::floats(i[j], jf);
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                rs[j][v] = sigmoid(rf[v]);
                lg[j][v] = there ? l.rate[v] * rs[j][v] : 0.f;
                a[j][v] = exp2_fast(lg[j][v]);
                if (GATE) zs[j][v] = sigmoid(zf[j][v]);
                go[j][v] = !there ? 0.f : GATE ? gv[j][v] * zf[j][v] * zs[j][v] : gv[j][v];
                mine.a[v] *= a[j][v];
                if (MODE == PAIRS) continue;
                b[j][v] = one_less_square(lg[j][v], a[j][v]);
                is[j][v] = sigmoid(jf[v]);
                ix[j][v] = is[j][v] * xf[v];
                mine.h[v] = fmaf(a[j][v], mine.h[v], there ? __builtin_amdgcn_sqrtf(b[j][v]) * ix[j][v] : 0.f);
            }
        }
#pragma unroll
        for (int j = K - 1; j >= 0; j--)
#pragma unroll
            for (int v = 0; v < V; v++) mine.g[v] = a[j][v] * (go[j][v] + mine.g[v]);
        ask(t0 - CHECK);
        pairs[which][wave][lane] = mine;
        lds_barrier();
        float g[V];
#pragma unroll
        for (int w = WAVES - 1; w >= 0; w--) {
            const Pair p = pairs[which][w][lane];
#pragma unroll
            for (int v = 0; v < V; v++) {
                if (w == wave) g[v] = c[v];
                c[v] = fmaf(p.a[v], c[v], p.g[v]);
                if (MODE == PAIRS) all[v] *= p.a[v];
            }
        }
        if (MODE == PAIRS) continue;
        for (int w = 0; w < wave; w++) {
            const Pair p = pairs[which][w][lane];
#pragma unroll
            for (int v = 0; v < V; v++) h[v] = fmaf(p.a[v], h[v], p.h[v]);
        }
        float hs[K][V];                       // the states before the tokens
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
            for (int v = 0; v < V; v++) {
                hs[j][v] = h[v];
                h[v] = fmaf(a[j][v], h[v], t0 + wave * K + j < l.len ? __builtin_amdgcn_sqrtf(b[j][v]) * ix[j][v] : 0.f);
            }
        float step[V];
#pragma unroll
        for (int v = 0; v < V; v++) step[v] = 0.f;
#pragma unroll
        for (int j = K - 1; j >= 0; j--) {
            const int t = t0 + wave * K + j;
            const bool there = t < l.len;
            float ox[V], orr[V], oi[V], oz[V];
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float gt = go[j][v] + g[v], ah = a[j][v] * hs[j][v], beta = __builtin_amdgcn_sqrtf(b[j][v]);
                // (where a is one, as at a shut gate, beta and what it changes by are nothing)
                const float turn = b[j][v] > 1e-37f ? a[j][v] * a[j][v] * __builtin_amdgcn_rsqf(b[j][v]) * ix[j][v] : 0.f;
                const float gl = gt * (ah - turn);
                ox[v] = there ? gt * beta * is[j][v] : 0.f;
                oi[v] = there ? gt * beta * ix[j][v] * (1.f - is[j][v]) : 0.f;
                orr[v] = there ? gl * (lg[j][v] * LN2) * (1.f - rs[j][v]) : 0.f;
                step[v] += there ? gl * rs[j][v] : 0.f;
                if (GATE) oz[v] = there ? gv[j][v] * fmaf(beta, ix[j][v], ah) * fmaf(zf[j][v] * zs[j][v], 1.f - zs[j][v], zs[j][v]) : 0.f;
                g[v] = a[j][v] * gt;
            }
            l.store(k.gx, t, ox);
            l.store(k.gr, t, orr);
            l.store(k.gi, t, oi);
            if (GATE) l.store(k.gz, t, oz);
        }
#pragma unroll
        for (int v = 0; v < V; v++) sum[v] += step[v];
    }
    if (MODE == PAIRS) {
        if (wave == 0) {
            l.put(l.pair(segment), all);
            l.put(l.pair(segment) + k.D, c);
        }
        return;
    }
    if (wave == 0 && segment == 0 && k.gstate_in) l.put(k.gstate_in + (size_t)l.b * k.D, c);
    // the decay's share: over the wavefronts
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; v++) pairs[0][wave][lane].a[v] = sum[v];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; w++)
#pragma unroll
        for (int v = 0; v < V; v++) sum[v] += pairs[0][w][lane].a[v];
    l.put(k.part + ((size_t)l.b * k.segments + segment) * k.D, sum);
}

// one token: an element per lane
template <class T> __global__ __launch_bounds__(256) void one(const Call k) {
    const size_t n = (size_t)blockIdx.x * 256 + threadIdx.x;
    const int b = (int)(n / k.D), d = (int)(n % k.D);
    if (b >= k.B) return;
    const bool there = !k.lengths || k.lengths[b] > 0;
    const float before = k.state_in ? k.state_in[n] : 0.f;
    float h = before, o = 0.f;
    if (there) {
        auto at = [&](const Rows &s) { return to_float(static_cast<const T *>(s.p)[b * s.batch + d]); };
        const float x = at(k.x), r = at(k.r), i = at(k.i), z = k.z.p ? at(k.z) : 0.f, lg = rate_of(k.decay[d], k.scale) * sigmoid(r), a = exp2_fast(lg);
        h = fmaf(a, before, __builtin_amdgcn_sqrtf(one_less_square(lg, a)) * sigmoid(i) * x);
        o = k.z.p ? h * z * sigmoid(z) : h;
    }
    static_cast<T *>(k.y)[n] = from_float<T>(o);
    k.state_out[n] = h;
}

// the sums over batch and time of l sigmoid(r) to the decay's gradient
struct ToDecay {
    float *out;
    const float *decay;
    float scale;
    __device__ __forceinline__ void operator()(size_t i, float v) const { out[i] = -scale * v * (1.f / (1.f + expf(-decay[i]))); }
};

// ---- launches
// Segments in time where whole sequences make too few workgroups
static inline int span_of(int B, int T, int D, int V) {
    const long long groups = (long long)B * ((D + 64 * V - 1) / (64 * V)), steps = (T + STEP - 1) / STEP;
    long long cut = std::min<long long>(cu_count() / groups, steps / 2);
    cut = std::max<long long>(1, std::min<long long>(cut, 64));
    return (int)((steps + cut - 1) / cut * STEP);
}
static inline int segments_of(int T, int span) { return (T + span - 1) / span; }
static inline size_t checkpoint_bytes(int B, int T, int D) { return (size_t)B * ((T + CHECK - 1) / CHECK) * D * 4; }
// (the larger of what a lane's possible channels need: how many a call takes depends on its pointers)
static inline size_t most_segments(int B, int T, int D) {
    size_t n = 1;
    for (int V : {1, 2}) n = std::max<size_t>(n, segments_of(T, span_of(B, T, D, V)));
    return n;
}
static inline size_t forward_scratch(int B, int T, int D) {
    const size_t n = most_segments(B, T, D);
    return n > 1 ? (size_t)B * n * 2 * D * 4 : 0;
}
static inline size_t backward_scratch(int B, int T, int D) { return (size_t)B * most_segments(B, T, D) * 3 * D * 4; }

template <class T, int V, bool GATE> static void forward_v(hipStream_t s, Call k) {
    k.span = span_of(k.B, k.T, k.D, V);
    k.segments = segments_of(k.T, k.span);
    const dim3 grid((k.D + 64 * V - 1) / (64 * V), k.B, k.segments);
    if (k.segments > 1) hipLaunchKernelGGL((forward<T, V, GATE, PAIRS>), grid, dim3(64 * WAVES), 0, s, k);
    hipLaunchKernelGGL((forward<T, V, GATE, FORWARD>), grid, dim3(64 * WAVES), 0, s, k);
}
template <class T, int V, bool GATE> static void backward_v(hipStream_t s, Call k, float *gdecay) {
    k.span = span_of(k.B, k.T, k.D, V);
    k.segments = segments_of(k.T, k.span);
    k.part = k.pairs + (k.segments > 1 ? (size_t)k.B * k.segments * 2 * k.D : 0);
    const dim3 grid((k.D + 64 * V - 1) / (64 * V), k.B, k.segments);
    if (k.segments > 1) hipLaunchKernelGGL((backward<T, V, GATE, PAIRS>), grid, dim3(64 * WAVES), 0, s, k);
    hipLaunchKernelGGL((backward<T, V, GATE, FORWARD>), grid, dim3(64 * WAVES), 0, s, k);
    Sums<ToDecay> sums;
    sums.add(k.B * k.segments, k.D, k.part, ToDecay{gdecay, k.decay, k.scale});
    sum_rows_launch(s, sums);
}
template <class T> static hipError_t forward_t(hipStream_t s, const Call &k, int v) {
    if (k.T == 1 && !k.checkpoints) hipLaunchKernelGGL(one<T>, dim3((unsigned)(((size_t)k.B * k.D + 255) / 256)), dim3(256), 0, s, k);
    else if (v == 2) k.z.p ? forward_v<T, 2, true>(s, k) : forward_v<T, 2, false>(s, k);
    else k.z.p ? forward_v<T, 1, true>(s, k) : forward_v<T, 1, false>(s, k);
    return hipGetLastError();
}
template <class T> static hipError_t backward_t(hipStream_t s, const Call &k, int v, float *gdecay) {
    if (v == 2) k.z.p ? backward_v<T, 2, true>(s, k, gdecay) : backward_v<T, 2, false>(s, k, gdecay);
    else k.z.p ? backward_v<T, 1, true>(s, k, gdecay) : backward_v<T, 1, false>(s, k, gdecay);
    return hipGetLastError();
}

}  // namespace gated
}  // namespace wkv
