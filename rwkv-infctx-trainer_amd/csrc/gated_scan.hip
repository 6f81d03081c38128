// The gated linear recurrence over the tokens, one state per channel:
//
//     a[t] = exp(-scale softplus(decay) sigmoid(r[t])),   h[t] = a[t] h[t-1] + sqrt(1 - a[t]^2) sigmoid(i[t]) x[t],   y[t] = h[t] silu(z[t]) or h[t]
//
// Backwards, with go = gy silu(z), b = sqrt(1 - a^2) and log a's slope l:
//
//     g[t] = go[t] + a[t+1] g[t+1],   gx = g b sigmoid(i),   gi = g b x sigmoid'(i),   l = g (a h[t-1] - a^2 / b sigmoid(i) x),
//     gr = l log a (1 - sigmoid(r)),   gdecay = -scale sigmoid(decay) sum of l sigmoid(r),   gz = gy h silu'(z)
//
// Bound by memory: every stream is read once and every result written once, where whole sequences make enough workgroups (B8 T4096 D4096 bf16, replayed: forward 277 us, 4.8 TB/s, backward
// 500, 4.8; as single calls under a profiler 292 and 540).  The recurrence is linear, so a run of tokens is the pair (product of a, its
// end from nothing), and pairs join.  A workgroup walks a sequence for 64 V channels, a step at a time: each of its wavefronts takes K tokens of the step for
// all of the channels, makes its run's pair and leaves it in LDS; behind one barrier every wavefront joins the pairs before its own and finishes
// its tokens from the state that gives, still in registers.  Where that makes too few workgroups the sequences are cut in time, and a pass over the decays
// and inputs alone leaves every segment's pair first: it reads x, r and i (backwards r, gy and z) once more, so that such calls stand at 1.5 to 3 times the streams' bytes
// (B1 T4096 D4096 58 / 93 us, B1 T8192 D512 27 / 38).  Backwards a step runs both ways at once: the states again, from one kept
// before every CHECK tokens, and their gradients.
//
// 1 - a^2 loses its digits where a is near one, the very channels that remember long: there it is formed from log a.
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

constexpr int WAVES = 16, BACK_WAVES = 16, CHECK = 64, STEP = 128;         // STEP: tokens of a forward step, and what a segment is a multiple of
constexpr int MAX_TOKEN_STRIDE = 1 << 24;               // a wavefront's tokens lie within 32-bit offsets
constexpr int OUTSIDE = (int)0x80000000u;                 // a lane's offset that is in no row's range

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }

// 1 - a^2 of a = 2^l: near one the polynomial of degree 4 in l nearest to (1 - 4^l) / l where 4^l is above exp(-1/2), right to 2^-22.2 of the value
__device__ __forceinline__ float one_less_square(float l, float a) {
    float p = fmaf(l, -0.03474162146449089f, -0.1514858603477478f);
    p = fmaf(p, l, -0.4437292814254761f);
    p = fmaf(p, l, -0.9608924984931946f);
    p = fmaf(p, l, -1.3862942457199097f);
    return l > -0.36067376f ? l * p : fmaf(-a, a, 1.f);
}
// log2 of a at an open gate; finite, so that a shut gate keeps the state whatever the decay is
__device__ __forceinline__ float rate_of(float decay, float scale) {
    const float soft = decay > 20.f ? decay : log1pf(expf(decay));
    const float rate = -scale * soft * LOG2E;
    return rate < -3e38f ? -3e38f : rate;
}

template <bool B> struct Bool { static constexpr bool value = B; };

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
        len = k.lengths ? min(max(__builtin_amdgcn_readfirstlane(k.lengths[b]), 0), k.T) : k.T;
#pragma unroll
        for (int v = 0; v < V; v++) rate[v] = d < k.D ? rate_of(k.decay[d + v], k.scale) : 0.f;
    }
    // a stream of this sequence, and up to `count` tokens of it from t on, those that there are before `end`: one range for all of them
    struct Stream { const char *p; int step; };
    struct Tokens { __amdgpu_buffer_rsrc_t range; int step; };
    __device__ __forceinline__ Stream in(const Rows &s) const {
        return {static_cast<const char *>(s.p) + (long long)b * s.batch * (long long)sizeof(T), (int)s.token * (int)sizeof(T)};
    }
    __device__ __forceinline__ Stream whole(const void *p) const { return in(Rows{p, (long long)k.T * k.D, k.D}); }
    __device__ __forceinline__ Tokens tokens(const Stream &s, int t, int count, int end) const {
        const int n = min(end - t, count);
        // (a scalar, which the compiler's choice of instructions loses: a range in vector registers is walked lane by lane)
        const int bytes = __builtin_amdgcn_readfirstlane(n > 0 ? (n - 1) * s.step + k.D * (int)sizeof(T) : 0);
        return {__builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(s.p + (long long)t * s.step), (short)0, bytes, 0x00027000), s.step};
    }
    __device__ __forceinline__ Raw load(const Tokens &s, int j) const { return R::load(s.range, at, j * s.step); }
    __device__ __forceinline__ void store(const Tokens &s, int j, const float (&v)[V]) const { R::store(s.range, at, j * s.step, v); }
    // V floats of a row of D, zeros where there is none
    __device__ __forceinline__ void floats(const float *row, float (&o)[V]) const { Row<float, V>::floats(Row<float, V>::load(row, row != nullptr, at32), o); }
    __device__ __forceinline__ void put(float *row, const float (&o)[V]) const { Row<float, V>::store(row, true, at32, o); }
    __device__ __forceinline__ const float *state_row(const float *p) const { return p ? p + (size_t)b * k.D : nullptr; }
    __device__ __forceinline__ float *pair(int segment) const { return k.pairs + ((size_t)b * k.segments + segment) * 2 * k.D; }
    // the pairs of the segments from `from` up to (not with) `to`, eight asked for at once
    __device__ __forceinline__ void join_segments(int from, int to, int step, float (&h)[V]) const {
        typedef Row<float, V> F;
        for (int s0 = from; s0 != to;) {
            const int n = min((to - s0) * step, 8);
            typename F::Raw a[8], e[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                a[j] = F::load(pair(s0 + j * step), j < n, at32);
                e[j] = F::load(pair(s0 + j * step) + k.D, j < n, at32);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float af[V], ef[V];
                F::floats(a[j], af);
                F::floats(e[j], ef);
                if (j < n)
#pragma unroll
                    for (int v = 0; v < V; v++) h[v] = fmaf(af[v], h[v], ef[v]);
            }
            s0 += n * step;
        }
    }
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
    typedef typename Lane<T, V>::Stream Stream;
    typedef typename Lane<T, V>::Tokens Tokens;
    const Stream xs = l.in(k.x), rs = l.in(k.r), is = l.in(k.i), zs = l.in(k.z), ys = l.whole(k.y);
    {
        const int t = begin + wave * K;
        const Tokens nx = l.tokens(xs, t, K, l.len), nr = l.tokens(rs, t, K, l.len), ni = l.tokens(is, t, K, l.len), nz = l.tokens(zs, t, K, l.len);
#pragma unroll
        for (int j = 0; j < K; j++) {
            x[j] = l.load(nx, j);
            r[j] = l.load(nr, j);
            i[j] = l.load(ni, j);
            if (GATE && MODE == FORWARD) z[j] = l.load(nz, j);
        }
    }
    float h[V], all[V];                       // the state before the step; PAIRS: from nothing, with the product of all a
#pragma unroll
    for (int v = 0; v < V; v++) h[v] = 0.f, all[v] = 1.f;
    if (MODE == FORWARD) {
        l.floats(l.state_row(k.state_in), h);
        l.join_segments(0, segment, 1, h);
    }
    // WHOLE: all of the wavefront's tokens are there (as they are but at a sequence's end)
    auto step = [&](auto whole, int t0, int which) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int t = t0 + wave * K;
        float a[K][V], u[K][V];
        Pair mine;
#pragma unroll
        for (int v = 0; v < V; v++) mine.a[v] = 1.f, mine.h[v] = 0.f;
        const Tokens nx = l.tokens(xs, t + STEP, K, l.len), nr = l.tokens(rs, t + STEP, K, l.len), ni = l.tokens(is, t + STEP, K, l.len);
#pragma unroll
        for (int j = 0; j < K; j++) {
            const bool there = WHOLE || t + j < l.len;
            float xf[V], rf[V], jf[V];
            R::floats(x[j], xf);
            R::floats(r[j], rf);
            R::floats(i[j], jf);
            // the next step's token into the place of this one's: as much is on its way at any time as a step takes
            x[j] = l.load(nx, j);
            r[j] = l.load(nr, j);
            i[j] = l.load(ni, j);
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float lg = l.rate[v] * sigmoid(rf[v]), e = exp2_fast(lg);
                a[j][v] = there ? e : 1.f;
                u[j][v] = there ? __builtin_amdgcn_sqrtf(one_less_square(lg, e)) * sigmoid(jf[v]) * xf[v] : 0.f;
                mine.a[v] *= a[j][v];
                mine.h[v] = fmaf(a[j][v], mine.h[v], u[j][v]);
            }
        }
        pairs[which][wave][lane] = mine;
        lds_barrier();
        float before[V];
        auto join = [&](int from, int to) {
#pragma unroll 4
            for (int w = from; w < to; w++) {
                const Pair p = pairs[which][w][lane];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    h[v] = fmaf(p.a[v], h[v], p.h[v]);
                    if (MODE == PAIRS) all[v] *= p.a[v];
                }
            }
        };
        join(0, wave);
#pragma unroll
        for (int v = 0; v < V; v++) before[v] = h[v];
        join(wave, WAVES);
        if (MODE == PAIRS) return;
        if (k.checkpoints && wave * K % CHECK == 0 && t < k.T)
            l.put(k.checkpoints + ((size_t)l.b * ((k.T + CHECK - 1) / CHECK) + t / CHECK) * k.D, before);
        const Tokens y = l.tokens(ys, t, K, k.T), nz = l.tokens(zs, t + STEP, K, l.len);
#pragma unroll
        for (int j = 0; j < K; j++) {
            const bool there = WHOLE || t + j < l.len;
            float o[V], zf[V];
            if (GATE) {
                R::floats(z[j], zf);
                z[j] = l.load(nz, j);
            }
#pragma unroll
            for (int v = 0; v < V; v++) {
                before[v] = fmaf(a[j][v], before[v], u[j][v]);
                o[v] = there ? GATE ? before[v] * (zf[v] * sigmoid(zf[v])) : before[v] : 0.f;
            }
            l.store(y, j, o);
        }
    };
    int which = 0, t0 = begin;
    for (; t0 < end && t0 + STEP <= l.len; t0 += STEP, which ^= 1) step(Bool<true>(), t0, which);
    for (; t0 < end; t0 += STEP, which ^= 1) step(Bool<false>(), t0, which);
    if (wave != 0) return;
    if (MODE == PAIRS) {
        l.put(l.pair(segment), all);
        l.put(l.pair(segment) + k.D, h);
    } else if (segment == k.segments - 1) {
        l.put(k.state_out + (size_t)l.b * k.D, h);
    }
}

template <class T, int V, bool GATE, int MODE>
__global__ __launch_bounds__(64 * BACK_WAVES) void backward(const Call k) {
    constexpr int K = CHECK / BACK_WAVES;
    typedef Row<T, V> R;
    typedef typename R::Raw Raw;
    struct Pair { float a[V], h[V], g[V]; };          // a run's product of a, its state from nothing, what it hands to the token before it from nothing
    __shared__ Pair pairs[2][BACK_WAVES][64];
    const Lane<T, V> l(k);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), segment = blockIdx.z;
    const int begin = segment * k.span, end = min(begin + k.span, k.T), checks = (k.T + CHECK - 1) / CHECK;
    Raw x[K], r[K], i[K], z[K], gy[K];
    float start[V];
    typedef typename Lane<T, V>::Stream Stream;
    typedef typename Lane<T, V>::Tokens Tokens;
    const Stream xs = l.in(k.x), rs = l.in(k.r), is = l.in(k.i), zs = l.in(k.z), gs = l.whole(k.gy);
    const Stream xo = l.whole(k.gx), ro = l.whole(k.gr), io = l.whole(k.gi), zo = l.whole(k.gz);
    Tokens nx, nr, ni, nz, ng;
    auto streams = [&](int t0) {
        const int t = max(t0, begin) + wave * K;
        nr = l.tokens(rs, t, K, l.len);
        ng = l.tokens(gs, t, K, l.len);
        if (GATE) nz = l.tokens(zs, t, K, l.len);
        if (MODE == PAIRS) return;
        nx = l.tokens(xs, t, K, l.len);
        ni = l.tokens(is, t, K, l.len);
        l.floats(k.checkpoints + ((size_t)l.b * checks + max(t0, begin) / CHECK) * k.D, start);
    };
    auto ask = [&](int j) {
        r[j] = l.load(nr, j);
        gy[j] = l.load(ng, j);
        if (GATE) z[j] = l.load(nz, j);
        if (MODE == PAIRS) return;
        x[j] = l.load(nx, j);
        i[j] = l.load(ni, j);
    };
    const int last = begin + (end - begin - 1) / CHECK * CHECK;
    streams(last);
#pragma unroll
    for (int j = 0; j < K; j++) ask(j);
    float c[V], all[V], sum[V];               // c: what the tokens behind the step hand to its last one
#pragma unroll
    for (int v = 0; v < V; v++) c[v] = sum[v] = 0.f, all[v] = 1.f;
    if (MODE == FORWARD) {
        l.floats(l.state_row(k.gstate_out), c);
        l.join_segments(k.segments - 1, segment, -1, c);
    }
    float slope[V];                           // of log a by sigmoid(r)
#pragma unroll
    for (int v = 0; v < V; v++) slope[v] = l.rate[v] * LN2;
    auto step = [&](auto whole, int t0, int which) {
        constexpr bool WHOLE = decltype(whole)::value;
        const int t = t0 + wave * K;
        // what the tokens' second half takes from the first; u: beta sigmoid(i) x
        float a[K][V], beta[K][V], u[K][V], rs[K][V], is[K][V], zs[K][V], hs[K + 1][V];
        Raw zk[K], gk[K];
        Pair mine;
#pragma unroll
        for (int v = 0; v < V; v++) mine.a[v] = 1.f, mine.h[v] = mine.g[v] = 0.f, hs[0][v] = start[v];
        streams(t0 - CHECK);
#pragma unroll
        for (int j = K - 1; j >= 0; j--) {
            const bool there = WHOLE || t + j < l.len;
            float xf[V], rf[V], jf[V], zf[V], gf[V];
            R::floats(r[j], rf);
            R::floats(gy[j], gf);
            if (GATE) R::floats(z[j], zf);
            if (MODE == FORWARD) {
                R::floats(x[j], xf);
                R::floats(i[j], jf);
                gk[j] = gy[j];
                if (GATE) zk[j] = z[j];
            }
            ask(j);          // the next step's token into the place of this one's
#pragma unroll
            for (int v = 0; v < V; v++) {
                rs[j][v] = sigmoid(rf[v]);
                const float lg = there ? l.rate[v] * rs[j][v] : 0.f;
                a[j][v] = exp2_fast(lg);
                if (GATE) zs[j][v] = sigmoid(zf[v]);
                mine.g[v] = a[j][v] * (GATE ? fmaf(gf[v], zf[v] * zs[j][v], mine.g[v]) : gf[v] + mine.g[v]);          // (what is not there came as zeros)
                mine.a[v] *= a[j][v];
                if (MODE == PAIRS) continue;
                const float b = one_less_square(lg, a[j][v]);
                is[j][v] = sigmoid(jf[v]);
                beta[j][v] = __builtin_amdgcn_sqrtf(b);
                u[j][v] = beta[j][v] * is[j][v] * xf[v];
            }
            __builtin_amdgcn_sched_barrier(0);          // (tokens all at once take more registers than there are)
        }
        if (MODE == FORWARD)
#pragma unroll
            for (int j = 0; j < K; j++)
#pragma unroll
                for (int v = 0; v < V; v++) mine.h[v] = fmaf(a[j][v], mine.h[v], u[j][v]);
        pairs[which][wave][lane] = mine;
        lds_barrier();
        float g[V];
        auto join = [&](int from, int to) {          // runs from .. to, the later first
#pragma unroll 4
            for (int w = from; w >= to; w--) {
                const Pair p = pairs[which][w][lane];
#pragma unroll
                for (int v = 0; v < V; v++) {
                    c[v] = fmaf(p.a[v], c[v], p.g[v]);
                    if (MODE == PAIRS) all[v] *= p.a[v];
                }
            }
        };
        join(BACK_WAVES - 1, wave + 1);
#pragma unroll
        for (int v = 0; v < V; v++) g[v] = c[v];
        join(wave, 0);
        if (MODE == PAIRS) return;
#pragma unroll 4
        for (int w = 0; w < wave; w++) {
            const Pair p = pairs[which][w][lane];
#pragma unroll
            for (int v = 0; v < V; v++) hs[0][v] = fmaf(p.a[v], hs[0][v], p.h[v]);
        }
        // (kept in 16 bits over the barrier, not widened before it)
        if constexpr (sizeof(T) == 2)
#pragma unroll
            for (int j = 0; j < K; j++) {
                asm("" : "+v"(gk[j]));
                if (GATE) asm("" : "+v"(zk[j]));
            }
        // hs[j]: the state before token j
#pragma unroll
        for (int j = 0; j < K; j++)
#pragma unroll
            for (int v = 0; v < V; v++) hs[j + 1][v] = fmaf(a[j][v], hs[j][v], u[j][v]);
        const Tokens gx = l.tokens(xo, t, K, k.T), gr = l.tokens(ro, t, K, k.T), gi = l.tokens(io, t, K, k.T), gz = l.tokens(zo, t, K, k.T);
        float part[V];
#pragma unroll
        for (int v = 0; v < V; v++) part[v] = 0.f;
#pragma unroll
        for (int j = K - 1; j >= 0; j--) {
            const bool there = WHOLE || t + j < l.len;
            float ox[V], orr[V], oi[V], oz[V], zf[V], gf[V];
            R::floats(gk[j], gf);
            if (GATE) R::floats(zk[j], zf);
#pragma unroll
            for (int v = 0; v < V; v++) {
                const float zz = GATE ? zf[v] * zs[j][v] : 1.f, gt = fmaf(gf[v], zz, g[v]);          // (last of all factors: it times a state or input alone may be infinite)
                // u changes by log a as -u times a^2 / beta^2: by a squared, for 1 / beta^2 - 1 has no digits left where a is small.  (Where a is one, as at a shut
                // gate, u is zero and so is that: the largest number stands for infinity.)
                const float less = a[j][v] * a[j][v] * fminf(__builtin_amdgcn_rcpf(beta[j][v] * beta[j][v]), 3e38f);
                const float gl = gt * (fmaf(-u[j][v], less, a[j][v] * hs[j][v]) * rs[j][v]);
                ox[v] = there ? gt * (beta[j][v] * is[j][v]) : 0.f;
                oi[v] = there ? gt * fmaf(-u[j][v], is[j][v], u[j][v]) : 0.f;
                orr[v] = there ? gl * (slope[v] * (1.f - rs[j][v])) : 0.f;
                part[v] += there ? gl : 0.f;
                if (GATE) oz[v] = there ? gf[v] * (hs[j + 1][v] * fmaf(zs[j][v], 1.f - zz, zz)) : 0.f;          // (gy h alone may be infinite)
                g[v] = a[j][v] * gt;
            }
            l.store(gx, j, ox);
            l.store(gr, j, orr);
            l.store(gi, j, oi);
            if (GATE) l.store(gz, j, oz);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int v = 0; v < V; v++) sum[v] += part[v];
    };
    // (a loop of each kind: both in one take more registers than there are)
    int which = 0, t0 = last;
    for (; t0 >= begin && t0 + CHECK > l.len; t0 -= CHECK, which ^= 1) step(Bool<false>(), t0, which);
    for (; t0 >= begin; t0 -= CHECK, which ^= 1) step(Bool<true>(), t0, which);
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
    for (int w = 1; w < BACK_WAVES; w++)
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
        o = k.z.p ? h * (z * sigmoid(z)) : h;          // (silu first, as a prompt's: h z may be infinite where it is zero)
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
// How a call is shared out: channels per lane, and segments in time where whole sequences make too few workgroups.  The weights rank the choices and are no times: a step of a
// workgroup counts 5.7 with two channels per lane and 3.6 with one, rounds of workgroups one after the other; a pass for the segments' pairs counts two thirds of the main one, and a
// launch and a walk over the pairs.  They are fitted to bf16 (forward) and hold the order of the others': replayed forward / backward in us, this rule's choice first:
// B4 T777 D4096 one channel 33 / 57, two 44 / 79, two in two segments 54 / 79; B1 T4096 D4096 two in eight 57 / 92, one in four 59 / 104; B5 T2048 D4096 two 112 / 213, one 141 / 256;
// B12 T2048 D4096 one 239 / 434, two 253 / 463; B1 T8192 D512 one in 32 27 / 38, two in 32 35 / 50; B8 T4096 D4096 two 277 / 500, one 308 / 558; fp32 B2 T301 D1001 in three 15.2 / 21.5, whole 15.2 /
// 22.5; B1 T4096 D4096 cut 98 / 167, in four 94 / 166, whole 155 / 283.  A step is 128 tokens (64 backwards) of a workgroup whatever T is, so many sequences of few tokens pay for
// tokens that are not there: 16M elements as B64 T64 D4096 68 / 98, B256 T16 217 / 290, B2048 T2 1665 / 2184 for 33 / 60 of bytes.
struct Plan { int v, span; };
static inline Plan plan_of(int B, int T, int D, bool two) {
    const long long cus = cu_count(), steps = (T + STEP - 1) / STEP;
    Plan best = {1, (int)(steps * STEP)};
    double least = 1e30;
    for (int v = 1; v <= (two ? 2 : 1); v++) {
        const long long groups = (long long)B * ((D + 64 * v - 1) / (64 * v));
        for (long long cut = 1; cut <= std::min<long long>(steps, 64); cut++) {
            const long long each = (steps + cut - 1) / cut, rounds = (groups * ((steps + each - 1) / each) + cus - 1) / cus;
            const double cost = (double)(rounds * each) * (v == 2 ? 5.7 : 3.6) * (cut > 1 ? 1.65 : 1.) + (cut > 1 ? 4. + 0.1 * (double)cut : 0.);
            if (cost < least) least = cost, best = {v, (int)(each * STEP)};
            if (groups * cut >= 2 * cus) break;
        }
    }
    return best;
}
static inline int segments_of(int T, int span) { return (T + span - 1) / span; }
static inline size_t checkpoint_bytes(int B, int T, int D) { return (size_t)B * ((T + CHECK - 1) / CHECK) * D * 4; }
// (the more of what a lane's possible channels need: whether two are possible depends on a call's pointers)
static inline size_t most_segments(int B, int T, int D) {
    return std::max(segments_of(T, plan_of(B, T, D, false).span), segments_of(T, plan_of(B, T, D, true).span));
}
static inline size_t forward_scratch(int B, int T, int D) {
    const size_t n = most_segments(B, T, D);
    return n > 1 ? (size_t)B * n * 2 * D * 4 : 0;
}
static inline size_t backward_scratch(int B, int T, int D) { return (size_t)B * most_segments(B, T, D) * 3 * D * 4; }

template <class T, int V, bool GATE> static void forward_v(hipStream_t s, Call k, int span) {
    k.span = span;
    k.segments = segments_of(k.T, k.span);
    const dim3 grid((k.D + 64 * V - 1) / (64 * V), k.B, k.segments);
    if (k.segments > 1) hipLaunchKernelGGL((forward<T, V, GATE, PAIRS>), grid, dim3(64 * WAVES), 0, s, k);
    hipLaunchKernelGGL((forward<T, V, GATE, FORWARD>), grid, dim3(64 * WAVES), 0, s, k);
}
template <class T, int V, bool GATE> static void backward_v(hipStream_t s, Call k, int span, float *gdecay) {
    k.span = span;
    k.segments = segments_of(k.T, k.span);
    k.part = k.pairs + (k.segments > 1 ? (size_t)k.B * k.segments * 2 * k.D : 0);
    const dim3 grid((k.D + 64 * V - 1) / (64 * V), k.B, k.segments);
    if (k.segments > 1) hipLaunchKernelGGL((backward<T, V, GATE, PAIRS>), grid, dim3(64 * BACK_WAVES), 0, s, k);
    hipLaunchKernelGGL((backward<T, V, GATE, FORWARD>), grid, dim3(64 * BACK_WAVES), 0, s, k);
    Sums<ToDecay> sums;
    sums.add(k.B * k.segments, k.D, k.part, ToDecay{gdecay, k.decay, k.scale});
    sum_rows_launch(s, sums);
}
// two: a lane may take two channels, which those of 16 bits do
template <class T> static hipError_t forward_t(hipStream_t s, const Call &k, bool two) {
    constexpr int PAIR = 4 / sizeof(T);
    const Plan p = plan_of(k.B, k.T, k.D, two && PAIR == 2);
    if (k.T == 1 && !k.checkpoints) hipLaunchKernelGGL(one<T>, dim3((unsigned)(((size_t)k.B * k.D + 255) / 256)), dim3(256), 0, s, k);
    else if (p.v == 2) k.z.p ? forward_v<T, PAIR, true>(s, k, p.span) : forward_v<T, PAIR, false>(s, k, p.span);
    else k.z.p ? forward_v<T, 1, true>(s, k, p.span) : forward_v<T, 1, false>(s, k, p.span);
    return hipGetLastError();
}
template <class T> static hipError_t backward_t(hipStream_t s, const Call &k, bool two, float *gdecay) {
    constexpr int PAIR = 4 / sizeof(T);
    const Plan p = plan_of(k.B, k.T, k.D, two && PAIR == 2);
    if (p.v == 2) k.z.p ? backward_v<T, PAIR, true>(s, k, p.span, gdecay) : backward_v<T, PAIR, false>(s, k, p.span, gdecay);
    else k.z.p ? backward_v<T, 1, true>(s, k, p.span, gdecay) : backward_v<T, 1, false>(s, k, p.span, gdecay);
    return hipGetLastError();
}

}  // namespace gated
}  // namespace wkv
