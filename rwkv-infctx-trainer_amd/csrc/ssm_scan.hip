// The selective state space scan.  For every channel d a state h of N values, started from what the caller hands in:
//
//     dt[t] = softplus(raw[t] + bias)                                   the step's length
//     h[t]  = exp(dt[t] A) h[t-1] + dt[t] x[t] B[t]                     A (N), B[t] (N): shared by the group's channels
//     y[t]  = (C[t] . h[t] + skip x[t]) silu(z[t])
//
// and backwards, with gy = gout silu(z) and g[t] = C[t] gy[t] + exp(dt[t+1] A) g[t+1]:
//
//     gx = dt (B . g) + skip gy            graw = ((B . g) x + A . (g p)) sigmoid(raw + bias),   p[t] = exp(dt[t] A) h[t-1]
//     gB = sum over channels of dt x g     gC = sum over channels of gy h     gA = sum over tokens of dt g p
//
// Layout.  A row of 16 lanes (the unit of a DPP) is one channel, its lanes are 16 states, and over a tile of 16 tokens
// the same lanes are the tokens: a lane reads, converts and finishes one token's values, the recurrence takes them from
// there by row broadcasts that ride on the multiplications, and the sums over the states come out one token per lane
// (reduce_row).  So nothing of a token's own arithmetic is done twice, and there are as many wavefronts as a quarter of
// the channels.  N above 16 takes J = 2 or 4 states per lane.  B[t] and C[t] go through LDS in fp32, [state][token].
//
// What bounds it: the exponentials and fp32 multiply-adds, an exponential and four to five instructions per token, channel
// and state, not the memory (which would take a third of the time).
#include "common.h"
#include "row_sums.h"

namespace wkv {
namespace scan {

constexpr int TILE = 16;                    // tokens per tile = states per lane row
constexpr int PITCH = TILE + 4;             // floats between two states' tokens in LDS: whole 16-byte pieces, every bank once
constexpr int MAX_STATES = 64;

struct Rows {                               // (B, T, .) with a contiguous last dimension; strides in elements
    const void *p;
    long long batch, token, group;
};

struct Call {
    int B, T, D, N, G, Dg, tiles, segments, seg_tiles, seg0;      // Dg channels per group; seg0: the launch's first segment
    Rows x, dt, z, b, c;
    const float *A, *skip, *bias, *state_in;
    const int *lengths;
    void *y;
    float *state_out;
    float *checkpoints;                     // (B, tiles, D, 16 J): the state before every tile, or NULL
    float *seg_state, *seg_dt;              // (B, segments, D, 16 J), (B, segments, D): what a segment makes of nothing, its total step
    // backward
    const void *gy;
    const float *gstate_out;
    void *gx, *gdt, *gz;
    float *gb_part, *gc_part;               // (channel tiles, B, T, G, N)
    float *ga_part, *gskip_part, *gbias_part;   // (B segments, D, N), (B segments, D) twice
    float *gstate_in;
};

template <int I> struct Int { static constexpr int value = I; };
template <int N, int I = 0, class F> __device__ __forceinline__ void unrolled(F f) {
    if constexpr (I < N) {
        f(Int<I>());
        unrolled<N, I + 1>(f);
    }
}
// lane `I` of every row of 16 lanes, to the whole row
template <int I> __device__ __forceinline__ float row_lane(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x150 + I, 0xf, 0xf, true));
}
template <int CTRL> __device__ __forceinline__ float dpp(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
constexpr int ROR8 = 0x128, ROR4 = 0x124, ROR12 = 0x12c, SWAP2 = 0x4e, SWAP1 = 0xb1;      // row_ror:n, quad_perm [2,3,0,1], [1,0,3,2]

// v[i] of 16 lanes summed over the row, the sum of v[n] in lane n: each step adds two registers' halves into one
__device__ __forceinline__ float reduce_row(float (&v)[TILE], int n) {
    float a[8], b[4], c[2];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float lo = v[i] + dpp<ROR8>(v[i]), hi = v[i + 8] + dpp<ROR8>(v[i + 8]);
        a[i] = n & 8 ? hi : lo;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float lo = a[i] + dpp<ROR12>(a[i]), hi = a[i + 4] + dpp<ROR4>(a[i + 4]);      // (lanes of the other half of eight are not read)
        b[i] = n & 4 ? hi : lo;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float lo = b[i] + dpp<SWAP2>(b[i]), hi = b[i + 2] + dpp<SWAP2>(b[i + 2]);
        c[i] = n & 2 ? hi : lo;
    }
    const float lo = c[0] + dpp<SWAP1>(c[0]), hi = c[1] + dpp<SWAP1>(c[1]);
    return n & 1 ? hi : lo;
}

// v[i] summed over the wavefront's four rows: out[i] holds token i + 4 row, state n
__device__ __forceinline__ void reduce_rows(const float (&v)[TILE], float (&out)[4]) {
    float a[8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 8]), false, false);
        a[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(a[i]), __float_as_uint(a[i + 4]), false, false);
        out[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
}

// log(1 + e^v), with the part of e that 1 + e rounds away
__device__ __forceinline__ float softplus(float v) {
    const float e = expf(fminf(v, 20.f)), u = 1.f + e;
    const float s = fmaf(__builtin_amdgcn_logf(u), LN2, (e - (u - 1.f)) * __builtin_amdgcn_rcpf(u));
    return v > 20.f ? v : v != v ? v : s;
}
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }

// Workgroups are handed to the eight XCDs in turn: neighbours in channels, which share lines of the streams and all of B
// and C, are given to one of them.
__device__ __forceinline__ int xcd_order(int i, int n) {
    const int each = n >> 3;
    return i < each << 3 ? (i & 7) * each + (i >> 3) : i;
}

// Where a workgroup is, and the B and C of its tiles on their way through LDS
template <class T, int J, int WAVES, bool NEEDS_C>
struct Work {
    static constexpr int THREADS = 64 * WAVES, CHANNELS = 4 * WAVES, STATES = 16 * J;
    static constexpr int PIECES = (TILE * STATES + THREADS - 1) / THREADS;
    const Call &k;
    int tid, row, n, wave, b, g, ct, seg, channel, len, first, last;      // channel: within all D; first .. last: tiles
    bool live;                                                             // the lane's channel exists
    float pb[PIECES], pc[PIECES];

    __device__ __forceinline__ Work(const Call &k_) : k(k_) {
        tid = threadIdx.x;
        wave = tid >> 6; row = (tid >> 4) & 3; n = tid & 15;
        const int cts = (k.Dg + CHANNELS - 1) / CHANNELS;
        int i = xcd_order(blockIdx.x, gridDim.x);
        ct = i % cts; i /= cts;
        g = i % k.G; i /= k.G;
        b = i % k.B; seg = k.seg0 + i / k.B;
        const int c = ct * CHANNELS + wave * 4 + row;
        live = c < k.Dg;
        channel = g * k.Dg + (live ? c : k.Dg - 1);
        len = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
        first = seg * k.seg_tiles;
        last = min(first + k.seg_tiles, k.tiles);
    }
    __device__ __forceinline__ float stream(const Rows &r, int t) const {
        return t < len ? to_float(static_cast<const T *>(r.p)[b * r.batch + t * r.token + channel]) : 0.f;
    }
    __device__ __forceinline__ float param(const float *p, float other) const { return p ? p[channel] : other; }
    __device__ __forceinline__ size_t state_at(int state) const { return ((size_t)b * k.D + channel) * k.N + state; }
    __device__ __forceinline__ void load_a(float (&a2)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++) a2[j] = n + 16 * j < k.N ? k.A[(size_t)channel * k.N + n + 16 * j] * LOG2E : 0.f;
    }
    __device__ __forceinline__ void load_state(const float *s, float (&h)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++) h[j] = s && n + 16 * j < k.N ? s[state_at(n + 16 * j)] : 0.f;
    }
    __device__ __forceinline__ void store_state(float *s, const float (&h)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++)
            if (live && n + 16 * j < k.N) s[state_at(n + 16 * j)] = h[j];
    }
    __device__ __forceinline__ float *wide(float *s, size_t index) const { return s + (index * k.D + channel) * STATES + n; }
    __device__ __forceinline__ void fetch(int tile) {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int at = tid + i * THREADS, token = at / STATES, state = at % STATES, t = tile * TILE + token;
            const bool in = (TILE * STATES % THREADS == 0 || token < TILE) && t < len && state < k.N && tile >= 0;
            pb[i] = in ? to_float(static_cast<const T *>(k.b.p)[b * k.b.batch + t * k.b.token + g * k.b.group + state]) : 0.f;
            if (NEEDS_C) pc[i] = in ? to_float(static_cast<const T *>(k.c.p)[b * k.c.batch + t * k.c.token + g * k.c.group + state]) : 0.f;
        }
    }
    __device__ __forceinline__ void stage(float *sb, float *sc) const {
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const int at = tid + i * THREADS, token = at / STATES, state = at % STATES;
            if (TILE * STATES % THREADS == 0 || token < TILE) {
                sb[state * PITCH + token] = pb[i];
                if (NEEDS_C) sc[state * PITCH + token] = pc[i];
            }
        }
    }
    __device__ __forceinline__ void read(const float *s, int j, float (&v)[TILE]) const {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const float4 f = *reinterpret_cast<const float4 *>(s + (n + 16 * j) * PITCH + 4 * q);
            v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
        }
    }
};

__device__ __forceinline__ float row_sum(float v) {
    v += dpp<ROR8>(v);
    v += dpp<ROR4>(v);
    v += dpp<SWAP2>(v);
    return v + dpp<SWAP1>(v);
}

// OUT: the outputs of every token; without it a segment's summary (its state from nothing, its total step) alone
template <class T, int J, bool OUT>
__global__ __launch_bounds__(256) void forward(const Call k) {
    typedef Work<T, J, 4, OUT> W;
    __shared__ __align__(16) float bc[2][OUT ? 2 : 1][W::STATES * PITCH];
    W w(k);
    float a2[J], h[J];
    w.load_a(a2);
    const float bias = w.param(k.bias, 0.f), skip = w.param(k.skip, 0.f);
    if (OUT) {
        w.load_state(k.state_in, h);
        for (int s = 0; s < w.seg; s++) {          // what the segments before this one make of it
            const size_t at = (size_t)w.b * k.segments + s;
            const float dt = k.seg_dt[at * k.D + w.channel];
#pragma unroll
            for (int j = 0; j < J; j++) h[j] = fmaf(exp2_fast(dt * a2[j]), h[j], w.wide(k.seg_state, at)[16 * j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < J; j++) h[j] = 0.f;
    }
    float total = 0.f;
    w.fetch(w.first);
    int t = w.first * TILE + w.n;
    float x = w.stream(k.x, t), raw = w.stream(k.dt, t), z = OUT && k.z.p ? w.stream(k.z, t) : 0.f;
    for (int tile = w.first; tile < w.last; tile++) {
        float *sb = bc[tile & 1][0], *sc = bc[tile & 1][OUT ? 1 : 0];
        w.stage(sb, sc);
        lds_barrier();
        const float xn = x, zn = z, dt = t < w.len ? softplus(raw + bias) : 0.f, dtx = dt * x;
        const int tn = t;
        t += TILE;
        w.fetch(tile + 1);
        x = w.stream(k.x, t); raw = w.stream(k.dt, t);
        if (OUT && k.z.p) z = w.stream(k.z, t);
        if (OUT && k.checkpoints && w.live) {
            float *to = w.wide(k.checkpoints, (size_t)w.b * k.tiles + tile);
#pragma unroll
            for (int j = 0; j < J; j++) to[16 * j] = h[j];
        }
        float y[TILE];
#pragma unroll
        for (int j = 0; j < J; j++) {
            float vb[TILE], vc[TILE];
            w.read(sb, j, vb);
            if (OUT) w.read(sc, j, vc);
            unrolled<TILE>([&](auto i) {
                constexpr int I = decltype(i)::value;
                const float a = exp2_fast(row_lane<I>(dt) * a2[j]);
                h[j] = fmaf(a, h[j], row_lane<I>(dtx) * vb[I]);
                if (OUT) y[I] = j == 0 ? vc[I] * h[j] : fmaf(vc[I], h[j], y[I]);
            });
        }
        if (OUT) {
            float out = fmaf(skip, xn, reduce_row(y, w.n));
            if (k.z.p) out *= zn * sigmoid(zn);
            if (w.live && tn < k.T) static_cast<T *>(k.y)[((size_t)w.b * k.T + tn) * k.D + w.channel] = from_float<T>(tn < w.len ? out : 0.f);
        } else {
            total += dt;
        }
    }
    if (OUT) {
        if (w.last == k.tiles) w.store_state(k.state_out, h);
    } else if (w.live) {
        total = row_sum(total);
        const size_t at = (size_t)w.b * k.segments + w.seg;
#pragma unroll
        for (int j = 0; j < J; j++) w.wide(k.seg_state, at)[16 * j] = h[j];
        if (w.n == 0) k.seg_dt[at * k.D + w.channel] = total;
    }
}

// The state's gradient that a segment hands to the one before it if none comes in: the backward's summary
template <class T, int J>
__global__ __launch_bounds__(256) void backward_summary(const Call k) {
    typedef Work<T, J, 4, true> W;
    __shared__ __align__(16) float bc[2][2][W::STATES * PITCH];
    W w(k);
    float a2[J], g[J];
    w.load_a(a2);
    const float bias = w.param(k.bias, 0.f);
#pragma unroll
    for (int j = 0; j < J; j++) g[j] = 0.f;
    float total = 0.f;
    for (int tile = w.last - 1; tile >= w.first; tile--) {
        const int t = tile * TILE + w.n;
        w.fetch(tile);
        const float raw = w.stream(k.dt, t);
        float gy = t < w.len ? to_float(static_cast<const T *>(k.gy)[((size_t)w.b * k.T + t) * k.D + w.channel]) : 0.f;
        if (k.z.p) {
            const float z = w.stream(k.z, t);
            gy *= z * sigmoid(z);
        }
        float *sb = bc[tile & 1][0], *sc = bc[tile & 1][1];
        w.stage(sb, sc);
        lds_barrier();
        const float dt = t < w.len ? softplus(raw + bias) : 0.f;
        total += dt;
#pragma unroll
        for (int j = 0; j < J; j++) {
            float vc[TILE];
            w.read(sc, j, vc);
            unrolled<TILE>([&](auto i) {
                constexpr int I = TILE - 1 - decltype(i)::value;
                g[j] = fmaf(row_lane<I>(gy), vc[I], g[j]) * exp2_fast(row_lane<I>(dt) * a2[j]);
            });
        }
    }
    if (w.live) {
        total = row_sum(total);
        const size_t at = (size_t)w.b * k.segments + w.seg;
#pragma unroll
        for (int j = 0; j < J; j++) w.wide(k.seg_state, at)[16 * j] = g[j];
        if (w.n == 0) k.seg_dt[at * k.D + w.channel] = total;
    }
}

// Tiles from the last to the first.  Within a tile the state runs forward again from its checkpoint, leaving every token's decay a
// and what is left of the state p in registers, then the gradient runs back over them.
constexpr int BACK_WAVES = 8;
template <class T, int J>
__global__ __launch_bounds__(64 * BACK_WAVES) void backward(const Call k) {
    typedef Work<T, J, BACK_WAVES, true> W;
    __shared__ __align__(16) float bc[2][2][W::STATES * PITCH];
    __shared__ __align__(16) float part[BACK_WAVES][2][16 * PITCH];
    W w(k);
    float a2[J], g[J], ga[J];
    w.load_a(a2);
    w.load_state(k.gstate_out, g);
    for (int s = k.segments - 1; s > w.seg; s--) {
        const size_t at = (size_t)w.b * k.segments + s;
        const float dt = k.seg_dt[at * k.D + w.channel];
#pragma unroll
        for (int j = 0; j < J; j++) g[j] = fmaf(exp2_fast(dt * a2[j]), g[j], w.wide(k.seg_state, at)[16 * j]);
    }
#pragma unroll
    for (int j = 0; j < J; j++) ga[j] = 0.f;
    const float bias = w.param(k.bias, 0.f), skip = w.param(k.skip, 0.f);
    float gskip = 0.f, gbias = 0.f;
    const T *gout = static_cast<const T *>(k.gy);
    const size_t bt = (size_t)w.b * k.T;
    for (int tile = w.last - 1; tile >= w.first; tile--) {
        const int t = tile * TILE + w.n;
        w.fetch(tile);
        const float x = w.stream(k.x, t), raw = w.stream(k.dt, t) + bias, z = k.z.p ? w.stream(k.z, t) : 0.f;
        const float go = t < w.len ? to_float(gout[(bt + t) * k.D + w.channel]) : 0.f;
        float h0[J];
        const float *from = w.wide(k.checkpoints, (size_t)w.b * k.tiles + tile);
#pragma unroll
        for (int j = 0; j < J; j++) h0[j] = from[16 * j];
        float *sb = bc[tile & 1][0], *sc = bc[tile & 1][1];
        w.stage(sb, sc);
        lds_barrier();
        const float dt = t < w.len ? softplus(raw) : 0.f, dtx = dt * x;
        const float sig = k.z.p ? sigmoid(z) : 1.f, gate = k.z.p ? z * sig : 1.f, gy = go * gate;
        float y[TILE], sx[TILE], sd[TILE];
#pragma unroll
        for (int j = 0; j < J; j++) {
            float vb[TILE], vc[TILE], a[TILE], p[TILE], gb[TILE], gc[TILE];
            w.read(sb, j, vb);
            w.read(sc, j, vc);
            float h = h0[j];
            unrolled<TILE>([&](auto i) {
                constexpr int I = decltype(i)::value;
                a[I] = exp2_fast(row_lane<I>(dt) * a2[j]);
                p[I] = a[I] * h;
                h = fmaf(row_lane<I>(dtx), vb[I], p[I]);
                y[I] = j == 0 ? vc[I] * h : fmaf(vc[I], h, y[I]);
                gc[I] = row_lane<I>(gy) * h;
            });
            const float an = a2[j] * LN2;
            unrolled<TILE>([&](auto i) {
                constexpr int I = TILE - 1 - decltype(i)::value;
                g[j] = fmaf(row_lane<I>(gy), vc[I], g[j]);
                gb[I] = row_lane<I>(dtx) * g[j];
                const float q = g[j] * p[I];
                sx[I] = j == 0 ? g[j] * vb[I] : fmaf(g[j], vb[I], sx[I]);
                sd[I] = j == 0 ? q * an : fmaf(q, an, sd[I]);
                ga[j] = fmaf(row_lane<I>(dt), q, ga[j]);
                g[j] *= a[I];
            });
            if (!w.live) {          // (its lanes repeat another channel)
#pragma unroll
                for (int i = 0; i < TILE; i++) gb[i] = gc[i] = 0.f;
            }
            float rb[4], rc[4];
            reduce_rows(gb, rb);
            reduce_rows(gc, rc);
            if (j) lds_barrier();
            *reinterpret_cast<float4 *>(&part[w.wave][0][w.n * PITCH + 4 * w.row]) = make_float4(rb[0], rb[1], rb[2], rb[3]);
            *reinterpret_cast<float4 *>(&part[w.wave][1][w.n * PITCH + 4 * w.row]) = make_float4(rc[0], rc[1], rc[2], rc[3]);
            lds_barrier();
            static_assert(W::THREADS == 512, "a thread per element of both sums");
            const int which = w.tid >> 8, token = (w.tid >> 4) & 15, state = w.tid & 15, tt = tile * TILE + token;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < BACK_WAVES; i++) s += part[i][which][state * PITCH + token];
            if (tt < k.T && state + 16 * j < k.N)
                (which ? k.gc_part : k.gb_part)[((((size_t)w.ct * k.B + w.b) * k.T + tt) * k.G + w.g) * k.N + state + 16 * j] = s;
        }
        const float ypre = fmaf(skip, x, reduce_row(y, w.n)), u = reduce_row(sx, w.n), d = reduce_row(sd, w.n);
        const float graw = fmaf(u, x, d) * sigmoid(raw), gx = fmaf(u, dt, gy * skip);
        if (t < w.len) {
            gskip = fmaf(gy, x, gskip);
            gbias += graw;
        }
        if (w.live && t < k.T) {
            const size_t at = (bt + t) * k.D + w.channel;
            const bool in = t < w.len;
            static_cast<T *>(k.gx)[at] = from_float<T>(in ? gx : 0.f);
            static_cast<T *>(k.gdt)[at] = from_float<T>(in ? graw : 0.f);
            if (k.z.p) static_cast<T *>(k.gz)[at] = from_float<T>(in ? go * ypre * (sig + gate * (1.f - sig)) : 0.f);
        }
    }
    gskip = row_sum(gskip);
    gbias = row_sum(gbias);
    if (w.live) {
        const size_t at = ((size_t)w.b * k.segments + w.seg) * k.D + w.channel;
#pragma unroll
        for (int j = 0; j < J; j++)
            if (w.n + 16 * j < k.N) k.ga_part[at * k.N + w.n + 16 * j] = ga[j];
        if (w.n == 0) {
            k.gskip_part[at] = gskip;
            k.gbias_part[at] = gbias;
        }
    }
    if (k.gstate_in && w.seg == 0) w.store_state(k.gstate_in, g);
}

// One token: bound by the states, read once and written once.  Q lanes per channel with four states each (N = 4 Q), or, for
// other N, a row of lanes as above.  state_out may be state_in: a lane writes what it has read.
template <class T, int Q>
__global__ __launch_bounds__(256) void decode(const Call k) {
    constexpr int V = Q ? 4 : 1, LANES = Q ? Q : 16, STEPS = Q ? 1 : (MAX_STATES + 15) / 16;
    const long long item = ((long long)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int lane = threadIdx.x % LANES;
    if (item >= (long long)k.B * k.D) return;
    const int b = (int)(item / k.D), d = (int)(item % k.D), g = d / k.Dg;
    const bool in = !k.lengths || k.lengths[b] > 0;
    const float x = in ? to_float(static_cast<const T *>(k.x.p)[b * k.x.batch + d]) : 0.f;
    const float dt = in ? softplus(to_float(static_cast<const T *>(k.dt.p)[b * k.dt.batch + d]) + (k.bias ? k.bias[d] : 0.f)) : 0.f;
    const T *pb = static_cast<const T *>(k.b.p) + b * k.b.batch + g * k.b.group, *pc = static_cast<const T *>(k.c.p) + b * k.c.batch + g * k.c.group;
    float y = 0.f;
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const int n = V * lane + 16 * s;
        if (n >= k.N) break;
        float a[V], h[V] = {};
        if constexpr (Q != 0) {
            load4(k.A + (size_t)d * k.N + n, a);
            if (k.state_in) load4(k.state_in + item * k.N + n, h);
        } else {
            a[0] = k.A[(size_t)d * k.N + n];
            if (k.state_in) h[0] = k.state_in[item * k.N + n];
        }
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float vb = in ? to_float(pb[n + v]) : 0.f, vc = in ? to_float(pc[n + v]) : 0.f;
            h[v] = fmaf(exp2_fast(dt * (a[v] * LOG2E)), h[v], dt * x * vb);
            y = fmaf(vc, h[v], y);
        }
        if constexpr (Q != 0) store4(k.state_out + item * k.N + n, h);
        else k.state_out[item * k.N + n] = h[0];
    }
#pragma unroll
    for (int m = LANES / 2; m > 0; m >>= 1) y += __shfl_xor(y, m);
    if (lane == 0) {
        y = fmaf(k.skip ? k.skip[d] : 0.f, x, y);
        if (k.z.p) {
            const float z = in ? to_float(static_cast<const T *>(k.z.p)[b * k.z.batch + d]) : 0.f;
            y *= z * sigmoid(z);
        }
        static_cast<T *>(k.y)[(size_t)b * k.D + d] = from_float<T>(in ? y : 0.f);
    }
}

// ---- plans
static inline int states_per_lane(int N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }
static inline long long workgroups(int B, int D, int G, int channels) { return (long long)B * G * ((D / G + channels - 1) / channels); }

// Segments of a sequence: as many as give every compute unit `per_cu` workgroups, none shorter than eight tiles (a segment's
// start costs it one summary per segment before it)
static inline int segments_for(long long groups, int tiles, int per_cu) {
    if (tiles < 16) return 1;
    const long long want = ((long long)per_cu * cu_count() + groups - 1) / groups;
    return (int)std::max(1ll, std::min({want, (long long)tiles / 8, 64ll}));
}
struct Plan { int tiles, segments, seg_tiles; };
static inline Plan plan(int B, int T, int D, int G, bool backward) {
    Plan p;
    p.tiles = (T + TILE - 1) / TILE;
    p.segments = segments_for(workgroups(B, D, G, backward ? 4 * BACK_WAVES : 16), p.tiles, backward ? 1 : 2);
    p.seg_tiles = (p.tiles + p.segments - 1) / p.segments;
    p.segments = (p.tiles + p.seg_tiles - 1) / p.seg_tiles;
    return p;
}
static inline size_t rounded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
static inline size_t summary_bytes(int B, int D, int N, int segments) {
    return segments > 1 ? rounded((size_t)B * segments * D * 16 * states_per_lane(N) * 4) + rounded((size_t)B * segments * D * 4) : 0;
}
static inline size_t checkpoint_bytes(int B, int T, int D, int N) { return (size_t)B * ((T + TILE - 1) / TILE) * D * 16 * states_per_lane(N) * 4; }
static inline size_t forward_scratch(int B, int T, int D, int N, int G) { return T == 1 ? 0 : summary_bytes(B, D, N, plan(B, T, D, G, false).segments); }
static inline size_t backward_scratch(int B, int T, int D, int N, int G) {
    const Plan p = plan(B, T, D, G, true);
    const size_t cts = (D / G + 4 * BACK_WAVES - 1) / (4 * BACK_WAVES), rows = (size_t)B * p.segments;
    return summary_bytes(B, D, N, p.segments) + 2 * rounded(cts * B * T * G * N * 4) + rounded(rows * D * N * 4) + 2 * rounded(rows * D * 4);
}

#define WKV_SCAN_J(KERNEL, GRID, BLOCK, ...)                                                             \
    do {                                                                                                 \
        const dim3 grid_((unsigned)(GRID)), block_(BLOCK);                                               \
        if (J == 1) hipLaunchKernelGGL((KERNEL<T, 1 __VA_ARGS__>), grid_, block_, 0, s, k);              \
        else if (J == 2) hipLaunchKernelGGL((KERNEL<T, 2 __VA_ARGS__>), grid_, block_, 0, s, k);         \
        else hipLaunchKernelGGL((KERNEL<T, 4 __VA_ARGS__>), grid_, block_, 0, s, k);                     \
    } while (0)
#define WKV_COMMA ,

template <class T> static hipError_t forward_t(hipStream_t s, Call k, void *scratch) {
    const int J = states_per_lane(k.N);
    if (k.T == 1 && !k.checkpoints) {
        const bool four = k.N % 4 == 0 && (k.N & (k.N - 1)) == 0;
        const int lanes = four ? k.N / 4 : 16;
        const long long blocks = ((long long)k.B * k.D * lanes + 255) / 256;
#define WKV_DECODE_SCAN(Q) hipLaunchKernelGGL((decode<T, Q>), dim3((unsigned)blocks), dim3(256), 0, s, k)
        switch (four ? lanes : 0) {
            case 1: WKV_DECODE_SCAN(1); break;
            case 2: WKV_DECODE_SCAN(2); break;
            case 4: WKV_DECODE_SCAN(4); break;
            case 8: WKV_DECODE_SCAN(8); break;
            case 16: WKV_DECODE_SCAN(16); break;
            default: WKV_DECODE_SCAN(0); break;
        }
#undef WKV_DECODE_SCAN
        return hipGetLastError();
    }
    const Plan p = plan(k.B, k.T, k.D, k.G, false);
    k.tiles = p.tiles; k.segments = p.segments; k.seg_tiles = p.seg_tiles;
    const long long groups = workgroups(k.B, k.D, k.G, 16);
    if (p.segments > 1) {
        k.seg_state = static_cast<float *>(scratch);
        k.seg_dt = reinterpret_cast<float *>(static_cast<char *>(scratch) + rounded((size_t)k.B * p.segments * k.D * 16 * J * 4));
        // (the last segment's summary is not needed)
        WKV_SCAN_J(forward, groups * (p.segments - 1), 256, WKV_COMMA false);
    }
    WKV_SCAN_J(forward, groups * p.segments, 256, WKV_COMMA true);
    return hipGetLastError();
}

// gradients as wkv_selective_scan_backward hands them out
struct Gradients { void *gb, *gc; float *ga, *gskip, *gbias; };
template <class T> static hipError_t backward_t(hipStream_t s, Call k, const Gradients &to, void *scratch) {
    const int J = states_per_lane(k.N);
    const Plan p = plan(k.B, k.T, k.D, k.G, true);
    k.tiles = p.tiles; k.segments = p.segments; k.seg_tiles = p.seg_tiles;
    char *at = static_cast<char *>(scratch);
    auto take = [&](size_t floats) {
        float *f = reinterpret_cast<float *>(at);
        at += rounded(floats * 4);
        return f;
    };
    const size_t rows = (size_t)k.B * p.segments, cts = (k.Dg + 4 * BACK_WAVES - 1) / (4 * BACK_WAVES), vectors = (size_t)k.B * k.T * k.G * k.N;
    if (p.segments > 1) {
        k.seg_state = take(rows * k.D * 16 * J);
        k.seg_dt = take(rows * k.D);
        k.seg0 = 1;          // (nothing lies before the first)
        WKV_SCAN_J(backward_summary, workgroups(k.B, k.D, k.G, 16) * (p.segments - 1), 256, );
        k.seg0 = 0;
    }
    k.gb_part = take(cts * vectors);
    k.gc_part = take(cts * vectors);
    // (one row of fp32 partial sums is the sum)
    k.ga_part = rows == 1 ? to.ga : take(rows * k.D * k.N);
    k.gskip_part = rows == 1 && to.gskip ? to.gskip : take(rows * k.D);
    k.gbias_part = rows == 1 && to.gbias ? to.gbias : take(rows * k.D);
    WKV_SCAN_J(backward, workgroups(k.B, k.D, k.G, 4 * BACK_WAVES) * p.segments, 64 * BACK_WAVES, );
    sum_rows_launch(s, (int)cts, vectors, k.gb_part, ToRow<T>{static_cast<T *>(to.gb)});
    sum_rows_launch(s, (int)cts, vectors, k.gc_part, ToRow<T>{static_cast<T *>(to.gc)});
    if (rows > 1) {
        sum_rows_launch(s, (int)rows, (size_t)k.D * k.N, k.ga_part, ToRow<float>{to.ga});
        if (to.gskip) sum_rows_launch(s, (int)rows, (size_t)k.D, k.gskip_part, ToRow<float>{to.gskip});
        if (to.gbias) sum_rows_launch(s, (int)rows, (size_t)k.D, k.gbias_part, ToRow<float>{to.gbias});
    }
    return hipGetLastError();
}

}  // namespace scan
}  // namespace wkv
