// The first half of a gated feed-forward block,  h = act(x Wg') * (x Wu')  with x (R, C) and both weights (F, C), and its backward:
//
//     g = x Wg',  u = x Wu',  h = act(g) u
//     dg = gh u act'(g),  du = gh act(g),  gx = dg Wg + du Wu,  gWg = dg' x,  gWu = du' x
//
// 4 R C F operations forward and 8 backward, on the matrix cores (matrix_tiles.h): bound by these with many rows (4096 rows of 4096 into 14336 columns bf16: forward
// 830 to 860 us, 1120 to 1160 TFLOP/s; gx 670 to 700 and weights' gradients 770 to 810, up to 1430 and 1250; the clock that power leaves decides), by the weights' bytes with few (1 row: 45 us, 5.2 TB/s).  Forward, a workgroup's tile of B is half of gate rows and
// half of the same up rows, so that a lane ends with g and u of the same places and the activation and product happen in registers: g and u
// never reach memory, except that a backward's are kept in fp32: rounded to 16 bits they would add as much to the gradients' error as each of the two
// roundings that are left, that of dg and du, which the matrix cores take in the streams' type, and that of the results (bf16, error of
// the 2-norm: 3.1e-3 against 2.4e-3).  Backward, one pass makes dg and du; the three products read
// them, x and the weights as they lie, with the index that is summed along memory or across it (gx: along dg and du, across the weights; gWg and gWu: across both).
#include <cmath>
#include <type_traits>

#include "matrix_tiles.h"
#include "vec.h"

namespace wkv {
namespace ffn {

using tiles::f4;
using tiles::i4;

enum { SILU = 0, GELU = 1, RELU = 2, ACTIVATIONS = 3 };

// widths in memory of this library's own are whole tiles of k, rows of 128 bytes
constexpr int ROUND = 64;
static inline long long rounded(long long n) { return (n + ROUND - 1) / ROUND * ROUND; }

__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }
constexpr float GELU_IN = 1.5957691216057308f, GELU_CUBE = 0.044715f;          // 2 sqrt(2 / pi): (1 + tanh v) / 2 = sigmoid(2 v)
__device__ __forceinline__ float activation(int kind, float g) {
    if (kind == RELU) return g > 0.f || g != g ? g : 0.f;
    return g * sigmoid(kind == SILU ? g : GELU_IN * fmaf(GELU_CUBE * g * g, g, g));
}
// the activation's value and slope
__device__ __forceinline__ void activation(int kind, float g, float &value, float &slope) {
    if (kind == RELU) {
        value = g > 0.f || g != g ? g : 0.f;
        slope = g > 0.f ? 1.f : 0.f;
        return;
    }
    const float s = sigmoid(kind == SILU ? g : GELU_IN * fmaf(GELU_CUBE * g * g, g, g));
    // g times the slope of what the sigmoid takes (past 1000 the sigmoid has none, but the cube would be infinite)
    const float c = fminf(fmaxf(g, -1000.f), 1000.f), inner = kind == SILU ? c : GELU_IN * fmaf(3.f * GELU_CUBE * c * c, c, c);
    value = g * s;
    slope = fmaf(inner * s, 1.f - s, s);
}

// four elements of a row from column n on, as far as the row goes
template <class T> __device__ __forceinline__ void put4(T *row, int n, int N, bool whole, const float (&v)[4]) {
    if (whole && n + 4 <= N) {
        store4(row + n, v);
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n + e < N) row[n + e] = from_float<T>(v[e]);
}

// Tiles of k ahead, and the wavefronts to a SIMD that LDS then leaves room for.  Tiles of 256 and 128 fill it with two tiles ahead.  Those of 64 leave room for four
// workgroups then, or for two with four tiles ahead, which is better where there are no more than two to a compute unit: nothing else hides what their loads wait for
// ((24, 2560) into 8192 columns bf16, weights out of the cache, 31 -> 21 us; (150, 1024) into 2816 13.0 -> 10.4; but (600, 512) into 2000 fp32 31.5 -> 35.7).
constexpr int DEEP = 4;
constexpr int waves_per_simd(int size, int ahead) { return  ahead == DEEP ? 2 : 256 / size; }
static inline bool deep_pays(long long groups) { return groups <= 2ll * cu_count(); }

// ---- forward
struct Forward {
    int R, K, F, kind;
    const void *x, *wg, *wu;
    long long xs, ws;                 // row strides
    void *h;
    float *kept;                      // (R, 2 Fs), g and u side by side, or NULL
    long long hs, Fs;
};

// LIE: rows are read as they lie, whole tiles of k straight to LDS and what is left behind them, if anything, before, by way of registers
template <class T, int BM, int BN, int WM, int WN, int AHEAD, bool LIE>
__global__ __launch_bounds__(64 * WM * WN, waves_per_simd(BM, AHEAD)) void forward(const Forward k, int rows, int columns, int width) {
    typedef tiles::Loop<T, tiles::Along<T, BM, 64 * WM * WN>, tiles::Along<T, BN / 2, 64 * WM * WN>, BM, BN, WM, WN, 2, AHEAD> L;
    __shared__ __align__(1024) char lds[L::LDS];
    int tm, tn;
    tiles::tile_of(blockIdx.x, rows, columns, tm, tn);
    const int m0 = tm * BM, n0 = tn * width, end = min(n0 + width, k.F);
    const int K = LIE ? k.K / tiles::depth<T>() * tiles::depth<T>() : k.K, live = min(BM, k.R - m0), columns_live = end - n0;
    const T *x = static_cast<const T *>(k.x) + m0 * k.xs, *wg = static_cast<const T *>(k.wg) + n0 * k.ws, *wu = static_cast<const T *>(k.wu) + n0 * k.ws;
    L l;
    l.a.place(x, k.xs, K, live);
    l.b[0].place(wg, k.ws, K, columns_live);
    l.b[1].place(wu, k.ws, K, columns_live);
    l.clear();
    if (LIE && K < k.K) {
        char *at_b = lds + (AHEAD + 1) * L::ABYTES;
        l.a.carry(x, k.xs, live, K, k.K, lds);
        l.b[0].carry(wg, k.ws, columns_live, K, k.K, at_b);
        l.b[1].carry(wu, k.ws, columns_live, K, k.K, at_b + L::BBYTES / 2);
        l.once(lds);
    }
    if (!LIE || K > 0) l.run(0, K, K, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    const bool whole = k.hs % 4 == 0;
    T *h = static_cast<T *>(k.h);
#pragma unroll
    for (int i = 0; i < L::MT; i++) {
        const int m = m0 + (wm * L::MT + i) * 16 + (lane & 15);
        if (m >= k.R) continue;
#pragma unroll
        for (int j = 0; j < L::NT / 2; j++) {
            const int n = n0 + (wn * (L::NT / 2) + j) * 16 + 4 * (lane >> 4);
            float g[4], u[4], o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                g[e] = l.acc[i][j][e];
                u[e] = l.acc[i][j + L::NT / 2][e];
                o[e] = activation(k.kind, g[e]) * u[e];
            }
            put4(h + m * k.hs, n, end, whole, o);
            if (k.kept) {
                put4(k.kept + m * (2 * k.Fs), n, end, true, g);
                put4(k.kept + m * (2 * k.Fs) + k.Fs, n, end, true, u);
            }
        }
    }
}

// fp16 has 5 bits of exponent: slopes that fp32 holds would be infinite from 65504 on and lose digits below 2^-14, where a mean loss' gradients lie.  So fp16 slopes are
// written times a power of two, the same for the whole call, that takes the largest finite one to 2^14 .. 2^15 (what is 2^-29 of it still has all its digits), and the
// products divide their fp32 sums by it.  A pass of its own finds the largest, by 256 workgroups, and reads what the slopes' pass reads again (the whole
// backward of 4096 rows of 4096 into 14336 columns 1656 -> 1775 us, of 777 of 2048 into 7168 140 -> 153, of 16 of 2560 into 8960 84 -> 88); bf16 and fp32 have no need of it.
template <class T> constexpr bool scaled() { return std::is_same<T, f16>::value; }
constexpr int LARGEST = 256;                  // workgroups, a number of each

// ---- a product of two operands
struct Product {
    int M, N, K;
    const void *a, *b, *b2;           // b2: B's rows of k from `turn` on
    long long as, bs;
    int turn, a_rows, b_rows;         // rows of k that are there, where k is across
    // out: rows below `split` (of which `live` are there) to out0, those from it on to out1; parts: fp32 sums over a share of k instead
    void *out0, *out1;
    long long os;
    int split, live;
    float *parts;
    int per;                          // of k to a share
    bool pairs;                       // every two rows of A are one number in two parts: rows of the result where they lie along memory, of k where across
    const int *exponent;              // fp16: A is times 2 to it
};
// what undoes it: asked for before a product's loop, for behind a store it would be asked for again
template <class T> struct Unscaled {
    int down = 0;
    __device__ __forceinline__ Unscaled(const Product &k) {
        if constexpr (scaled<T>()) down = -*k.exponent;
    }
    __device__ __forceinline__ float operator()(float v) const {
        if constexpr (scaled<T>()) return ldexpf(v, down);
        return v;
    }
};

// ACROSS_A: k lies across memory in A, as it does in B
template <class T, int BM, int BN, int WM, int WN, int AHEAD, bool ACROSS_A>
__global__ __launch_bounds__(64 * WM * WN, waves_per_simd(BM, AHEAD)) void product(const Product k, int rows, int columns) {
    typedef std::conditional_t<ACROSS_A, tiles::Across<T, BM, 64 * WM * WN>, tiles::Along<T, BM, 64 * WM * WN>> A;
    typedef tiles::Across<T, BN, 64 * WM * WN> B;
    typedef tiles::Loop<T, A, B, BM, BN, WM, WN, 1, AHEAD> L;
    __shared__ __align__(1024) char lds[L::LDS];
    int tm, tn;
    tiles::tile_of(blockIdx.x, rows, columns, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    L l;
    const T *a = static_cast<const T *>(k.a), *b = static_cast<const T *>(k.b), *b2 = static_cast<const T *>(k.b2);
    constexpr int E = tiles::piece<T>();          // (rows are whole pieces, what they hold may not be)
    if constexpr (ACROSS_A) l.a.place(a, a, 0x7fffffff, k.as, m0, k.a_rows, (k.M + E - 1) / E * E);
    else l.a.place(a + m0 * k.as, k.as, k.K, min(BM, k.M - m0));
    l.b[0].place(b, b2, k.turn, k.bs, n0, k.b_rows, (k.N + E - 1) / E * E, ACROSS_A && k.pairs);
    const int k0 = blockIdx.y * k.per;
    const Unscaled<T> unscaled(k);
    l.clear();
    l.run(k0, min(k0 + k.per, k.K), k.K, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    const bool whole = k.os % 4 == 0, pairs = !ACROSS_A && k.pairs;
    const int M = pairs ? k.M / 2 : k.M;
#pragma unroll
    for (int i = 0; i < L::MT; i++) {
        const int in = m0 + (wm * L::MT + i) * 16 + (lane & 15), m = pairs ? in >> 1 : in, r = m < k.split ? m : m - k.split;
        if (pairs)
#pragma unroll
            for (int j = 0; j < L::NT; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) l.acc[i][j][e] += __shfl_xor(l.acc[i][j][e], 1);
        if (m >= M || r >= k.live || (pairs && in & 1)) continue;
#pragma unroll
        for (int j = 0; j < L::NT; j++) {
            const int n = n0 + (wn * L::NT + j) * 16 + 4 * (lane >> 4);
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = k.parts ? l.acc[i][j][e] : unscaled(l.acc[i][j][e]);
            if (k.parts) put4(k.parts + ((size_t)blockIdx.y * M + m) * k.os, n, k.N, whole, o);
            else put4(static_cast<T *>(m < k.split ? k.out0 : k.out1) + r * k.os, n, k.N, whole, o);
        }
    }
}
// the shares' sums, in their order
template <class T> __global__ __launch_bounds__(256) void join(const Product k, int M, int shares) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)M * k.os;
    if (i >= n) return;
    float s = k.parts[i];
    for (int p = 1; p < shares; p++) s += k.parts[p * n + i];
    const int m = (int)(i / k.os), r = m < k.split ? m : m - k.split;
    if (r < k.live) static_cast<T *>(m < k.split ? k.out0 : k.out1)[r * k.os + i % k.os] = from_float<T>(Unscaled<T>(k)(s));
}

// ---- layouts
// rows of C elements -> rows of Cs, zeros behind; up to three arrays in a launch
struct Widen {
    struct { const void *in; void *out; long long stride; size_t end; } array[3];          // end: of the elements written, over the arrays
    int C, Cs;
};
template <class T> __global__ __launch_bounds__(256) void widen(const Widen k) {
    constexpr int V = tiles::piece<T>();
    size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * V, first = 0;
    int j = 0;
    while (j < 2 && i >= k.array[j].end) first = k.array[j++].end;
    if (i >= k.array[j].end) return;
    i -= first;
    const size_t r = i / k.Cs;
    const int c = (int)(i - r * k.Cs);
    const T *in = static_cast<const T *>(k.array[j].in) + r * k.array[j].stride;
    uint4 raw;
    if (c + V <= k.C) {
        __builtin_memcpy(&raw, in + c, 16);          // (one load, whatever the alignment)
    } else {
        T e[V];
#pragma unroll
        for (int q = 0; q < V; q++) e[q] = c + q < k.C ? in[c + q] : from_float<T>(0.f);
        __builtin_memcpy(&raw, e, 16);
    }
    *reinterpret_cast<uint4 *>(static_cast<T *>(k.array[j].out) + i) = raw;
}
// dg and du of four places of a row from column f on, zeros past F
template <class T, bool WHOLE> __device__ __forceinline__ void slopes_at(const float *row, const T *gh, int kind, int f, int F, long long Fs, float (&dg)[4], float (&du)[4]) {
    float g[4], u[4], o[4];
    load4(row + f, g);
    load4(row + Fs + f, u);
    if (WHOLE && f + 4 <= F) load4(gh + f, o);
    else
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = f + e < F ? to_float(gh[f + e]) : 0.f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float value, slope;
        activation(kind, g[e], value, slope);
        // (what is kept past F was never written; gh u alone may be infinite)
        dg[e] = f + e < F ? o[e] * (u[e] * slope) : 0.f;
        du[e] = f + e < F ? o[e] * value : 0.f;
    }
}
template <class T, bool WHOLE> __global__ __launch_bounds__(1024) void largest(int R, int F, int kind, const float *kept, const T *gh, long long Fs, float *most) {
    __shared__ float wave_most[16];
    const int pieces = (int)(Fs / 4), first = blockIdx.x * 1024 + threadIdx.x, rows = LARGEST * 1024 / pieces, rest = LARGEST * 1024 % pieces;
    float m = 0.f;
    for (int r = first / pieces, c = first % pieces; r < R;) {
        float dg[4], du[4];
        slopes_at<T, WHOLE>(kept + r * 2 * Fs, gh + (long long)r * F, kind, c * 4, F, Fs, dg, du);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float v = fmaxf(fabsf(dg[e]), 0.f), w = fmaxf(fabsf(du[e]), 0.f);          // (NaN: zero)
            m = fmaxf(m, fmaxf(v < INFINITY ? v : 0.f, w < INFINITY ? w : 0.f));
        }
        r += rows;
        c += rest;
        if (c >= pieces) c -= pieces, r++;
    }
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    if ((threadIdx.x & 63) == 0) wave_most[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x != 0) return;
#pragma unroll
    for (int w = 1; w < 16; w++) m = fmaxf(m, wave_most[w]);
    most[blockIdx.x] = m;
}
// the exponent of the call's power of two, for every lane of a wavefront
__device__ __forceinline__ int exponent_of(const float *most) {
    float v[4];
    static_assert(LARGEST == 4 * 64, "four numbers to a lane");
    load4(most + 4 * (threadIdx.x & 63), v);
    float m = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
#pragma unroll
    for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
    return m > 0.f ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
}
// dg and du (R, 2 Fs) from g, u and gh, zeros past F; a row per workgroup of y.  pairs: (2 R, 2 Fs), what a row's rounding leaves in the row behind it.  fp16: times 2 to the
// exponent, which is left for the products
template <class T, bool WHOLE> __global__ __launch_bounds__(256) void slopes(int R, int F, int kind, const float *kept, const T *gh, T *d, long long Fs, bool pairs, const float *most, int *exponent) {
    const int f = (blockIdx.x * 256 + threadIdx.x) * 4;
    int up = 0;
    if constexpr (scaled<T>()) {
        up = exponent_of(most);
        if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *exponent = up;
    }
    if (f >= Fs) return;
    for (int r = blockIdx.y; r < R; r += gridDim.y) {
        float dg[4], du[4];
        slopes_at<T, WHOLE>(kept + r * 2 * Fs, gh + (long long)r * F, kind, f, F, Fs, dg, du);
        if constexpr (scaled<T>())
#pragma unroll
            for (int e = 0; e < 4; e++) dg[e] = ldexpf(dg[e], up), du[e] = ldexpf(du[e], up);
        T *to = d + (long long)r * (pairs ? 4 : 2) * Fs + f;
        store4(to, dg);
        store4(to + Fs, du);
        if (!pairs) continue;
        // (infinity is all in the first part)
        auto left = [](float v) {
            const float rounded = to_float(from_float<T>(v));
            return fabsf(rounded) < INFINITY ? v - rounded : 0.f;
        };
#pragma unroll
        for (int e = 0; e < 4; e++) dg[e] = left(dg[e]), du[e] = left(du[e]);
        store4(to + 2 * Fs, dg);
        store4(to + 3 * Fs, du);
    }
}

// ---- few rows: a serving loop's single tokens.  What they cost is the weights, read once: a workgroup takes 16 gate rows and the same 16 up rows,
// its four wavefronts every fourth tile of k; operands go straight from memory to registers, so that nothing waits for a barrier or for LDS (1 row of 1002
// into 2731 columns bf16, weights out of the cache: 7.2 us with the launch).
constexpr int FEW = 64, FEW_WAVES = 4;
template <class T, int GROUPS, bool WHOLE>                    // GROUPS of 16 rows of x; WHOLE: rows are whole pieces of 16 bytes
__global__ __launch_bounds__(64 * FEW_WAVES) void few(const Forward k) {
    constexpr int E = tiles::piece<T>(), D = tiles::depth<T>(), STEP = FEW_WAVES * D, AHEAD = GROUPS == 1 ? 4 : 2;
    __shared__ f4 part[FEW_WAVES][GROUPS][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16, in = lane & 15;
    const int f = min(n0 + in, k.F - 1);
    const T *wg = static_cast<const T *>(k.wg) + f * k.ws, *wu = static_cast<const T *>(k.wu) + f * k.ws, *x[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; i++) x[i] = static_cast<const T *>(k.x) + min(i * 16 + in, k.R - 1) * k.xs;
    f4 g[GROUPS], u[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; i++) g[i] = u[i] = f4{0.f, 0.f, 0.f, 0.f};
    enum { PIECES, INSIDE, ELEMENTS };          // pieces that are there or not; all of them inside the rows, at any alignment; any end
    auto load = [&](auto how, const T *p, int at) -> i4 {
        i4 v = {0, 0, 0, 0};
        if constexpr (decltype(how)::value == PIECES) {
            const i4 there = *reinterpret_cast<const i4 *>(p + (at < k.K ? at : 0));
            if (at < k.K) v = there;
        } else if constexpr (decltype(how)::value == INSIDE) {
            __builtin_memcpy(&v, p + at, 16);
        } else {
            T e[E];
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = at + q < k.K ? p[at + q] : from_float<T>(0.f);
            __builtin_memcpy(&v, e, 16);
        }
        return v;
    };
    // `N` of the wavefront's tiles of k from t on
    auto tiles_at = [&](auto how, auto many, int t) {
        constexpr int N = decltype(many)::value;
        i4 a[N][2], b[N][2], y[N][2][GROUPS];
#pragma unroll
        for (int q = 0; q < N; q++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int at = t + q * STEP + ((lane >> 4) + 4 * s) * E;
                a[q][s] = load(how, wg, at);
                b[q][s] = load(how, wu, at);
#pragma unroll
                for (int i = 0; i < GROUPS; i++) y[q][s][i] = load(how, x[i], at);
            }
#pragma unroll
        for (int q = 0; q < N; q++)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < GROUPS; i++) {
                    g[i] = tiles::mma<T>(a[q][s], y[q][s][i], g[i]);
                    u[i] = tiles::mma<T>(b[q][s], y[q][s][i], u[i]);
                }
    };
    typedef std::integral_constant<int, AHEAD> Many;
    typedef std::integral_constant<int, 1> One;
    int t = wave * D;
    if (WHOLE) {
        for (; t < k.K; t += STEP * AHEAD) tiles_at(std::integral_constant<int, PIECES>(), Many(), t);
    } else {
        for (; t + STEP * (AHEAD - 1) + D <= k.K; t += STEP * AHEAD) tiles_at(std::integral_constant<int, INSIDE>(), Many(), t);
        for (; t + D <= k.K; t += STEP) tiles_at(std::integral_constant<int, INSIDE>(), One(), t);
        if (t < k.K) tiles_at(std::integral_constant<int, ELEMENTS>(), One(), t);
    }
#pragma unroll
    for (int i = 0; i < GROUPS; i++) {
        part[wave][i][0][lane] = g[i];
        part[wave][i][1][lane] = u[i];
    }
    __syncthreads();
    const int i = wave, m = i * 16 + in, n = n0 + 4 * (lane >> 4);
    if (i >= GROUPS || m >= k.R) return;
    f4 a = part[0][i][0][lane], b = part[0][i][1][lane];
#pragma unroll
    for (int w = 1; w < FEW_WAVES; w++) {
        a += part[w][i][0][lane];
        b += part[w][i][1][lane];
    }
    const float gv[4] = {a[0], a[1], a[2], a[3]}, uv[4] = {b[0], b[1], b[2], b[3]};
    float o[4];
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = activation(k.kind, gv[e]) * uv[e];
    put4(static_cast<T *>(k.h) + m * k.hs, n, k.F, k.hs % 4 == 0, o);
    if (k.kept) {
        float *kept = k.kept + m * 2 * k.Fs;
        put4(kept, n, k.F, true, gv);
        put4(kept + k.Fs, n, k.F, true, uv);
    }
}

// ---- launches
struct Layout {
    Widen k = {};
    size_t all = 0;
    int count = 0;
    explicit Layout(int C) { k.C = C; k.Cs = (int)rounded(C); }
    // from here on p is the copy at `to`
    template <class T> void add(const T *&p, long long stride, int rows, void *to) {
        all += (size_t)rows * k.Cs;
        k.array[count++] = {p, to, stride, all};
        p = static_cast<const T *>(to);
    }
    template <class T> void launch(hipStream_t s) {
        for (int j = count; j < 3; j++) k.array[j].end = all;
        if (all) hipLaunchKernelGGL(widen<T>, dim3((unsigned)((all / tiles::piece<T>() + 255) / 256)), dim3(256), 0, s, k);
    }
};
static inline int tiles_of(long long n, int size) { return (int)((n + size - 1) / size); }
// What `groups` workgroups of tiles of a size take, each `steps` tiles deep, in us: in rounds of one tile of 256, two of 128 or four of 64 to a compute unit, as many as LDS has room for (fp32
// is bound by the matrix cores, and a unit's groups add up).  Fitted to shapes in bf16, fp16 and fp32 from 16 to 4096 rows, where the choice by these is the
// fastest or within 10 % of it: by 256, 128, 64 x (200, 4096) into 14336 columns bf16 105, 79, 113, (300, 4096) 107, 128, 159, (400, 2560) into 8960 72, 81, 86,
// (777, 2048) into 5632 53, 59, 69, (300, 1024) into 4096 28, 14, 12; (301, 1001) into 2731 fp32 258, 86, 54.
template <class T> static double cost_of(int size, long long groups, long long steps) {
    const long long cus = cu_count();
    const double share = (double)groups / (double)cus, n = (double)steps;
    if (sizeof(T) == 4) {
        if (size == 256) return (double)((groups + cus - 1) / cus) * (7.6 * n + 10);
        if (size == 128) return std::max(2.3 * n + 4, share * (2.0 * n + 2));
        return std::max(0.8 * n + 2, share * (0.55 * n + 0.6));
    }
    if (size == 256) return (double)((groups + cus - 1) / cus) * (1.5 * n + 6);
    if (size == 64) return std::max(0.48 * n + 2, std::ceil(share) * (0.235 * n + 0.6));
    const long long rest = groups % (2 * cus);
    return (double)(groups / (2 * cus)) * (1.08 * n + 2) + (rest == 0 ? 0 : rest <= cus ? 0.8 * n + 3 : 1.08 * n + 2);
}
// How a product is shared out: the tiles' size, and k cut into shares where the tiles do not fill the compute units, their sums joined by another launch
struct Plan { int size, rows, columns, shares, per; double cost; };
template <class T> static Plan plan_of(long long M, long long N, long long K, bool cut) {
    Plan best = {};
    const long long steps = (K + tiles::depth<T>() - 1) / tiles::depth<T>();
    double least = 1e30;
    for (int size : {256, 128, 64})
        for (long long shares = 1; shares <= (cut && size < 256 ? 16 : 1) && steps >= 4 * shares - 3; shares *= 2) {
            const long long rows = tiles_of(M, size), columns = tiles_of(N, size), each = (steps + shares - 1) / shares, all = (steps + each - 1) / each;
            const double cost = cost_of<T>(size, rows * columns * all, each) + (all > 1 ? 5 + (double)(all * M * N) * 8 / 4e6 : 0);
            if (cost < least) least = cost, best = {size, (int)rows, (int)columns, (int)all, (int)(each * tiles::depth<T>()), cost};
        }
    return best;
}
// Up to 64 rows: whether to take their kernel.  It reads the weights at what memory gives and waits for nothing, but reads x again for every 16 columns (weights out of
// the cache, in us with the launch by it and by tiles: bf16 (4096, 14336) 1 row 50 and 46, 16 rows 62 and 47, 64 rows 102 and 52; (1002, 2731) 7.2 and 9.8, 7.4 and 10.1, 10.2 and 13.8; fp32
// (1001, 2731) 9 and 27, 11 and 27, 18 and 28; (4095, 14335) 118 and 160, 147 and 156, 255 and 170; (1024, 8960) 26 and 42, 28 and 42, 62 and 43).  Rows that begin between 4 bytes cost it twice
// a row's loads: bf16 (4095, 14335) 102 and 60, 148 and 59, 294 and 79, rows that begin at 4 ((4094, 14335)) 68 and 65, 82 and 62, 143 and 80.
template <class T> static bool few_pays(int R, int C, int F) {
    if (R > FEW) return false;
    const double mb = 2. * F * C * sizeof(T) / 1e6, groups = R <= 16 ? 1 : R <= 32 ? 2 : 4;
    const bool narrow = sizeof(T) == 2, whole = C % tiles::piece<T>() == 0;
    const double few = 3 + mb * (!narrow ? 0.15 + 0.14 * groups : whole ? 0.22 + 0.0033 * R : C % 2 == 0 ? 0.26 + 0.0055 * R : 0.5 + 0.015 * R);
    const double tiled = std::max((narrow ? 0.22 : 0.33) * mb, cost_of<T>(64, tiles_of(F, 32), (C + tiles::depth<T>() - 1) / tiles::depth<T>()));
    return few < (narrow && !whole ? 1.2 : 1.) * tiled;
}
// Rows that are not whole pieces of 16 bytes: read as they lie (pieces that lie across lines take the memory pipe longer, by a third of the whole call's time with 16-bit elements,
// next to nothing with fp32), or copied to rows that are, by another launch.  In us so and copied, bf16: (4095, 14335) 64 rows 83 and 158, 777 rows 267 and 317; (1001, 2731) 128 rows 11 and 18,
// 777 rows 33 and 30, 4096 rows 92 and 70; (2050, 5001) 1500 rows 77 and 85, 4096 rows 217 and 205; fp32 (1001, 2731) 300 rows 48 and 57, 4096 rows 406 and 404.
struct Choice { bool few, lie, copy; Plan plan; };
// Columns of a tile (gate and up rows each).  One row of tiles of 64 that is more than one to a compute unit and up to one and a half leaves some with twice the work, all of it loads:
// there every compute unit takes its share of the columns as one tile of up to 48, as wide as that (x (64, 2560) into 8960 columns bf16 34.7 -> 24.6 us, 16 rows 27.0 -> 21.3,
// (64, 4096) into 11008 46.3 -> 41.0; but 1 row of 4096 into 14336, seven quarters to a compute unit, 45 -> 49, and (64, 2048) into 7168, less than one, 16.7 -> 19.0; fp32 is bound by
// the matrix cores, 45 and 45 us for (64, 1024) into 8960).
template <class T> static int width_of(const Plan &p, int F) {
    const int cus = cu_count(), small = tiles_of(F, 32);
    return sizeof(T) == 2 && p.size == 64 && p.rows == 1 && small > cus && 2 * small <= 3 * cus ? (tiles_of(F, cus) + 3) / 4 * 4 : p.size / 2;
}
template <class T> static Choice choose(int R, int C, int F) {
    Choice c = {few_pays<T>(R, C, F), false, false, plan_of<T>(R, 2ll * F, C, false)};          // (a tile's columns are half gate, half up)
    if (!c.few && C % tiles::piece<T>()) {
        c.lie = (sizeof(T) == 2 ? 0.3 : 0.04) * c.plan.cost < 3 + ((double)R + 2. * F) * C * 2 * sizeof(T) / 5e6;
        c.copy = !c.lie;
    }
    return c;
}
template <class T> static size_t forward_scratch(int R, int C, int F) {
    return choose<T>(R, C, F).copy ? ((size_t)R + 2 * (size_t)F) * rounded(C) * sizeof(T) : 0;
}
template <class T> static hipError_t forward_t(hipStream_t s, Forward k, void *scratch) {
    const Choice c = choose<T>(k.R, k.K, k.F);
    if (c.few) {
        const bool whole = k.K % tiles::piece<T>() == 0;
        const dim3 grid(tiles_of(k.F, 16));
        const int groups = tiles_of(k.R, 16);
#define WKV_FEW(G)                                                                                             \
    do {                                                                                                       \
        if (whole) hipLaunchKernelGGL((few<T, G, true>), grid, dim3(64 * FEW_WAVES), 0, s, k);                 \
        else hipLaunchKernelGGL((few<T, G, false>), grid, dim3(64 * FEW_WAVES), 0, s, k);                      \
    } while (0)
        if (groups == 1) WKV_FEW(1);
        else if (groups == 2) WKV_FEW(2);
        else WKV_FEW(4);
#undef WKV_FEW
        return hipGetLastError();
    }
    if (c.copy) {
        Layout l(k.K);
        const int Cs = l.k.Cs;
        T *to = static_cast<T *>(scratch);
        const T *x = static_cast<const T *>(k.x), *wg = static_cast<const T *>(k.wg), *wu = static_cast<const T *>(k.wu);
        l.add(x, k.xs, k.R, to);
        l.add(wg, k.ws, k.F, to + (size_t)k.R * Cs);
        l.add(wu, k.ws, k.F, to + (size_t)(k.R + k.F) * Cs);
        l.launch<T>(s);
        k.x = x; k.wg = wg; k.wu = wu;
        k.xs = k.ws = k.K = Cs;
    }
    const Plan &p = c.plan;
    const int width = width_of<T>(p, k.F), columns = tiles_of(k.F, width);
    const dim3 grid(p.rows * columns);
#define WKV_FORWARD(BM, BN, WN, AHEAD, WAVES)                                                                                                    \
    do {                                                                                                                                         \
        if (c.lie) hipLaunchKernelGGL((forward<T, BM, BN, 2, WN, AHEAD, true>), grid, dim3(64 * WAVES), 0, s, k, p.rows, columns, width);         \
        else hipLaunchKernelGGL((forward<T, BM, BN, 2, WN, AHEAD, false>), grid, dim3(64 * WAVES), 0, s, k, p.rows, columns, width);              \
    } while (0)
    if (p.size == 256) WKV_FORWARD(256, 256, 4, 2, 8);
    else if (p.size == 128) WKV_FORWARD(128, 128, 2, 2, 4);
    else if (width > 32) {
        if constexpr (sizeof(T) == 2) WKV_FORWARD(64, 128, 2, DEEP, 4);
    } else if (deep_pays(p.rows * columns)) WKV_FORWARD(64, 64, 2, DEEP, 4);
    else WKV_FORWARD(64, 64, 2, 2, 4);
#undef WKV_FORWARD
    return hipGetLastError();
}

struct Backward {
    int R, C, F, kind;
    const void *x, *wg, *wu, *gh;
    const float *kept;
    long long xs, ws;
    void *gx, *gwg, *gwu;             // gx, or gwg and gwu, may be NULL: not wanted
};
// Whether the slopes go into the products in two parts, rounded and what that leaves.  With few rows nothing averages their rounding (2 or 3 rows in bf16: results up to half as far again
// off the 64-bit ones as their own rounding makes them; in two parts that alone is left), and while the parts' rows fill no more than a tile the weights, which bound such calls, pay
// for them ((16, 2560) into 8960 columns gx 31.5 -> 34.4 us, weights' gradients 36.2 -> 36.8; (64, 2560) would be 41 -> 50, 38 -> 42).
constexpr int PAIRED = 32;
template <class T> constexpr bool in_pairs(int R) { return sizeof(T) == 2 && R <= PAIRED; }
struct Regions { size_t d, x, wg, wu, most, exponent, parts, all; };
template <class T> static Regions regions(int R, int C, int F, bool want_x, bool want_w) {
    const size_t Fs = rounded(F), Cs = C % tiles::piece<T>() ? rounded(C) : 0;
    Regions r;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t was = at; at += (n + 255) / 256 * 256; return was; };
    const int pairs = in_pairs<T>(R) ? 2 : 1;
    r.d = take((size_t)pairs * R * 2 * Fs * sizeof(T));
    r.x = take(want_w ? (size_t)R * Cs * sizeof(T) : 0);
    r.wg = take(want_x ? (size_t)F * Cs * sizeof(T) : 0);
    r.wu = take(want_x ? (size_t)F * Cs * sizeof(T) : 0);
    r.most = take(scaled<T>() ? LARGEST * 4 : 0);
    r.exponent = take(scaled<T>() ? 4 : 0);
    size_t parts = 0;
    if (want_x) {
        const Plan p = plan_of<T>(pairs * R, C, 2 * Fs, true);
        if (p.shares > 1) parts = std::max(parts, (size_t)p.shares * R * C * 4);
    }
    if (want_w) {
        const Plan p = plan_of<T>(2 * Fs, C, rounded(pairs * R), true);
        if (p.shares > 1) parts = std::max(parts, (size_t)p.shares * 2 * Fs * C * 4);
    }
    r.parts = take(parts);
    r.all = at;
    return r;
}
template <class T, bool ACROSS_A> static void product_launch(hipStream_t s, Product k, const Plan &p) {
    k.per = p.per;
    if (p.shares == 1) k.parts = nullptr;
    const dim3 grid(p.rows * p.columns, p.shares);
    if (p.size == 256) hipLaunchKernelGGL((product<T, 256, 256, 2, 4, 2, ACROSS_A>), grid, dim3(512), 0, s, k, p.rows, p.columns);
    else if (p.size == 128) hipLaunchKernelGGL((product<T, 128, 128, 2, 2, 2, ACROSS_A>), grid, dim3(256), 0, s, k, p.rows, p.columns);
    else if (deep_pays((long long)p.rows * p.columns * p.shares)) hipLaunchKernelGGL((product<T, 64, 64, 2, 2, DEEP, ACROSS_A>), grid, dim3(256), 0, s, k, p.rows, p.columns);
    else hipLaunchKernelGGL((product<T, 64, 64, 2, 2, 2, ACROSS_A>), grid, dim3(256), 0, s, k, p.rows, p.columns);
    const int M = !ACROSS_A && k.pairs ? k.M / 2 : k.M;
    if (p.shares > 1) hipLaunchKernelGGL(join<T>, dim3((unsigned)(((size_t)M * k.os + 255) / 256)), dim3(256), 0, s, k, M, p.shares);
}
template <class T> static hipError_t backward_t(hipStream_t s, const Backward &k, void *scratch) {
    const int Fs = (int)rounded(k.F), R2 = in_pairs<T>(k.R) ? 2 * k.R : k.R;
    const bool pairs = R2 != k.R;
    const bool want_x = k.gx, want_w = k.gwg;
    const Regions r = regions<T>(k.R, k.C, k.F, want_x, want_w);
    char *ws = static_cast<char *>(scratch);
    T *d = reinterpret_cast<T *>(ws + r.d);
    const T *x = static_cast<const T *>(k.x), *wg = static_cast<const T *>(k.wg), *wu = static_cast<const T *>(k.wu);
    long long xs = k.xs, ld = k.ws;
    if (k.C % tiles::piece<T>()) {
        Layout l(k.C);
        if (want_w) l.add(x, xs, k.R, ws + r.x);
        if (want_x) {
            l.add(wg, ld, k.F, ws + r.wg);
            l.add(wu, ld, k.F, ws + r.wu);
        }
        l.launch<T>(s);
        xs = ld = rounded(k.C);
    }
    float *parts = reinterpret_cast<float *>(ws + r.parts);
    const dim3 grid(tiles_of(Fs, 1024), std::min(k.R, 32768));
    float *most = reinterpret_cast<float *>(ws + r.most);
    int *exponent = reinterpret_cast<int *>(ws + r.exponent);
    const T *gh = static_cast<const T *>(k.gh);
    auto both = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
        if constexpr (scaled<T>()) hipLaunchKernelGGL((largest<T, WHOLE>), dim3(LARGEST), dim3(1024), 0, s, k.R, k.F, k.kind, k.kept, gh, Fs, most);
        hipLaunchKernelGGL((slopes<T, WHOLE>), grid, dim3(256), 0, s, k.R, k.F, k.kind, k.kept, gh, d, Fs, pairs, most, exponent);
    };
    if (k.F % 4 == 0) both(std::true_type());
    else both(std::false_type());
    if (want_x) {
        Product p = {};
        p.M = R2; p.N = k.C; p.K = 2 * Fs; p.pairs = pairs; p.exponent = exponent;
        p.a = d; p.as = 2 * Fs;
        p.b = wg; p.b2 = wu; p.bs = ld; p.turn = Fs; p.b_rows = k.F;
        p.out0 = p.out1 = k.gx; p.os = k.C; p.split = p.live = k.R;
        p.parts = parts;
        product_launch<T, false>(s, p, plan_of<T>(p.M, p.N, p.K, true));
    }
    if (want_w) {
        Product p = {};
        p.M = 2 * Fs; p.N = k.C; p.K = (int)rounded(R2); p.pairs = pairs; p.exponent = exponent;
        p.a = d; p.as = 2 * Fs;
        p.b = p.b2 = x; p.bs = xs; p.turn = 0x7fffffff; p.a_rows = R2; p.b_rows = k.R;
        p.out0 = k.gwg; p.out1 = k.gwu; p.os = k.C; p.split = Fs; p.live = k.F;
        p.parts = parts;
        product_launch<T, true>(s, p, plan_of<T>(p.M, p.N, p.K, true));
    }
    return hipGetLastError();
}

}  // namespace ffn
}  // namespace wkv
