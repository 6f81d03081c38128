// The first half of a gated feed-forward block,  h = act(x Wg') * (x Wu')  with x (R, C) and both weights (F, C), and its backward:
//
//     g = x Wg',  u = x Wu',  h = act(g) u
//     dg = gh u act'(g),  du = gh act(g),  gx = dg Wg + du Wu,  gWg = dg' x,  gWu = du' x
//
// R C F 4 operations forward and 8 backward, on the matrix cores (matrix_tiles.h).  Forward, a workgroup's tile of B is half of gate rows and
// half of the same up rows, so that a lane ends with g and u of the same places and the activation and product happen in registers: g and u
// never reach memory, except that a backward's are kept in fp32: rounded to 16 bits they would add as much to the gradients' error as each of the two
// roundings that cannot be left out, that of dg and du, which the matrix cores take in the streams' type, and that of the results (bf16, error of
// the 2-norm: 3.1e-3 against 2.4e-3).  Backward, one pass makes dg and du, as rows and as columns; x and the weights are laid out with their
// other index along memory, and then the three products are the same loop.
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

// ---- forward
struct Forward {
    int R, K, F, kind;
    const void *x, *wg, *wu;
    long long xs, ws;                 // row strides
    void *h;
    float *kept;                      // (R, 2 Fs), g and u side by side, or NULL
    long long hs, Fs;
};

template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void forward(const Forward k, int rows, int columns) {
    typedef tiles::Loop<T, BM, BN, WM, WN, 2> L;
    __shared__ __align__(1024) char lds[L::LDS];
    int tm, tn;
    tiles::tile_of(blockIdx.x, rows, columns, tm, tn);
    const int m0 = tm * BM, n0 = tn * (BN / 2);
    L l;
    l.a.place(static_cast<const T *>(k.x) + m0 * k.xs, k.xs, k.K, min(BM, k.R - m0));
    l.b[0].place(static_cast<const T *>(k.wg) + n0 * k.ws, k.ws, k.K, min(BN / 2, k.F - n0));
    l.b[1].place(static_cast<const T *>(k.wu) + n0 * k.ws, k.ws, k.K, min(BN / 2, k.F - n0));
    l.run(0, k.K, k.K, lds);
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
            put4(h + m * k.hs, n, k.F, whole, o);
            if (k.kept) {
                put4(k.kept + m * (2 * k.Fs), n, k.F, true, g);
                put4(k.kept + m * (2 * k.Fs) + k.Fs, n, k.F, true, u);
            }
        }
    }
}

// ---- a product of two operands with k along memory
struct Product {
    int M, N, K;
    const void *a, *b;
    long long as, bs;
    // out: rows below `split` (of which `live` are there) to out0, those from it on to out1; parts: fp32 sums over a share of k instead
    void *out0, *out1;
    long long os;
    int split, live;
    float *parts;
    int per;                          // of k to a share
};

template <class T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product(const Product k, int rows, int columns) {
    typedef tiles::Loop<T, BM, BN, WM, WN, 1> L;
    __shared__ __align__(1024) char lds[L::LDS];
    int tm, tn;
    tiles::tile_of(blockIdx.x, rows, columns, tm, tn);
    const int m0 = tm * BM, n0 = tn * BN;
    L l;
    l.a.place(static_cast<const T *>(k.a) + m0 * k.as, k.as, k.K, min(BM, k.M - m0));
    l.b[0].place(static_cast<const T *>(k.b) + n0 * k.bs, k.bs, k.K, min(BN, k.N - n0));
    const int k0 = blockIdx.y * k.per;
    l.run(k0, min(k0 + k.per, k.K), k.K, lds);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    const bool whole = k.os % 4 == 0;
#pragma unroll
    for (int i = 0; i < L::MT; i++) {
        const int m = m0 + (wm * L::MT + i) * 16 + (lane & 15);
        const int r = m < k.split ? m : m - k.split;
        if (m >= k.M || r >= k.live) continue;
#pragma unroll
        for (int j = 0; j < L::NT; j++) {
            const int n = n0 + (wn * L::NT + j) * 16 + 4 * (lane >> 4);
            float o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = l.acc[i][j][e];
            if (k.parts) put4(k.parts + ((size_t)blockIdx.y * k.M + m) * k.os, n, k.N, whole, o);
            else put4(static_cast<T *>(m < k.split ? k.out0 : k.out1) + r * k.os, n, k.N, whole, o);
        }
    }
}
// the shares' sums, in their order
template <class T> __global__ __launch_bounds__(256) void join(const Product k, int shares) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x, n = (size_t)k.M * k.os;
    if (i >= n) return;
    float s = k.parts[i];
    for (int p = 1; p < shares; p++) s += k.parts[p * n + i];
    const int m = (int)(i / k.os), r = m < k.split ? m : m - k.split;
    if (r < k.live) static_cast<T *>(m < k.split ? k.out0 : k.out1)[r * k.os + i % k.os] = from_float<T>(s);
}

// ---- layouts
// rows of C elements -> rows of Cs, zeros behind
template <class T> __global__ __launch_bounds__(256) void widen(const T *in, long long stride, int R, int C, T *out, int Cs) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    const size_t r = i / Cs, c = i % Cs;
    if (r < (size_t)R) out[i] = (int)c < C ? in[r * stride + c] : from_float<T>(0.f);
}
// (R, C) -> (C, ld): out[c][r], zeros where r is past R; ld: R in whole tiles.  64 x 64 at a time through LDS
template <class T> __global__ __launch_bounds__(256) void turn(const T *in, long long stride, int R, int C, T *out, long long ld) {
    __shared__ T tile[64][66];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int r = wave * 16 + i;
        tile[r][lane] = r0 + r < R && c0 + lane < C ? in[(r0 + r) * stride + c0 + lane] : from_float<T>(0.f);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int c = wave * 16 + i;
        if (c0 + c < C) out[(c0 + c) * ld + r0 + lane] = tile[lane][c];
    }
}
// dg and du from g, u and gh: rows (R, 2 Fs) and columns (2 Fs, Rs), zeros outside
template <class T> __global__ __launch_bounds__(256) void slopes(int R, int F, int kind, const float *kept, const T *gh, T *d, T *turned, long long Fs, long long Rs) {
    __shared__ T tile[2][64][66];
    const int r0 = blockIdx.x * 64, c0 = blockIdx.y * 64, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, f = c0 + lane;
#pragma unroll 4
    for (int i = 0; i < 16; i++) {
        const int r = r0 + wave * 16 + i;
        float dg = 0.f, du = 0.f;
        if (r < R) {
            if (f < F) {
                const float g = kept[r * 2 * Fs + f], u = kept[r * 2 * Fs + Fs + f], o = to_float(gh[(long long)r * F + f]);
                float value, slope;
                activation(kind, g, value, slope);
                dg = o * u * slope;
                du = o * value;
            }
            d[r * 2 * Fs + f] = from_float<T>(dg);
            d[r * 2 * Fs + Fs + f] = from_float<T>(du);
        }
        tile[0][wave * 16 + i][lane] = from_float<T>(dg);
        tile[1][wave * 16 + i][lane] = from_float<T>(du);
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll 4
        for (int i = 0; i < 16; i++) {
            const int c = wave * 16 + i;
            turned[(p * Fs + c0 + c) * Rs + r0 + lane] = tile[p][lane][c];
        }
}

// ---- few rows: a serving loop's single tokens.  What they cost is the weights, read once: a workgroup takes 16 gate rows and the same 16 up rows,
// its four wavefronts every fourth tile of k; operands go straight from memory to registers.
constexpr int FEW = 64, FEW_WAVES = 4;
template <class T, int GROUPS, bool WHOLE>                    // GROUPS of 16 rows of x; WHOLE: rows are whole pieces of 16 bytes
__global__ __launch_bounds__(64 * FEW_WAVES) void few(const Forward k) {
    constexpr int E = tiles::piece<T>(), D = tiles::depth<T>(), AHEAD = !WHOLE ? 1 : GROUPS == 1 ? 4 : 2;
    __shared__ f4 part[FEW_WAVES][GROUPS][2][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n0 = blockIdx.x * 16, in = lane & 15;
    const int f = min(n0 + in, k.F - 1);
    const T *wg = static_cast<const T *>(k.wg) + f * k.ws, *wu = static_cast<const T *>(k.wu) + f * k.ws, *x[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; i++) x[i] = static_cast<const T *>(k.x) + min(i * 16 + in, k.R - 1) * k.xs;
    f4 g[GROUPS], u[GROUPS];
#pragma unroll
    for (int i = 0; i < GROUPS; i++) g[i] = u[i] = f4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const T *p, int at) -> i4 {
        if constexpr (WHOLE) {
            const i4 v = *reinterpret_cast<const i4 *>(p + (at < k.K ? at : 0));
            return at < k.K ? v : i4{0, 0, 0, 0};
        } else {
            T e[E];
#pragma unroll
            for (int q = 0; q < E; q++) e[q] = at + q < k.K ? p[at + q] : from_float<T>(0.f);
            i4 v;
            __builtin_memcpy(&v, e, 16);
            return v;
        }
    };
    for (int t = wave * D; t < k.K; t += FEW_WAVES * D * AHEAD) {
        i4 a[AHEAD][2], b[AHEAD][2], y[AHEAD][2][GROUPS];
#pragma unroll
        for (int q = 0; q < AHEAD; q++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const int at = t + q * FEW_WAVES * D + ((lane >> 4) + 4 * s) * E;
                a[q][s] = load(wg, at);
                b[q][s] = load(wu, at);
#pragma unroll
                for (int i = 0; i < GROUPS; i++) y[q][s][i] = load(x[i], at);
            }
#pragma unroll
        for (int q = 0; q < AHEAD; q++)
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
                for (int i = 0; i < GROUPS; i++) {
                    g[i] = tiles::mma<T>(a[q][s], y[q][s][i], g[i]);
                    u[i] = tiles::mma<T>(b[q][s], y[q][s][i], u[i]);
                }
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
static inline int tiles_of(long long n, int size) { return (int)((n + size - 1) / size); }
template <class T> static size_t forward_scratch(int R, int C, int F) {
    if (C % tiles::piece<T>() == 0 || R <= FEW) return 0;
    return ((size_t)R + 2 * (size_t)F) * rounded(C) * sizeof(T);
}
template <class T> static hipError_t forward_t(hipStream_t s, Forward k, void *scratch) {
    const bool whole = k.K % tiles::piece<T>() == 0;
    if (k.R <= FEW) {
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
    if (!whole) {
        const int Cs = (int)rounded(k.K);
        T *to = static_cast<T *>(scratch);
        auto lay = [&](const void *&p, long long stride, int rows) {
            hipLaunchKernelGGL(widen<T>, dim3((unsigned)(((size_t)rows * Cs + 255) / 256)), dim3(256), 0, s, static_cast<const T *>(p), stride, rows, k.K, to, Cs);
            p = to;
            to += (size_t)rows * Cs;
        };
        lay(k.x, k.xs, k.R);
        lay(k.wg, k.ws, k.F);
        lay(k.wu, k.ws, k.F);
        k.xs = k.ws = k.K = Cs;
    }
    const int big = tiles_of(k.R, 256) * tiles_of(k.F, 128);
    if (big >= cu_count()) {
        const int rows = tiles_of(k.R, 256), columns = tiles_of(k.F, 128);
        hipLaunchKernelGGL((forward<T, 256, 256, 2, 4>), dim3(rows * columns), dim3(512), 0, s, k, rows, columns);
    } else {
        const int rows = tiles_of(k.R, 128), columns = tiles_of(k.F, 64);
        hipLaunchKernelGGL((forward<T, 128, 128, 2, 2>), dim3(rows * columns), dim3(256), 0, s, k, rows, columns);
    }
    return hipGetLastError();
}

struct Backward {
    int R, C, F, kind;
    const void *x, *wg, *wu, *gh;
    const float *kept;
    long long xs, ws;
    void *gx, *gwg, *gwu;             // gx, or gwg and gwu, may be NULL: not wanted
};
// How a product is shared out: tiles of 256 or 128, and k cut where the tiles do not fill the compute units
struct Plan { int size, rows, columns, shares, per; };
template <class T> static Plan plan_of(long long M, long long N, long long K) {
    Plan p;
    const int cus = cu_count();
    p.size = (long long)tiles_of(M, 256) * tiles_of(N, 256) >= cus * 3 / 4 ? 256 : 128;
    p.rows = tiles_of(M, p.size);
    p.columns = tiles_of(N, p.size);
    const long long steps = (K + tiles::depth<T>() - 1) / tiles::depth<T>();
    long long shares = 1;
    while (p.size == 128 && (long long)p.rows * p.columns * shares * 2 <= 2 * cus && steps >= 16 * shares) shares *= 2;
    const long long each = (steps + shares - 1) / shares;
    p.shares = (int)((steps + each - 1) / each);
    p.per = (int)(each * tiles::depth<T>());
    return p;
}
struct Regions { size_t d, turned, x, w, parts, all; };
template <class T> static Regions regions(int R, int C, int F, bool want_x, bool want_w) {
    const size_t Fs = rounded(F), Rs = rounded(R);
    Regions r;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t was = at; at += (n + 255) / 256 * 256; return was; };
    r.d = take((size_t)R * 2 * Fs * sizeof(T));
    r.turned = take(2 * Fs * Rs * sizeof(T));
    r.x = take(want_w ? (size_t)C * Rs * sizeof(T) : 0);
    r.w = take(want_x ? (size_t)C * 2 * Fs * sizeof(T) : 0);
    size_t parts = 0;
    if (want_x) {
        const Plan p = plan_of<T>(R, C, 2 * Fs);
        if (p.shares > 1) parts = std::max(parts, (size_t)p.shares * R * C * 4);
    }
    if (want_w) {
        const Plan p = plan_of<T>(2 * Fs, C, Rs);
        if (p.shares > 1) parts = std::max(parts, (size_t)p.shares * 2 * Fs * C * 4);
    }
    r.parts = take(parts);
    r.all = at;
    return r;
}
template <class T> static void product_launch(hipStream_t s, Product k, const Plan &p) {
    k.per = p.per;
    if (p.shares == 1) k.parts = nullptr;
    const dim3 grid(p.rows * p.columns, p.shares);
    if (p.size == 256) hipLaunchKernelGGL((product<T, 256, 256, 2, 4>), grid, dim3(512), 0, s, k, p.rows, p.columns);
    else hipLaunchKernelGGL((product<T, 128, 128, 2, 2>), grid, dim3(256), 0, s, k, p.rows, p.columns);
    if (p.shares > 1) hipLaunchKernelGGL(join<T>, dim3((unsigned)(((size_t)k.M * k.os + 255) / 256)), dim3(256), 0, s, k, p.shares);
}
template <class T> static hipError_t backward_t(hipStream_t s, const Backward &k, void *scratch) {
    const long long Fs = rounded(k.F), Rs = rounded(k.R);
    const bool want_x = k.gx, want_w = k.gwg;
    const Regions r = regions<T>(k.R, k.C, k.F, want_x, want_w);
    char *ws = static_cast<char *>(scratch);
    T *d = reinterpret_cast<T *>(ws + r.d), *turned = reinterpret_cast<T *>(ws + r.turned), *xt = reinterpret_cast<T *>(ws + r.x), *wt = reinterpret_cast<T *>(ws + r.w);
    float *parts = reinterpret_cast<float *>(ws + r.parts);
    const dim3 wide(256);
    hipLaunchKernelGGL(slopes<T>, dim3((unsigned)(Rs / 64), (unsigned)(Fs / 64)), wide, 0, s, k.R, k.F, k.kind, k.kept, static_cast<const T *>(k.gh), d, turned, Fs, Rs);
    if (want_x) {
        const dim3 grid((unsigned)(Fs / 64), tiles_of(k.C, 64));
        hipLaunchKernelGGL(turn<T>, grid, wide, 0, s, static_cast<const T *>(k.wg), k.ws, k.F, k.C, wt, 2 * Fs);
        hipLaunchKernelGGL(turn<T>, grid, wide, 0, s, static_cast<const T *>(k.wu), k.ws, k.F, k.C, wt + Fs, 2 * Fs);
        const Product p = {k.R, k.C, (int)(2 * Fs), d, wt, 2 * Fs, 2 * Fs, k.gx, k.gx, k.C, k.R, k.R, parts, 0};
        product_launch<T>(s, p, plan_of<T>(k.R, k.C, 2 * Fs));
    }
    if (want_w) {
        hipLaunchKernelGGL(turn<T>, dim3((unsigned)(Rs / 64), tiles_of(k.C, 64)), wide, 0, s, static_cast<const T *>(k.x), k.xs, k.R, k.C, xt, Rs);
        const Product p = {(int)(2 * Fs), k.C, (int)Rs, turned, xt, Rs, Rs, k.gwg, k.gwu, k.C, (int)Fs, k.F, parts, 0};
        product_launch<T>(s, p, plan_of<T>(2 * Fs, k.C, Rs));
    }
    return hipGetLastError();
}

}  // namespace ffn
}  // namespace wkv
