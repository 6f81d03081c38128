// One token per row of logits, from a random number u per row:
//
//     s[i] = (max - l[i]) log2(e) / temperature         w[i] = 2^-s[i], in whole 2^-31ths
//
// Tokens stand in the order of s, ties by index.  Kept are the first top_k of them, of those the ones with w >= min_p, of
// those the shortest beginning with a share top_p of their weight; drawn is the first token, by index, at which the sum of the kept
// weights passes u times their total.  Temperature below 1e-6: the likeliest token.  NaN counts as -infinity; a row with nothing but
// -infinity has no token (-1).
//
// The weights are whole numbers so that every sum is exact: no order of adding, no split over lanes changes a token.
//
// A workgroup of 16 wavefronts holds a row's s in registers (65536 elements; wider rows are read again for every pass) and
// never sorts: the two cuts are found from counts and weights in 1024 bins of s, then in 1024 bins of the bin with the cut, then, between the
// elements left there (for 16-bit logits mostly one value), by bisection of the value's bits.
#include "common.h"

namespace wkv {
namespace sampling {

constexpr int THREADS = 1024, WAVES = THREADS / 64, PIECE = 8, CHUNK = THREADS * PIECE;
constexpr int BINS = 1024;
constexpr float MOST = 32.f, PER_OCTAVE = 32.f;      // weights vanish at s = 32, in bin BINS; a power of two: products with it are exact
constexpr int MAX_VOCABULARY = 1 << 20;        // totals stay below 2^53: exact in fp64
constexpr int MAX_CHUNKS = MAX_VOCABULARY / CHUNK + 1;
typedef unsigned long long u64;
constexpr double ONE = 2147483648.0;

struct Call {
    int rows, V;
    long long stride;
    const void *logits;
    const float *u, *temperature, *top_p, *min_p;      // per row, or NULL and the value below
    const int *top_k;
    float temperature_value, top_p_value, min_p_value;
    int top_k_value;
    long long *token;
    float *logprob;
};

__device__ __forceinline__ u64 shfl_up(u64 v, int d) {
    const unsigned lo = __shfl_up((unsigned)v, d), hi = __shfl_up((unsigned)(v >> 32), d);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 up_to(u64 v) {          // inclusive sum over the wavefront's lanes
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = shfl_up(v, d);
        if (lane >= d) v += o;
    }
    return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    return (u64)__builtin_amdgcn_readlane((unsigned)(v >> 32), 63) << 32 | (unsigned)__builtin_amdgcn_readlane((unsigned)v, 63);
}

// N chunks of a row in registers, as s; N = 0: read again for every pass
template <class T, int N> struct Row {
    const T *p;
    int V, head, chunks;           // head: the row's first element's place in its aligned 16 bytes' (two of them for fp32) piece
    float top, scale;
    float s[N ? N : 1][PIECE];

    __device__ __forceinline__ Row(const Call &k) {
        p = static_cast<const T *>(k.logits) + blockIdx.x * k.stride;
        V = k.V;
        head = (int)((reinterpret_cast<uintptr_t>(p) / sizeof(T)) % PIECE);
        chunks = (V + head + CHUNK - 1) / CHUNK;
    }
    __device__ __forceinline__ int first(int c) const { return c * CHUNK + (int)threadIdx.x * PIECE - head; }      // index of a piece's first element
    __device__ __forceinline__ void raw(int c, float (&o)[PIECE]) const {
        const int at = first(c);
        if (at >= 0 && at + PIECE <= V) {
            T e[PIECE];
            if constexpr (sizeof(T) == 2) {
                const uint4 q = *reinterpret_cast<const uint4 *>(p + at);
                __builtin_memcpy(e, &q, 16);
            } else {
                const float4 q = *reinterpret_cast<const float4 *>(p + at), r = *reinterpret_cast<const float4 *>(p + at + 4);
                __builtin_memcpy(e, &q, 16);
                __builtin_memcpy(e + 4, &r, 16);
            }
#pragma unroll
            for (int i = 0; i < PIECE; i++) o[i] = to_float(e[i]);
        } else {
#pragma unroll
            for (int i = 0; i < PIECE; i++) o[i] = at + i >= 0 && at + i < V ? to_float(p[at + i]) : -INFINITY;
        }
#pragma unroll
        for (int i = 0; i < PIECE; i++) o[i] = o[i] != o[i] ? -INFINITY : o[i];
    }
    __device__ __forceinline__ void place(float (&o)[PIECE]) const {
#pragma unroll
        for (int i = 0; i < PIECE; i++) o[i] = o[i] == -INFINITY ? INFINITY : o[i] == top ? 0.f : (top - o[i]) * scale;
    }
    // f(chunk, its piece's s)
    template <class F> __device__ __forceinline__ void each(F f) {
        if constexpr (N > 0) {
#pragma unroll
            for (int c = 0; c < N; c++) f(c, s[c]);
        } else {
            for (int c = 0; c < chunks; c++) {
                raw(c, s[0]);
                place(s[0]);
                f(c, s[0]);
            }
        }
    }
};

__device__ __forceinline__ unsigned weight(float s) { return (unsigned)rintf(exp2_fast(-s) * (float)ONE); }

struct Shared {
    u64 bin_weight[2][BINS];
    unsigned bin_count[2][BINS];
    u64 sums[WAVES * MAX_CHUNKS];          // by chunk and wavefront
    unsigned ties[WAVES * MAX_CHUNKS];
    u64 red[2][WAVES];
    float redf[2][WAVES];
    // what a scan found
    int bin;
    u64 before;
};

// sum over the workgroup; `turn` alternates between two barriers
__device__ __forceinline__ u64 over_all(u64 v, Shared &sh, int &turn) {
    v = last_lane(up_to(v));
    if ((threadIdx.x & 63) == 0) sh.red[turn][threadIdx.x >> 6] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int i = 0; i < WAVES; i++) s += sh.red[turn][i];
    turn ^= 1;
    return s;
}

// The first bin at which the sum of `in` reaches `need` (1 <= need <= the sum of all), and the sum before it
template <class E> __device__ __forceinline__ void find_bin(const E *in, u64 need, Shared &sh, int &bin, u64 &before) {
    if (threadIdx.x < 64) {
        constexpr int EACH = BINS / 64;
        u64 own = 0;
        for (int i = 0; i < EACH; i++) own += in[threadIdx.x * EACH + i];
        const u64 upto = up_to(own);
        if (upto >= need && upto - own < need) {
            u64 s = upto - own;
            int i = threadIdx.x * EACH;
            while (s + in[i] < need) s += in[i++];
            sh.bin = i;
            sh.before = s;
        }
    }
    __syncthreads();
    bin = sh.bin;
    before = sh.before;
    __syncthreads();
}

struct Cut {
    unsigned key;          // kept: the values below, and the first `ties` of those equal
    u64 ties;
    u64 before;            // what the values below come to
    u64 here;              // what all the equal ones do
};

// Where the first `need` (of tokens, or of weight) in the order of s end; the first level's bins are filled.
// limit: tokens of larger s do not count
template <bool WEIGHT, class R>
__device__ __forceinline__ Cut find_cut(R &row, u64 need, float limit, Shared &sh, int &turn) {
    int b1, b2;
    u64 before, inner;
    if (WEIGHT) find_bin(sh.bin_weight[0], need, sh, b1, before);
    else find_bin(sh.bin_count[0], need, sh, b1, before);
    for (int i = threadIdx.x; i < BINS; i += THREADS) {
        sh.bin_weight[1][i] = 0;
        sh.bin_count[1][i] = 0;
    }
    __syncthreads();
    const float base = (float)b1;
    row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
        for (int i = 0; i < PIECE; i++) {
            const float x = s[i] * PER_OCTAVE - base;
            if (x >= 0.f && x < 1.f && s[i] <= limit) {
                const int b = (int)(x * BINS);
                if (WEIGHT) atomicAdd(&sh.bin_weight[1][b], (u64)weight(s[i]));
                else atomicAdd(&sh.bin_count[1][b], 1u);
            }
        }
    });
    __syncthreads();
    if (WEIGHT) find_bin(sh.bin_weight[1], need - before, sh, b2, inner);
    else find_bin(sh.bin_count[1], need - before, sh, b2, inner);
    before += inner;
    // the values left: those with x in [b2, b2 + 1) / BINS; their smallest and largest bits
    auto inside = [&](float s) {
        const float x = s * PER_OCTAVE - base;
        return x >= 0.f && x < 1.f && s <= limit && (int)(x * BINS) == b2;
    };
    unsigned lo = 0xffffffffu, hi = 0;
    row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
        for (int i = 0; i < PIECE; i++)
            if (inside(s[i])) {
                lo = min(lo, __float_as_uint(s[i]));
                hi = max(hi, __float_as_uint(s[i]));
            }
    });
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        lo = min(lo, (unsigned)__shfl_xor((int)lo, m));
        hi = max(hi, (unsigned)__shfl_xor((int)hi, m));
    }
    if ((threadIdx.x & 63) == 0) sh.red[turn][threadIdx.x >> 6] = (u64)hi << 32 | lo;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        const u64 r = sh.red[turn][i];
        lo = min(lo, (unsigned)r);
        hi = max(hi, (unsigned)(r >> 32));
    }
    turn ^= 1;
    // the smallest value up to which there is enough
    auto upto = [&](unsigned key) {
        u64 n = 0;
        row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
            for (int i = 0; i < PIECE; i++)
                if (__float_as_uint(s[i]) <= key && inside(s[i])) n += WEIGHT ? weight(s[i]) : 1;
        });
        return over_all(n, sh, turn);
    };
    while (lo < hi) {
        const unsigned mid = lo + ((hi - lo) >> 1);
        if (before + upto(mid) >= need) hi = mid;
        else lo = mid + 1;
    }
    Cut cut;
    cut.key = lo;
    u64 below = 0, equal = 0;
    row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
        for (int i = 0; i < PIECE; i++)
            if (inside(s[i])) {
                if (__float_as_uint(s[i]) < lo) below += WEIGHT ? weight(s[i]) : 1;
                if (__float_as_uint(s[i]) == lo) equal += 1;
            }
    });
    cut.before = before + over_all(below, sh, turn);
    cut.here = over_all(equal, sh, turn);
    const u64 left = need - cut.before, each = WEIGHT ? max(weight(__uint_as_float(lo)), 1u) : 1u;
    cut.ties = (left + each - 1) / each;
    return cut;
}

template <class T, int N>
__global__ __launch_bounds__(THREADS) void sample(const Call k) {
    __shared__ Shared sh;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const size_t r = blockIdx.x;
    Row<T, N> row(k);
    const float temperature = k.temperature ? k.temperature[r] : k.temperature_value;
    const float top_p = k.top_p ? k.top_p[r] : k.top_p_value, min_p = k.min_p ? k.min_p[r] : k.min_p_value;
    const bool warm = temperature >= 1e-6f;
    const int top_k = !warm ? 1 : k.top_k ? k.top_k[r] : k.top_k_value;
    // the largest logit
    float top = -INFINITY;
    if constexpr (N > 0) {
#pragma unroll
        for (int c = 0; c < N; c++) {
            row.raw(c, row.s[c]);
#pragma unroll
            for (int i = 0; i < PIECE; i++) top = fmaxf(top, row.s[c][i]);
        }
    } else {
        for (int c = 0; c < row.chunks; c++) {
            row.raw(c, row.s[0]);
#pragma unroll
            for (int i = 0; i < PIECE; i++) top = fmaxf(top, row.s[0][i]);
        }
    }
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
    if (lane == 0) sh.redf[0][wave] = top;
    for (int i = tid; i < BINS; i += THREADS) {
        sh.bin_weight[0][i] = 0;
        sh.bin_count[0][i] = 0;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) top = fmaxf(top, sh.redf[0][i]);
    if (top == -INFINITY) {
        if (tid == 0) {
            k.token[r] = -1;
            k.logprob[r] = -INFINITY;
        }
        return;
    }
    row.top = top;
    row.scale = LOG2E / (warm ? temperature : 1.f);
    if constexpr (N > 0) {
#pragma unroll
        for (int c = 0; c < N; c++) row.place(row.s[c]);
    }
    // counts and weights in bins of s; a token lighter than `least` does not count
    const double share = (double)min_p * ONE;
    const unsigned least = share > 1.0 ? share < ONE ? (unsigned)ceil(share) : (unsigned)ONE : 1u;
    int turn = 0;
    u64 own = 0, count = 0;
    float limit = 0.f;          // the largest s that counts (weights fall with s)
    row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
        for (int i = 0; i < PIECE; i++)
            if (s[i] < MOST) {
                const unsigned w = weight(s[i]);
                if (w >= least) {
                    const int b = (int)(s[i] * PER_OCTAVE);
                    atomicAdd(&sh.bin_weight[0][b], (u64)w);
                    atomicAdd(&sh.bin_count[0][b], 1u);
                    own += w;
                    count++;
                    limit = fmaxf(limit, s[i]);
                }
            }
    });
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) limit = fmaxf(limit, __shfl_xor(limit, m));
    if (lane == 0) sh.redf[1][wave] = limit;
    u64 total = over_all(own, sh, turn);
    count = over_all(count, sh, turn);
#pragma unroll
    for (int i = 0; i < WAVES; i++) limit = fmaxf(limit, sh.redf[1][i]);
    unsigned key = __float_as_uint(limit);
    u64 ties = ~0ull;
    if (top_k > 0 && (u64)top_k < count) {
        const Cut c = find_cut<false>(row, (u64)top_k, limit, sh, turn);
        u64 lighter = 0;          // the weight of what is kept
        row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
            for (int i = 0; i < PIECE; i++)
                if (__float_as_uint(s[i]) < c.key) lighter += weight(s[i]);
        });
        total = over_all(lighter, sh, turn) + c.ties * weight(__uint_as_float(c.key));
        key = c.key;
        ties = c.ties < c.here ? c.ties : ~0ull;
    }
    if (top_p < 1.f) {
        const double share_p = ceil((double)top_p * (double)total);
        const u64 need = share_p > 1.0 ? (u64)share_p : 1;
        if (need < total) {
            const Cut c = find_cut<true>(row, need, limit, sh, turn);
            key = c.key;
            ties = c.ties < c.here ? c.ties : ~0ull;
        }
    }
    // ties by index: how many of the values equal to the cut lie before each wavefront's piece of each chunk
    const int entries = row.chunks * WAVES;
    const bool some_ties = ties != ~0ull;
    auto equal = [&](const float (&s)[PIECE]) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < PIECE; i++) n += __float_as_uint(s[i]) == key;
        return n;
    };
    if (some_ties) {
        row.each([&](int c, const float (&s)[PIECE]) {
            const u64 all = last_lane(up_to(equal(s)));
            if (lane == 0 && c < row.chunks) sh.ties[c * WAVES + wave] = (unsigned)all;
        });
        __syncthreads();
        if (wave == 0) {
            u64 carried = 0;
            for (int e0 = 0; e0 < entries; e0 += 64) {
                const u64 v = e0 + lane < entries ? sh.ties[e0 + lane] : 0, upto = up_to(v) + carried;
                if (e0 + lane < entries) sh.ties[e0 + lane] = (unsigned)(upto - v);
                carried = last_lane(upto);
            }
        }
        __syncthreads();
    }
    // the kept weights by index
    auto kept = [&](int c, const float (&s)[PIECE], unsigned (&w)[PIECE]) {
        u64 rank = 0, all = 0;
        if (some_ties && c < row.chunks) {
            const int n = equal(s);
            rank = sh.ties[c * WAVES + wave] + up_to(n) - n;
        }
#pragma unroll
        for (int i = 0; i < PIECE; i++) {
            const unsigned bits = __float_as_uint(s[i]);
            w[i] = bits <= key && (bits < key || rank++ < ties) ? weight(s[i]) : 0;
            all += w[i];
        }
        return all;
    };
    row.each([&](int c, const float (&s)[PIECE]) {
        unsigned w[PIECE];
        const u64 all = last_lane(up_to(kept(c, s, w)));
        if (lane == 0 && c < row.chunks) sh.sums[c * WAVES + wave] = all;
    });
    __syncthreads();
    // the entry with the target, by wavefront 0
    if (wave == 0) {
        u64 carried = 0;
        for (int e0 = 0; e0 < entries; e0 += 64) {
            const u64 v = e0 + lane < entries ? sh.sums[e0 + lane] : 0, upto = up_to(v) + carried;
            if (e0 + lane < entries) sh.sums[e0 + lane] = upto;
            carried = last_lane(upto);
        }
    }
    __syncthreads();
    total = sh.sums[entries - 1];
    const float u = k.u[r];
    u64 target = u > 0.f ? (u64)fmin((double)u * (double)total, 9007199254740991.0) : 0;
    target = target < total ? target : total - 1;
    row.each([&](int c, const float (&s)[PIECE]) {
        if (c >= row.chunks) return;
        const int e = c * WAVES + wave;
        const u64 before = e ? sh.sums[e - 1] : 0;
        if (target < before || target >= sh.sums[e]) return;          // (the wavefront's)
        unsigned w[PIECE];
        const u64 own = kept(c, s, w), upto = up_to(own) + before;
        if (target < upto - own || target >= upto) return;            // one lane is left
        u64 at = upto - own;
        bool done = false;
#pragma unroll
        for (int i = 0; i < PIECE; i++) {
            at += w[i];
            if (!done && target < at) {
                done = true;
                k.token[r] = row.first(c) + i;
                k.logprob[r] = (float)log((double)w[i] / (double)total);
            }
        }
    });
}

template <class T> static hipError_t launch(hipStream_t s, const Call &k) {
    // (a row may start anywhere in its first piece unless all of them start on one)
    const bool whole = k.stride % PIECE == 0 && reinterpret_cast<uintptr_t>(k.logits) % (PIECE * sizeof(T)) == 0;
    const int chunks = (k.V + (whole ? 0 : PIECE - 1) + CHUNK - 1) / CHUNK;
    const dim3 grid(k.rows), block(THREADS);
    if (chunks <= 1) hipLaunchKernelGGL((sample<T, 1>), grid, block, 0, s, k);
    else if (chunks <= 2) hipLaunchKernelGGL((sample<T, 2>), grid, block, 0, s, k);
    else if (chunks <= 4) hipLaunchKernelGGL((sample<T, 4>), grid, block, 0, s, k);
    else if (chunks <= 8) hipLaunchKernelGGL((sample<T, 8>), grid, block, 0, s, k);
    else hipLaunchKernelGGL((sample<T, 0>), grid, block, 0, s, k);
    return hipGetLastError();
}

}  // namespace sampling
}  // namespace wkv
