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
// never sorts.  Each of the two cuts is found from a histogram over 4096 bins of s, of tokens for top_k and of weights for top_p, and
// then among the elements of the bin it falls into, which one wavefront searches by the bits of s.  What bounds it is the passes over
// the registers and the histograms' atomics in LDS, so these take only what a cut can reach: for top_k what is not
// below every lane's best (1024 such there are), for top_p what the rest of the vocabulary could not outweigh.  B1 V65536 fp32, one compute
// unit's work: 13 us without cuts, 7 at temperature 0, 14 with min_p, 19 with top_k, 27 to 33 with top_p; a row per compute unit, B200 V50277 bf16: 14, 8.5
// (temperature 0), 23 and 31 to 35.
#include "common.h"

namespace wkv {
namespace sampling {

constexpr int THREADS = 1024, WAVES = THREADS / 64, PIECE = 8, CHUNK = THREADS * PIECE;
constexpr int BINS = 4096, PER_THREAD = BINS / THREADS;
constexpr float MOST = 32.f, PER_OCTAVE = 128.f;     // weights vanish at s = 32, in bin BINS; a power of two: products with it are exact
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

// v of the lane that a DPP names, 0 where there is none
template <int CTRL, int ROWS> __device__ __forceinline__ u64 from_lane(u64 v) {
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 up_to(u64 v) {          // inclusive sum over the wavefront's lanes
    v += from_lane<0x111, 0xf>(v);                     // row_shr:1, 2, 4, 8
    v += from_lane<0x112, 0xf>(v);
    v += from_lane<0x114, 0xf>(v);
    v += from_lane<0x118, 0xf>(v);
    v += from_lane<0x142, 0xa>(v);                     // row_bcast:15 to the second and the fourth row
    v += from_lane<0x143, 0xc>(v);                     // row_bcast:31 to the upper two
    return v;
}
__device__ __forceinline__ u64 last_lane(u64 v) {
    return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), 63) << 32 | (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, 63);
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
        for (int i = 0; i < PIECE; i++) o[i] = fmaxf(o[i], -INFINITY);          // (of a NaN and a number the number)
    }
    __device__ __forceinline__ void place(float (&o)[PIECE]) const {
        if (top == INFINITY) {
#pragma unroll
            for (int i = 0; i < PIECE; i++) o[i] = o[i] == INFINITY ? 0.f : INFINITY;
        } else {
#pragma unroll
            for (int i = 0; i < PIECE; i++) o[i] = (top - o[i]) * scale;          // (-infinity: infinity)
        }
    }
    // f(chunk, its piece's s), from the registers where they hold it
    template <class F> __device__ __forceinline__ void each(F f) {
        if constexpr (N > 0) {
#pragma unroll
            for (int c = 0; c < N; c++) f(c, s[c]);
        } else {
            each_again(f);
        }
    }
    // the same read again, in a short loop: for what is rare
    template <class F> __device__ __forceinline__ void each_again(F f) const {
#pragma unroll 1
        for (int c = 0; c < chunks; c++) {
            float o[PIECE];
            read(c, o);
            f(c, o);
        }
    }
    __device__ __forceinline__ void read(int c, float (&o)[PIECE]) const {
        raw(c, o);
        place(o);
    }
};

__device__ __forceinline__ unsigned weight(float s) { return (unsigned)rintf(exp2_fast(-s) * (float)ONE); }

// the largest bits of s whose weight is at least `least`: 64 of them tried at once
__device__ __forceinline__ unsigned last_of_weight(unsigned least) {
    unsigned lo = 0, hi = __float_as_uint(MOST);          // it lies in [lo, hi)
    while (hi - lo > 1) {
        const unsigned step = (hi - lo + 63) / 64, at = lo + (threadIdx.x & 63) * step;
        const u64 reached = __ballot(at < hi && weight(__uint_as_float(at)) >= least);
        const int last = 63 - __clzll((long long)reached);          // (lane 0's does: that of lo)
        hi = min(hi, lo + (last + 1) * step);
        lo += last * step;
    }
    return lo;
}

constexpr int LIST = 1024;                     // elements of one bin that one wavefront searches
struct Shared {
    u64 bin_weight[BINS];
    unsigned bin_count[BINS];
    float list[LIST];
    unsigned list_weight[LIST], listed;
    u64 sums[WAVES * MAX_CHUNKS];          // by chunk and wavefront
    unsigned ties[WAVES * MAX_CHUNKS + 1];
    u64 red[2][WAVES];
    float redf[2][WAVES];
    // what a search found
    int bin;
    unsigned key;
    u64 before, equal, total;
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

// The first bin at which the sum of `in` reaches `need` (at least 1), and the sum before it; false if it does not
template <class E> __device__ __forceinline__ bool find_bin(const E *in, u64 need, Shared &sh, int &turn, int &bin, u64 &before) {
    const int wave = threadIdx.x >> 6;
    u64 own = 0;
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) own += in[threadIdx.x * PER_THREAD + i];
    u64 upto = up_to(own), total = 0;
    if ((threadIdx.x & 63) == 63) sh.red[turn][wave] = upto;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        if (i < wave) upto += sh.red[turn][i];
        total += sh.red[turn][i];
    }
    turn ^= 1;
    if (total < need) return false;
    if (upto >= need && upto - own < need) {
        u64 sum = upto - own;
        int i = threadIdx.x * PER_THREAD;
        while (sum + in[i] < need) sum += in[i++];
        sh.bin = i;
        sh.before = sum;
    }
    __syncthreads();
    bin = sh.bin;
    before = sh.before;
    return true;
}

struct Cut {
    unsigned key;          // kept: the values below, and the first `ties` of those equal
    u64 ties;
    u64 before;            // the weight (tokens) of the values below
    u64 equal;             // how many are equal
};

// Where the first `need` (of tokens, or of weight) in the order of s end, from the histogram `in` of the elements up to `most` (bits of s); false if
// there is less than that
template <bool WEIGHT, class E, class R>
__device__ __forceinline__ bool find_cut(R &row, const E *in, u64 need, unsigned most, Shared &sh, int &turn, Cut &cut) {
    int bin;
    u64 before;
    if (threadIdx.x == 0) sh.listed = 0;
    if (!find_bin(in, need, sh, turn, bin, before)) return false;
    // the bin's values (the products are exact)
    const unsigned first = __float_as_uint(bin * (1.f / PER_OCTAVE)), span = min(__float_as_uint((bin + 1) * (1.f / PER_OCTAVE)) - 1, most) - first;
    auto inside = [&](float s) { return __float_as_uint(s) - first <= span; };
    row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
        for (int i = 0; i < PIECE; i++)
            if (inside(s[i])) {
                const unsigned at = atomicAdd(&sh.listed, 1u);
                if (at < LIST) sh.list[at] = s[i];
            }
    });
    __syncthreads();
    const unsigned m = sh.listed;
    if (m <= 64) {          // an element per lane of one wavefront: each is held against all
        if (threadIdx.x < 64) {
            const bool there = threadIdx.x < m;
            const float s = there ? sh.list[threadIdx.x] : 0.f;
            const unsigned own = __float_as_uint(s), w = WEIGHT ? weight(s) : 1;
            u64 below = 0;
            unsigned equal = 0;
            for (unsigned i = 0; i < m; i++) {
                const unsigned bits = __builtin_amdgcn_readlane(own, i), each = __builtin_amdgcn_readlane(w, i);
                below += bits < own ? each : 0u;
                equal += bits == own;
            }
            below += before;
            // (equal ones agree, so whichever writes)
            if (there && below < need && below + (u64)equal * w >= need) {
                sh.key = own;
                sh.equal = equal;
                sh.total = below;
            }
        }
        __syncthreads();
        cut.key = sh.key;
        cut.equal = sh.equal;
        cut.before = sh.total;
    } else if (m <= LIST) {
        if (threadIdx.x < 64) {
            unsigned lo = 0xffffffffu, hi = 0;
            for (unsigned i = threadIdx.x; i < m; i += 64) {
                const float s = sh.list[i];
                if (WEIGHT) sh.list_weight[i] = weight(s);
                lo = min(lo, __float_as_uint(s));
                hi = max(hi, __float_as_uint(s));
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) {
                lo = min(lo, (unsigned)__shfl_xor((int)lo, d));
                hi = max(hi, (unsigned)__shfl_xor((int)hi, d));
            }
            auto sum = [&](unsigned from, unsigned to, bool weights) {          // of the values from .. to (a lane reads what it has written)
                u64 n = 0;
                for (unsigned i = threadIdx.x; i < m; i += 64) {
                    const unsigned bits = __float_as_uint(sh.list[i]);
                    n += bits >= from && bits <= to ? (weights ? sh.list_weight[i] : 1u) : 0u;
                }
                return last_lane(up_to(n));
            };
            while (lo < hi) {
                const unsigned mid = lo + ((hi - lo) >> 1);
                if (before + sum(0, mid, WEIGHT) >= need) hi = mid;
                else lo = mid + 1;
            }
            const u64 n = sum(lo, lo, false), below = lo ? sum(0, lo - 1, WEIGHT) : 0;
            if (threadIdx.x == 0) {
                sh.key = lo;
                sh.equal = n;
                sh.total = before + below;
            }
        }
        __syncthreads();
        cut.key = sh.key;
        cut.equal = sh.equal;
        cut.before = sh.total;
    } else {          // too many for that, most likely equal ones: the same search by all, over the registers
        unsigned lo = 0xffffffffu, hi = 0;
        row.each_again([&](int, const float (&s)[PIECE]) {
#pragma unroll
            for (int i = 0; i < PIECE; i++)
                if (inside(s[i])) {
                    lo = min(lo, __float_as_uint(s[i]));
                    hi = max(hi, __float_as_uint(s[i]));
                }
        });
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            lo = min(lo, (unsigned)__shfl_xor((int)lo, d));
            hi = max(hi, (unsigned)__shfl_xor((int)hi, d));
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
        auto sum = [&](unsigned from, unsigned to, bool weights) {          // of the values from .. to
            u64 n = 0;
            row.each_again([&](int, const float (&s)[PIECE]) {
#pragma unroll
                for (int i = 0; i < PIECE; i++)
                    if (__float_as_uint(s[i]) >= from && __float_as_uint(s[i]) <= to && inside(s[i])) n += weights ? weight(s[i]) : 1;
            });
            return over_all(n, sh, turn);
        };
        while (lo < hi) {
            const unsigned mid = lo + ((hi - lo) >> 1);
            if (before + sum(0, mid, WEIGHT) >= need) hi = mid;
            else lo = mid + 1;
        }
        cut.key = lo;
        cut.equal = sum(lo, lo, false);
        cut.before = before + (lo ? sum(0, lo - 1, WEIGHT) : 0);
    }
    const u64 left = need - cut.before, each = WEIGHT ? max(weight(__uint_as_float(cut.key)), 1u) : 1u;
    cut.ties = (left + each - 1) / each;
    return true;
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
    const int top_k = k.top_k ? k.top_k[r] : k.top_k_value;
    // the largest logit of the lane and of all
    float best = -INFINITY;
    if constexpr (N > 0) {
#pragma unroll
        for (int c = 0; c < N; c++) {
            row.raw(c, row.s[c]);
#pragma unroll
            for (int i = 0; i < PIECE; i++) best = fmaxf(best, row.s[c][i]);
        }
    } else {
        for (int c = 0; c < row.chunks; c++) {
            row.raw(c, row.s[0]);
#pragma unroll
            for (int i = 0; i < PIECE; i++) best = fmaxf(best, row.s[0][i]);
        }
    }
    float top = best, least_best = best;
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) {
        top = fmaxf(top, __shfl_xor(top, m));
        least_best = fminf(least_best, __shfl_xor(least_best, m));
    }
    if (lane == 0) {
        sh.redf[0][wave] = top + 0.f;          // (-0, which a maximum of zeros of both signs may be, is +0 from here on: less +0 it would be -0, whose bits lie past every cut)
        sh.redf[1][wave] = least_best;
    }
#pragma unroll
    for (int i = 0; i < PER_THREAD; i++) {
        sh.bin_weight[tid + i * THREADS] = 0;
        sh.bin_count[tid + i * THREADS] = 0;
    }
    __syncthreads();
    top = sh.redf[0][0];
#pragma unroll
    for (int i = 0; i < WAVES; i++) {
        top = fmaxf(top, sh.redf[0][i]);
        least_best = fminf(least_best, sh.redf[1][i]);
    }
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
    if (!warm) {          // the first of the likeliest
        unsigned at = ~0u;
        row.each([&](int c, const float (&s)[PIECE]) {
#pragma unroll
            for (int i = 0; i < PIECE; i++)
                if (s[i] == 0.f) at = min(at, (unsigned)(row.first(c) + i));
        });
#pragma unroll
        for (int m = 32; m > 0; m >>= 1) at = min(at, (unsigned)__shfl_xor((int)at, m));
        if (lane == 0) sh.red[0][wave] = at;
        __syncthreads();
        if (tid == 0) {
            for (int i = 1; i < WAVES; i++) at = min(at, (unsigned)sh.red[0][i]);
            k.token[r] = at;
            k.logprob[r] = 0.f;
        }
        return;
    }
    // a token counts from a weight of 1, or of min_p's share: up to the bits `most` of s
    const double share = (double)min_p * ONE;
    const unsigned least = share > 1.0 ? share < ONE ? (unsigned)ceil(share) : (unsigned)ONE : 1u;
    const unsigned most = least == 1 ? __float_as_uint(MOST) - 1 : last_of_weight(least);
    int turn = 0;
    unsigned key = most;
    u64 ties = ~0ull;
    bool cut_k = false;
    if (top_k > 0 && top_k < k.V) {
        // every lane has an element within `far`: the first 1024 are there
        float far[PIECE];
#pragma unroll
        for (int i = 0; i < PIECE; i++) far[i] = least_best;
        row.place(far);
        const unsigned near = top_k <= THREADS ? min(most, __float_as_uint(far[0])) : most;
        row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
            for (int i = 0; i < PIECE; i++)
                if (__float_as_uint(s[i]) <= near) atomicAdd(&sh.bin_count[(int)(s[i] * PER_OCTAVE)], 1u);
        });
        __syncthreads();
        Cut c;
        if (find_cut<false>(row, sh.bin_count, (u64)top_k, near, sh, turn, c)) {
            cut_k = true;
            key = c.key;
            ties = c.ties < c.equal ? c.ties : ~0ull;
        }
    }
    if (top_p < 1.f) {
        // the weight of what is left; where top_k has left little, its histogram too
        u64 own = 0;
        if (cut_k) {
            row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
                for (int i = 0; i < PIECE; i++)
                    if (__float_as_uint(s[i]) <= key) {
                        const unsigned w = weight(s[i]);
                        atomicAdd(&sh.bin_weight[(int)(s[i] * PER_OCTAVE)], (u64)w);
                        if (__float_as_uint(s[i]) < key || ties == ~0ull) own += w;
                    }
            });
        } else {
            row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
                for (int i = 0; i < PIECE; i++)
                    if (__float_as_uint(s[i]) <= key) own += weight(s[i]);
            });
        }
        u64 total = over_all(own, sh, turn);
        if (ties != ~0ull) total += ties * weight(__uint_as_float(key));
        const double share_p = ceil((double)top_p * (double)total);
        const u64 need = share_p > 1.0 ? (u64)share_p : 1;
        if (need < total) {
            unsigned near = key;
            if (!cut_k) {
                // what lies beyond weighs less than what top_p leaves out, even if all of the vocabulary lies there
                const float each = (float)(total - need) / (float)k.V - 1.f;
                if (each > 1.f) near = min(near, __float_as_uint(31.01f - __builtin_amdgcn_logf(each)));
                row.each([&](int, const float (&s)[PIECE]) {
#pragma unroll
                    for (int i = 0; i < PIECE; i++)
                        if (__float_as_uint(s[i]) <= near) atomicAdd(&sh.bin_weight[(int)(s[i] * PER_OCTAVE)], (u64)weight(s[i]));
                });
                __syncthreads();
            }
            Cut c;
            if (find_cut<true>(row, sh.bin_weight, need, near, sh, turn, c)) {
                key = c.key;
                ties = c.ties < c.equal ? c.ties : ~0ull;
            }
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
            unsigned n = 0;
#pragma unroll
            for (int i = 0; i < PIECE; i++) n += __popcll(__ballot(__float_as_uint(s[i]) == key));
            if (lane == 0 && c < row.chunks) sh.ties[c * WAVES + wave] = n;
        });
        __syncthreads();
        if (wave == 0) {
            u64 carried = 0;
            for (int e0 = 0; e0 < entries; e0 += 64) {
                const u64 v = e0 + lane < entries ? sh.ties[e0 + lane] : 0, upto = up_to(v) + carried;
                if (e0 + lane < entries) sh.ties[e0 + lane] = (unsigned)(upto - v);
                carried = last_lane(upto);
            }
            if (lane == 0) sh.ties[entries] = (unsigned)carried;
        }
        __syncthreads();
    }
    // the kept weights by index
    auto kept = [&](int c, const float (&s)[PIECE], unsigned (&w)[PIECE]) {
        const int n = equal(s);
        u64 rank = sh.ties[c * WAVES + wave] + up_to(n) - n, all = 0;
#pragma unroll
        for (int i = 0; i < PIECE; i++) {
            // (selections: as branches around weight() the compiler lost the weight of the ties that stay)
            const unsigned bits = __float_as_uint(s[i]), each = weight(fminf(s[i], MOST));
            const bool tie = bits == key, stays = (bits < key) | (tie & (!some_ties | (rank < ties)));
            rank += tie;
            w[i] = stays ? each : 0;
            all += w[i];
        }
        return all;
    };
    row.each([&](int c, const float (&s)[PIECE]) {
        if (c >= row.chunks) return;
        // of the wavefront's equal ones all stay, or none, or (in one place of the row) some
        const int e = c * WAVES + wave;
        u64 all = 0;
        unsigned below = key + 1;
        if (some_ties && sh.ties[e + 1] > ties) {
            below = key;
            if (sh.ties[e] < ties) {
                unsigned w[PIECE];
                all = kept(c, s, w);
                below = 0;
            }
        }
        if (below) {
#pragma unroll
            for (int i = 0; i < PIECE; i++)
                if (__float_as_uint(s[i]) < below) all += weight(s[i]);
        }
        all = last_lane(up_to(all));
        if (lane == 0) sh.sums[e] = all;
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
    const u64 total = sh.sums[entries - 1];
    const float u = k.u[r];
    u64 target = u > 0.f ? (u64)fmin((double)u * (double)total, 9007199254740991.0) : 0;
    target = target < total ? target : total - 1;
    for (int c = 0; c < row.chunks; c++) {
        const int e = c * WAVES + wave;
        const u64 before = e ? sh.sums[e - 1] : 0;
        if (target < before || target >= sh.sums[e]) continue;          // (the same for the wavefront)
        float s[PIECE];
        unsigned w[PIECE];
        row.read(c, s);
        const u64 own = kept(c, s, w), upto = up_to(own) + before;
        if (target < upto - own || target >= upto) break;               // one lane is left
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
        break;
    }
}

constexpr int ROWS_PER_LAUNCH = 1 << 21;          // (a grid has fewer than 2^32 threads)
template <class T> static hipError_t launch(hipStream_t s, const Call &all) {
    // (a row may start anywhere in its first piece unless all of them start on one)
    const bool whole = all.stride % PIECE == 0 && reinterpret_cast<uintptr_t>(all.logits) % (PIECE * sizeof(T)) == 0;
    const int chunks = (all.V + (whole ? 0 : PIECE - 1) + CHUNK - 1) / CHUNK;
    for (int done = 0; done < all.rows; done += std::min(all.rows - done, ROWS_PER_LAUNCH)) {
        Call k = all;
        auto on = [&](auto *p) { return p ? p + done : p; };
        k.rows = std::min(all.rows - done, ROWS_PER_LAUNCH);
        k.logits = static_cast<const T *>(all.logits) + done * all.stride;
        k.u = on(all.u); k.temperature = on(all.temperature); k.top_p = on(all.top_p); k.min_p = on(all.min_p); k.top_k = on(all.top_k);
        k.token = on(all.token); k.logprob = on(all.logprob);
        const dim3 grid(k.rows), block(THREADS);
        if (chunks <= 1) hipLaunchKernelGGL((sample<T, 1>), grid, block, 0, s, k);
        else if (chunks <= 2) hipLaunchKernelGGL((sample<T, 2>), grid, block, 0, s, k);
        else if (chunks <= 4) hipLaunchKernelGGL((sample<T, 4>), grid, block, 0, s, k);
        else if (chunks <= 8) hipLaunchKernelGGL((sample<T, 8>), grid, block, 0, s, k);
        else hipLaunchKernelGGL((sample<T, 0>), grid, block, 0, s, k);
    }
    return hipGetLastError();
}

}  // namespace sampling
}  // namespace wkv
