// Products  out[m][n] = sum over k of A[m][k] B[n][k]  tile by tile on the matrix cores: the loop that the
// gated feed-forward's products share.  A workgroup makes BM x BN outputs; 128 bytes of every row of A and B at a time (64 16-bit elements, 32 of
// fp32: a tile of k) go from memory straight to LDS, two to four tiles ahead of the one that is multiplied.
//
// In LDS a row's eight pieces of 16 bytes are exchanged by the row's low three bits, so that sixteen rows' equal pieces, which the
// matrix instructions take, lie over all banks.  A piece is a matrix instruction's whole operand of one lane: eight 16-bit elements for
// v_mfma_f32_16x16x32, four fp32 ones for four v_mfma_f32_16x16x4_f32 (whatever the order of k, it is A's and B's alike).
#pragma once
#include "common.h"

namespace wkv {
namespace tiles {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

template <class T> constexpr int piece() { return 16 / (int)sizeof(T); }             // elements in 16 bytes
template <class T> constexpr int depth() { return 128 / (int)sizeof(T); }            // of k at a time

template <class T> __device__ __forceinline__ f4 mma(i4 a, i4 b, f4 c);
template <> __device__ __forceinline__ f4 mma<bf16>(i4 a, i4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f4 mma<f16>(i4 a, i4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f4 mma<float>(i4 a, i4 b, f4 c) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
}

// 16 bytes per lane from memory to LDS, the lanes' side by side from `lds` on; nothing waits for them here.  What lies outside the range comes as zeros; the memory's
// addresses may be of any alignment (rows at every even one, by odd widths and sliced operands, are what the feed-forward's tests read), LDS' are whole pieces.
__device__ __forceinline__ void to_lds(i4 range, unsigned offset, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane((int)lds)), "v"(offset), "s"(range) : "memory", "m0");
}
__device__ __forceinline__ i4 range_of(const void *p, long long bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(p);
    const unsigned n = (unsigned)__builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : bytes > 0x7fffffff ? 0x7fffffff : bytes));
    return i4{__builtin_amdgcn_readfirstlane((int)a), __builtin_amdgcn_readfirstlane((int)((a >> 32) & 0xffff)), (int)n, 0x00027000};
}
constexpr unsigned NOWHERE = 0xfffffff0u;

// One operand's share of a workgroup's tile, ROWS rows with k along memory: `live` rows of K elements from `base` on, `ld` apart.
template <class T, int ROWS, int THREADS> struct Along {
    static constexpr int ROUNDS = ROWS * 8 / THREADS;
    const char *p;
    long long bytes;                  // from p to the last live row's end
    unsigned at[ROUNDS];
    int column;                       // of the lane's piece, in elements
    __device__ __forceinline__ void place(const T *base, long long ld, int K, int live) {
        p = reinterpret_cast<const char *>(base);
        bytes = live > 0 ? ((long long)(live - 1) * ld + K) * (long long)sizeof(T) : 0;
        const int row = threadIdx.x >> 3, c = (threadIdx.x & 7) ^ (row & 7);
        column = c * piece<T>();
#pragma unroll
        for (int j = 0; j < ROUNDS; j++) at[j] = (unsigned)((row + j * (THREADS / 8)) * ld * (long long)sizeof(T)) + c * 16;
    }
    // the tile of k from `k` on into LDS at `lds`, round by round
    i4 range;
    bool there;
    __device__ __forceinline__ void ask(int k, int K) {
        const long long skip = (long long)k * sizeof(T);
        range = range_of(p + skip, bytes - skip);
        there = k + column < K;                      // (K is whole pieces)
    }
    __device__ __forceinline__ void fetch(int j, unsigned lds) const {
        to_lds(range, there ? at[j] : NOWHERE, lds + j * (THREADS * 16) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024);
    }
    // the same by way of registers, of a tile of k that ends at any element: zeros from `end` on
    __device__ __forceinline__ void carry(const T *base, long long ld, int live, int k, int end, char *lds) const {
#pragma unroll
        for (int j = 0; j < ROUNDS; j++) {
            const int row = (threadIdx.x >> 3) + j * (THREADS / 8);
            const T *from = base + row * ld + k + column;
            T e[piece<T>()];
#pragma unroll
            for (int q = 0; q < piece<T>(); q++) e[q] = row < live && k + column + q < end ? from[q] : from_float<T>(0.f);
            __builtin_memcpy(lds + j * (THREADS * 16) + threadIdx.x * 16, e, 16);
        }
    }
    // the operands of sixteen rows: `first` the lane's, the same for every sixteen; half: of the tile of k
    struct Reader {
        int first;
        __device__ __forceinline__ Reader() {
            const int lane = threadIdx.x & 63;
            first = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
        }
        __device__ __forceinline__ i4 read(const char *tile, int sixteen, int half) const {
            return *reinterpret_cast<const i4 *>(tile + sixteen * (16 * 128) + (first ^ (half * 64)));
        }
    };
};
// The same of an operand with k across: ROWS columns of rows that are `ld` apart, a row per k; what lies between `end` and the end of the last row is not
// there.  In LDS a row of k is ROWS elements; the pieces that one instruction takes of its rows are exchanged by the row, so that they lie over all banks.  16-bit
// elements turn on their way to the registers (a transposing read gives a lane four of k of one column), fp32 ones are read one by one.
template <class T, int ROWS, int THREADS> struct Across {
    static constexpr int BYTES = ROWS * (int)sizeof(T), PIECES = BYTES / 16, PER = THREADS / PIECES, ROUNDS = depth<T>() / PER;
    const char *p, *second;           // rows of k from `turn` on: second's, from its first
    long long bytes, ld;              // from p to the end
    int turn;
    int shift;                        // 1: every row is taken for two of k
    unsigned at[ROUNDS];
    // of the pieces' numbers in row k: an instruction takes two pieces (fp32: four) of each of rows 8 g .. 8 g + 3 (fp32: of rows 4 g)
    static __device__ __forceinline__ int exchange(int k) {
        if (sizeof(T) == 4) return (k >> 2 & 3) << 2;
        return (PIECES >= 16 ? (k & 3) | (k >> 1 & 4) : (k >> 1 & 1) | (k >> 2 & 2)) << 1;
    }
    // column n0 of rows that are there up to `rows`, `width` elements wide
    __device__ __forceinline__ void place(const T *base, const T *base2, int turn_, long long ld_, int n0, int rows, int width, int shift_ = 0) {
        p = reinterpret_cast<const char *>(base + n0);
        second = reinterpret_cast<const char *>(base2 + n0);
        turn = turn_;
        shift = shift_;
        ld = ld_ * (long long)sizeof(T);
        bytes = (long long)(rows - 1) * ld + (long long)(width - n0) * (long long)sizeof(T);
#pragma unroll
        for (int j = 0; j < ROUNDS; j++) {
            const int k = threadIdx.x / PIECES + j * PER, c = (threadIdx.x % PIECES) ^ exchange(k);
            at[j] = (unsigned)((k >> shift) * ld) + c * 16;
        }
    }
    i4 range;
    __device__ __forceinline__ void ask(int k, int) {
        k >>= shift;
        const bool behind = k >= turn;
        const long long skip = (long long)(behind ? k - turn : k) * ld;
        range = range_of((behind ? second : p) + skip, bytes - skip);
    }
    __device__ __forceinline__ void fetch(int j, unsigned lds) const {
        to_lds(range, at[j], lds + j * (THREADS * 16) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024);
    }
    struct Reader {
        int first, mix;
        __device__ __forceinline__ Reader() {
            const int lane = threadIdx.x & 63, a = lane & 15, g = lane >> 4;
            if constexpr (sizeof(T) == 2) {
                first = (8 * g + (a >> 2)) * BYTES + 8 * (a & 3);
                mix = exchange(8 * g + (a >> 2)) << 4;
            } else {
                first = 4 * g * BYTES + 4 * a;
                mix = exchange(4 * g) << 4;
            }
        }
        __device__ __forceinline__ i4 read(const char *tile, int sixteen, int half) const {
            typedef short s4 __attribute__((ext_vector_type(4)));
            typedef s4 __attribute__((address_space(3))) lds_s4;
            const char *at = tile + first + ((sixteen * (sizeof(T) == 2 ? 32 : 64)) ^ mix) + half * (depth<T>() / 2) * BYTES;
            if constexpr (sizeof(T) == 2) {
                s4 o[2];
#pragma unroll
                for (int q = 0; q < 2; q++) o[q] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4 *)(at + q * 4 * BYTES));
                return __builtin_bit_cast(i4, o);
            } else {
                float o[4];
#pragma unroll
                for (int q = 0; q < 4; q++) o[q] = *reinterpret_cast<const float *>(at + q * BYTES);
                return __builtin_bit_cast(i4, o);
            }
        }
    };
};

// A launch's tiles in the order in which they are worked: the eight XCDs (a workgroup's number modulo 8) each take a run of
// tiles, and a run goes down eight rows of tiles before it goes on to the next column, so that the workgroups that share an L2 share operands.
__device__ __forceinline__ void tile_of(int index, int rows, int columns, int &row, int &column) {
    const int all = rows * columns, x = index & 7, i = index >> 3, q = all >> 3, rest = all & 7;
    const int t = x * q + (x < rest ? x : rest) + i;
    const int band = 8 * columns, b = t / band, first = b * 8, high = rows - first < 8 ? rows - first : 8, in = t - b * band;
    row = first + in % high;
    column = in / high;
}

// The loop over k of a workgroup of WM x WN wavefronts, on top of what acc holds: acc[i][j] is the sum of 16 rows of A and 16 of B, a lane's element e the one of A's row
// (lane & 15) and B's row 4 (lane >> 4) + e.  B's rows come in PARTS parts of BN / PARTS rows; a wavefront takes its share of each.  LDS holds AHEAD + 1
// of A's tiles and AHEAD of B's.
template <class T, class A, class B, int BM, int BN, int WM, int WN, int PARTS, int AHEAD> struct Loop {
    static constexpr int MT = BM / WM / 16, NT = BN / WN / 16, ABYTES = BM * 128, BBYTES = BN * 128, LDS = (AHEAD + 1) * ABYTES + AHEAD * BBYTES;
    static constexpr int LOADS = A::ROUNDS + PARTS * B::ROUNDS;          // of a lane and tile
    A a;
    B b[PARTS];
    f4 acc[MT][NT];

    __device__ __forceinline__ void ask_b(int k, int K) {
#pragma unroll
        for (int p = 0; p < PARTS; p++) b[p].ask(k, K);
    }
    // share `g` of `of` of a tile's loads
    __device__ __forceinline__ void fetch_a(int g, int of, unsigned lds) const {
#pragma unroll
        for (int q = g * A::ROUNDS / of; q < (g + 1) * A::ROUNDS / of; q++) a.fetch(q, lds);
    }
    __device__ __forceinline__ void fetch_b(int g, int of, unsigned lds) const {
        constexpr int ALL = PARTS * B::ROUNDS;
#pragma unroll
        for (int q = g * ALL / of; q < (g + 1) * ALL / of; q++) b[q / B::ROUNDS].fetch(q % B::ROUNDS, lds + q / B::ROUNDS * (BN / PARTS) * 128);
    }
    // a half tile's operands
    struct Half { i4 x[MT], y[NT]; };
    // share `g` of `of` of a half's reads: those that the multiplications begin with first
    __device__ __forceinline__ void read(const typename A::Reader &ra, const typename B::Reader &rb, const char *at_a, const char *at_b, int wm, int wn, int half, int g, int of, Half &h) const {
#pragma unroll
        for (int q = 0; q < MT + NT; q++) {
            if (q < g * (MT + NT) / of || q >= (g + 1) * (MT + NT) / of) continue;
            if (q < NT) {
                const int part = q / (NT / PARTS), jj = q % (NT / PARTS);
                h.y[q] = rb.read(at_b + part * (BN / PARTS) * 128, wn * (NT / PARTS) + jj, half);
            } else {
                h.x[q - NT] = ra.read(at_a, wm * MT + q - NT, half);
            }
        }
    }
    __device__ __forceinline__ void multiply(const Half &h, int i) {
#pragma unroll
        for (int j = 0; j < NT; j++) acc[i][j] = mma<T>(h.y[j], h.x[i], acc[i][j]);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
            for (int j = 0; j < NT; j++) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    }
    // a tile of k that lies in LDS, where the first of A's and of B's go
    __device__ __forceinline__ void once(char *lds) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
        const typename A::Reader ra;
        const typename B::Reader rb;
        __syncthreads();
#pragma unroll
        for (int half = 0; half < 2; half++) {
            Half h;
            read(ra, rb, lds, lds + (AHEAD + 1) * ABYTES, wm, wn, half, 0, 1, h);
#pragma unroll
            for (int i = 0; i < MT; i++) multiply(h, i);
        }
        __syncthreads();
    }
    // k from k0 (whole tiles) to k1.  Half a tile's operands are multiplied while the next half's are on their way from LDS; the one barrier of a tile stands
    // between its halves, where every wavefront has read all of the tile and the next has come, so that there is work in registers on both sides of it.  A's tile
    // AHEAD from this one is asked for in a tile's first half, B's in the second, in the place of this one's.  Reads and loads are issued between the
    // multiplications, a few at a time: issued together they hold the matrix instructions behind them up (a tile's loads take the memory pipe half a tile's time).
    __device__ __forceinline__ void run(int k0, int k1, int K, char *lds) {
        constexpr int D = depth<T>();
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave / WN, wn = wave % WN;
        const unsigned base = (unsigned)reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds);
        const typename A::Reader ra;
        const typename B::Reader rb;
        Half first, second;
        int at_a[AHEAD + 1], at_b[AHEAD];          // this tile's, the next one's ...
#pragma unroll
        for (int q = 0; q <= AHEAD; q++) at_a[q] = q * ABYTES;
#pragma unroll
        for (int q = 0; q < AHEAD; q++) at_b[q] = (AHEAD + 1) * ABYTES + q * BBYTES;
#pragma unroll
        for (int q = 0; q < AHEAD; q++) {
            a.ask(k0 + q * D, K);          // (past K: zeros, which nobody reads)
            ask_b(k0 + q * D, K);
            fetch_a(0, 1, base + at_a[q]);
            fetch_b(0, 1, base + at_b[q]);
        }
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((AHEAD - 1) * LOADS) : "memory");
        read(ra, rb, lds + at_a[0], lds + at_b[0], wm, wn, 0, 0, 1, first);
        // (the last tile apart: behind a branch the compiler waits for what either side may have asked for)
        for (int k = k0; k + D < k1; k += D) {
            a.ask(k + AHEAD * D, K);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                read(ra, rb, lds + at_a[0], lds + at_b[0], wm, wn, 1, i, MT, second);
                __builtin_amdgcn_sched_barrier(0);
                multiply(first, i);
                __builtin_amdgcn_sched_barrier(0);
                fetch_a(i, MT, base + at_a[AHEAD]);
            }
            // (all but what was asked for after the next tile's: A's and B's of the ones behind it, A's of the last)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((AHEAD - 2) * LOADS + A::ROUNDS) : "memory");
            ask_b(k + AHEAD * D, K);
#pragma unroll
            for (int i = 0; i < MT; i++) {
                read(ra, rb, lds + at_a[1], lds + at_b[1], wm, wn, 0, i, MT, first);
                __builtin_amdgcn_sched_barrier(0);
                multiply(second, i);
                __builtin_amdgcn_sched_barrier(0);
                fetch_b(i, MT, base + at_b[0]);
            }
            const int was_a = at_a[0], was_b = at_b[0];
#pragma unroll
            for (int q = 0; q < AHEAD; q++) at_a[q] = at_a[q + 1];
#pragma unroll
            for (int q = 0; q + 1 < AHEAD; q++) at_b[q] = at_b[q + 1];
            at_a[AHEAD] = was_a, at_b[AHEAD - 1] = was_b;
        }
        read(ra, rb, lds + at_a[0], lds + at_b[0], wm, wn, 1, 0, 1, second);
#pragma unroll
        for (int i = 0; i < MT; i++) multiply(first, i);
#pragma unroll
        for (int i = 0; i < MT; i++) multiply(second, i);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // (nothing may come into LDS behind the workgroup's end)
    }
};

}  // namespace tiles
}  // namespace wkv
