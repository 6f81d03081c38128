// Rows of a table by token, scaled, and the table's gradient:
//
//     out[n] = scale table[token[n]],      gtable[v] = scale (sum over the n with token[n] = v of gout[n])
//
// A token outside the table is a place without one: a row of zeros, no gradient.  Both directions are bound by memory (32768 places of 2560 channels bf16, 65536 tokens: lookup 55 us,
// 6 TB/s from the last-level cache's share; sums and zeros 101, 5 TB/s, behind 30 of sorting in small launches).  The gradient is written
// whole (V C, most of it zeros) from the places sorted by token: no atomics on sums, fp32 ones in the places' order within a chunk and in the chunks' order over them, the same bits every time.  Sorting: stable
// passes over ten bits of the token at most, counts per tile of places, then each tile's places to where the tiles and digits before leave off; up
// to one tile's worth in a single launch.  Sums: a workgroup takes a chunk of up to 64 sorted places, whoever they belong to, so that it does not matter how often a token
// comes; a token that lies within them is written as it ends, one that crosses their border leaves a part for a second launch.  The zeros are written beside what waits: of one tile,
// the whole table beside the sorting (the few rows that have a sum are written again), else the tokens' that no place has beside the sums, whose gathers wait for memory.
#include <type_traits>

#include "common.h"
#include "vec.h"

namespace wkv {
namespace embedding {

// ---- lookup: 16 bytes (or an element) per lane
struct Lookup { size_t count; int V, C; long long ws; float scale; const void *tokens, *table; void *out; };
template <class I> __device__ __forceinline__ long long token_at(const void *p, size_t n) { return static_cast<const I *>(p)[n]; }

constexpr int EACH = 4;                       // pieces per lane
template <class T, class I, int W> __global__ __launch_bounds__(256) void lookup(const Lookup k) {
    const unsigned pieces = k.C / W;
    const size_t first = (size_t)blockIdx.x * (256 * EACH), n0 = first / pieces, total = k.count * pieces;
    const unsigned start = (unsigned)(first - n0 * pieces);
    float v[EACH][W];
    bool there[EACH];
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const unsigned at = start + e * 256 + threadIdx.x, r = at / pieces, c = at - r * pieces;
#pragma unroll
        for (int w = 0; w < W; w++) v[e][w] = 0.f;
        there[e] = false;
        if (first + e * 256 + threadIdx.x >= total) continue;
        const long long t = token_at<I>(k.tokens, n0 + r);
        there[e] = t >= 0 && t < k.V;
        if (there[e]) load_vec(static_cast<const T *>(k.table) + t * k.ws + c * W, v[e]);
    }
#pragma unroll
    for (int e = 0; e < EACH; e++) {
        const size_t at = first + e * 256 + threadIdx.x;
        if (at >= total) continue;
#pragma unroll
        for (int w = 0; w < W; w++) v[e][w] = there[e] ? v[e][w] * k.scale : 0.f;          // (zeros whatever the scale is)
        store_vec(static_cast<T *>(k.out) + at * W, v[e]);
    }
}

// ---- zeros: groups of 256 threads, each a run of the table as one row of elements, whatever its width, 16 bytes per lane.  E: an element's bits
constexpr int ZEROS = 8;                      // pieces per lane
struct Zeros {
    void *out;
    const int *starts;                        // by token, as find_starts leaves them; NULL: the whole table
    int V, C;
};
static inline size_t groups_of_zeros(int V, int C, size_t size) { return ((size_t)V * C * size + 256 * ZEROS * 16 - 1) / (256 * ZEROS * 16); }
template <class E> __device__ __forceinline__ void put_zeros(const Zeros &k, size_t group) {
    constexpr int W = 16 / sizeof(E);
    const size_t first = group * (256 * ZEROS * W), v0 = first / k.C, total = (size_t)k.V * k.C;
    const unsigned start = (unsigned)(first - v0 * k.C);
    E *out = static_cast<E *>(k.out);
    auto empty = [&](size_t v) { return !k.starts || k.starts[v] == k.starts[v + 1]; };
#pragma unroll
    for (int z = 0; z < ZEROS; z++) {
        const unsigned in = (z * 256 + (threadIdx.x & 255)) * W, at = start + in, r = at / k.C, last = (at + W - 1) / k.C;
        const size_t i = first + in;
        if (i >= total) return;
        const bool one = i + W <= total && empty(v0 + r);
        if (one && (last == r || (last == r + 1 && empty(v0 + last)))) {
            *reinterpret_cast<uint4 *>(out + i) = make_uint4(0, 0, 0, 0);
            continue;
        }
        if (i + W <= total && last == r) continue;          // (a row that has a sum)
        for (int w = 0; w < W && i + w < total; w++)
            if (empty(v0 + (at + w) / k.C)) out[i + w] = 0;
    }
}
// ---- sorting
constexpr int SORT_THREADS = 1024, SORT_WAVES = 16, MAX_BITS = 10, BINS = 1 << MAX_BITS, TILE = 4 * SORT_THREADS;          // TILE: places of a large tile
struct Sort {
    int count, V;                             // keys: tokens, V for none
    const void *tokens;                       // the first pass's keys; their places are 0, 1, ..
    const int *keys, *places;                 // the later passes'
    int *to_keys, *to_places, *counts;        // counts (tiles + 1, BINS)
    int shift, bits;
};
template <class I> __device__ __forceinline__ int key_at(const Sort &k, int n) {
    if (!k.tokens) return k.keys[n];
    const long long t = token_at<I>(k.tokens, n);
    return t >= 0 && t < k.V ? (int)t : k.V;
}
template <class I, int ROUNDS> __global__ __launch_bounds__(SORT_THREADS) void count(const Sort k) {
    __shared__ int bin[BINS];
    bin[threadIdx.x] = 0;
    __syncthreads();
    const int mask = (1 << k.bits) - 1;
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {
        const long long n = (long long)blockIdx.x * (ROUNDS * SORT_THREADS) + j * SORT_THREADS + threadIdx.x;
        if (n < k.count) atomicAdd(&bin[key_at<I>(k, (int)n) >> k.shift & mask], 1);          // (whole numbers: the order is nothing)
    }
    __syncthreads();
    k.counts[(size_t)blockIdx.x * BINS + threadIdx.x] = bin[threadIdx.x];
}

// Many tiles' counts turned into those of the tiles before, with all tiles' behind the last: 64 digits per workgroup, its wavefronts a share of the tiles each.  Few
// tiles' are added up by every tile for itself, which saves the launch (the whole gradient of 2^17, 2^18, 2^20, 2^24 places of 8 channels by 32, 64, 256, 4096 tiles, so and with
// this launch: 66 and 68 us, 78 and 77, 187 and 159, 6991 and 1872).
constexpr int MANY = 48;
static __global__ __launch_bounds__(SORT_THREADS) void sum_tiles(int *counts, int tiles) {
    __shared__ int share[SORT_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (tiles + SORT_WAVES - 1) / SORT_WAVES, from = min(wave * per, tiles), to = min(from + per, tiles);
    int *row = counts + blockIdx.x * 64 + lane, s = 0;
#pragma unroll 8
    for (int t = from; t < to; t++) s += row[(size_t)t * BINS];
    share[wave][lane] = s;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; w++) before += share[w][lane];
    for (int t0 = from; t0 < to; t0 += 8) {
        int n[8];
#pragma unroll
        for (int j = 0; j < 8; j++) n[j] = t0 + j < to ? row[(size_t)(t0 + j) * BINS] : 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            if (t0 + j < to) row[(size_t)(t0 + j) * BINS] = before;
            before += n[j];
        }
    }
    if (wave == SORT_WAVES - 1) row[(size_t)tiles * BINS] = before;
}

struct SortLds {
    int base[BINS];                           // where the tile's first place of a digit goes
    int wave_sum[SORT_WAVES];
    unsigned short seen[SORT_WAVES][BINS];    // places of a digit in a wavefront, then in those before it
};
// an exclusive sum over the workgroup's 1024 values
__device__ __forceinline__ int sum_before(SortLds &m, int v) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int o = __shfl_up(s, d);
        s += lane >= d ? o : 0;
    }
    if (lane == 63) m.wave_sum[wave] = s;
    __syncthreads();
    int before = 0;
    for (int w = 0; w < wave; w++) before += m.wave_sum[w];
    return before + s - v;
}
// One tile's stable ranks by digit: keys[j] is place (wave * ROUNDS + j) * 64 + lane of it, `there` of them exist.  rank[j]: the places of the same digit before it
// in its wavefront; seen: those in the wavefronts before.  total: of digit threadIdx.x in the tile.
template <int ROUNDS> __device__ __forceinline__ void ranks(SortLds &m, const int (&digit)[ROUNDS], const bool (&there)[ROUNDS], int bits, int (&rank)[ROUNDS], int &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++) m.seen[w][threadIdx.x] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {
        unsigned long long same = __ballot(there[j]);
        for (int b = 0; b < bits; b++) {
            const unsigned long long set = __ballot(digit[j] >> b & 1);
            same &= digit[j] >> b & 1 ? set : ~set;
        }
        const int before = __popcll(same & ((1ull << lane) - 1));
        if (there[j]) {
            rank[j] = m.seen[wave][digit[j]] + before;
            // (the digit's last place in this round, after all of them have read: a wavefront's LDS accesses are in order)
            if (__popcll(same >> lane) == 1) m.seen[wave][digit[j]] = (unsigned short)(rank[j] + 1);
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; w++) {
        const int n = m.seen[w][threadIdx.x];
        m.seen[w][threadIdx.x] = (unsigned short)total;
        total += n;
    }
}
template <class I, int ROUNDS> __global__ __launch_bounds__(SORT_THREADS) void scatter(const Sort k, int tiles) {
    __shared__ SortLds m;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mask = (1 << k.bits) - 1;
    int key[ROUNDS], place[ROUNDS], digit[ROUNDS], rank[ROUNDS], total;
    bool there[ROUNDS];
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {
        const long long n = (long long)blockIdx.x * (ROUNDS * SORT_THREADS) + wave * (64 * ROUNDS) + j * 64 + lane;
        there[j] = n < k.count;
        key[j] = there[j] ? key_at<I>(k, (int)n) : 0;
        place[j] = k.tokens || !there[j] ? (int)n : k.places[n];
        digit[j] = key[j] >> k.shift & mask;
        rank[j] = 0;
    }
    // of digit threadIdx.x: in the tiles before, and in all
    int before = 0, all = 0;
    if (tiles > MANY) {
        before = k.counts[(size_t)blockIdx.x * BINS + threadIdx.x];
        all = k.counts[(size_t)tiles * BINS + threadIdx.x];
    } else {
        for (int t0 = 0; t0 < tiles; t0 += 8) {
            int n[8];
#pragma unroll
            for (int j = 0; j < 8; j++) n[j] = t0 + j < tiles ? k.counts[(size_t)(t0 + j) * BINS + threadIdx.x] : 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                before += t0 + j < (int)blockIdx.x ? n[j] : 0;
                all += n[j];
            }
        }
    }
    m.base[threadIdx.x] = sum_before(m, all) + before;
    ranks(m, digit, there, k.bits, rank, total);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ROUNDS; j++)
        if (there[j]) {
            const int to = m.base[digit[j]] + m.seen[wave][digit[j]] + rank[j];
            k.to_keys[to] = key[j];
            k.to_places[to] = place[j];
        }
}
// up to one tile: every pass in one workgroup, and the zeros of the whole table in those behind it
template <class I, class E> __global__ __launch_bounds__(SORT_THREADS) void sort_few(const Sort k, int passes, const Zeros zeros) {
    __shared__ SortLds m;
    constexpr int ROUNDS = TILE / SORT_THREADS;
    __shared__ int keys[TILE], places[TILE];
    if (blockIdx.x > 0) {
        put_zeros<E>(zeros, (size_t)(blockIdx.x - 1) * (SORT_THREADS / 256) + (threadIdx.x >> 8));
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, mask = (1 << k.bits) - 1;
    for (int p = 0; p < passes; p++) {
        int key[ROUNDS], place[ROUNDS], digit[ROUNDS], rank[ROUNDS], total;
        bool there[ROUNDS];
#pragma unroll
        for (int j = 0; j < ROUNDS; j++) {
            const int n = wave * (64 * ROUNDS) + j * 64 + lane;
            there[j] = n < k.count;
            key[j] = !there[j] ? 0 : p ? keys[n] : key_at<I>(k, n);
            place[j] = p ? places[n] : n;
            digit[j] = key[j] >> (p * k.bits) & mask;
            rank[j] = 0;
        }
        __syncthreads();
        ranks(m, digit, there, k.bits, rank, total);
        m.base[threadIdx.x] = sum_before(m, total);
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ROUNDS; j++)
            if (there[j]) {
                const int to = m.base[digit[j]] + m.seen[wave][digit[j]] + rank[j];
                keys[to] = key[j];
                places[to] = place[j];
            }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {
        const int n = j * SORT_THREADS + threadIdx.x;
        if (n < k.count) {
            k.to_keys[n] = keys[n];
            k.to_places[n] = places[n];
        }
    }
}
// starts[v]: the first place whose token is v or later, v up to V (what has no token lies behind)
static __global__ __launch_bounds__(256) void find_starts(const int *keys, int count, int V, int *starts) {
    const int v = blockIdx.x * 256 + threadIdx.x;
    if (v > V) return;
    int lo = 0, hi = count;
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (keys[mid] < v) lo = mid + 1;
        else hi = mid;
    }
    starts[v] = lo;
}

// ---- sums
constexpr int CHUNK = 64, AHEAD = 8;          // the most places of a chunk, and those asked for together
// A chunk is worked through one place after the other, so few places are cut finer, until there are enough to fill the machine; many are better off with fewer parts to join
// (the whole gradient of 2^9 places of 512 channels by chunks of 8, 16, 32, 64: 22, 24, 28, 37 us, 2^14 53, 53, 53, 59, 2^17 95, 86, 81, 77).
constexpr int chunk_of(long long count, int C) {
    count *= (C + 1023) / 1024;
    return count <= 1 << 12 ? 8 : count <= 1 << 14 ? 16 : count <= 1 << 16 ? 32 : CHUNK;
}
struct Gradient {
    int count, V, C, slices, chunk, chunks;   // slices: of the channels, one per workgroup
    long long gs;                             // gout's row stride
    float scale;
    const int *keys, *places;
    const void *gout;
    float *parts;                             // (chunks, 2, C): sums of a chunk's first token where it began before, and of its last where it goes on behind
    void *out;
};
template <class T, int W> __device__ __forceinline__ void put_row(const Gradient &k, int v, int c, float (&s)[W]) {
#pragma unroll
    for (int w = 0; w < W; w++) s[w] *= k.scale;
    store_vec(static_cast<T *>(k.out) + (size_t)v * k.C + c, s);
}
// a chunk's tokens, W channels per lane
template <class T, int W> __device__ __forceinline__ void sum_chunk(const Gradient &k, int chunk, int c) {
    __shared__ int keys[CHUNK + 2], places[CHUNK];          // keys[0], keys[n + 1]: the neighbours'
    const int p0 = chunk * k.chunk, n = min(k.chunk, k.count - p0);
    if ((int)threadIdx.x < k.chunk + 2) {
        const int p = p0 - 1 + (int)threadIdx.x;
        keys[threadIdx.x] = p >= 0 && p < k.count ? k.keys[p] : -1;
        if (threadIdx.x < n) places[threadIdx.x] = k.places[p0 + threadIdx.x];
    }
    __syncthreads();
    if (c >= k.C) return;
    float s[W];
    int begun = 0;                            // where the token in hand begins
    for (int g = 0; g < n; g += AHEAD) {
        float v[AHEAD][W];
#pragma unroll
        for (int j = 0; j < AHEAD; j++) load_vec(static_cast<const T *>(k.gout) + places[min(g + j, n - 1)] * k.gs + c, v[j]);
#pragma unroll
        for (int j = 0; j < AHEAD; j++) {
            const int at = g + j, key = __builtin_amdgcn_readfirstlane(keys[min(at, n - 1) + 1]);
            if (at >= n || key == k.V) break;
            if (at == 0 || key != keys[at]) {
                begun = at;
#pragma unroll
                for (int w = 0; w < W; w++) s[w] = 0.f;
            }
#pragma unroll
            for (int w = 0; w < W; w++) s[w] += v[j][w];
            const bool ends = keys[at + 2] != key;
            if (!ends && at + 1 < n) continue;
            const bool before = begun == 0 && keys[0] == key;
            if (before || !ends) {
                float *to = k.parts + ((size_t)chunk * 2 + !before) * k.C + c;
#pragma unroll
                for (int w = 0; w < W; w++) to[w] = s[w];
            } else {
                put_row<T>(k, key, c, s);
            }
        }
    }
}
template <class T, class E, int W> __global__ __launch_bounds__(256) void sums(const Gradient k, const Zeros zeros) {
    const long long work = (long long)k.chunks * k.slices;
    if ((long long)blockIdx.x < work) sum_chunk<T, W>(k, blockIdx.x / k.slices, (int)((blockIdx.x % k.slices) * 256 + threadIdx.x) * W);
    else put_zeros<E>(zeros, blockIdx.x - work);
}
// a token that goes on behind the chunk it begins in: its sums over the chunks, in their order
template <class T, int W> __global__ __launch_bounds__(256) void join(const Gradient k) {
    const int chunk = blockIdx.x, last = (chunk + 1) * k.chunk - 1, c = (blockIdx.y * 256 + threadIdx.x) * W;
    const int key = k.keys[last];
    if (key == k.V || k.keys[last + 1] != key || (chunk > 0 && k.keys[chunk * k.chunk - 1] == key) || c >= k.C) return;
    // the last chunk that begins with it: strides that double until they leave it, then halve
    int end = chunk + 1, stride = 1;
    auto has = [&](int j) { return j < k.chunks && k.keys[j * k.chunk] == key; };
    while (has(end + stride)) {
        end += stride;
        stride *= 2;
    }
    for (; stride > 0; stride /= 2)
        if (has(end + stride)) end += stride;
    float s[W];
    load_vec(k.parts + ((size_t)chunk * 2 + 1) * k.C + c, s);
    for (int j = chunk + 1; j <= end; j += AHEAD) {
        float v[AHEAD][W];
#pragma unroll
        for (int q = 0; q < AHEAD; q++) load_vec(k.parts + (size_t)min(j + q, end) * 2 * k.C + c, v[q]);
#pragma unroll
        for (int q = 0; q < AHEAD; q++)
#pragma unroll
            for (int w = 0; w < W; w++) s[w] += j + q <= end ? v[q][w] : 0.f;
    }
    put_row<T>(k, key, c, s);
}

// ---- launches
// Rounds of 1024 places to a tile: one, which is sooner done, as long as the tiles' counts are few (the gradient of 2^13, 2^15, 2^18, 2^20 places of 8 channels by one and by
// four: 31 and 41 us, 42 and 49, 70 and 77, 179 and 162).
static inline int rounds_of(int count) { return count <= 1 << 18 ? 1 : TILE / SORT_THREADS; }
static inline int tiles_of(int count) { return (count + rounds_of(count) * SORT_THREADS - 1) / (rounds_of(count) * SORT_THREADS); }
static inline int chunks_of(int count, int C) { return (count + chunk_of(count, C) - 1) / chunk_of(count, C); }
struct Regions { size_t keys[2], places[2], counts, starts, parts, all; };
static inline Regions regions(int count, int V, int C) {
    Regions r;
    size_t at = 0;
    auto take = [&](size_t n) { const size_t was = at; at += (n + 255) / 256 * 256; return was; };
    for (int i = 0; i < 2; i++) {
        r.keys[i] = take((size_t)count * 4);
        r.places[i] = take((size_t)count * 4);
    }
    r.counts = take(((size_t)tiles_of(count) + 1) * BINS * 4);
    r.starts = take(((size_t)V + 1) * 4);
    r.parts = take((size_t)chunks_of(count, C) * 2 * C * 4);
    r.all = at;
    return r;
}
// elements per lane: 16 bytes where rows are whole pieces, else one
template <class T, class I> static hipError_t forward_t(hipStream_t s, const Lookup &k, bool whole) {
    constexpr int W = 16 / sizeof(T);
    const size_t pieces = k.count * (whole ? k.C / W : k.C);
    const dim3 grid((unsigned)((pieces + 256 * EACH - 1) / (256 * EACH)));
    if (whole) hipLaunchKernelGGL((lookup<T, I, W>), grid, dim3(256), 0, s, k);
    else hipLaunchKernelGGL((lookup<T, I, 1>), grid, dim3(256), 0, s, k);
    return hipGetLastError();
}
template <class I, class E> static void sort(hipStream_t s, const Gradient &g, const void *tokens, char *ws, const Regions &r, int &at) {
    int bits = 1;
    while ((g.V >> bits) != 0) bits++;          // V itself is a key
    const int passes = (bits + MAX_BITS - 1) / MAX_BITS, tiles = tiles_of(g.count);
    Sort k = {};
    k.count = g.count; k.V = g.V; k.tokens = tokens;
    k.bits = (bits + passes - 1) / passes;
    k.counts = reinterpret_cast<int *>(ws + r.counts);
    auto region = [&](size_t o) { return reinterpret_cast<int *>(ws + o); };
    at = 0;
    if (g.count <= TILE) {
        constexpr int GROUPS = SORT_THREADS / 256;
        const Zeros zeros = {g.out, nullptr, g.V, g.C};
        k.to_keys = region(r.keys[0]);
        k.to_places = region(r.places[0]);
        hipLaunchKernelGGL((sort_few<I, E>), dim3((unsigned)(1 + (groups_of_zeros(g.V, g.C, sizeof(E)) + GROUPS - 1) / GROUPS)), dim3(SORT_THREADS), 0, s, k, passes, zeros);
        return;
    }
    for (int p = 0; p < passes; p++) {
        k.shift = p * k.bits;
        k.to_keys = region(r.keys[p & 1]);
        k.to_places = region(r.places[p & 1]);
        if (rounds_of(g.count) == 1) hipLaunchKernelGGL((count<I, 1>), dim3(tiles), dim3(SORT_THREADS), 0, s, k);
        else hipLaunchKernelGGL((count<I, TILE / SORT_THREADS>), dim3(tiles), dim3(SORT_THREADS), 0, s, k);
        if (tiles > MANY) hipLaunchKernelGGL(sum_tiles, dim3(BINS / 64), dim3(SORT_THREADS), 0, s, k.counts, tiles);
        if (rounds_of(g.count) == 1) hipLaunchKernelGGL((scatter<I, 1>), dim3(tiles), dim3(SORT_THREADS), 0, s, k, tiles);
        else hipLaunchKernelGGL((scatter<I, TILE / SORT_THREADS>), dim3(tiles), dim3(SORT_THREADS), 0, s, k, tiles);
        k.tokens = nullptr;
        k.keys = k.to_keys;
        k.places = k.to_places;
        at = p & 1;
    }
}
template <class T, class E, int W> static void sums_w(hipStream_t s, Gradient k, const Zeros &zeros) {
    k.slices = (k.C + 256 * W - 1) / (256 * W);
    const size_t groups = zeros.starts ? groups_of_zeros(k.V, k.C, sizeof(E)) : 0;
    hipLaunchKernelGGL((sums<T, E, W>), dim3((unsigned)((size_t)k.chunks * k.slices + groups)), dim3(256), 0, s, k, zeros);
    if (k.chunks > 1) hipLaunchKernelGGL((join<T, W>), dim3(k.chunks - 1, k.slices), dim3(256), 0, s, k);
}
template <class T> static hipError_t backward_t(hipStream_t s, Gradient k, const void *tokens, bool wide, bool whole, void *workspace) {
    char *ws = static_cast<char *>(workspace);
    const Regions r = regions(k.count, k.V, k.C);
    int at;
    typedef std::conditional_t<sizeof(T) == 2, unsigned short, unsigned> E;
    if (wide) sort<long long, E>(s, k, tokens, ws, r, at);
    else sort<int, E>(s, k, tokens, ws, r, at);
    k.keys = reinterpret_cast<int *>(ws + r.keys[at]);
    k.places = reinterpret_cast<int *>(ws + r.places[at]);
    k.parts = reinterpret_cast<float *>(ws + r.parts);
    k.chunk = chunk_of(k.count, k.C);
    k.chunks = chunks_of(k.count, k.C);
    Zeros zeros = {k.out, nullptr, k.V, k.C};
    if (k.count > TILE) {
        int *starts = reinterpret_cast<int *>(ws + r.starts);
        hipLaunchKernelGGL(find_starts, dim3(k.V / 256 + 1), dim3(256), 0, s, k.keys, k.count, k.V, starts);
        zeros.starts = starts;
    }
    if (whole) sums_w<T, E, 4>(s, k, zeros);
    else sums_w<T, E, 1>(s, k, zeros);
    return hipGetLastError();
}

}  // namespace embedding
}  // namespace wkv
