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
// the same lanes are the tokens: the recurrence takes a token's values from its lane by row broadcasts that ride on the
// multiplications, and the sums over the states come out one token per lane (reduce_row).  So nothing of a token's own
// arithmetic is done twice, and there are as many wavefronts as a quarter of the channels.  N above 16 takes J = 2 or 4
// states per lane.  B[t] and C[t] go through LDS in fp32, [state][token].
//
// That arithmetic (softplus, gate, what leaves) is done in the order of memory instead, lane 4 token + channel, so that four neighbouring lanes
// touch one line: in the order of the rows every lane of an access is an L1 access of its own, and those were what
// bounded the forward.  to_rows and to_memory are the two permutations between the orders.
//
// What bounds it: vector instructions, not the memory.  Per token, channel and state the forward takes an exponential (two issue
// slots) and four multiplications or multiply-adds, the backward an exponential and twelve; with the sums over the rows and a token's own arithmetic
// that is 165 and 472 instructions per wavefront and tile, and the vector unit is busy 83 % of the time in both (B8 T2048 D4096 N16 bf16: 455 us
// forward with checkpoints, 0.8 GB, which memory alone would take 160 us for; 1188 us backward).  The recurrence by itself has 5 and 13 of them per token,
// 80 and 208 per tile; the rest are the sums over states and channels (33 and 99 + 48) and a token's own arithmetic.
#include "common.h"
#include "row_sums.h"
#include "vec.h"

namespace wkv {
namespace scan {

constexpr int TILE = 16;                    // tokens per tile = states per lane row
constexpr int PITCH = TILE + 4;             // floats between two states' tokens in LDS: whole 16-byte pieces, every bank once
constexpr int MAX_STATES = 64, MAX_TOKEN_STRIDE = 1 << 24;       // (a tile's tokens are addressed with 32-bit byte offsets)

struct Rows {                               // (B, T, .) with a contiguous last dimension; strides in elements
    const void *p;
    long long batch, token, group;
};

struct Call {
    int B, T, D, N, G, Dg, tiles, segments, seg_tiles, seg0;      // Dg channels per group; seg0: the first segment there is work for
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
    int first, workgroups;                  // the launch's first workgroup, and of how many in all (at the end: the other operands' places cost a single token 0.2 us of 11.7)
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
// (a value the compiler does not connect with `v`: a broadcast of it is made where it is used and held in no register)
__device__ __forceinline__ float again(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

// v[i] of 16 lanes summed over the row, the sum of v[n] in lane n: each step adds two registers' halves into one.  A DPP's bank mask
// writes a register's groups of four lanes one by one, so the steps of eight and four lanes need no selection: 33 instructions
// instead of 45.  (Written out because the compiler selects; a register is not to be read by a DPP within two instructions of its
// write, which the s_nop and the order see to.)
__device__ __forceinline__ float reduce_row(float (&v)[TILE]) {
#define WKV_HALVES(a, b, c, d, e, f, g, h)                                                                               \
    asm("s_nop 1\n"                                                                                                      \
        "v_add_f32_dpp %0, %0, %0 row_ror:8 row_mask:0xf bank_mask:0x3\nv_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0xc\n" \
        "v_add_f32_dpp %1, %1, %1 row_ror:8 row_mask:0xf bank_mask:0x3\nv_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0xc\n" \
        "v_add_f32_dpp %2, %2, %2 row_ror:8 row_mask:0xf bank_mask:0x3\nv_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0xc\n" \
        "v_add_f32_dpp %3, %3, %3 row_ror:8 row_mask:0xf bank_mask:0x3\nv_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0xc"   \
        : "+v"(a), "+v"(b), "+v"(c), "+v"(d) : "v"(e), "v"(f), "v"(g), "v"(h))
    WKV_HALVES(v[0], v[1], v[2], v[3], v[8], v[9], v[10], v[11]);
    WKV_HALVES(v[4], v[5], v[6], v[7], v[12], v[13], v[14], v[15]);
#undef WKV_HALVES
    const uint64_t m2 = 0xccccccccccccccccull, m1 = 0xaaaaaaaaaaaaaaaaull;      // the lanes whose token has the bit
    asm("s_nop 1\n"
        "v_add_f32_dpp %0, %0, %0 row_ror:12 row_mask:0xf bank_mask:0x5\nv_add_f32_dpp %0, %4, %4 row_ror:4 row_mask:0xf bank_mask:0xa\n"
        "v_add_f32_dpp %1, %1, %1 row_ror:12 row_mask:0xf bank_mask:0x5\nv_add_f32_dpp %1, %5, %5 row_ror:4 row_mask:0xf bank_mask:0xa\n"
        "v_add_f32_dpp %2, %2, %2 row_ror:12 row_mask:0xf bank_mask:0x5\nv_add_f32_dpp %2, %6, %6 row_ror:4 row_mask:0xf bank_mask:0xa\n"
        "v_add_f32_dpp %3, %3, %3 row_ror:12 row_mask:0xf bank_mask:0x5\nv_add_f32_dpp %3, %7, %7 row_ror:4 row_mask:0xf bank_mask:0xa\n"
        "v_add_f32_dpp %0, %0, %0 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        "v_add_f32_dpp %2, %2, %2 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        "v_add_f32_dpp %1, %1, %1 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        "v_add_f32_dpp %3, %3, %3 quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf\n"
        "v_cndmask_b32_e64 %0, %0, %2, %8\n"
        "v_cndmask_b32_e64 %1, %1, %3, %8\n"
        "s_nop 1\n"
        "v_add_f32_dpp %0, %0, %0 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
        "v_add_f32_dpp %1, %1, %1 quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf\n"
        "v_cndmask_b32_e64 %0, %0, %1, %9"
        : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]) : "v"(v[4]), "v"(v[5]), "v"(v[6]), "v"(v[7]), "s"(m2), "s"(m1));
    return v[0];
}

// v[i] summed over the wavefront's four rows: out[i] holds token 4 row + i.  (As a matrix product with one-hot operands, which would take the
// broadcast along, it cost more: an fp32 MFMA keeps the vector unit from issuing, 1602 us for the backward of B8 T2048 D4096 against 1203.)
typedef float f4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f4 reduce_rows(const float (&v)[TILE]) {
    float a[8];
    f4 out;
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
    return out;
}
// v += (lane I of every row of w) u.  (The compiler makes the broadcast a move of its own here.  The s_nop: a register is not to be read by a DPP
// within two instructions of its write.)
template <int I> __device__ __forceinline__ void add_lane(float &v, float w, float u) {
    asm("s_nop 1\nv_fmac_f32_dpp %0, %1, %2 row_newbcast:%3 row_mask:0xf bank_mask:0xf" : "+v"(v) : "v"(w), "v"(u), "n"(I));
}

// log(1 + e^v): e^v with what v log2(e) rounds away, the logarithm with what 1 + e^v does
__device__ __forceinline__ float softplus(float v) {
    const float c = fminf(fmaxf(v, -100.f), 20.f), t = c * LOG2E, low = fmaf(c, 1.925963033e-8f, fmaf(c, LOG2E, -t));
    float e = exp2_fast(t);
    e = fmaf(e, low * LN2, e);
    const float u = 1.f + e, s = fmaf(__builtin_amdgcn_logf(u), LN2, (e - (u - 1.f)) * __builtin_amdgcn_rcpf(u));
    return v <= 20.f ? s : v;
}
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + exp2_fast(-LOG2E * v)); }
// A as the exponentials of two take it.  An infinite one becomes the largest number: times a step of zero, as of a token that is not there, it is to be zero.
__device__ __forceinline__ float octaves(float a) {
    a *= LOG2E;
    return fabsf(a) < INFINITY || a != a ? a : copysignf(3.40282347e38f, a);
}

// Workgroups are handed to the eight XCDs in turn: neighbours in channels, which share lines of the streams and all of B
// and C, are given to one of them.
__device__ __forceinline__ int xcd_order(int i, int n) {
    const int each = n >> 3;
    return i < each << 3 ? (i & 7) * each + (i >> 3) : i;
}

// Streams are read and written by buffer instructions from a base that moves on with the tile: a lane's offset is the same for every
// tile, what is not there (past the sequence's end, past the channels) is at NOWHERE, read as zero and not written.  Without
// branches around them the loads of the next tile can stay in flight over a tile, and no wait for them waits for a store.
typedef __amdgpu_buffer_rsrc_t Buffer;
constexpr unsigned NOWHERE = 0x80000000u;
__device__ __forceinline__ Buffer buffer_at(const void *p) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, (int)NOWHERE, 0x00027000);
}
template <class T> __device__ __forceinline__ float buffer_load(Buffer b, unsigned at) {
    if constexpr (sizeof(T) == 4) return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(b, (int)at, 0, 0));
    else return to_float(__builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(b, (int)at, 0, 0)));
}
template <class T> __device__ __forceinline__ void buffer_store(Buffer b, unsigned at, float v) {
    const T t = from_float<T>(v);
    if constexpr (sizeof(T) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, t), b, (int)at, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(__builtin_bit_cast(unsigned short, t), b, (int)at, 0, 0);
}

// an operand with strides: where the tile at hand begins, and a lane's element from there
template <class T> struct Stream {
    const char *at;                // of the workgroup's channels
    int step;                      // from a tile to the next (below 2^31 by MAX_TOKEN_STRIDE)
    unsigned lane;
    __device__ __forceinline__ Stream(const void *p, long long offset, long long token, int own, int n, int tile)          // n, own: the lane's token and channel
        : at(static_cast<const char *>(p) + (offset + tile * TILE * token) * (long long)sizeof(T)), step((int)(TILE * token * (long long)sizeof(T))),
          lane((unsigned)((n * token + own) * sizeof(T))) {}
    __device__ __forceinline__ float load(bool in) const { return buffer_load<T>(buffer_at(at), in ? lane : NOWHERE); }
    __device__ __forceinline__ void next() { at += step; }
    __device__ __forceinline__ void back() { at -= step; }
};
// the same of all contiguous (B, T, D) operands and results
template <class T> struct Packed {
    long long at;
    int step;
    unsigned lane;
    __device__ __forceinline__ Packed(long long offset, int D, int own, int n, int tile)
        : at((offset + (long long)tile * TILE * D) * (long long)sizeof(T)), step(TILE * D * (int)sizeof(T)), lane((unsigned)((n * D + own) * sizeof(T))) {}
    __device__ __forceinline__ float load(const void *p, bool in) const { return buffer_load<T>(buffer_at(static_cast<const char *>(p) + at), in ? lane : NOWHERE); }
    __device__ __forceinline__ void store(void *p, bool in, float v) const { buffer_store<T>(buffer_at(static_cast<char *>(p) + at), in ? lane : NOWHERE, v); }
    __device__ __forceinline__ void next() { at += step; }
    __device__ __forceinline__ void back() { at -= step; }
};

// Where a workgroup is, and the B and C of its tiles on their way through LDS
template <class T, int J, int WAVES, bool NEEDS_B, bool NEEDS_C>
struct Work {
    static constexpr int THREADS = 64 * WAVES, CHANNELS = 4 * WAVES, STATES = 16 * J;
    static constexpr int PIECES = (TILE * STATES + THREADS - 1) / THREADS;
    const Call &k;
    int tid, row, n, wave, own, b, g, ct, seg, channel, len, first, last, end;      // own: the row's channel within the workgroup's, channel: within all D
    int token, other, mine;                                                         // in the order of memory: the lane's token, its channel likewise
    bool live, mine_live;                                                           // they exist
    int from_row, from_memory;
    unsigned at_b[PIECES], at_c[PIECES];
    float pb[PIECES], pc[PIECES];
    const char *from_b, *from_c;                // of the tile that fetch takes next

    __device__ __forceinline__ Work(const Call &k_) : k(k_) {
        tid = threadIdx.x;
        wave = tid >> 6; row = (tid >> 4) & 3; n = tid & 15;
        const int cts = (k.Dg + CHANNELS - 1) / CHANNELS;
        int i = xcd_order(k.first + (int)blockIdx.x, k.workgroups);
        ct = i % cts; i /= cts;
        g = i % k.G; i /= k.G;
        b = i % k.B; seg = k.seg0 + i / k.B;
        own = wave * 4 + row;
        live = ct * CHANNELS + own < k.Dg;
        channel = live ? base_channel() + own : 0;
        token = (tid & 63) >> 2;
        other = wave * 4 + (tid & 3);
        mine_live = ct * CHANNELS + other < k.Dg;
        mine = mine_live ? base_channel() + other : 0;
        from_memory = 4 * (n * 4 + row);
        from_row = 4 * ((tid & 3) * 16 + token);
        len = k.lengths ? min(max(k.lengths[b], 0), k.T) : k.T;
        first = seg * k.seg_tiles;
        last = min(first + k.seg_tiles, k.tiles);
        end = max(first, min(last, (len + TILE - 1) / TILE));          // first .. end: tiles with tokens, end .. last: those without
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            const int at = tid + p * THREADS, token = at / STATES, state = at % STATES;
            const bool in = token < TILE && state < k.N;
            at_b[p] = in ? (unsigned)((token * k.b.token + state) * sizeof(T)) : NOWHERE;
            at_c[p] = in ? (unsigned)((token * k.c.token + state) * sizeof(T)) : NOWHERE;
        }
    }
    __device__ __forceinline__ int base_channel() const { return g * k.Dg + ct * CHANNELS; }
    __device__ __forceinline__ Stream<T> stream(const Rows &r, int tile) const { return Stream<T>(r.p, b * r.batch + base_channel(), r.token, other, token, tile); }
    __device__ __forceinline__ Packed<T> packed(int tile) const { return Packed<T>((long long)b * k.T * k.D + base_channel(), k.D, other, token, tile); }
    __device__ __forceinline__ bool in(int tile) const { return mine_live && token < len - tile * TILE; }
    __device__ __forceinline__ bool exists(int tile) const { return mine_live && token < k.T - tile * TILE; }
    __device__ __forceinline__ float param(const float *p) const { return p ? p[mine] : 0.f; }
    __device__ __forceinline__ float to_rows(float v) const { return __int_as_float(__builtin_amdgcn_ds_bpermute(from_memory, __float_as_int(v))); }
    __device__ __forceinline__ float to_memory(float v) const { return __int_as_float(__builtin_amdgcn_ds_bpermute(from_row, __float_as_int(v))); }
    __device__ __forceinline__ size_t state_at(int state) const { return ((size_t)b * k.D + channel) * k.N + state; }
    // (a row without a channel has nothing, not the first channel's: what it adds to its group's gB and gC is to be zero whatever that holds)
    __device__ __forceinline__ void load_a(float (&a2)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++) a2[j] = live && n + 16 * j < k.N ? octaves(k.A[(size_t)channel * k.N + n + 16 * j]) : 0.f;
    }
    __device__ __forceinline__ void load_state(const float *s, float (&h)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++) h[j] = s && live && n + 16 * j < k.N ? s[state_at(n + 16 * j)] : 0.f;
    }
    __device__ __forceinline__ void store_state(float *s, const float (&h)[J]) const {
#pragma unroll
        for (int j = 0; j < J; j++)
            if (live && n + 16 * j < k.N) s[state_at(n + 16 * j)] = h[j];
    }
    // (. , D, 16 J) arrays: the workgroup's first channel, and the lane's element from there
    __device__ __forceinline__ Buffer wide(const float *s, size_t index) const { return buffer_at(s + (index * k.D + base_channel()) * STATES); }
    __device__ __forceinline__ unsigned wide_lane() const { return live ? (unsigned)((own * STATES + n) * 4) : NOWHERE; }
    __device__ __forceinline__ void load_wide(const float *s, size_t index, float (&h)[J]) const {
        const Buffer from = wide(s, index);
        const unsigned at = wide_lane();
#pragma unroll
        for (int j = 0; j < J; j++) h[j] = buffer_load<float>(from, at + 64 * j);
    }
    __device__ __forceinline__ void store_wide(float *s, size_t index, const float (&h)[J]) const {
        const Buffer to = wide(s, index);
        const unsigned at = wide_lane();
#pragma unroll
        for (int j = 0; j < J; j++) buffer_store<float>(to, at + 64 * j, h[j]);
    }
    // what the segments on one side make of an incoming state (or its gradient): v <- decay v + theirs.  (A > 0: a growth past 2^127 is applied in
    // two steps and to nothing not at all, since what it makes may be finite where it itself is not.)
    __device__ __forceinline__ void pass(int s, const float (&a2)[J], float (&v)[J]) const {
        const size_t at = (size_t)b * k.segments + s;
        const float dt = live ? k.seg_dt[at * k.D + channel] : 0.f;
        float theirs[J];
        load_wide(k.seg_state, at, theirs);
#pragma unroll
        for (int j = 0; j < J; j++) {
            float e = dt * a2[j];
            if (e > 127.f) {
                if (v[j] != 0.f) v[j] *= exp2_fast(e - 127.f);
                e = 127.f;
            }
            v[j] = fmaf(exp2_fast(e), v[j], theirs[j]);
        }
    }
    __device__ __forceinline__ void from(int tile) {
        from_b = static_cast<const char *>(k.b.p) + (b * k.b.batch + tile * TILE * k.b.token + g * k.b.group) * (long long)sizeof(T);
        from_c = static_cast<const char *>(k.c.p) + (b * k.c.batch + tile * TILE * k.c.token + g * k.c.group) * (long long)sizeof(T);
    }
    // a tile's B and C, `step` tokens on from there next
    __device__ __forceinline__ void fetch(int left, int step) {
        const Buffer fb = buffer_at(from_b), fc = buffer_at(from_c);
        from_b += step * k.b.token * (long long)sizeof(T);
        from_c += step * k.c.token * (long long)sizeof(T);
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            const bool there = (tid + p * THREADS) / STATES < left;
            if (NEEDS_B) pb[p] = buffer_load<T>(fb, there ? at_b[p] : NOWHERE);
            if (NEEDS_C) pc[p] = buffer_load<T>(fc, there ? at_c[p] : NOWHERE);
        }
    }
    __device__ __forceinline__ void stage(float *sb, float *sc) const {
#pragma unroll
        for (int p = 0; p < PIECES; p++) {
            const int at = tid + p * THREADS, token = at / STATES, state = at % STATES;
            if (TILE * STATES % THREADS == 0 || token < TILE) {
                if (NEEDS_B) sb[state * PITCH + token] = pb[p];
                if (NEEDS_C) sc[state * PITCH + token] = pc[p];
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

// over a channel's lanes in the order of memory
__device__ __forceinline__ float token_sum(float v) {
#pragma unroll
    for (int m = 4; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// OUT: the outputs of every token; without it a segment's summary (its state from nothing, its total step) alone
template <class T, int J, bool OUT>
__global__ __launch_bounds__(256, J == 1 ? 8 : 4) void forward(const Call k) {
    typedef Work<T, J, 4, true, OUT> W;
    __shared__ __align__(16) float bc[2][OUT ? 2 : 1][W::STATES * PITCH];
    W w(k);
    float a2[J], h[J];
    w.load_a(a2);
    const float bias = w.param(k.bias), skip = w.param(k.skip);
    const bool gated = OUT && k.z.p;
    Stream<T> sx = w.stream(k.x, w.first), sdt = w.stream(k.dt, w.first), sz = w.stream(gated ? k.z : k.x, w.first);
    Packed<T> out_at = w.packed(w.first);
    if (OUT) {
        w.load_state(k.state_in, h);
        for (int s = 0; s < w.seg; s++) w.pass(s, a2, h);
    } else {
#pragma unroll
        for (int j = 0; j < J; j++) h[j] = 0.f;
    }
    float total = 0.f, x, raw, z = 0.f;
    auto fetch = [&](int tile) {
        const bool in = w.in(tile);
        w.fetch(w.len - tile * TILE, TILE);
        x = sx.load(in);
        raw = sdt.load(in);
        if (gated) z = sz.load(in);
        sx.next(); sdt.next(); sz.next();
    };
    w.from(w.first);
    fetch(w.first);
    for (int tile = w.first; tile < w.end; tile++) {
        float *sb = bc[tile & 1][0], *sc = bc[tile & 1][OUT ? 1 : 0];
        w.stage(sb, sc);
        lds_barrier();
        const bool in = w.in(tile);
        const float xn = x, zn = z, step = in ? softplus(raw + bias) : 0.f, dt = w.to_rows(step), dtx = w.to_rows(step * x);
        fetch(tile + 1);          // (past the end: nothing is there)
        if (OUT && k.checkpoints) w.store_wide(k.checkpoints, (size_t)w.b * k.tiles + tile, h);
        float y[TILE];
#pragma unroll
        for (int j = 0; j < J; j++) {
            float vb[TILE], vc[TILE];
            w.read(sb, j, vb);
            if (OUT) w.read(sc, j, vc);
            const float dtj = again(dt), dtxj = again(dtx);
            unrolled<TILE>([&](auto i) {
                constexpr int I = decltype(i)::value;
                const float a = exp2_fast(row_lane<I>(dtj) * a2[j]);
                h[j] = fmaf(a, h[j], row_lane<I>(dtxj) * vb[I]);
                if (OUT) y[I] = j == 0 ? vc[I] * h[j] : fmaf(vc[I], h[j], y[I]);
            });
        }
        if (OUT) {
            float out = fmaf(skip, xn, w.to_memory(reduce_row(y)));
            if (gated) out *= zn * sigmoid(zn);
            out_at.store(k.y, w.exists(tile), in ? out : 0.f);
            out_at.next();
        } else {
            total += step;
        }
    }
    if (OUT) {
        for (int tile = w.end; tile < w.last; tile++, out_at.next()) out_at.store(k.y, w.exists(tile), 0.f);
        if (w.last == k.tiles) w.store_state(k.state_out, h);
    } else {
        total = token_sum(total);
        const size_t at = (size_t)w.b * k.segments + w.seg;
        w.store_wide(k.seg_state, at, h);
        if (w.mine_live && w.token == 0) k.seg_dt[at * k.D + w.mine] = total;
    }
}

// The state's gradient that a segment hands to the one before it if none comes in: the backward's summary
template <class T, int J>
__global__ __launch_bounds__(256) void backward_summary(const Call k) {
    typedef Work<T, J, 4, false, true> W;
    __shared__ __align__(16) float cs[2][W::STATES * PITCH];
    W w(k);
    float a2[J], g[J];
    w.load_a(a2);
    const float bias = w.param(k.bias);
    const bool gated = k.z.p;
    const int begin = max(w.end - 1, w.first);
    Stream<T> sdt = w.stream(k.dt, begin), sz = w.stream(gated ? k.z : k.x, begin);
    Packed<T> in_at = w.packed(begin);
#pragma unroll
    for (int j = 0; j < J; j++) g[j] = 0.f;
    float total = 0.f, raw, go, z = 0.f;
    auto fetch = [&](int tile) {
        const bool there = tile >= w.first, in = there && w.in(tile);
        w.fetch(there ? w.len - tile * TILE : 0, -TILE);
        raw = sdt.load(in);
        go = in_at.load(k.gy, in);
        if (gated) z = sz.load(in);
        sdt.back(); sz.back(); in_at.back();
    };
    w.from(begin);
    fetch(w.end - 1);
    for (int tile = w.end - 1; tile >= w.first; tile--) {
        w.stage(nullptr, cs[tile & 1]);
        lds_barrier();
        const float step = w.in(tile) ? softplus(raw + bias) : 0.f, dt = w.to_rows(step), gy = w.to_rows(gated ? go * (z * sigmoid(z)) : go);
        total += step;
        fetch(tile - 1);
#pragma unroll
        for (int j = 0; j < J; j++) {
            float vc[TILE];
            w.read(cs[tile & 1], j, vc);
            const float dtj = again(dt), gyj = again(gy);
            unrolled<TILE>([&](auto i) {
                constexpr int I = TILE - 1 - decltype(i)::value;
                g[j] = fmaf(row_lane<I>(gyj), vc[I], g[j]) * exp2_fast(row_lane<I>(dtj) * a2[j]);
            });
        }
    }
    total = token_sum(total);
    const size_t at = (size_t)w.b * k.segments + w.seg;
    w.store_wide(k.seg_state, at, g);
    if (w.mine_live && w.token == 0) k.seg_dt[at * k.D + w.mine] = total;
}

// Tiles from the last to the first.  Within a tile the state runs forward again from its checkpoint, leaving every token's decay a
// and the state before it in registers, then the gradient runs back over them.  A tile's shares of gB and gC are added up over the
// workgroup's channels in LDS after the next tile's barrier.
// Eight wavefronts share a workgroup's sums, two workgroups a compute unit (128 registers) up to 16 states; with four states per lane
// 256 registers do not hold a tile (B2 T2048 D4096 N64: 3658 us), so four wavefronts have 512 each.
constexpr int back_waves(int J) { return J == 4 ? 4 : 8; }
template <class T, int J>
__global__ __launch_bounds__(64 * back_waves(J), J == 1 ? 4 : J == 2 ? 2 : 1) void backward(const Call k) {
    constexpr int BACK_WAVES = back_waves(J);
    typedef Work<T, J, BACK_WAVES, true, true> W;
    constexpr int TURNS = J == 1 ? 2 : 1;
    __shared__ __align__(16) float bc[2][2][W::STATES * PITCH];
    __shared__ __align__(16) float part[TURNS][BACK_WAVES][2][16 * PITCH];
    W w(k);
    float a2[J], g[J], ga[J];
    w.load_a(a2);
    w.load_state(k.gstate_out, g);
    for (int s = k.segments - 1; s > w.seg; s--) w.pass(s, a2, g);
#pragma unroll
    for (int j = 0; j < J; j++) ga[j] = 0.f;
    const float bias = w.param(k.bias), skip = w.param(k.skip);
    const bool gated = k.z.p;
    float gskip = 0.f, gbias = 0.f;
    const int begin = max(w.end - 1, w.first);
    Stream<T> sx = w.stream(k.x, begin), sdt = w.stream(k.dt, begin), sz = w.stream(gated ? k.z : k.x, begin);
    Packed<T> in_at = w.packed(begin), out_at = w.packed(w.last - 1);
    // the elements of the workgroup's gB and gC: 256 of each per tile and 16 states
    auto elements = [&](int tile, int j, auto f) {
#pragma unroll
        for (int e = w.tid; e < 512; e += W::THREADS) {
            const int which = e >> 8, token = (e >> 4) & 15, state = e & 15, t = tile * TILE + token;
            const float v = f(which, token, state);
            // (behind the sequence's end a step or gradient of zero times a state or gradient that is not finite is still to be zero)
            if (t < k.T && state + 16 * j < k.N)
                (which ? k.gc_part : k.gb_part)[((((size_t)w.ct * k.B + w.b) * k.T + t) * k.G + w.g) * k.N + state + 16 * j] = t < w.len ? v : 0.f;
        }
    };
    auto add_up = [&](const float (&p)[BACK_WAVES][2][16 * PITCH], int tile, int j) {
        elements(tile, j, [&](int which, int token, int state) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < BACK_WAVES; i++) s += p[i][which][state * PITCH + token];
            return s;
        });
    };
    auto nothing = [&](int tile) {
        for (int j = 0; j < J; j++) elements(tile, j, [](int, int, int) { return 0.f; });
        const bool there = w.exists(tile);
        out_at.store(k.gx, there, 0.f);
        out_at.store(k.gdt, there, 0.f);
        if (gated) out_at.store(k.gz, there, 0.f);
        out_at.back();
    };
    for (int tile = w.last - 1; tile >= w.end; tile--) nothing(tile);
    float x, raw, go, z = 0.f, h0[J];
    auto fetch = [&](int tile) {
        const bool there = tile >= w.first, in = there && w.in(tile);
        w.fetch(there ? w.len - tile * TILE : 0, -TILE);
        x = sx.load(in);
        raw = sdt.load(in);
        go = in_at.load(k.gy, in);
        if (gated) z = sz.load(in);
        w.load_wide(k.checkpoints, (size_t)w.b * k.tiles + max(tile, w.first), h0);
        sx.back(); sdt.back(); sz.back(); in_at.back();
    };
    w.from(begin);
    fetch(w.end - 1);
    for (int tile = w.end - 1; tile >= w.first; tile--) {
        float *sb = bc[tile & 1][0], *sc = bc[tile & 1][1];
        w.stage(sb, sc);
        lds_barrier();
        const bool in = w.in(tile), there = w.exists(tile);
        const float xn = x, rawn = raw + bias, gon = go, zn = z, step = in ? softplus(rawn) : 0.f;
        const float sig = gated ? sigmoid(zn) : 1.f, gate = gated ? zn * sig : 1.f, gyn = gon * gate;
        const float dt = w.to_rows(step), dtx = w.to_rows(step * xn), gy = w.to_rows(gyn);
        float hn[J];
#pragma unroll
        for (int j = 0; j < J; j++) hn[j] = h0[j];
        fetch(tile - 1);
        if (J == 1 && tile + 1 < w.end) add_up(part[(tile + 1) & 1], tile + 1, 0);
        float y[TILE], sums[TILE], slopes[TILE], ysum = 0.f;
#pragma unroll
        for (int j = 0; j < J; j++) {
            float a[TILE], before[TILE];
            float h = hn[j];
            {
                float vb[TILE], vc[TILE];
                w.read(sb, j, vb);
                w.read(sc, j, vc);
                float gc[TILE];
                const float gy1 = again(gy), dt1 = again(dt), dtx1 = again(dtx);
                unrolled<TILE>([&](auto i) {
                    constexpr int I = decltype(i)::value;
                    before[I] = h;
                    a[I] = exp2_fast(row_lane<I>(dt1) * a2[j]);
                    h = fmaf(a[I], h, row_lane<I>(dtx1) * vb[I]);
                    y[I] = j == 0 ? vc[I] * h : fmaf(vc[I], h, y[I]);
                    gc[I] = row_lane<I>(gy1) * h;
                });
                if (j) lds_barrier();
                *reinterpret_cast<f4 *>(&part[J == 1 ? tile & 1 : 0][w.wave][1][w.n * PITCH + 4 * w.row]) = reduce_rows(gc);
            }
            if (j == J - 1) ysum = reduce_row(y);
            __builtin_amdgcn_sched_barrier(0);
            {
                float vb[TILE], vc[TILE];
                w.read(sb, j, vb);
                w.read(sc, j, vc);
                float gb[TILE], share = 0.f;          // share: a tile's of gA, so that its sum over the tokens rounds T / 16 + 16 times in a row, not T
                const float an = a2[j] * LN2, dtx2 = again(dtx);
                unrolled<TILE>([&](auto i) {
                    constexpr int I = TILE - 1 - decltype(i)::value;
                    add_lane<I>(g[j], gy, vc[I]);
                    gb[I] = row_lane<I>(dtx2) * g[j];
                    sums[I] = j == 0 ? g[j] * vb[I] : fmaf(g[j], vb[I], sums[I]);
                    g[j] *= a[I];
                    const float q = g[j] * before[I];
                    slopes[I] = j == 0 ? q * an : fmaf(q, an, slopes[I]);
                    add_lane<I>(share, dt, q);
                });
                ga[j] += share;
                *reinterpret_cast<f4 *>(&part[J == 1 ? tile & 1 : 0][w.wave][0][w.n * PITCH + 4 * w.row]) = reduce_rows(gb);
            }
            __builtin_amdgcn_sched_barrier(0);
            if (J > 1) {
                lds_barrier();
                add_up(part[0], tile, j);
            }
        }
        const float ypre = fmaf(skip, xn, w.to_memory(ysum)), u = w.to_memory(reduce_row(sums)), d = w.to_memory(reduce_row(slopes));
        const float graw = fmaf(u, xn, d) * sigmoid(rawn), gx = fmaf(u, step, gyn * skip);
        if (in) {
            gskip = fmaf(gyn, xn, gskip);
            gbias += graw;
        }
        out_at.store(k.gx, there, in ? gx : 0.f);
        out_at.store(k.gdt, there, in ? graw : 0.f);
        if (gated) out_at.store(k.gz, there, in ? gon * ypre * (sig + gate * (1.f - sig)) : 0.f);
        out_at.back();
    }
    if (J == 1 && w.end > w.first) {
        lds_barrier();
        add_up(part[w.first & 1], w.first, 0);
    }
    gskip = token_sum(gskip);
    gbias = token_sum(gbias);
    const size_t at = (size_t)w.b * k.segments + w.seg;
    if (w.live)
#pragma unroll
        for (int j = 0; j < J; j++)
            if (w.n + 16 * j < k.N) k.ga_part[(at * k.D + w.channel) * k.N + w.n + 16 * j] = ga[j];
    if (w.mine_live && w.token == 0) {
        k.gskip_part[at * k.D + w.mine] = gskip;
        k.gbias_part[at * k.D + w.mine] = gbias;
    }
    if (k.gstate_in && w.seg == 0) w.store_state(k.gstate_in, g);
}

// One token: bound by the states, read once and written once (B64 D5120: 42 MB in 12.8 us; B1 D4096: 3.5 us, a launch).  Q lanes per channel with four states each (N = 4 Q), or, for
// other N, a row of lanes as above; a lane takes NB sequences, whose loads are all in flight together, with one read of its A.  VEC: four of
// B or C are one load.  state_out may be state_in: a lane writes what it has read.
template <class T, int Q, int NB, bool VEC>
__global__ __launch_bounds__(256) void decode(const Call k) {
    constexpr int V = Q ? 4 : 1, LANES = Q ? Q : 16, STEPS = Q ? 1 : (MAX_STATES + 15) / 16;
    const int d = (int)(((long long)blockIdx.x * 256 + threadIdx.x) / LANES), lane = threadIdx.x % LANES, b0 = blockIdx.y * NB;
    if (d >= k.D) return;
    const int g = d / k.Dg;
    const float bias = k.bias ? k.bias[d] : 0.f, skip = k.skip ? k.skip[d] : 0.f;
    float x[NB], raw[NB], z[NB], y[NB], step[NB];
    bool in[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) {
        const int b = min(b0 + i, k.B - 1);
        in[i] = !k.lengths || k.lengths[b] > 0;
        x[i] = in[i] ? to_float(static_cast<const T *>(k.x.p)[b * k.x.batch + d]) : 0.f;
        raw[i] = in[i] ? to_float(static_cast<const T *>(k.dt.p)[b * k.dt.batch + d]) : 0.f;
        z[i] = in[i] && k.z.p ? to_float(static_cast<const T *>(k.z.p)[b * k.z.batch + d]) : 0.f;
        y[i] = 0.f;
    }
#pragma unroll
    for (int s = 0; s < STEPS; s++) {
        const int n = V * lane + 16 * s;
        if (n >= k.N) break;
        float a[V], h[NB][V], vb[NB][V], vc[NB][V];
        load_vec(k.A + (size_t)d * k.N + n, a);
#pragma unroll
        for (int i = 0; i < NB; i++) {
            const int b = min(b0 + i, k.B - 1);
            const T *pb = static_cast<const T *>(k.b.p) + b * k.b.batch + g * k.b.group + n, *pc = static_cast<const T *>(k.c.p) + b * k.c.batch + g * k.c.group + n;
#pragma unroll
            for (int v = 0; v < V; v++) h[i][v] = 0.f;
            if (k.state_in) load_vec(k.state_in + ((size_t)b * k.D + d) * k.N + n, h[i]);
            if constexpr (VEC) {
                load_vec(pb, vb[i]);
                load_vec(pc, vc[i]);
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) {
                    vb[i][v] = to_float(pb[v]);
                    vc[i][v] = to_float(pc[v]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NB; i++) {
            if (s == 0) step[i] = in[i] ? softplus(raw[i] + bias) : 0.f;
            const float dtx = step[i] * x[i];
            if (in[i])          // (else the state stays as it is)
#pragma unroll
                for (int v = 0; v < V; v++) {
                    h[i][v] = fmaf(exp2_fast(step[i] * (a[v] * LOG2E)), h[i][v], dtx * vb[i][v]);
                    y[i] = fmaf(vc[i][v], h[i][v], y[i]);
                }
            if (b0 + i < k.B) store_vec(k.state_out + ((size_t)(b0 + i) * k.D + d) * k.N + n, h[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < NB; i++) {
#pragma unroll
        for (int m = LANES / 2; m > 0; m >>= 1) y[i] += __shfl_xor(y[i], m);
        if (lane == 0 && b0 + i < k.B) {
            float out = fmaf(skip, x[i], y[i]);
            if (k.z.p) out *= z[i] * sigmoid(z[i]);
            static_cast<T *>(k.y)[(size_t)(b0 + i) * k.D + d] = from_float<T>(in[i] ? out : 0.f);
        }
    }
}

// ---- plans
static inline int states_per_lane(int N) { return N <= 16 ? 1 : N <= 32 ? 2 : 4; }
static inline long long workgroups(int B, int D, int G, int channels) { return (long long)B * G * ((D / G + channels - 1) / channels); }

// Segments of a sequence: as many as give every compute unit `per_cu` workgroups, of eight tiles or more (of four up to four segments).
// A cut costs a pass over the inputs without outputs, so it pays where workgroups are few: forward B1 T4096 D4096 271 us with one per compute unit,
// 221 with two, 159 with four, but B4 T777 D4096 84 us uncut and 101 in two segments; forward and backward B1 T4096 D4096 (128 workgroups of
// the backward) 847, 666 and 562 us with one, two and four of them, B1 T2048 D1536 (48) 203, 163, 132, B4 T1024 D4096 (512) 431 uncut, 487 in two.
static inline int segments_for(long long groups, int tiles, int per_cu) {
    const long long want = ((long long)per_cu * cu_count() + groups - 1) / groups;
    return (int)std::max(1ll, std::min({want, (long long)std::max(tiles / 8, std::min(4, tiles / 4)), 64ll}));
}
struct Plan { int tiles, segments, seg_tiles; };
static inline Plan plan(int B, int T, int D, int N, int G, bool backward) {
    Plan p;
    p.tiles = (T + TILE - 1) / TILE;
    const long long groups = workgroups(B, D, G, backward ? 4 * back_waves(states_per_lane(N)) : 16);
    p.segments = segments_for(groups, p.tiles, !backward || 2 * groups < cu_count() ? 4 : 2);
    p.seg_tiles = (p.tiles + p.segments - 1) / p.segments;
    p.segments = (p.tiles + p.seg_tiles - 1) / p.seg_tiles;
    return p;
}
static inline size_t rounded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
static inline size_t summary_bytes(int B, int D, int N, int segments) {
    return segments > 1 ? rounded((size_t)B * segments * D * 16 * states_per_lane(N) * 4) + rounded((size_t)B * segments * D * 4) : 0;
}
static inline size_t checkpoint_bytes(int B, int T, int D, int N) { return (size_t)B * ((T + TILE - 1) / TILE) * D * 16 * states_per_lane(N) * 4; }
static inline size_t forward_scratch(int B, int T, int D, int N, int G) { return T == 1 ? 0 : summary_bytes(B, D, N, plan(B, T, D, N, G, false).segments); }
static inline size_t backward_scratch(int B, int T, int D, int N, int G) {
    const Plan p = plan(B, T, D, N, G, true);
    const int channels = 4 * back_waves(states_per_lane(N));
    const size_t cts = (D / G + channels - 1) / channels, rows = (size_t)B * p.segments;
    return summary_bytes(B, D, N, p.segments) + 2 * rounded(cts * B * T * G * N * 4) + rounded(rows * D * N * 4) + 2 * rounded(rows * D * 4);
}

constexpr long long WORKGROUPS_PER_LAUNCH = 1 << 22;          // (a grid has fewer than 2^32 threads)
#define WKV_SCAN_J(KERNEL, GRID, BLOCK, ...)                                                             \
    do {                                                                                                 \
        const long long all_ = GRID;                                                                     \
        k.workgroups = (int)all_;                                                                        \
        for (long long at_ = 0; at_ < all_; at_ += WORKGROUPS_PER_LAUNCH) {                              \
            const dim3 grid_((unsigned)std::min(all_ - at_, WORKGROUPS_PER_LAUNCH)), block_(BLOCK);      \
            k.first = (int)at_;                                                                          \
            if (J == 1) hipLaunchKernelGGL((KERNEL<T, 1 __VA_ARGS__>), grid_, block_, 0, s, k);          \
            else if (J == 2) hipLaunchKernelGGL((KERNEL<T, 2 __VA_ARGS__>), grid_, block_, 0, s, k);     \
            else hipLaunchKernelGGL((KERNEL<T, 4 __VA_ARGS__>), grid_, block_, 0, s, k);                 \
        }                                                                                                \
    } while (0)
#define WKV_COMMA ,

template <class T> static hipError_t forward_t(hipStream_t s, Call k, void *scratch) {
    const int J = states_per_lane(k.N);
    if (k.T == 1 && !k.checkpoints) {
        const bool four = k.N % 4 == 0 && (k.N & (k.N - 1)) == 0;
        auto whole = [](const Rows &r) { return reinterpret_cast<uintptr_t>(r.p) % (4 * sizeof(T)) == 0 && r.batch % 4 == 0 && r.group % 4 == 0; };
        const bool vec = whole(k.b) && whole(k.c);
        const int lanes = four ? k.N / 4 : 16;
        const unsigned blocks = (unsigned)(((long long)k.D * lanes + 255) / 256);
        // four sequences per lane where that leaves every compute unit its wavefronts (B64 D5120: 17.2 us with one, 12.8 with four; below that
        // one token's latency counts and the lanes are spread)
        const bool many = (long long)blocks * ((k.B + 3) / 4) >= 2ll * cu_count();
#define WKV_DECODE_SCAN(Q)                                                                                                         \
    do {                                                                                                                           \
        if (many && vec) hipLaunchKernelGGL((decode<T, Q, 4, true>), dim3(blocks, (k.B + 3) / 4), dim3(256), 0, s, k);             \
        else if (many) hipLaunchKernelGGL((decode<T, Q, 4, false>), dim3(blocks, (k.B + 3) / 4), dim3(256), 0, s, k);              \
        else if (vec) hipLaunchKernelGGL((decode<T, Q, 1, true>), dim3(blocks, k.B), dim3(256), 0, s, k);                          \
        else hipLaunchKernelGGL((decode<T, Q, 1, false>), dim3(blocks, k.B), dim3(256), 0, s, k);                                  \
    } while (0)
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
    const Plan p = plan(k.B, k.T, k.D, k.N, k.G, false);
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
    const Plan p = plan(k.B, k.T, k.D, k.N, k.G, true);
    k.tiles = p.tiles; k.segments = p.segments; k.seg_tiles = p.seg_tiles;
    char *at = static_cast<char *>(scratch);
    auto take = [&](size_t floats) {
        float *f = reinterpret_cast<float *>(at);
        at += rounded(floats * 4);
        return f;
    };
    const int channels = 4 * back_waves(J);
    const size_t rows = (size_t)k.B * p.segments, cts = (k.Dg + channels - 1) / channels, vectors = (size_t)k.B * k.T * k.G * k.N;
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
    WKV_SCAN_J(backward, workgroups(k.B, k.D, k.G, channels) * p.segments, 16 * channels, );
    Sums<ToRow<T>> sums;
    sums.add((int)cts, vectors, k.gb_part, {to.gb, false});
    sums.add((int)cts, vectors, k.gc_part, {to.gc, false});
    if (rows > 1) {
        sums.add((int)rows, (size_t)k.D * k.N, k.ga_part, {to.ga, true});
        if (to.gskip) sums.add((int)rows, (size_t)k.D, k.gskip_part, {to.gskip, true});
        if (to.gbias) sums.add((int)rows, (size_t)k.D, k.gbias_part, {to.gbias, true});
    }
    sum_rows_launch(s, sums);
    return hipGetLastError();
}

}  // namespace scan
}  // namespace wkv
