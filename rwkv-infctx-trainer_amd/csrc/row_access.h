// Accesses to rows that may not be there.
#pragma once
#include "common.h"

namespace wkv {

// A row's V elements of one lane as they lie in memory, read and written by buffer instructions whose range is a scalar: of a row that is not there it
// is nothing, which reads as zero and is not written.  So no branch stands between a load and its use a group of tokens later.
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
template <class T> struct is_bf16 { static constexpr bool value = false; };
template <> struct is_bf16<bf16> { static constexpr bool value = true; };
template <int BYTES> struct RawOf;
template <> struct RawOf<2> { typedef unsigned short type; };
template <> struct RawOf<4> { typedef unsigned type; };
template <> struct RawOf<8> { typedef u2 type; };
template <> struct RawOf<16> { typedef u4 type; };
template <class T, int V> struct Row {
    typedef typename RawOf<V * sizeof(T)>::type Raw;
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t range(const void *p, bool there) {
        return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), (short)0, there ? (int)0x80000000u : 0, 0x00027000);
    }
    // `at` is the lane's offset in bytes and `row` the row's; the range covers their sum
    static __device__ __forceinline__ Raw load(__amdgpu_buffer_rsrc_t b, int at, int row) {
        if constexpr (sizeof(Raw) == 2) return __builtin_amdgcn_raw_buffer_load_b16(b, at, row, 0);
        else if constexpr (sizeof(Raw) == 4) return __builtin_amdgcn_raw_buffer_load_b32(b, at, row, 0);
        else if constexpr (sizeof(Raw) == 8) return __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b64(b, at, row, 0));
        else return __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b128(b, at, row, 0));
    }
    static __device__ __forceinline__ Raw packed(const float (&v)[V]) {
        Raw raw;
        if constexpr (is_bf16<T>::value && V % 2 == 0) {          // a pair in one instruction (rounded one by one it takes four)
            unsigned w[V / 2];
#pragma unroll
            for (int i = 0; i < V / 2; i++) w[i] = bf16_pack2(v[2 * i], v[2 * i + 1]);
            __builtin_memcpy(&raw, w, sizeof(raw));
        } else {
            T e[V];
#pragma unroll
            for (int i = 0; i < V; i++) e[i] = from_float<T>(v[i]);
            __builtin_memcpy(&raw, e, sizeof(raw));
        }
        return raw;
    }
    static __device__ __forceinline__ void store(__amdgpu_buffer_rsrc_t b, int at, int row, const float (&v)[V]) {
        const Raw raw = packed(v);
        if constexpr (sizeof(Raw) == 2) __builtin_amdgcn_raw_buffer_store_b16(raw, b, at, row, 0);
        else if constexpr (sizeof(Raw) == 4) __builtin_amdgcn_raw_buffer_store_b32(raw, b, at, row, 0);
        else if constexpr (sizeof(Raw) == 8) __builtin_amdgcn_raw_buffer_store_b64(raw, b, at, row, 0);
        else __builtin_amdgcn_raw_buffer_store_b128(raw, b, at, row, 0);
    }
    static __device__ __forceinline__ Raw load(const T *p, bool there, int at) { return load(range(p, there), at, 0); }
    static __device__ __forceinline__ void store(T *p, bool there, int at, const float (&v)[V]) { store(range(p, there), at, 0, v); }
    static __device__ __forceinline__ void floats(const Raw &raw, float (&o)[V]) {
        T e[V];
        __builtin_memcpy(e, &raw, sizeof(raw));
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = to_float(e[i]);
    }
};

}  // namespace wkv
