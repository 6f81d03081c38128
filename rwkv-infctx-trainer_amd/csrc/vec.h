// V consecutive elements as floats: one, as many as make 4 or 8 bytes, or whole 16-byte pieces (p aligned to 4, 8 or 16 bytes then).
#pragma once
#include "common.h"

namespace wkv {

template <class T, int V> __device__ __forceinline__ void load_vec(const T *p, float (&o)[V]) {
    if constexpr (V == 1) {
        o[0] = to_float(*p);
    } else if constexpr (V * sizeof(T) == 4) {
        const unsigned raw = *reinterpret_cast<const unsigned *>(p);
        T e[V];
        __builtin_memcpy(e, &raw, 4);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = to_float(e[i]);
    } else if constexpr (V * sizeof(T) == 8) {
        const uint2 raw = *reinterpret_cast<const uint2 *>(p);
        T e[V];
        __builtin_memcpy(e, &raw, 8);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = to_float(e[i]);
    } else {
        constexpr int EACH = 16 / sizeof(T);
        static_assert(V % EACH == 0, "whole 16-byte pieces");
#pragma unroll
        for (int q = 0; q < V; q += EACH) {
            const uint4 raw = *reinterpret_cast<const uint4 *>(p + q);
            T e[EACH];
            __builtin_memcpy(e, &raw, 16);
#pragma unroll
            for (int i = 0; i < EACH; i++) o[q + i] = to_float(e[i]);
        }
    }
}
template <class T, int V> __device__ __forceinline__ void store_vec(T *p, const float (&o)[V]) {
    if constexpr (V == 1) {
        *p = from_float<T>(o[0]);
    } else if constexpr (V * sizeof(T) == 4) {
        T e[V];
#pragma unroll
        for (int i = 0; i < V; i++) e[i] = from_float<T>(o[i]);
        unsigned raw;
        __builtin_memcpy(&raw, e, 4);
        *reinterpret_cast<unsigned *>(p) = raw;
    } else if constexpr (V * sizeof(T) == 8) {
        T e[V];
#pragma unroll
        for (int i = 0; i < V; i++) e[i] = from_float<T>(o[i]);
        uint2 raw;
        __builtin_memcpy(&raw, e, 8);
        *reinterpret_cast<uint2 *>(p) = raw;
    } else {
        constexpr int EACH = 16 / sizeof(T);
#pragma unroll
        for (int q = 0; q < V; q += EACH) {
            T e[EACH];
#pragma unroll
            for (int i = 0; i < EACH; i++) e[i] = from_float<T>(o[q + i]);
            uint4 raw;
            __builtin_memcpy(&raw, e, 16);
            *reinterpret_cast<uint4 *>(p + q) = raw;
        }
    }
}

}  // namespace wkv
