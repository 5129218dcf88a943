// V consecutive values of type T (float or raw bf16; V = 8, 4 or 1) moved in 16- or 8-byte accesses. The address is aligned to
// min(16, V sizeof(T)) bytes; vec_width() picks V from what a call's addresses and row length allow.
#pragma once
#include "common.h"

// V consecutive values as they lie in memory
template <typename T, int V> struct Vec {
    static constexpr int N = V * (int)sizeof(T) / 16;   // 16-byte pieces; 0: one 8-byte piece (bf16 x 4); V = 1: one value
    uint4 r[N ? N : 1];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (V == 1) r[0].x = __float_as_uint(OpT<T>::to(p[0]));
        else if constexpr (N == 0) { const uint2 u = *reinterpret_cast<const uint2*>(p); r[0].x = u.x; r[0].y = u.y; }
        else
#pragma unroll
            for (int i = 0; i < N; ++i) r[i] = reinterpret_cast<const uint4*>(p)[i];
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
        if constexpr (V == 1) v[0] = __uint_as_float(r[0].x);
        else {
            const unsigned* w = reinterpret_cast<const unsigned*>(r);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                if constexpr (sizeof(T) == 4) v[e] = __uint_as_float(w[e]);
                else v[e] = __uint_as_float(e & 1 ? w[e >> 1] & 0xffff0000u : w[e >> 1] << 16);
            }
        }
    }
};
template <typename T, int V> __device__ __forceinline__ void vec_store(T* p, const float (&v)[V]) {
    if constexpr (V == 1) p[0] = OpT<T>::from(v[0]);
    else if constexpr (sizeof(T) == 2 && V == 8) {
        *reinterpret_cast<uint4*>(p) = make_uint4(f2bf2(v[0], v[1]), f2bf2(v[2], v[3]), f2bf2(v[4], v[5]), f2bf2(v[6], v[7]));
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) { const float q[4] = {v[i], v[i + 1], v[i + 2], v[i + 3]}; Op4<T>::store(p + i, q); }
    }
}


// 16-byte accesses of the narrower type where rows of n values and every address allow them, else 4 values, else one by one
static inline int vec_width(long long n, const void* a, int a_bf16, const void* b, int b_bf16) {
    for (int v = a_bf16 && b_bf16 ? 8 : 4; v >= 4; v >>= 1) {
        const size_t ma = (a_bf16 ? 2 * v : 16) - 1, mb = (b_bf16 ? 2 * v : 16) - 1;
        if (n % v == 0 && !((size_t)a & ma) && !((size_t)b & mb)) return v;
    }
    return 1;
}
