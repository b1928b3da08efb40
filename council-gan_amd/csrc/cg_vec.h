// Element types and row-chunk access of the channel-MLP operators (channel_mlp.hip, gated.hip): fp32, fp16 and bf16 tensors whose
// rows may start at any element (an odd row length).  gfx950 loads and stores 16 bytes from any address the element type allows
// (unaligned access mode of the HSA ABI), so a chunk is one instruction on aligned and unaligned rows alike; only the last,
// partial chunk of a row goes element by element.
#pragma once
#include "cg_common.h"

typedef _Float16 cg_h16;
typedef __bf16 cg_b16;

template <typename T> struct CgT;
template <> struct CgT<float> { static constexpr int N = 4; typedef float V __attribute__((ext_vector_type(4), aligned(4))); };
template <> struct CgT<cg_h16> { static constexpr int N = 8; typedef cg_h16 V __attribute__((ext_vector_type(8), aligned(2))); };
template <> struct CgT<cg_b16> { static constexpr int N = 8; typedef cg_b16 V __attribute__((ext_vector_type(8), aligned(2))); };

// v[0..N) = p[0..n) widened to fp32, zeros behind; n <= 0 reads nothing
template <typename T, int N = CgT<T>::N>
__device__ __forceinline__ void cg_load(const T* p, int n, float (&v)[N]) {
    constexpr int W = CgT<T>::N;
    if (n >= N) {
#pragma unroll
        for (int q = 0; q < N; q += W) {
            const typename CgT<T>::V t = *(const typename CgT<T>::V*)(p + q);
#pragma unroll
            for (int i = 0; i < W; ++i) v[q + i] = (float)t[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
}

// p[0..min(n, N)) = v rounded to T (round to nearest even: one rounding of the fp32 result)
template <typename T, int N = CgT<T>::N>
__device__ __forceinline__ void cg_store(T* p, int n, const float (&v)[N]) {
    constexpr int W = CgT<T>::N;
    if (n >= N) {
#pragma unroll
        for (int q = 0; q < N; q += W) {
            typename CgT<T>::V t;
#pragma unroll
            for (int i = 0; i < W; ++i) t[i] = (T)v[q + i];
            *(typename CgT<T>::V*)(p + q) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (T)v[i];
    }
}

#define CG_DISPATCH_DT(dt, T, ...)                                        \
    do {                                                                  \
        if ((dt) == CG_DT_F32) { using T = float; __VA_ARGS__; }          \
        else if ((dt) == CG_DT_F16) { using T = cg_h16; __VA_ARGS__; }    \
        else { using T = cg_b16; __VA_ARGS__; }                           \
    } while (0)
