// Element types of the sequence kernels: conversion to the type the arithmetic runs in and back, and
// aligned groups of V elements that move with one load or store.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

namespace sigb200 {

template <typename T> struct Element { using Acc = float; };
template <> struct Element<double> { using Acc = double; };
template <typename T> using Acc = typename Element<T>::Acc;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T narrow(Acc<T> v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ double narrow<double>(double v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// V results rounded to T; pairs of 16-bit values by one conversion.
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> narrow_pack(const Acc<T> (&v)[V]) {
    Pack<T, V> r;
    if constexpr (sizeof(T) == 2 && V % 2 == 0) {
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            if constexpr (std::is_same_v<T, __half>) {
                const __half2 two = __floats2half2_rn(v[i], v[i + 1]);
                r.v[i] = __low2half(two);
                r.v[i + 1] = __high2half(two);
            } else {
                const __nv_bfloat162 two = __floats2bfloat162_rn(v[i], v[i + 1]);
                r.v[i] = __low2bfloat16(two);
                r.v[i + 1] = __high2bfloat16(two);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = narrow<T>(v[i]);
    }
    return r;
}

template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
    return *reinterpret_cast<const Pack<T, V>*>(p);
}

template <typename T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) {
    *reinterpret_cast<Pack<T, V>*>(p) = v;
}

}  // namespace sigb200
