// Element types of the packed-layer operators: conversion to and from float32 (rounded once, to nearest even) and loads
// of several elements at once.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dllm_hip {

enum ElementType : int64_t { kFloat32 = 0, kBFloat16 = 1, kFloat16 = 2 };

inline size_t element_bytes(int64_t dtype) { return dtype == kFloat32 ? 4 : 2; }

template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
    T v[N];
};

// N elements of p as floats. N * sizeof(T) is a load's width where p is aligned to it, else N is 1.
template <typename T, int N>
__device__ __forceinline__ void load_as_float(const T* p, float (&out)[N]) {
    const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<float>(a.v[i]);
}

template <typename T, int N>
__device__ __forceinline__ void store_from_float(T* p, const float (&in)[N]) {
    Pack<T, N> a;
#pragma unroll
    for (int i = 0; i < N; ++i) a.v[i] = static_cast<T>(in[i]);
    *reinterpret_cast<Pack<T, N>*>(p) = a;
}

template <typename T>
constexpr int kChunk = 16 / sizeof(T);  // elements of a 16-byte access

inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

}  // namespace dllm_hip
