// Element types of the operators that take float32, float16 and bfloat16 tensors, and their vectors of V elements.
#pragma once
#include <hip/hip_runtime.h>

namespace raftcorr {

// V elements that are only aligned as one element is: global loads and stores take any such address, 16 bytes at a time.
template <typename T, int V> struct alignas(sizeof(T)) Vec {
    T e[V];
    __device__ __forceinline__ T& operator[](int i) { return e[i]; }
    __device__ __forceinline__ const T& operator[](int i) const { return e[i]; }
};

template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_vec(const T* p)
{
    Vec<T, V> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}

template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& v) { __builtin_memcpy(p, &v, sizeof(v)); }

template <typename T> __device__ __forceinline__ float to_float(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_float(float x) { return (T)x; }      // nearest, ties to even

}  // namespace raftcorr
