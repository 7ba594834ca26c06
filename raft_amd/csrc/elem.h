// Element types of the operators that take float32, float16 and bfloat16 tensors, and their vectors of V elements.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace raftcorr {

// V elements that are only aligned as one element is: global loads and stores take any such address, 16 bytes at a time.
template <typename T, int V> struct alignas(sizeof(T)) Vec {
    T e[V];
    __device__ __forceinline__ T& operator[](int i) { return e[i]; }
    __device__ __forceinline__ const T& operator[](int i) const { return e[i]; }
};

// words of BYTES bytes that are aligned to ALIGN
template <int BYTES, int ALIGN> struct Word;
#define RAFTCORR_WORD(BYTES, ALIGN, ...) template <> struct Word<BYTES, ALIGN> { typedef __VA_ARGS__ type __attribute__((aligned(ALIGN))); }
typedef uint32_t word2 __attribute__((ext_vector_type(2)));
typedef uint32_t word4 __attribute__((ext_vector_type(4)));
RAFTCORR_WORD(16, 4, word4);
RAFTCORR_WORD(16, 2, word4);
RAFTCORR_WORD(8, 1, word2);
RAFTCORR_WORD(4, 4, uint32_t);
RAFTCORR_WORD(2, 2, uint16_t);
#undef RAFTCORR_WORD

template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_vec(const T* p)
{
    Vec<T, V> v;
    __builtin_memcpy(&v, p, sizeof(v));
    return v;
}

template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& v) { __builtin_memcpy(p, &v, sizeof(v)); }

// The same for what is read or written once and not soon again: it does not displace what the caches hold.
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_vec_once(const T* p)
{
    constexpr int B = sizeof(T) * V < 16 ? sizeof(T) * V : 16;
    typedef typename Word<B, sizeof(T)>::type W;
    Vec<T, V> v;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * V); i += B) {
        const W w = __builtin_nontemporal_load((const W*)((const char*)p + i));
        __builtin_memcpy((char*)&v + i, &w, B);
    }
    return v;
}

template <typename T, int V> __device__ __forceinline__ void store_vec_once(T* p, const Vec<T, V>& v)
{
    constexpr int B = sizeof(T) * V < 16 ? sizeof(T) * V : 16;
    typedef typename Word<B, sizeof(T)>::type W;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) * V); i += B) {
        W w;
        __builtin_memcpy(&w, (const char*)&v + i, B);
        __builtin_nontemporal_store(w, (W*)((char*)p + i));
    }
}

// Holds the compiler to the vector as it is: 16-bit values that are used again later are converted again, not kept in 32 bits each.
template <typename T, int V> __device__ __forceinline__ void keep_packed(Vec<T, V>& v)
{
    if constexpr (sizeof(T) == 2 && V == 8) {
        word4 w;
        __builtin_memcpy(&w, &v, 16);
        asm volatile("" : "+v"(w));
        __builtin_memcpy(&v, &w, 16);
    }
}

template <typename T> __device__ __forceinline__ float to_float(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T from_float(float x) { return (T)x; }      // nearest, ties to even

}  // namespace raftcorr
