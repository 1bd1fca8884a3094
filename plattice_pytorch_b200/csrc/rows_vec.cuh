// rows_vec.cuh -- accesses of V neighbouring elements at a time, and labels.
#pragma once
#include "rows_common.cuh"

namespace plr {

// V elements as they lie in memory, one access of V sizeof(T) <= 16 bytes (or
// more, in pieces of 16), which the address must allow.
template <typename T, int V> struct Vec {
    static constexpr int kBytes = V * (int)sizeof(T);
    static constexpr int kPiece = kBytes < 16 ? kBytes : 16;
    struct alignas(kPiece) Raw { T e[V]; };
    Raw r;
    __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const Raw*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = r; }
    __device__ __forceinline__ float at(int i) const { return to_f32(r.e[i]); }
    __device__ __forceinline__ void set(int i, float v) { r.e[i] = from_f32<T>(v); }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < V; ++i) r.e[i] = from_f32<T>(0.f);
    }
};

// The widest access (in elements: 16 bytes, half, ... one) that rows of c
// elements and the pointers' joined bits allow.
inline int widest(int64_t c, size_t element, uintptr_t bits) {
    int v = (int)(16 / element);
    while (v > 1 && (c % v || bits % (v * element))) v >>= 1;
    return v;
}

// Labels: int64 or int32; outside 0..n-1 stands for "none" (-1 here).
struct Labels {
    const void* p;
    int wide;
    __device__ __forceinline__ int at(int64_t i, int64_t n) const {
        const int64_t v = wide ? static_cast<const long long*>(p)[i] : (int64_t)static_cast<const int*>(p)[i];
        return v >= 0 && v < n ? (int)v : -1;
    }
};

}  // namespace plr
