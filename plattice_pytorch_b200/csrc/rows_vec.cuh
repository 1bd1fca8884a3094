// rows_vec.cuh -- accesses of V neighbouring elements at a time, and labels.
#pragma once
#include <type_traits>

#include "rows_common.cuh"

namespace plr {

// V elements as they lie in memory, one access of V sizeof(T) <= 16 bytes (or
// more, in pieces of 16), which the address must allow.  Held in whole registers:
// a pair of 16-bit elements is one.
template <typename T, int V> struct Vec {
    static constexpr int kBytes = V * (int)sizeof(T), kPiece = kBytes < 16 ? kBytes : 16;
    static constexpr int kWords = (kBytes + 3) / 4;
    typedef typename std::conditional<kBytes == 2, uint16_t, uint32_t>::type Word;
    struct alignas(kPiece) Raw { Word w[kWords]; };
    Raw r;
    __device__ __forceinline__ void load(const T* p) { r = *reinterpret_cast<const Raw*>(p); }
    __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = r; }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) r.w[i] = 0;
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
        else if constexpr (kBytes == 2) return to_f32(bits(r.w[0]));
        else if constexpr (std::is_same<T, __nv_bfloat16>::value)
            return __uint_as_float(i % 2 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
        else return to_f32(bits((uint16_t)(r.w[i / 2] >> (i % 2 * 16))));
    }
    __device__ __forceinline__ void from(const float (&v)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < V; ++i) r.w[i] = __float_as_uint(v[i]);
        } else if constexpr (kBytes == 2) {
            const T t = from_f32<T>(v[0]);
            r.w[0] = *reinterpret_cast<const uint16_t*>(&t);
        } else {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                typename Pair<T>::type t;
                pair_from(t, v[i], v[i + 1]);
                r.w[i / 2] = *reinterpret_cast<const uint32_t*>(&t);
            }
        }
    }

private:
    static __device__ __forceinline__ T bits(uint16_t u) { return *reinterpret_cast<const T*>(&u); }
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
    __device__ __forceinline__ long long raw(int64_t i) const {
        return wide ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
    }
    __device__ __forceinline__ int at(int64_t i, int64_t n) const {
        const int64_t v = raw(i);
        return v >= 0 && v < n ? (int)v : -1;
    }
};

}  // namespace plr
