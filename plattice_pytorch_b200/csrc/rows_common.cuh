// rows_common.cuh -- what the row operators share: element types, loads and
// stores of 8 consecutive channels, the 8-bit row format, the activations.
//
// 8-bit rows: a [rows][c] tensor as e4m3 codes [rows][cp], cp = c rounded up
// to 32 (codes behind the last channel are 0), and one byte per 32 channels,
// 127 + s: the codes stand for code * 2^s.  2^s is the smallest power of two
// with amax <= 448 * 2^s (448: the largest e4m3 value), so nothing saturates
// (but for values next to float32's largest, held8) and a block's largest value
// keeps at least 3 mantissa bits.  A power of two
// makes code * 2^s exact in bfloat16 and float32 (4 significant bits), so a
// product of bfloat16 operands reads the checkpoint without a further
// rounding.  s is clamped to [-110, 120]: the smallest non-zero value is then
// 2^-119, a normal number in both types.  A value that is not finite becomes
// the NaN code and does not enter amax, so its neighbours keep their values.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/plattice.h"

namespace plr {

constexpr int kBlock8 = 32;          // channels that share one scale
constexpr int kScaleMin = -110, kScaleMax = 120;

__host__ __device__ inline int64_t width8(int64_t c) { return (c + kBlock8 - 1) / kBlock8 * kBlock8; }

// ------------------------------------------------------------- element types

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// The value a parameter (gain, bias) of either type holds.
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t i) {
    if (dtype == PLATTICE_F32) return static_cast<const float*>(p)[i];
    if (dtype == PLATTICE_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
    return to_f32(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
    if (dtype == PLATTICE_F32) static_cast<float*>(p)[i] = v;
    else if (dtype == PLATTICE_BF16) static_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
    else static_cast<__half*>(p)[i] = from_f32<__half>(v);
}

// 8 consecutive elements; `vec`: 16-byte accesses are aligned and all 8 exist,
// otherwise the first n (n <= 8, also <= 0) are accessed one by one and the
// others read as 0.
__device__ __forceinline__ void load8(float (&v)[8], const float* p, bool vec, int n) {
    if (vec) {
        const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? p[i] : 0.f;
    }
}

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <> struct Pair<__half> { typedef __half2 type; };
__device__ __forceinline__ float2 pair_f32(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 pair_f32(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ void pair_from(__nv_bfloat162& o, float a, float b) { o = __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ void pair_from(__half2& o, float a, float b) { o = __floats2half2_rn(a, b); }

template <typename T>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, bool vec, int n) {
    if (vec) {
        union { uint4 u; typename Pair<T>::type h[4]; } r;
        r.u = *reinterpret_cast<const uint4*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = pair_f32(r.h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.f;
    }
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8], bool vec, int n) {
    if (vec) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v[i];
    }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], bool vec, int n) {
    if (vec) {
        union { uint4 u; typename Pair<T>::type h[4]; } r;
#pragma unroll
        for (int i = 0; i < 4; ++i) pair_from(r.h[i], v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(p) = r.u;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

// ------------------------------------------------------ pairs of float32 values

// Two multiply-adds in one instruction (f32x2).
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void pair_to(uint64_t p, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t both(float a) { return pair_of(a, a); }
__device__ __forceinline__ void mul2(float& a, float& b, float x, float y) { pair_to(mul2(pair_of(a, b), pair_of(x, y)), a, b); }
__device__ __forceinline__ void add2(float& a, float& b, float x, float y) { pair_to(add2(pair_of(a, b), pair_of(x, y)), a, b); }

// 8 elements as loaded, to be widened when they are used: what a kernel holds
// while the loads of its next row are in flight.
template <typename T> struct Raw8 {
    uint4 u;
    __device__ __forceinline__ void load(const T* p, bool vec, int n) {
        if (vec) {
            u = *reinterpret_cast<const uint4*>(p);
        } else {
            union { uint4 w; T h[8]; } r;
            r.w = make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) r.h[i] = p[i];
            u = r.w;
        }
    }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
        union { uint4 w; typename Pair<T>::type h[4]; } r;
        r.w = u;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = pair_f32(r.h[i]);
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
};
template <> struct Raw8<float> {
    float v8[8];
    __device__ __forceinline__ void load(const float* p, bool vec, int n) { load8(v8, p, vec, n); }
    __device__ __forceinline__ void widen(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v8[i];
    }
};

// --------------------------------------------------------------- 8-bit rows

// NaN stays NaN in both
__device__ __forceinline__ float min_nan(float a, float b) {
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// s of a block whose largest finite magnitude is amax: amax = 1.f * 2^e needs
// 2^(e-8) when 1.f <= 1.75 (448 = 1.75 * 2^8), twice that otherwise.
__device__ __forceinline__ int block_exponent(float amax) {
    const int b = __float_as_int(amax);
    const int s = (b >> 23) - 135 + ((b & 0x7fffff) > 0x600000);
    return min(max(s, kScaleMin), kScaleMax);
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

__device__ __forceinline__ bool is_infinite(float a) { return a > 3.402823466e38f; }   // of a magnitude

// Largest finite magnitude of v (fmaxf passes over NaN by itself).  Infinities
// become NaN on the way, which is the code they get.
template <int N>
__device__ __forceinline__ float finite_amax(float (&v)[N]) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) amax = fmaxf(amax, fabsf(v[i]));
    if (is_infinite(amax)) {   // rare: look at each
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if (is_infinite(fabsf(v[i]))) v[i] = __int_as_float(0x7fffffff);
            amax = fmaxf(amax, fabsf(v[i]));
        }
    }
    return amax;
}

// The same of values that must stay: infinities are passed over in amax and
// codes_of gives them the NaN code.
template <int N>
__device__ __forceinline__ float finite_amax_of(const float (&v)[N], bool& infinite) {
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) amax = fmaxf(amax, fabsf(v[i]));
    infinite = is_infinite(amax);
    if (infinite) {
        amax = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) amax = is_infinite(fabsf(v[i])) ? amax : fmaxf(amax, fabsf(v[i]));
    }
    return amax;
}

// At the largest scale codes of 256 stand for infinity: values that would round to
// them (from 248 2^120 on) are held at the code below, within 2^-4 of them.
__device__ __forceinline__ bool largest_scale(float inv) { return inv == pow2(-kScaleMax); }
__device__ __forceinline__ float held8(float v) {
    const float most = 240.f * pow2(kScaleMax);
    return max_nan(min_nan(v, most), -most);
}

// Codes of 8 values, finite or NaN, times 2^-s (multiplying by a power of two
// is exact, so the one rounding is the conversion's).
__device__ __forceinline__ uint2 codes8_below(const float* v, float inv) {   // below the largest scale
    unsigned w[2];
    const uint64_t m = both(inv);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float2 lo, hi;
        pair_to(mul2(pair_of(v[4 * i], v[4 * i + 1]), m), lo.x, lo.y);
        pair_to(mul2(pair_of(v[4 * i + 2], v[4 * i + 3]), m), hi.x, hi.y);
        w[i] = __nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
               ((unsigned)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16);
    }
    return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ uint2 codes8(const float* v, float inv) {
    if (!largest_scale(inv)) return codes8_below(v, inv);
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = held8(v[i]);
    return codes8_below(t, inv);
}

// Codes of 8 N values that must stay.
template <int N>
__device__ __forceinline__ void codes_of(uint2 (&q)[N], const float* v, float inv, bool infinite) {
    if (!infinite && !largest_scale(inv)) {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = codes8_below(v + 8 * i, inv);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = is_infinite(fabsf(v[8 * i + j])) ? __int_as_float(0x7fffffff) : v[8 * i + j];
        q[i] = codes8(t, inv);
    }
}

__device__ __forceinline__ void values4(float* v, unsigned codes, float scale) {
    const __half2 a(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffff), __NV_E4M3));
    const __half2 b(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3));
    const float2 fa = __half22float2(a), fb = __half22float2(b);
    const uint64_t s = both(scale);
    pair_to(mul2(pair_of(fa.x, fa.y), s), v[0], v[1]);
    pair_to(mul2(pair_of(fb.x, fb.y), s), v[2], v[3]);
}

__device__ __forceinline__ float value1(uint8_t code, float scale) {
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(code, __NV_E4M3))) * scale;
}

__device__ __forceinline__ void values8(float (&v)[8], uint2 codes, float scale) {
    values4(v, codes.x, scale);
    values4(v + 4, codes.y, scale);
}

__device__ __forceinline__ float scale_of(uint8_t byte) { return pow2((int)byte - 127); }

// float16 ends at 65504; a block's largest value may round to the next code
// above it, which stays the largest number rather than becoming infinite.
template <typename T> __device__ __forceinline__ float within(float v) { return v; }
template <> __device__ __forceinline__ float within<__half>(float v) {
    return fabsf(v) <= 3.402823466e38f ? fminf(fmaxf(v, -65504.f), 65504.f) : v;
}

// -------------------------------------------------------------- activations

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal_fast(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Phi(-|z|) and exp(-z^2 / 2).  Phi(-x) = exp(-x^2 / 2) R(x) with R smooth and
// falling like 1 / x: R(x) is t times a polynomial of degree 7 in t = 1 / (1 + 0.3
// x), whose coefficients are the minimax fit of the relative error over 0 <= x <=
// 16, computed as a linear program (1.9e-7; evaluated in float32 5.2e-7, and the
// exponential's argument adds u z^2, u = 2^-24).  So the tail is good relative to
// itself as far as float32 holds it.  The product's epilogue computes this for
// every output on the way out, beside the matrix instructions.
__device__ __forceinline__ uint64_t tail2(float z0, float z1, uint64_t& e) {
    const uint64_t t = pair_of(reciprocal_fast(fmaf(0.3f, fabsf(z0), 1.f)), reciprocal_fast(fmaf(0.3f, fabsf(z1), 1.f)));
    const uint64_t z = pair_of(z0, z1);
    float x0, x1;
    pair_to(mul2(mul2(z, both(-0.72134752044448170f)), z), x0, x1);   // log2(e) / 2
    e = pair_of(exp2_fast(x0), exp2_fast(x1));
    uint64_t q = fma2(both(0.03468257764877231f), t, both(-0.15303787828018373f));
    q = fma2(q, t, both(0.1991376515281999f));
    q = fma2(q, t, both(-0.04702725808130784f));
    q = fma2(q, t, both(0.12504815173945477f));
    q = fma2(q, t, both(0.10096930636298611f));
    q = fma2(q, t, both(0.12058744223124965f));
    q = fma2(q, t, both(0.11963991150309353f));
    return mul2(mul2(q, t), e);
}

// The activation of a pair.  gelu: z Phi(z) = max(z, 0) - |z| Phi(-|z|), with
// |z| held at 16, where the tail is 0, so that an infinite z has its limit.
template <int kAct> __device__ __forceinline__ void act2(float& a, float& b) {
    if (kAct == PLATTICE_ACT_RELU) {
        a = max_nan(a, 0.f);
        b = max_nan(b, 0.f);
    } else if (kAct == PLATTICE_ACT_GELU) {
        uint64_t e;
        const uint64_t q = tail2(a, b, e);
        pair_to(fma2(pair_of(-min_nan(fabsf(a), 16.f), -min_nan(fabsf(b), 16.f)), q,
                     pair_of(fmaxf(a, 0.f), fmaxf(b, 0.f))),
                a, b);
    } else if (kAct == PLATTICE_ACT_SILU) {
        float x, y;
        pair_to(mul2(pair_of(a, b), both(-1.4426950408889634f)), x, y);
        pair_to(add2(pair_of(exp2_fast(x), exp2_fast(y)), both(1.f)), x, y);
        mul2(a, b, reciprocal_fast(x), reciprocal_fast(y));
    }
}

// d act / d z of a pair.  gelu: Phi(z) + z phi(z), z held in -16..16 (there
// both have reached their limits).
template <int kAct> __device__ __forceinline__ void slope2(float& a, float& b) {
    if (kAct == PLATTICE_ACT_RELU) {
        a = a > 0.f ? 1.f : (a == a ? 0.f : a);
        b = b > 0.f ? 1.f : (b == b ? 0.f : b);
    } else if (kAct == PLATTICE_ACT_GELU) {
        const float x = max_nan(min_nan(a, 16.f), -16.f), y = max_nan(min_nan(b, 16.f), -16.f);
        uint64_t e;
        const uint64_t q = tail2(x, y, e);
        float q0, q1, p0, p1;
        pair_to(q, q0, q1);
        pair_to(fma2(q, both(-1.f), both(1.f)), p0, p1);
        const uint64_t p = pair_of(x < 0.f ? q0 : p0, y < 0.f ? q1 : p1);   // Phi(z)
        pair_to(fma2(mul2(pair_of(x, y), both(0.39894228040143268f)), e, p), a, b);
    } else if (kAct == PLATTICE_ACT_SILU) {
        float x, y;
        const uint64_t z = pair_of(a, b);
        pair_to(mul2(z, both(-1.4426950408889634f)), x, y);
        pair_to(add2(pair_of(exp2_fast(x), exp2_fast(y)), both(1.f)), x, y);
        const uint64_t s = pair_of(reciprocal_fast(x), reciprocal_fast(y));
        // s (1 + z (1 - s))
        pair_to(mul2(s, fma2(z, fma2(s, both(-1.f), both(1.f)), both(1.f))), a, b);
    }
}

template <int kAct, int N> __device__ __forceinline__ void activations(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) act2<kAct>(v[i], v[i + 1]);
}
template <int kAct, int N> __device__ __forceinline__ void slopes(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 2) slope2<kAct>(v[i], v[i + 1]);
}
__device__ __forceinline__ void slope16(float (&v)[16], int act) {
    if (act == PLATTICE_ACT_RELU) slopes<PLATTICE_ACT_RELU>(v);
    else if (act == PLATTICE_ACT_GELU) slopes<PLATTICE_ACT_GELU>(v);
    else slopes<PLATTICE_ACT_SILU>(v);
}
template <int N> __device__ __forceinline__ void activate(float (&v)[N], int act) {
    if (act == PLATTICE_ACT_RELU) activations<PLATTICE_ACT_RELU>(v);
    else if (act == PLATTICE_ACT_GELU) activations<PLATTICE_ACT_GELU>(v);
    else if (act == PLATTICE_ACT_SILU) activations<PLATTICE_ACT_SILU>(v);
}

}  // namespace plr
