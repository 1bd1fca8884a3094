// rows_split.cuh -- float32 operands of the tensor cores as bfloat16 parts.
#pragma once
#include <math.h>

#include "rows_common.cuh"

namespace plr {

// Two float32 values as kParts bfloat16 each, packed as they lie in memory.  A
// part is what is left of the value, rounded to the nearest (8 significant bits;
// what would round past bfloat16's largest number is held there), so that the
// remainders are exact and three parts are the value.  The second part is at
// most 2^-8 of the first's binade and the third 2^-17: products of parts below
// the sixth are within 2^-24 of the whole, and change their sign from value to
// value.  (Cutting instead of rounding left 2^-21, always of the value's sign.)
//
// An infinity has its first part held, too, and gives NaN where it meets small
// parts: split_any is for values that may not be finite.
template <int kParts>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t (&o)[kParts]) {
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        if (i < kParts - 1) asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(b), "f"(a));
        else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[i]) : "f"(b), "f"(a));
        a -= __uint_as_float(o[i] << 16);
        b -= __uint_as_float(o[i] & 0xffff0000u);
    }
}

// 1 of their sign in place of values that are not finite, which become packed
// bfloat16; 0 when both are finite.
__device__ __forceinline__ uint32_t take_not_finite(float& a, float& b) {
    uint32_t taken = 0;
    if (fabsf(a) + fabsf(b) < INFINITY) return taken;
    if (!(fabsf(a) < INFINITY)) {
        taken = __float_as_uint(a) >> 16 | (a == a ? 0u : 0x40u);
        a = copysignf(1.f, a);
    }
    if (!(fabsf(b) < INFINITY)) {
        taken |= (__float_as_uint(b) & 0xffff0000u) | (b == b ? 0u : 0x400000u);
        b = copysignf(1.f, b);
    }
    return taken;
}

// The same of any values: one that is not finite is the last part, which meets
// only the other operand's first, and the first part a 1 of its sign, so that
// two infinities meet something, too.  Sums over an infinity come out as those of
// one product.
template <int kParts>
__device__ __forceinline__ void split_any(float a, float b, uint32_t (&o)[kParts]) {
    const uint32_t last = kParts > 1 ? take_not_finite(a, b) : 0;
    split_pair(a, b, o);
    o[kParts - 1] |= last;   // 0 so far
}

// Two parts for products with an operand of a single part, which may itself be
// infinite: both parts have the value's sign and neither is 0 where the value is
// not (2^-20 of it goes to the second), so that infinity times them is not NaN.
// The first is cut, the second rounded: off by at most 2^-16 + 2^-20.
template <bool kAny>
__device__ __forceinline__ void split_one_sign(float a, float b, uint32_t (&o)[2]) {
    const uint32_t first = kAny ? take_not_finite(a, b) : 0;
    const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
    o[0] = ua >> 16 | ub | first;   // a 1's bits are among an infinity's
    const float ra = fmaf(a, 1.f + 9.5367432e-7f, -__uint_as_float(ua)), rb = fmaf(b, 1.f + 9.5367432e-7f, -__uint_as_float(ub));
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(o[1]) : "f"(rb), "f"(ra));
}

// NaN where one of the values is not finite, else 0 (added up over many pairs).
__device__ __forceinline__ void watch(uint64_t& w, float a, float b) { w = fma2(pair_of(a, b), 0ull, w); }
__device__ __forceinline__ bool not_finite(uint64_t w) {
    float a, b;
    pair_to(w, a, b);
    return !(a + b == 0.f);
}

}  // namespace plr
