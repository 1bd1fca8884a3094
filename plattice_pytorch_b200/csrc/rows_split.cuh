// rows_split.cuh -- float32 operands of the tensor cores as bfloat16 parts.
#pragma once
#include "rows_common.cuh"

namespace plr {

// Two float32 values as kParts bfloat16 each, packed as they lie in memory.  A
// part is what is left of the value, rounded to the nearest (8 significant bits;
// what would round past bfloat16's largest number is held there), so that the
// remainders are exact and three parts are the value.  The second part is at
// most 2^-8 of the first's binade and the third 2^-17: products of parts below
// the sixth are within 2^-24 of the whole, and change their sign from value to
// value.  (Cutting instead of rounding left 2^-21, always of the value's sign.)
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

}  // namespace plr
