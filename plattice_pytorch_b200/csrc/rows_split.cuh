// rows_split.cuh -- float32 operands of the tensor cores as bfloat16 parts.
#pragma once
#include "rows_common.cuh"

namespace plr {

// A float32 value as three bfloat16 whose sum it is: each takes the leading 8
// significant bits of what is left (cut, not rounded, so that none overflows
// and the remainders are exact).  What is not finite stays in the first part.
__device__ __forceinline__ void split3(float v, __nv_bfloat16 (&o)[3]) {
    const bool fine = fabsf(v) <= 3.402823466e38f;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        // cutting a NaN's low bits could leave an infinity: round those
        const __nv_bfloat16 h = fine ? __ushort_as_bfloat16((unsigned short)(__float_as_uint(v) >> 16))
                                     : __float2bfloat16_rn(i == 0 ? v : 0.f);
        o[i] = h;
        v = fine ? v - __bfloat162float(h) : v;
    }
}

// The same of two finite values into packed parts; a value that is not finite
// makes all its products NaN (infinity minus infinity in the second part).
__device__ __forceinline__ void split3_pair(float a, float b, uint32_t (&o)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const uint32_t ua = __float_as_uint(a) & 0xffff0000u, ub = __float_as_uint(b) & 0xffff0000u;
        o[i] = (ua >> 16) | ub;
        a -= __uint_as_float(ua);
        b -= __uint_as_float(ub);
    }
}

}  // namespace plr
