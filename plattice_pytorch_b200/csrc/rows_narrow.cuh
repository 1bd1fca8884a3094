// rows_narrow.cuh -- the linear map where one side is small: at most 32 output
// channels (the projections to the filter's features and values), or few rows.
// Both read what they need once and are bound by that read; a
// 128-row tensor-memory tile would be mostly padding, and staging it costs
// more than the product.
#pragma once
#include "plattice_runtime.h"
#include "rows_common.cuh"
#include "rows_host.h"
#include "rows_narrow.h"
#include "rows_split.cuh"

namespace plr {

enum XType { kX8 = 0, kXBf16 = 1, kXHalf = 2, kXFloat = 3 };

// ------------------------------------------------------- at most 32 channels
//
// A warp takes 16 kM rows at a time and keeps their sums in registers; the
// weights lie in shared memory in the fragment order of the warp's matrix
// instruction (m16n8k16).  The sum's order is free, so lane (g, t) of a quad
// group is given 16 neighbouring channels t 16.. of each 64 instead of the
// instruction's pairs: 16 bytes of codes (32 of a 16-bit type, 64 of float32)
// per row and load, straight into the operand's registers.
//
// float32 runs as three bfloat16 parts (split_pair), six products, small first.
//
// 8-bit rows go in as float16, one conversion a pair of codes and exact, with
// their scales left out: a step then stays within a block of 32 channels (lane
// t holds t 8.. of each), whose sum is multiplied by the row's scale.  The
// weights are float16 too, each output channel's times the power of two that
// takes its largest to 2^14: 11 significant bits hold a bfloat16 weight down
// to 2^-28 of that largest, and below lose at most 2^-39 of it; a float32
// weight takes three parts.  (Widening codes to bfloat16 instead, scales
// included, took five instructions a pair: 35 against 25 us for 1048576 rows,
// 64 -> 8.)
//
// 25 us for those 1048576 rows (103 MB, 15.7 us at the copy rate), where tiles of
// 128 rows took 109.  500 instructions a block of 32 rows, issued in 65 % of the
// cycles: bound by that and by what 24 warps an SM, all that the registers leave,
// cannot hide.

template <int kXT> struct NarrowShape {
    static constexpr int kM = kXT == kX8 ? 2 : 1;                               // 16-row fragments
    static constexpr int kRaw = kXT == kX8 ? 1 : kXT == kXFloat ? 4 : 2;        // 16-byte loads per row and 64 channels
};

constexpr int kNarrowWarps = 8;
constexpr int kNarrowPitch = 33;
__host__ inline int64_t narrow_staging(int m) { return (int64_t)kNarrowWarps * 16 * m * kNarrowPitch * 4; }

// CTAs that the registers let share an SM (more would spill).
__host__ __device__ constexpr int narrow_ctas(int xt, int nf) { return xt == kXFloat || (xt == kX8 && nf > 1) ? 2 : 3; }

template <bool kHalf>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint2 b) {
    if (kHalf)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b.x), "r"(b.y));
}

// What a lane loads of 64 channels of kM x 2 rows (g and g + 8 of each fragment).
template <int kXT> struct NarrowRaw {
    uint4 v[NarrowShape<kXT>::kM][2][NarrowShape<kXT>::kRaw];
    uint8_t scale[NarrowShape<kXT>::kM][2];
};

// The same of 8-bit rows for k_narrow: 8 channels of each of the two blocks.
struct NarrowCodes {
    uint2 v[2][2][2];   // fragment, row, block
    uint8_t scale[2][2][2];
};

// Rows behind the last read the last one again (what they give is not stored),
// a missing second block reads the first: no load hangs on a branch.
__device__ __forceinline__ void narrow_load(NarrowCodes& r, const SmallArgs& a, int64_t row0, int chunk, int lane) {
    const int g = lane >> 2, t = lane & 3;
    const int width = (a.k + 31) & ~31, blocks = width >> 5;
    const int last = (int)min((int64_t)31, a.rows - 1 - row0);
    const int second = chunk * 64 + 32 < width ? 1 : 0;
    const uint8_t* src = static_cast<const uint8_t*>(a.x) + row0 * width + chunk * 64 + t * 8;
    const uint8_t* scale = a.x_scale + row0 * blocks + chunk * 2;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = min(m * 16 + h * 8 + g, last);
            const uint8_t *p = src + row * width, *q = scale + row * blocks;
            r.v[m][h][0] = *reinterpret_cast<const uint2*>(p);
            r.v[m][h][1] = *reinterpret_cast<const uint2*>(p + second * 32);
            r.scale[m][h][0] = q[0];
            r.scale[m][h][1] = q[second];
        }
}

// 4 codes as two pairs of float16
__device__ __forceinline__ void codes_to_half(uint32_t codes, uint32_t& lo, uint32_t& hi) {
    asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(codes));
}

// Float16 parts of a pair, rounded: 11 + 11 + 2 and more bits.  Of several, what
// is not finite is the last and the first a 1 (see split_any).
template <int kParts>
__device__ __forceinline__ void half_parts(float a, float b, uint32_t (&o)[3]) {
    union { __half2 h; uint32_t u; } x, last;
    last.u = 0;
    if (kParts > 1 && !(fabsf(a) + fabsf(b) < INFINITY)) {
        const bool fa = fabsf(a) < INFINITY, fb = fabsf(b) < INFINITY;
        last.h = __floats2half2_rn(fa ? 0.f : a, fb ? 0.f : b);
        a = fa ? a : copysignf(1.f, a);
        b = fb ? b : copysignf(1.f, b);
    }
#pragma unroll
    for (int i = 0; i < kParts; ++i) {
        x.h = __floats2half2_rn(a, b);
        o[i] = x.u;
        a -= __low2float(x.h);
        b -= __high2float(x.h);
    }
    o[kParts - 1] |= last.u;
}

template <int kXT, int kFragments = NarrowShape<kXT>::kM>
__device__ __forceinline__ void narrow_load(NarrowRaw<kXT>& r, const SmallArgs& a, int64_t row0, int chunk, int lane) {
    const int g = lane >> 2, ch = chunk * 64 + (lane & 3) * 16;
    const int pitch = kXT == kX8 ? (a.k + 31) & ~31 : a.k;
    const int last = (int)min((int64_t)(16 * kFragments - 1), a.rows - 1 - row0);
    constexpr int kSize = kXT == kX8 ? 1 : kXT == kXFloat ? 4 : 2;
    constexpr int kPer = 16 / kSize;   // elements of a 16-byte load
    const char* src = static_cast<const char*>(a.x) + row0 * pitch * kSize;
#pragma unroll
    for (int m = 0; m < kFragments; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = min(m * 16 + h * 8 + g, last);
            const char* p = src + (int64_t)row * pitch * kSize;
            if (kXT == kX8) {
                const int c = ch < pitch ? ch : 0;
                r.v[m][h][0] = *reinterpret_cast<const uint4*>(p + c);
                r.scale[m][h] = a.x_scale[(row0 + row) * (pitch >> 5) + (c >> 5)];
            } else if (a.vec_x) {
#pragma unroll
                for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) {
                    const int c = ch + i * kPer;
                    // below 2^32: at most 2^30 channels
                    r.v[m][h][i] = *reinterpret_cast<const uint4*>(p + (uint32_t)(c < a.k ? c : 0) * (uint32_t)kSize);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) {
                    union { uint4 u; uint32_t w[4]; uint16_t f[8]; } o;
#pragma unroll
                    for (int j = 0; j < kPer; ++j) {
                        const int c = ch + i * kPer + j, at = c < a.k ? c : 0;
                        if (kXT == kXFloat) o.w[j & 3] = reinterpret_cast<const uint32_t*>(p)[at];
                        else o.f[j & 7] = reinterpret_cast<const uint16_t*>(p)[at];
                    }
                    r.v[m][h][i] = o.u;
                }
            }
        }
}

// Zeros in place of what lies behind the last channel (narrow_load reads
// channel 0 there): when the values are used, so that no load is waited for.
template <int kXT, int kFragments = NarrowShape<kXT>::kM>
__device__ __forceinline__ void narrow_mask(NarrowRaw<kXT>& r, int k, int chunk, int lane) {
    if (chunk * 64 + 64 <= k) return;
    const int left = k - chunk * 64 - (lane & 3) * 16;
#pragma unroll
    for (int m = 0; m < kFragments; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) {
                union { uint4 u; uint32_t w[4]; } o;
                o.u = r.v[m][h][i];
                constexpr int kPer = kXT == kX8 ? 4 : kXT == kXFloat ? 1 : 2;   // elements of a word
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = left - (i * 4 + j) * kPer;   // that are there
                    if (n <= 0) o.w[j] = 0;
                    else if (kPer == 2 && n == 1) o.w[j] &= 0xffff;   // 8-bit rows hold zeros there
                }
                r.v[m][h][i] = o.u;
            }
}

// The operand registers of step s (4 of the lane's 16 channels), part p of kPA;
// kAny: float32 values may not be finite.
template <int kXT, int kPA, bool kAny>
__device__ __forceinline__ void narrow_operand(const NarrowRaw<kXT>& r, int m, int s, uint32_t (&o)[kPA][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (kXT == kXFloat) {
            const uint4& q = r.v[m][h][s];
            uint32_t lo[3], hi[3];
            if constexpr (kAny) {
                split_any(__uint_as_float(q.x), __uint_as_float(q.y), lo);
                split_any(__uint_as_float(q.z), __uint_as_float(q.w), hi);
            } else {
                split_pair(__uint_as_float(q.x), __uint_as_float(q.y), lo);
                split_pair(__uint_as_float(q.z), __uint_as_float(q.w), hi);
            }
#pragma unroll
            for (int p = 0; p < kPA; ++p) {
                o[p][h] = lo[p];
                o[p][2 + h] = hi[p];
            }
        } else {
            const uint4& q = r.v[m][h][s >> 1];
            o[0][h] = s & 1 ? q.z : q.x;
            o[0][2 + h] = s & 1 ? q.w : q.y;
        }
    }
}

// float32's products are made as if all values were finite.  Where one is not, or
// one of their products is past float32's range, the products of small parts say
// so: they are made again from split_any's parts.
template <bool kValue> struct Fixed { static constexpr bool value = kValue; };

template <int kM, int kN>
__device__ __forceinline__ bool small_not_finite(const float (&low)[kM][kN][4]) {
    uint64_t w = 0;
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int f = 0; f < kN; ++f) {
            watch(w, low[m][f][0], low[m][f][1]);
            watch(w, low[m][f][2], low[m][f][3]);
        }
    return not_finite(w);
}

// A sum that is infinite without its small parts stays so (those of a product
// far past the range may be infinite the other way).
template <int kM, int kN>
__device__ __forceinline__ void drop_beside_infinity(float (&low)[kM][kN][4], const float (&sum)[kM][kN][4]) {
#pragma unroll
    for (int m = 0; m < kM; ++m)
#pragma unroll
        for (int f = 0; f < kN; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (is_infinite(fabsf(sum[m][f][i]))) low[m][f][i] = 0.f;
}

// Copies a run of `count` staged values to elements at.. of a tensor, `add`'s
// elements added: 16 bytes a lane where the run starts on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void narrow_copy_as(const float* st, T* dst, int count, const T* add, bool vec, int lane) {
    constexpr int kPer = 16 / sizeof(T);
    int done = 0;
    if (vec) {
        for (int t = lane * kPer; t + kPer <= count; t += 32 * kPer) {
            float v[kPer];
#pragma unroll
            for (int i = 0; i < kPer; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(st + t + i);
            union { uint4 u; T e[kPer]; } o;
            if (add) {
                o.u = *reinterpret_cast<const uint4*>(add + t);
#pragma unroll
                for (int i = 0; i < kPer; ++i) v[i] += to_f32(o.e[i]);
            }
#pragma unroll
            for (int i = 0; i < kPer; ++i) o.e[i] = from_f32<T>(v[i]);
            *reinterpret_cast<uint4*>(dst + t) = o.u;
        }
        done = count / kPer * kPer;
    }
    for (int t = done + lane; t < count; t += 32) dst[t] = from_f32<T>(st[t] + (add ? to_f32(add[t]) : 0.f));
}

__device__ __forceinline__ void narrow_copy(const float* st, void* dst, int dtype, int64_t at, int count, const void* add,
                                            bool vec, int lane) {
    if (dtype == PLATTICE_F32)
        narrow_copy_as(st, static_cast<float*>(dst) + at, count, add ? static_cast<const float*>(add) + at : nullptr, vec, lane);
    else if (dtype == PLATTICE_BF16)
        narrow_copy_as(st, static_cast<__nv_bfloat16*>(dst) + at, count,
                       add ? static_cast<const __nv_bfloat16*>(add) + at : nullptr, vec, lane);
    else
        narrow_copy_as(st, static_cast<__half*>(dst) + at, count, add ? static_cast<const __half*>(add) + at : nullptr, vec,
                       lane);
}

template <int kXT> struct NarrowLoad { typedef NarrowRaw<kXT> type; };
template <> struct NarrowLoad<kX8> { typedef NarrowCodes type; };
template <int kXT>
__device__ __forceinline__ void narrow_fetch(NarrowRaw<kXT>& r, const SmallArgs& a, int64_t row0, int chunk, int lane) {
    narrow_load<kXT>(r, a, row0, chunk, lane);
}
__device__ __forceinline__ void narrow_fetch(NarrowCodes& r, const SmallArgs& a, int64_t row0, int chunk, int lane) {
    narrow_load(r, a, row0, chunk, lane);
}
__device__ __forceinline__ float lane_finite(float v) { return is_infinite(fabsf(v)) ? 0.f : fmaxf(fabsf(v), 0.f); }

// The type of the weights.
template <int kXT, bool kFloat> struct WeightType { typedef __nv_bfloat16 type; };
template <int kXT> struct WeightType<kXT, true> { typedef float type; };
template <> struct WeightType<kXHalf, false> { typedef __half type; };

// kSplit: few rows and many channels: the CTA's warps take turns over the
// channels of the same rows and their sums are added in shared memory, in order.
// kPlain: float32 results without activation, residual and kept z, as the
// filter takes them: none of those is asked for at every block of rows.
template <int kXT, int kNF, bool kW3, bool kSplit, bool kPlain>
__global__ void __launch_bounds__(32 * kNarrowWarps, narrow_ctas(kXT, kNF)) k_narrow(const SmallArgs a) {
    constexpr int kM = NarrowShape<kXT>::kM, kPA = kXT == kXFloat ? 3 : 1, kPB = kW3 ? 3 : 1;
    extern __shared__ __align__(16) char smem_raw[];
    __shared__ float sbias[32];
    __shared__ float column[32];   // 8-bit rows: the power of two that undoes a channel's
    typedef typename NarrowLoad<kXT>::type Raw;
    const typename WeightType<kXT, kW3>::type* weights = static_cast<const typename WeightType<kXT, kW3>::type*>(a.w);
    const int steps = narrow_steps(a.k), chunks = steps / 4;
    uint2* frag = reinterpret_cast<uint2*>(smem_raw);   // [kPB][steps][kNF][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float* st = reinterpret_cast<float*>(smem_raw + (size_t)kPB * steps * kNF * 256) + warp * 16 * kM * kNarrowPitch;

    if (threadIdx.x < 32)
        sbias[threadIdx.x] = a.bias && (int)threadIdx.x < a.n ? load_param(a.bias, a.bias_dtype, threadIdx.x) : 0.f;
    if (kXT == kX8) {
        for (int c = warp; c < 32; c += kNarrowWarps) {
            float most = 0.f;
            if (c < a.n)
                for (int ch = lane; ch < a.k; ch += 32) most = fmaxf(most, lane_finite(to_f32(weights[(int64_t)c * a.k + ch])));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int e = min(max((__float_as_int(most) >> 23) - 127 - 14, -120), 120);
            if (lane == 0) column[c] = pow2(e);
        }
        __syncthreads();
    }
    for (int i = threadIdx.x; i < steps * kNF * 32; i += blockDim.x) {
        const int l = i & 31, f = (i >> 5) % kNF, s = (i >> 5) / kNF;
        const int col = f * 8 + (l >> 2);
        const int ch = (s >> 2) * 64 + (kXT == kX8 ? ((s >> 1) & 1) * 32 + (l & 3) * 8 + (s & 1) * 4 : (l & 3) * 16 + (s & 3) * 4);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = col < a.n && ch + j < a.k ? to_f32(weights[(int64_t)col * a.k + ch + j]) : 0.f;
        uint32_t lo[3], hi[3];
        if (kXT == kX8) {
            const float up = 1.f / column[col];   // a power of two
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] *= up;
            half_parts<kPB>(v[0], v[1], lo);
            half_parts<kPB>(v[2], v[3], hi);
        } else if (kW3) {
            split_any(v[0], v[1], lo);
            split_any(v[2], v[3], hi);
        } else if (kXT == kXHalf) {
            union { __half2 h; uint32_t u; } x, y;
            x.h = __floats2half2_rn(v[0], v[1]);
            y.h = __floats2half2_rn(v[2], v[3]);
            lo[0] = x.u;
            hi[0] = y.u;
        } else {
            union { __nv_bfloat162 h; uint32_t u; } x, y;
            x.h = __floats2bfloat162_rn(v[0], v[1]);
            y.h = __floats2bfloat162_rn(v[2], v[3]);
            lo[0] = x.u;
            hi[0] = y.u;
        }
#pragma unroll
        for (int p = 0; p < kPB; ++p) frag[p * steps * kNF * 32 + i] = make_uint2(lo[p], hi[p]);
    }
    __syncthreads();

    const int64_t blocks = (a.rows + 16 * kM - 1) / (16 * kM);
    const int64_t stride = kSplit ? gridDim.x : (int64_t)gridDim.x * kNarrowWarps;
    int64_t block = kSplit ? blockIdx.x : (int64_t)blockIdx.x * kNarrowWarps + warp;
    const int chunk0 = kSplit ? warp : 0, chunk_step = kSplit ? kNarrowWarps : 1;

    // where a lane's columns go in the staged output: the rows of y0 one after
    // the other, then y1's (a split), each as it will lie in memory
    const int w0 = a.split ? a.split : a.n, w1 = a.n - w0;
    int put[kNF][2], width[kNF][2];
#pragma unroll
    for (int f = 0; f < kNF; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int c = f * 8 + t * 2 + i;
            width[f][i] = c < w0 ? w0 : w1;
            put[f][i] = c < w0 ? c : c < a.n ? 16 * kM * w0 + c - w0 : -1;
        }
    uint64_t undo[kNF];
#pragma unroll
    for (int f = 0; f < kNF; ++f) undo[f] = kXT == kX8 ? pair_of(column[f * 8 + t * 2], column[f * 8 + t * 2 + 1]) : 0;

    Raw next;
    if (block < blocks && chunk0 < chunks) narrow_fetch(next, a, block * (16 * kM), chunk0, lane);
    for (; block < blocks; block += stride) {
        const int64_t row0 = block * (16 * kM);
        float acc[kM][kNF][4];
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int f = 0; f < kNF; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][f][i] = 0.f;
        for (int c = chunk0; c < chunks; c += chunk_step) {
            Raw raw = next;
            const bool more = c + chunk_step < chunks;   // of this block; else the next block's first
            if (more || block + stride < blocks)
                narrow_fetch(next, a, more ? row0 : row0 + stride * (16 * kM), more ? c + chunk_step : chunk0, lane);
            if constexpr (kXT == kX8) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    if (blk && c * 64 + 32 >= a.k) break;   // no second block of 32 channels here
                    float sum[kM][kNF][4];
#pragma unroll
                    for (int m = 0; m < kM; ++m)
#pragma unroll
                        for (int f = 0; f < kNF; ++f)
#pragma unroll
                            for (int i = 0; i < 4; ++i) sum[m][f][i] = 0.f;
#pragma unroll
                    for (int s = 0; s < 2; ++s) {
                        uint32_t o[kM][4];
#pragma unroll
                        for (int m = 0; m < kM; ++m)
#pragma unroll
                            for (int h = 0; h < 2; ++h)
                                codes_to_half(s ? raw.v[m][h][blk].y : raw.v[m][h][blk].x, o[m][h], o[m][2 + h]);
#pragma unroll
                        for (int p = kPB - 1; p >= 0; --p)   // small parts first
#pragma unroll
                            for (int f = 0; f < kNF; ++f) {
                                const uint2 b = frag[((p * steps + c * 4 + blk * 2 + s) * kNF + f) * 32 + lane];
#pragma unroll
                                for (int m = 0; m < kM; ++m) mma16816<true>(sum[m][f], o[m][0], o[m][1], o[m][2], o[m][3], b);
                            }
                    }
#pragma unroll
                    for (int m = 0; m < kM; ++m)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const uint64_t sc = both(scale_of(raw.scale[m][h][blk]));
#pragma unroll
                            for (int f = 0; f < kNF; ++f) {
                                // the channel's power first: neither product leaves float32's range by itself
                                const uint64_t v = mul2(pair_of(sum[m][f][2 * h], sum[m][f][2 * h + 1]), undo[f]);
                                pair_to(fma2(v, sc, pair_of(acc[m][f][2 * h], acc[m][f][2 * h + 1])), acc[m][f][2 * h],
                                        acc[m][f][2 * h + 1]);
                            }
                        }
                }
                continue;
            } else {
            narrow_mask<kXT>(raw, a.k, c, lane);
            // the sum of these 64 channels by itself, and float32's products of small
            // parts apart from it: the matrix instruction cuts where an addition
            // rounds, by which a long chain of them drifts
            float sum[kM][kNF][4], low[kM][kNF][4];
            auto clear = [&] {
#pragma unroll
                for (int m = 0; m < kM; ++m)
#pragma unroll
                    for (int f = 0; f < kNF; ++f)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sum[m][f][i] = low[m][f][i] = 0.f;
            };
            auto step = [&](int m, int s, const uint32_t (&o)[kPA][4]) {
#pragma unroll
                for (int size = 2; size >= 0; --size)   // small products first
#pragma unroll
                    for (int pa = 0; pa < kPA; ++pa) {
                        const int pb = size - pa;
                        if (pb < 0 || pb >= kPB) continue;
#pragma unroll
                        for (int f = 0; f < kNF; ++f)
                            mma16816<kXT == kXHalf>(size ? low[m][f] : sum[m][f], o[pa][0], o[pa][1], o[pa][2], o[pa][3],
                                                    frag[((pb * steps + c * 4 + s) * kNF + f) * 32 + lane]);
                    }
            };
            clear();
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    uint32_t o[kPA][4];
                    narrow_operand<kXT, kPA, false>(raw, m, s, o);
                    step(m, s, o);
                }
            if constexpr (kPA == 3) {
                if (__any_sync(0xffffffffu, small_not_finite(low))) {   // rare: from memory again, 4 channels at a time
                    clear();
#pragma unroll 1
                    for (int s = 0; s < 4; ++s) {
                        uint32_t o[kPA][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int64_t row = min(row0 + h * 8 + g, a.rows - 1);
                            const int ch = c * 64 + t * 16 + s * 4;
                            float v[8];
                            load8(v, static_cast<const float*>(a.x) + row * a.k + ch, false, min(a.k - ch, 4));
                            uint32_t lo[3], hi[3];
                            split_any(v[0], v[1], lo);
                            split_any(v[2], v[3], hi);
#pragma unroll
                            for (int p = 0; p < kPA; ++p) {
                                o[p][h] = lo[p];
                                o[p][2 + h] = hi[p];
                            }
                        }
                        step(0, s, o);
                    }
                    drop_beside_infinity(low, sum);
                }
            }
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f) {
                    if (kPA == 3) {
                        add2(sum[m][f][0], sum[m][f][1], low[m][f][0], low[m][f][1]);
                        add2(sum[m][f][2], sum[m][f][3], low[m][f][2], low[m][f][3]);
                    }
                    add2(acc[m][f][0], acc[m][f][1], sum[m][f][0], sum[m][f][1]);
                    add2(acc[m][f][2], acc[m][f][3], sum[m][f][2], sum[m][f][3]);
                }
            }
        }
        const int rows = (int)min((int64_t)(16 * kM), a.rows - row0);
        if (kSplit) {
            __syncthreads();   // the staging has been read
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        st[(m * 16 + (i >> 1) * 8 + g) * kNarrowPitch + f * 8 + t * 2 + (i & 1)] = acc[m][f][i];
            __syncthreads();
            if (warp != 0) continue;
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = acc[m][f][i];
                        for (int w = 1; w < kNarrowWarps; ++w)
                            v += st[w * 16 * kM * kNarrowPitch + (m * 16 + (i >> 1) * 8 + g) * kNarrowPitch + f * 8 +
                                    t * 2 + (i & 1)];
                        acc[m][f][i] = v;
                    }
        }
#pragma unroll
        for (int m = 0; m < kM; ++m)
#pragma unroll
            for (int f = 0; f < kNF; ++f)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][f][i] += sbias[f * 8 + t * 2 + (i & 1)];
        if (!kPlain && a.z_scale) {   // the whole row is one block; 16 columns a lane
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        st[(m * 16 + (i >> 1) * 8 + g) * kNarrowPitch + f * 8 + t * 2 + (i & 1)] = acc[m][f][i];
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kM; ++m) {
                const int r = m * 16 + (lane >> 1), c0 = (lane & 1) * 16;
                float v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = c0 + i < a.n ? st[r * kNarrowPitch + c0 + i] : 0.f;
                bool infinite;
                float amax = finite_amax_of(v, infinite);
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                const int e = block_exponent(amax);
                if (r < rows) {
                    const float inv = pow2(-e);
                    uint2 q[2];
                    codes_of(q, v, inv, infinite);
                    reinterpret_cast<uint4*>(a.z)[(row0 + r) * 2 + (lane & 1)] = make_uint4(q[0].x, q[0].y, q[1].x, q[1].y);
                    if ((lane & 1) == 0) a.z_scale[row0 + r] = (uint8_t)(e + 127);
                }
            }
        }
        const bool full_z = !kPlain && a.z && !a.z_scale;   // without a split (forward_way)
        for (int pass = full_z ? 0 : 1; pass < 2; ++pass) {   // a kept z, then y
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f) {
                    if (!kPlain && pass == 1) activate(acc[m][f], a.act);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (put[f][i & 1] >= 0) st[(m * 16 + (i >> 1) * 8 + g) * width[f][i & 1] + put[f][i & 1]] = acc[m][f][i];
                }
            __syncwarp();
            if (kPlain) {
                narrow_copy_as<float>(st, static_cast<float*>(a.y0) + row0 * w0, rows * w0, nullptr, a.vec_y, lane);
                if (a.split)
                    narrow_copy_as<float>(st + 16 * kM * w0, static_cast<float*>(a.y1) + row0 * w1, rows * w1, nullptr,
                                          a.vec_y, lane);
            } else if (pass == 0) {
                narrow_copy(st, a.z, a.out_dtype, row0 * a.n, rows * a.n, nullptr, a.vec_y, lane);
            } else {
                narrow_copy(st, a.y0, a.out_dtype, row0 * w0, rows * w0, a.residual, a.vec_y, lane);
                if (a.split) narrow_copy(st + 16 * kM * w0, a.y1, a.out_dtype, row0 * w1, rows * w1, nullptr, a.vec_y, lane);
            }
        }
    }
}

// ------------------------------------ backward, at most 32 output channels
//
// One pass: a warp takes 16 rows and a slice of 64 input channels, makes gz
// (grad_y act'(z)) once in shared memory, and
// from it the rows' grad_x (gz w) and its share of grad_w (x^T gz, kept in
// registers over all of the warp's rows) and grad_bias.  What a CTA gathered
// goes to `partial`, one line of n k + n sums per CTA of a slice's column;
// k_sum_lines adds those in order.  Read once: grad_y and z per slice, x;
// written once: grad_x.  Bound by the latency of its phases (12 warps an SM is
// what the registers of the sums leave): 262144 rows, 64 -> 24 from 8 bits and
// float32 gradients 29 us and 4 for the sums (76 MB, 11.6 us at the copy rate),
// where the gradient's pass and two tiled products took 72.
constexpr int kTilePitch = 72;   // 16-bit elements: rows 144 bytes apart, no bank conflicts for ldmatrix

// kParts: of the weights: 3 with float32 ones, 1 or 2 with 16-bit ones.
//
// gz = grad_y act'(z) is made here in float32 and has two parts beside 16-bit
// operands: 28 more matrix instructions a block of rows, 8 % of the pass, keep what
// rounding it to one would add to both gradients' errors.  float16 holds only a
// small part of what gz can be:
// * behind float32 gradients (of 1e-8 or 1e6) float16 operands run as two bfloat16
//   parts each (kParts 2, exact; gz's two hold 16 bits), three products;
// * a float16 gradient is one float16 part as it came, or behind an activation two,
//   the first held at the type's largest number (a slope of up to 1.13 can take gz
//   past it).
template <int kXT, int kParts> struct NarrowGradShape {
    static constexpr bool kHalf = kXT == kXHalf && kParts == 1;                       // float16 matrix instructions
    static constexpr int kPX = kXT == kXFloat ? 3 : kParts == 2 ? 2 : 1;
    static constexpr int kPZ = kParts == 3 ? 3 : 2;
    static constexpr int kFragBytes = kParts * 2 * 8 * 32 * 8;                        // weights of the slice
    static constexpr int kStaged = 16 * kNarrowPitch + 4;   // gz of 16 rows, and a place for what is behind them
    static constexpr int kWarpBytes = kStaged * 4 + kPX * 16 * kTilePitch * 2;
    static constexpr int kBytes = kFragBytes + kGradWarps * kWarpBytes + 64 * 33 * 4;
};

// a and b as kP packed parts, bfloat16 or float16 (rounded).  kAny: they may not be
// finite (float16: one part then); kLone: they meet operands of a single part.
template <int kP, bool kHalf, bool kAny, bool kLone = false>
__device__ __forceinline__ void to_parts(float a, float b, uint32_t (&o)[kP]) {
    if constexpr (kHalf) {
#pragma unroll
        for (int i = 0; i < kP; ++i) {
            union { __half2 h; uint32_t u; } x;
            if (i < kP - 1) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(x.u) : "f"(b), "f"(a));
            else x.h = __floats2half2_rn(a, b);
            o[i] = x.u;
            a -= __low2float(x.h);
            b -= __high2float(x.h);
        }
    } else if constexpr (kLone && kP == 2) {
        split_one_sign<kAny>(a, b, o);
    } else if constexpr (kAny) {
        split_any(a, b, o);
    } else {
        split_pair(a, b, o);
    }
}

template <int kXT, bool kG32> struct GradType { typedef __nv_bfloat16 type; };
template <int kXT> struct GradType<kXT, true> { typedef float type; };
template <> struct GradType<kXHalf, false> { typedef __half type; };

// kXT: the type of x (and, for 16-bit ones, of everything); kNF: output channels / 8;
// kG32: float32 gradients.
template <int kXT, int kParts, int kNF, bool kG32>
__global__ void __launch_bounds__(32 * kGradWarps, narrow_grad_ctas(kParts, kNF)) k_narrow_grad(const SmallGradArgs a) {
    typedef NarrowGradShape<kXT, kParts> Shape;
    typedef typename GradType<kXT, kG32>::type TG;
    constexpr int kPX = Shape::kPX, kPZ = Shape::kPZ, kKS = kNF > 2 ? 2 : 1;   // steps of 16 output channels in grad_x's sum
    constexpr bool kHalf = Shape::kHalf;
    extern __shared__ __align__(16) char smem_raw[];
    uint2* frag = reinterpret_cast<uint2*>(smem_raw);   // [kParts][kKS][8][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    char* mine = smem_raw + Shape::kFragBytes + warp * Shape::kWarpBytes;
    float* st = reinterpret_cast<float*>(mine);                                       // gz, 16 x 33
    uint16_t* tile = reinterpret_cast<uint16_t*>(mine + Shape::kStaged * 4);          // x, [kPX][16][72]
    float* gather = reinterpret_cast<float*>(smem_raw + Shape::kFragBytes + kGradWarps * Shape::kWarpBytes);
    const int ch0 = blockIdx.y * 64, n = a.s.n, k = a.s.k;
    const int cols_per_lane = kKS * 4;   // output channels of lane t in grad_x's sum: t cols_per_lane..

    // fragment f, column c of the weights is channel (c >> 1) 16 + 2 f + (c & 1)
    // of the slice, so that a lane ends up with 16 neighbouring channels
    bool odd = false;   // float16: weights that are not finite
    if (a.need_x) {
        typedef typename WeightType<kXT, kParts == 3>::type TW;
        const TW* weights = static_cast<const TW*>(a.s.w);
        for (int i = threadIdx.x; i < kKS * 8 * 32; i += blockDim.x) {
            const int l = i & 31, f = (i >> 5) & 7, s = i >> 8;
            const int ch = ch0 + (l >> 3) * 16 + 2 * f + ((l >> 2) & 1), o = (l & 3) * cols_per_lane + s * 4;
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = o + j < n && ch < k ? to_f32(weights[(int64_t)(o + j) * k + ch]) : 0.f;
            uint32_t lo[kParts], hi[kParts];
            if (kHalf)
#pragma unroll
                for (int j = 0; j < 4; ++j) odd |= !(fabsf(v[j]) < INFINITY);
            to_parts<kParts, kHalf, true>(v[0], v[1], lo);
            to_parts<kParts, kHalf, true>(v[2], v[3], hi);
#pragma unroll
            for (int p = 0; p < kParts; ++p) frag[p * kKS * 256 + i] = make_uint2(lo[p], hi[p]);
        }
    }
    for (int i = lane; i < 16 * kNarrowPitch; i += 32) st[i] = 0.f;   // columns behind n stay 0
    // float16: one part of gz where it is a gradient as it came, or meets what is
    // not finite (a second part of 0 would make NaN of it)
    const bool single = kHalf && (__syncthreads_or(odd) || !a.s.z);
    if (!kHalf) __syncthreads();

    float dw[4][kNF][4];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int f = 0; f < kNF; ++f)
#pragma unroll
            for (int i = 0; i < 4; ++i) dw[m][f][i] = 0.f;
    float db = 0.f;

    const int64_t blocks = (a.s.rows + 15) / 16, stride = (int64_t)gridDim.x * kGradWarps;
    int64_t block = (int64_t)blockIdx.x * kGradWarps + warp;
    // The rows' gradients are the run of g0's 16 rows, then g1's.  A lane takes
    // kPer elements (16 bytes) from (32 i + lane) kPer on; where each goes in
    // the staged rows is the same for every 16 rows.
    constexpr int kPer = 16 / (int)sizeof(TG), kVecs = (16 * 8 * kNF / kPer + 31) / 32, kRun = kVecs * kPer;
    const int w0 = a.s.split ? a.s.split : n, w1 = n - w0, run0 = 16 * w0;
    uint16_t place[kRun];
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
        const int e = (i / kPer * 32 + lane) * kPer + i % kPer;
        place[i] = 16 * kNarrowPitch;
        if (e < run0) place[i] = (uint16_t)(e / w0 * kNarrowPitch + e % w0);
        else if (e < 16 * n) place[i] = (uint16_t)((e - run0) / w1 * kNarrowPitch + w0 + (e - run0) % w1);
    }
    union { uint4 v[kVecs]; TG e[kRun]; } gn;   // the next rows' gradients, x and z, loaded ahead
    NarrowRaw<kXT> xn;
    uint4 zn = make_uint4(0, 0, 0, 0);
    uint8_t zs = 127;
    auto load_rows = [&](int64_t b) {
        const TG* p0 = static_cast<const TG*>(a.g0) + b * 16 * w0;
        const TG* p1 = static_cast<const TG*>(a.g1) + b * 16 * w1 - run0;
        const int rows = (int)min((int64_t)16, a.s.rows - b * 16);
        if (a.vec_g && rows == 16) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) {
                const int e = (i * 32 + lane) * kPer;
                gn.v[i] = *reinterpret_cast<const uint4*>(e < run0 ? p0 + e : e < 16 * n ? p1 + e : p0);
            }
        } else {   // rows on other boundaries, and the last ones
            const int limit = rows * kNarrowPitch;
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const int e = (i / kPer * 32 + lane) * kPer + i % kPer;
                gn.e[i] = *(place[i] < limit ? e < run0 ? p0 + e : p1 + e : p0);
            }
        }
        if (a.s.z_scale) {   // a lane per half row
            const int64_t row = min(b * 16 + (lane >> 1), a.s.rows - 1);   // behind the last: its own, times 0
            zn = reinterpret_cast<const uint4*>(a.s.z)[row * 2 + (lane & 1)];
            zs = a.s.z_scale[row];
        }
        if (!a.need_w) return;
        narrow_load<kXT, 1>(xn, a.s, b * 16, blockIdx.y, lane);
    };
    if (block < blocks) load_rows(block);
    for (; block < blocks; block += stride) {
        const int64_t row0 = block * 16;
        const int rows = (int)min((int64_t)16, a.s.rows - row0);
        __syncwarp();
        if (rows == 16) {
#pragma unroll
            for (int i = 0; i < kRun; ++i) st[place[i]] = to_f32(gn.e[i]);
        } else {   // 0 behind the last row
#pragma unroll
            for (int i = 0; i < kRun; ++i) st[place[i]] = place[i] < rows * kNarrowPitch ? to_f32(gn.e[i]) : 0.f;
        }
        odd = false;
        if (a.need_w) {   // x, widened, into the tile
            narrow_mask<kXT, 1>(xn, k, blockIdx.y, lane);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (rows < 16 && g + 8 * h >= rows)   // what was read is the last row again: times 0, were it finite
#pragma unroll
                    for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) xn.v[0][h][i] = make_uint4(0, 0, 0, 0);
                uint16_t* row = tile + (g + 8 * h) * kTilePitch + t * 16;
                if (kXT == kX8) {
                    float v[16];
                    const float sc = scale_of(xn.scale[0][h]);
                    values4(v, xn.v[0][h][0].x, sc);
                    values4(v + 4, xn.v[0][h][0].y, sc);
                    values4(v + 8, xn.v[0][h][0].z, sc);
                    values4(v + 12, xn.v[0][h][0].w, sc);
                    union { uint4 u[2]; __nv_bfloat162 b[8]; } o;   // exact
#pragma unroll
                    for (int i = 0; i < 8; ++i) o.b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    reinterpret_cast<uint4*>(row)[0] = o.u[0];
                    reinterpret_cast<uint4*>(row)[1] = o.u[1];
                } else if (kXT == kXFloat) {
                    auto put = [&](auto any) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint4& q = xn.v[0][h][i % NarrowShape<kXT>::kRaw];
                            uint32_t lo[3], hi[3];
                            to_parts<3, false, decltype(any)::value>(__uint_as_float(q.x), __uint_as_float(q.y), lo);
                            to_parts<3, false, decltype(any)::value>(__uint_as_float(q.z), __uint_as_float(q.w), hi);
#pragma unroll
                            for (int p = 0; p < 3; ++p)
                                *reinterpret_cast<uint2*>(row + (p % kPX) * 16 * kTilePitch + i * 4) = make_uint2(lo[p], hi[p]);
                        }
                    };
                    uint64_t w = 0;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4& q = xn.v[0][h][i % NarrowShape<kXT>::kRaw];
                        watch(w, __uint_as_float(q.x), __uint_as_float(q.y));
                        watch(w, __uint_as_float(q.z), __uint_as_float(q.w));
                    }
                    if (!not_finite(w)) put(Fixed<false>());
                    else put(Fixed<true>());
                } else if (kPX == 2) {   // float16 as two bfloat16
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        union { uint4 u; __half2 h[4]; } q;
                        q.u = xn.v[0][h][i % NarrowShape<kXT>::kRaw];
                        uint32_t o[4][2];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 f = __half22float2(q.h[j]);
                            split_any(f.x, f.y, o[j]);
                        }
#pragma unroll
                        for (int p = 0; p < 2; ++p)
                            reinterpret_cast<uint4*>(row + (p % kPX) * 16 * kTilePitch)[i] =
                                make_uint4(o[0][p], o[1][p], o[2][p], o[3][p]);
                    }
                } else {
                    reinterpret_cast<uint4*>(row)[0] = xn.v[0][h][0];
                    reinterpret_cast<uint4*>(row)[1] = xn.v[0][h][1 % NarrowShape<kXT>::kRaw];
                    if (kHalf && !single) {
                        const __half2* q = reinterpret_cast<const __half2*>(row);   // its own 16 again
                        __half2 w = __float2half2_rn(0.f);
#pragma unroll
                        for (int i = 0; i < 8; ++i) w = __hfma2(q[i], __float2half2_rn(0.f), w);
                        odd |= !(__low2float(w) + __high2float(w) == 0.f);
                    }
                }
            }
        }
        const uint4 zc = zn;
        const float zscale = scale_of(zs);
        if (block + stride < blocks) load_rows(block + stride);
        __syncwarp();
        if (a.s.z_scale) {
            float v[16];
            values4(v, zc.x, zscale);
            values4(v + 4, zc.y, zscale);
            values4(v + 8, zc.z, zscale);
            values4(v + 12, zc.w, zscale);
            slope16(v, a.s.act);
            float* row = st + (lane >> 1) * kNarrowPitch + (lane & 1) * 16;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if ((lane & 1) * 16 + i < n) row[i] *= v[i];
            __syncwarp();
        } else if (a.s.z) {
            const unsigned inv = 65536u / (unsigned)n + 1;
            for (int e = lane; e < rows * n; e += 32) {
                const int r = (int)((e * inv) >> 16);
                float v[16] = {load_param(a.s.z, a.s.out_dtype, row0 * n + e)};
                slope16(v, a.s.act);
                st[r * kNarrowPitch + e - r * n] *= v[0];
            }
            __syncwarp();
        }
        // sums of the columns, for the bias's gradient and to see whether all is finite
        float column = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 8) {   // short chains: many rows drift less
            float t[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) t[i] = st[(r + i) * kNarrowPitch + lane];
            const float part = ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
            column += part;
            db += part;
        }
        auto products = [&](auto any) {
            constexpr bool kAny = decltype(any)::value;
            constexpr int kZ = kHalf && kAny ? 1 : kPZ;
            if (a.need_x) {
                uint32_t o[kKS][kZ][4];
#pragma unroll
                for (int s = 0; s < kKS; ++s)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float* p = st + (g + 8 * h) * kNarrowPitch + t * cols_per_lane + s * 4;
                        uint32_t lo[kZ], hi[kZ];
                        to_parts<kZ, kHalf, kAny, kPX == 1 && kParts == 1>(p[0], p[1], lo);
                        to_parts<kZ, kHalf, kAny, kPX == 1 && kParts == 1>(p[2], p[3], hi);
#pragma unroll
                        for (int q = 0; q < kZ; ++q) {
                            o[s][q][h] = lo[q];
                            o[s][q][2 + h] = hi[q];
                        }
                    }
                float dx[8][4];
#pragma unroll
                for (int f = 0; f < 8; ++f) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) dx[f][i] = 0.f;
#pragma unroll
                    for (int sum = kZ - 1; sum >= 0; --sum)   // small products first
#pragma unroll
                        for (int pa = 0; pa < kZ; ++pa) {
                            const int pb = sum - pa;
                            if (pb < 0 || pb >= kParts) continue;
#pragma unroll
                            for (int s = 0; s < kKS; ++s)
                                mma16816<kHalf>(dx[f], o[s][pa][0], o[s][pa][1], o[s][pa][2], o[s][pa][3],
                                                frag[((pb * kKS + s) * 8 + f) * 32 + lane]);
                        }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {   // 16 neighbouring channels of rows g and g + 8
                    if (g + 8 * h >= rows) continue;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const int ch = ch0 + t * 16 + q * 8, left = k - ch;
                        if (left <= 0) continue;
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = dx[q * 4 + (i >> 1)][h * 2 + (i & 1)];
                        const int64_t at = (row0 + g + 8 * h) * k + ch;
                        const bool vec = a.vec_gx && left >= 8;
                        if (kXT == kXHalf) store8(static_cast<__half*>(a.grad_x) + at, v, vec, left);
                        else if (kParts == 3) store8(static_cast<float*>(a.grad_x) + at, v, vec, left);
                        else store8(static_cast<__nv_bfloat16*>(a.grad_x) + at, v, vec, left);
                    }
                }
            }
            if (a.need_w) {
                uint32_t b[kZ][kNF][2];
#pragma unroll
                for (int f = 0; f < kNF; ++f)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const float* p = st + (2 * t + 8 * h) * kNarrowPitch + f * 8 + g;
                        uint32_t o[kZ];
                        to_parts<kZ, kHalf, kAny, kPX == 1 && kParts == 1>(p[0], p[kNarrowPitch], o);
#pragma unroll
                        for (int q = 0; q < kZ; ++q) b[q][f][h] = o[q];
                    }
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    uint32_t x[kPX][4];
#pragma unroll
                    for (int q = 0; q < kPX; ++q) {
                        const uint16_t* src = tile + q * 16 * kTilePitch + ((lane >> 4) * 8 + (lane & 7)) * kTilePitch +
                                              m * 16 + ((lane >> 3) & 1) * 8;
                        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                     : "=r"(x[q][0]), "=r"(x[q][1]), "=r"(x[q][2]), "=r"(x[q][3])
                                     : "r"((uint32_t)__cvta_generic_to_shared(src))
                                     : "memory");
                    }
                    // float32: the sum of these rows by itself (see k_narrow)
                    float rows16[kNF][4];
                    if (kParts == 3) {
#pragma unroll
                        for (int f = 0; f < kNF; ++f)
#pragma unroll
                            for (int i = 0; i < 4; ++i) rows16[f][i] = 0.f;
                    }
#pragma unroll
                    for (int sum = kZ - 1; sum >= 0; --sum)
#pragma unroll
                        for (int px = 0; px < kPX; ++px) {
                            const int pb = sum - px;
                            if (pb < 0 || pb > kZ - 1) continue;
#pragma unroll
                            for (int f = 0; f < kNF; ++f)
                                mma16816<kHalf>(kParts == 3 ? rows16[f] : dw[m][f], x[px][0], x[px][1], x[px][2], x[px][3],
                                                make_uint2(b[pb][f][0], b[pb][f][1]));
                        }
                    if (kParts == 3) {
#pragma unroll
                        for (int f = 0; f < kNF; ++f) {
                            add2(dw[m][f][0], dw[m][f][1], rows16[f][0], rows16[f][1]);
                            add2(dw[m][f][2], dw[m][f][3], rows16[f][2], rows16[f][3]);
                        }
                    }
                }
            }
        };
        if (!single && !__any_sync(0xffffffffu, odd || !(fabsf(column) < INFINITY))) products(Fixed<false>());
        else products(Fixed<true>());
    }

    // the CTA's sums, warp after warp
    float* line = a.partial + (int64_t)blockIdx.x * ((int64_t)n * k + n);
    if (a.need_w) {
        for (int w = 0; w < kGradWarps; ++w) {
            __syncthreads();
            if (warp != w) continue;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float* p = gather + (m * 16 + (i >> 1) * 8 + g) * 33 + f * 8 + t * 2 + (i & 1);
                        *p = w ? *p + dw[m][f][i] : dw[m][f][i];
                    }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 64 * n; i += blockDim.x) {
            const int col = i >> 6, ch = i & 63;
            if (ch0 + ch < k) line[(int64_t)col * k + ch0 + ch] = gather[ch * 33 + col];
        }
    }
    if (a.need_b && blockIdx.y == 0) {
        __syncthreads();
        gather[warp * 32 + lane] = db;
        __syncthreads();
        if (threadIdx.x < n) {
            float v = 0.f;
            for (int w = 0; w < kGradWarps; ++w) v += gather[w * 32 + threadIdx.x];
            line[(int64_t)n * k + threadIdx.x] = v;
        }
    }
}

// -------------------------------------------------------------- few rows
//
// The same products with the sides changed over: 16 output channels are the
// rows of the matrix instruction and 8 or 16 input rows its columns.  Both
// operands' registers are loaded from memory as they lie there (neither has a
// second reader in a warp), 32 bytes of a 16-bit type per row and load; a CTA
// takes 32 channels, the block of a kept 8-bit pre-activation, and its warps
// take turns over the input channels, 64 at a time, whose sums are added in
// shared memory in order.  Bound by the read of w and its latency: 1024 -> 4096 in bfloat16 (8.4
// MB, 1.3 us at the copy rate) takes 3.5 us with 1 row, 4.6 with 16, of which
// launching is 2.2; 4096 -> 4096 (33.5 MB, 5.1 us) 6.0 and 9.6.
constexpr int few_splits(int wt) { return wt == kXFloat ? 8 : 16; }   // warps that share the input channels

template <int kWT, bool kX8In, int kN>
__global__ void __launch_bounds__(64 * few_splits(kWT)) k_few(const SmallArgs a) {
    constexpr int kSplits = few_splits(kWT), kPW = kWT == kXFloat ? 3 : 1, kXT = kX8In ? (int)kX8 : kWT;
    constexpr int kPX = kXT == kXFloat ? 3 : 1;
    __shared__ float part[kSplits][8 * kN][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int half = warp & 1, split = warp >> 1, chunks = narrow_steps(a.k) / 4;
    SmallArgs w = a;   // the weights as the rows of a load
    w.x = a.w;
    w.rows = a.n;
    w.vec_x = a.vec_w;
    const int64_t col0 = (int64_t)blockIdx.x * 32 + half * 16, row0 = (int64_t)blockIdx.y * (8 * kN);
    float acc[kN][4];
#pragma unroll
    for (int j = 0; j < kN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[j][i] = 0.f;
    if (col0 < a.n) {
        for (int c = split; c < chunks; c += kSplits) {
            NarrowRaw<kWT> wr;
            NarrowRaw<kXT> xr;
            narrow_load<kWT, 1>(wr, w, col0, c, lane);
            narrow_load<kXT, 1>(xr, a, row0, c, lane);
            narrow_mask<kWT, 1>(wr, a.k, c, lane);
            narrow_mask<kXT, 1>(xr, a.k, c, lane);
            float sum[1][kN][4], low[1][kN][4];   // low: float32's products of small parts (see k_narrow)
            auto products = [&](const NarrowRaw<kWT>& wr, const NarrowRaw<kXT>& xr, auto any) {
#pragma unroll
                for (int j = 0; j < kN; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sum[0][j][i] = low[0][j][i] = 0.f;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t o[kPW][4], b[kPX][4];
                    narrow_operand<kWT, kPW, decltype(any)::value>(wr, 0, s, o);
                    if constexpr (kX8In) {
#pragma unroll
                        for (int h = 0; h < kN; ++h) {
                            const uint4& q = xr.v[0][h][0];
                            float v[4];   // exact in bfloat16
                            values4(v, s == 0 ? q.x : s == 1 ? q.y : s == 2 ? q.z : q.w, scale_of(xr.scale[0][h]));
                            union { __nv_bfloat162 p; uint32_t u; } x, y;
                            x.p = __floats2bfloat162_rn(v[0], v[1]);
                            y.p = __floats2bfloat162_rn(v[2], v[3]);
                            b[0][h] = x.u;
                            b[0][2 + h] = y.u;
                        }
                    } else {
                        narrow_operand<kXT, kPX, decltype(any)::value>(xr, 0, s, b);
                    }
#pragma unroll
                    for (int size = 2; size >= 0; --size)   // small products first
#pragma unroll
                        for (int pw = 0; pw < kPW; ++pw) {
                            const int px = size - pw;
                            if (px < 0 || px >= kPX) continue;
#pragma unroll
                            for (int j = 0; j < kN; ++j)
                                mma16816<kWT == kXHalf>(size ? low[0][j] : sum[0][j], o[pw][0], o[pw][1], o[pw][2], o[pw][3],
                                                        make_uint2(b[px][j], b[px][2 + j]));
                        }
                }
            };
            products(wr, xr, Fixed<false>());
            if constexpr (kPW == 3)
                if (__any_sync(0xffffffffu, small_not_finite(low))) {   // rare
                    NarrowRaw<kWT> w2;
                    NarrowRaw<kXT> x2;
                    narrow_load<kWT, 1>(w2, w, col0, c, lane);
                    narrow_load<kXT, 1>(x2, a, row0, c, lane);
                    narrow_mask<kWT, 1>(w2, a.k, c, lane);
                    narrow_mask<kXT, 1>(x2, a.k, c, lane);
                    products(w2, x2, Fixed<true>());
                    drop_beside_infinity(low, sum);
                }
#pragma unroll
            for (int j = 0; j < kN; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[j][i] += kPW == 3 ? sum[0][j][i] + low[0][j][i] : sum[0][j][i];
        }
    }
#pragma unroll
    for (int j = 0; j < kN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) part[split][j * 8 + t * 2 + (i & 1)][half * 16 + (i >> 1) * 8 + g] = acc[j][i];
    __syncthreads();
    const int64_t row = row0 + warp;
    if (warp >= 8 * kN || row >= a.rows) return;
    // a warp per row, a lane per channel
    const int c = blockIdx.x * 32 + lane;
    const bool have = c < a.n;
    float z = 0.f;
    if (have && a.bias) z = load_param(a.bias, a.bias_dtype, c);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < kSplits; ++i) sum += part[i][warp][lane];
    z = have ? z + sum : 0.f;
    if (a.z_scale) {
        float amax = lane_finite(z);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int e = block_exponent(amax);
        const float v[8] = {z, 0, 0, 0, 0, 0, 0, 0};
        const int64_t at = row * ((a.n + 31) / 32) + blockIdx.x;
        uint2 q[1];
        codes_of(q, v, pow2(-e), is_infinite(fabsf(z)));
        static_cast<uint8_t*>(a.z)[at * 32 + lane] = (uint8_t)q[0].x;
        if (lane == 0) a.z_scale[at] = (uint8_t)(e + 127);
    } else if (a.z && have) {
        store_param(a.z, a.out_dtype, row * a.n + c, z);
    }
    if (!have) return;
    float y[2] = {z, 0.f};
    activate(y, a.act);
    if (a.residual) y[0] += load_param(a.residual, a.out_dtype, row * a.n + c);
    if (c < a.split) store_param(a.y0, a.out_dtype, row * a.split + c, y[0]);
    else if (a.split) store_param(a.y1, a.out_dtype, row * (a.n - a.split) + c - a.split, y[0]);
    else store_param(a.y0, a.out_dtype, row * a.n + c, y[0]);
}

}  // namespace plr
