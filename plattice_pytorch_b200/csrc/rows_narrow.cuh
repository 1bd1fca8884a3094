// rows_narrow.cuh -- the linear map where one side is small: at most 32 output
// channels (the projections to the filter's features and values), or at most
// 8 rows.  Both read what they need once and are bound by that read; a
// 128-row tensor-memory tile would be mostly padding, and staging it costs
// more than the product.
#pragma once
#include "rows_common.cuh"

namespace plr {

enum XType { kX8 = 0, kXBf16 = 1, kXHalf = 2, kXFloat = 3 };

struct SmallArgs {
    const void* x;
    const uint8_t* x_scale;
    const void* w;
    const void* bias;
    const void* residual;
    void* y0;
    void* y1;
    void* z;
    uint8_t* z_scale;
    int64_t rows;
    int k, n, split, act;
    int w_dtype, out_dtype, bias_dtype;
    bool vec_x;    // 16-byte accesses to x's rows
    bool vec_w;    // the same for w's
};

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

// ------------------------------------------------------- at most 32 channels
//
// A warp takes 16 kM rows at a time and keeps their sums in registers; the
// weights lie in shared memory in the fragment order of the warp's matrix
// instruction (m16n8k16).  The sum's order is free, so lane (g, t) of a quad
// group is given 16 neighbouring channels t 16.. of each 64 instead of the
// instruction's pairs: 16 bytes of codes (32 of a 16-bit type, 64 of float32)
// per row and load, straight into the operand's registers.
//
// float32 runs as three bfloat16 parts (split3), six products, small first.

template <int kXT> struct NarrowShape {
    static constexpr int kM = kXT == kX8 ? 2 : 1;                               // 16-row fragments
    static constexpr int kRaw = kXT == kX8 ? 1 : kXT == kXFloat ? 4 : 2;        // 16-byte loads per row and 64 channels
};

__host__ __device__ inline int narrow_steps(int k) { return (k + 63) / 64 * 4; }   // of 16 channels
__host__ inline int64_t narrow_fragments(int k, int nf, int parts) { return (int64_t)parts * narrow_steps(k) * nf * 256; }
constexpr int kNarrowWarps = 8;
constexpr int kNarrowPitch = 33;
__host__ inline int64_t narrow_staging(int m) { return (int64_t)kNarrowWarps * 16 * m * kNarrowPitch * 4; }
constexpr int64_t kNarrowMost = 64 * 1024;   // bytes of weights: two CTAs then share an SM

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

template <int kXT, int kFragments = NarrowShape<kXT>::kM>
__device__ __forceinline__ void narrow_load(NarrowRaw<kXT>& r, const SmallArgs& a, int64_t row0, int chunk, int lane) {
    const int g = lane >> 2, ch = chunk * 64 + (lane & 3) * 16;
#pragma unroll
    for (int m = 0; m < kFragments; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int64_t row = row0 + m * 16 + h * 8 + g;
            const bool live = row < a.rows;
#pragma unroll
            for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) r.v[m][h][i] = make_uint4(0, 0, 0, 0);
            if (kXT == kX8) {
                const int width = (a.k + 31) / 32 * 32;
                r.scale[m][h] = 127;
                if (live && ch < width) {
                    const int64_t at = row * width + ch;
                    r.v[m][h][0] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(a.x) + at);
                    r.scale[m][h] = a.x_scale[at >> 5];
                }
                continue;
            }
            constexpr int kPer = kXT == kXFloat ? 4 : 8;   // elements of a 16-byte load
#pragma unroll
            for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) {
                const int c = ch + i * kPer;
                if (!live || c >= a.k) continue;
                if (a.vec_x) {
                    r.v[m][h][i] = kXT == kXFloat
                        ? *reinterpret_cast<const uint4*>(static_cast<const float*>(a.x) + row * a.k + c)
                        : *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.x) + row * a.k + c);
                } else if (kXT == kXFloat) {
                    union { uint4 u; float f[4]; } o;
#pragma unroll
                    for (int j = 0; j < 4; ++j) o.f[j] = c + j < a.k ? static_cast<const float*>(a.x)[row * a.k + c + j] : 0.f;
                    r.v[m][h][i] = o.u;
                } else {
                    union { uint4 u; uint16_t f[8]; } o;
#pragma unroll
                    for (int j = 0; j < 8; ++j) o.f[j] = c + j < a.k ? static_cast<const uint16_t*>(a.x)[row * a.k + c + j] : 0;
                    r.v[m][h][i] = o.u;
                }
            }
        }
}

// The operand registers of step s (4 of the lane's 16 channels), part p of kPA.
template <int kXT, int kPA>
__device__ __forceinline__ void narrow_operand(const NarrowRaw<kXT>& r, int m, int s, uint32_t (&o)[kPA][4]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (kXT == kX8) {
            const uint4& q = r.v[m][h][0];
            float f[4];
            values4(f, s == 0 ? q.x : s == 1 ? q.y : s == 2 ? q.z : q.w, scale_of(r.scale[m][h]));
            union { __nv_bfloat162 b; uint32_t u; } lo, hi;   // exact
            lo.b = __floats2bfloat162_rn(f[0], f[1]);
            hi.b = __floats2bfloat162_rn(f[2], f[3]);
            o[0][h] = lo.u;
            o[0][2 + h] = hi.u;
        } else if (kXT == kXFloat) {
            const uint4& q = r.v[m][h][s];
            uint32_t lo[3], hi[3];
            split3_pair(__uint_as_float(q.x), __uint_as_float(q.y), lo);
            split3_pair(__uint_as_float(q.z), __uint_as_float(q.w), hi);
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

// Stores columns [c0, c0 + w) of `rows` staged rows to a tensor of w columns
// whose rows they are: one run of rows x w elements.
__device__ __forceinline__ void narrow_run(const float* st, void* dst, int dtype, int64_t row0, int rows, int c0, int w,
                                           const void* add, int lane) {
    const unsigned inv = 65536u / (unsigned)w + 1;   // t / w for t < 1024, w <= 32
    for (int t = lane; t < rows * w; t += 32) {
        const int r = (int)((t * inv) >> 16), c = t - r * w;
        float v = st[r * kNarrowPitch + c0 + c];
        if (add) v += load_param(add, dtype, row0 * w + t);
        store_param(dst, dtype, row0 * w + t, v);
    }
}

// kSplit: few rows and many channels: the CTA's warps take turns over the
// channels of the same rows and their sums are added in shared memory, in order.
template <int kXT, int kNF, bool kW3, bool kSplit>
__global__ void __launch_bounds__(32 * kNarrowWarps, 2) k_narrow(const SmallArgs a) {
    constexpr int kM = NarrowShape<kXT>::kM, kPA = kXT == kXFloat ? 3 : 1, kPB = kW3 ? 3 : 1;
    extern __shared__ __align__(16) char smem_raw[];
    __shared__ float sbias[32];
    const int steps = narrow_steps(a.k), chunks = steps / 4;
    uint2* frag = reinterpret_cast<uint2*>(smem_raw);   // [kPB][steps][kNF][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    float* st = reinterpret_cast<float*>(smem_raw + (size_t)kPB * steps * kNF * 256) + warp * 16 * kM * kNarrowPitch;

    if (threadIdx.x < 32)
        sbias[threadIdx.x] = a.bias && (int)threadIdx.x < a.n ? load_param(a.bias, a.bias_dtype, threadIdx.x) : 0.f;
    for (int i = threadIdx.x; i < steps * kNF * 32; i += blockDim.x) {
        const int l = i & 31, f = (i >> 5) % kNF, s = (i >> 5) / kNF;
        const int col = f * 8 + (l >> 2), ch = (s >> 2) * 64 + (l & 3) * 16 + (s & 3) * 4;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = col < a.n && ch + j < a.k ? load_param(a.w, a.w_dtype, (int64_t)col * a.k + ch + j) : 0.f;
        uint32_t lo[3], hi[3];
        if (kW3) {
            split3_pair(v[0], v[1], lo);
            split3_pair(v[2], v[3], hi);
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

    NarrowRaw<kXT> next;
    if (block < blocks && chunk0 < chunks) narrow_load<kXT>(next, a, block * (16 * kM), chunk0, lane);
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
            const NarrowRaw<kXT> raw = next;
            if (c + chunk_step < chunks) narrow_load<kXT>(next, a, row0, c + chunk_step, lane);
            else if (block + stride < blocks) narrow_load<kXT>(next, a, row0 + stride * (16 * kM), chunk0, lane);
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                uint2 b[kPB][kNF];
#pragma unroll
                for (int p = 0; p < kPB; ++p)
#pragma unroll
                    for (int f = 0; f < kNF; ++f) b[p][f] = frag[((p * steps + c * 4 + s) * kNF + f) * 32 + lane];
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    uint32_t o[kPA][4];
                    narrow_operand<kXT, kPA>(raw, m, s, o);
#pragma unroll
                    for (int sum = 2; sum >= 0; --sum)   // small products first
#pragma unroll
                        for (int pa = 0; pa < kPA; ++pa) {
                            const int pb = sum - pa;
                            if (pb < 0 || pb >= kPB) continue;
#pragma unroll
                            for (int f = 0; f < kNF; ++f)
                                mma16816<kXT == kXHalf>(acc[m][f], o[pa][0], o[pa][1], o[pa][2], o[pa][3], b[pb][f]);
                        }
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
        const bool keep = a.z != nullptr;
        for (int pass = keep ? 0 : 1; pass < 2; ++pass) {   // z, then y
            __syncwarp();
#pragma unroll
            for (int m = 0; m < kM; ++m)
#pragma unroll
                for (int f = 0; f < kNF; ++f) {
                    if (pass == 0 || !keep) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[m][f][i] += sbias[f * 8 + t * 2 + (i & 1)];
                    }
                    if (pass == 1) activate(acc[m][f], a.act);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        st[(m * 16 + (i >> 1) * 8 + g) * kNarrowPitch + f * 8 + t * 2 + (i & 1)] = acc[m][f][i];
                }
            __syncwarp();
            if (pass == 0 && a.z_scale) {   // the whole row is one block; 16 columns a lane
#pragma unroll
                for (int m = 0; m < kM; ++m) {
                    const int r = m * 16 + (lane >> 1), c0 = (lane & 1) * 16;
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        v[i] = c0 + i < kNF * 8 ? st[r * kNarrowPitch + c0 + i] : 0.f;
                    bool infinite;
                    float amax = finite_amax_of(v, infinite);
                    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                    const int e = block_exponent(amax);
                    if (r < rows) {
                        const float inv = pow2(-e);
                        const uint2 x = codes8_of(v, inv, infinite), y = codes8_of(v + 8, inv, infinite);
                        reinterpret_cast<uint4*>(a.z)[(row0 + r) * 2 + (lane & 1)] = make_uint4(x.x, x.y, y.x, y.y);
                        if ((lane & 1) == 0) a.z_scale[row0 + r] = (uint8_t)(e + 127);
                    }
                }
            } else if (pass == 0) {
                narrow_run(st, a.z, a.out_dtype, row0, rows, 0, a.n, nullptr, lane);
            } else if (a.split) {
                narrow_run(st, a.y0, a.out_dtype, row0, rows, 0, a.split, nullptr, lane);
                narrow_run(st, a.y1, a.out_dtype, row0, rows, a.split, a.n - a.split, nullptr, lane);
            } else {
                narrow_run(st, a.y0, a.out_dtype, row0, rows, 0, a.n, a.residual, lane);
            }
        }
    }
}

// ------------------------------------ backward, at most 32 output channels
//
// One pass: a warp takes 16 rows and a slice of 64 input channels, makes gz
// (grad_y act'(z), rounded to the operands' type) once in shared memory, and
// from it the rows' grad_x (gz w) and its share of grad_w (x^T gz, kept in
// registers over all of the warp's rows) and grad_bias.  What a CTA gathered
// goes to `partial`, one line of n k + n sums per CTA of a slice's column;
// k_sum_lines adds those in order.  Read once: grad_y and z per slice, x;
// written once: grad_x.
struct SmallGradArgs {
    SmallArgs s;          // x, x_scale, w, z, z_scale, rows, k, n, split, act, types, alignments
    const void* g0;
    const void* g1;
    void* grad_x;
    float* partial;       // [gridDim.x][n k + n]: grad_w [n][k], then grad_bias [n]
    bool need_x, need_w, need_b;
    bool vec_gx;          // 16-byte accesses to grad_x's rows
};

constexpr int kGradWarps = 4;
constexpr int kTilePitch = 72;   // 16-bit elements: rows 144 bytes apart, no bank conflicts for ldmatrix

template <int kXT, int kParts> struct NarrowGradShape {
    static constexpr int kPX = kXT == kXFloat ? 3 : 1;
    static constexpr int kFragBytes = kParts * 2 * 8 * 32 * 8;                        // weights of the slice
    static constexpr int kWarpBytes = 16 * kNarrowPitch * 4 + kPX * 16 * kTilePitch * 2;
    static constexpr int kBytes = kFragBytes + kGradWarps * kWarpBytes + 64 * 33 * 4;
};

template <int kP>
__device__ __forceinline__ void to_parts(float a, float b, bool half, uint32_t (&o)[kP]) {
    if (kP == 3) {
        uint32_t t[3];
        split3_pair(a, b, t);
#pragma unroll
        for (int i = 0; i < kP; ++i) o[i] = t[i];
    } else if (half) {
        union { __half2 h; uint32_t u; } x;
        x.h = __floats2half2_rn(a, b);
        o[0] = x.u;
    } else {
        union { __nv_bfloat162 h; uint32_t u; } x;
        x.h = __floats2bfloat162_rn(a, b);
        o[0] = x.u;
    }
}

// Element e of the 16 rows' gradients, g0's run first, then g1's: its place
// (row, column) and value.
struct GradRun {
    const void *g0, *g1;
    int dtype, w0, w1, rows;
    unsigned inv0, inv1;
    int64_t row0;
    __device__ __forceinline__ GradRun(const SmallGradArgs& a, int64_t row0_)
        : g0(a.g0), g1(a.g1), dtype(a.s.out_dtype), w0(a.s.split ? a.s.split : a.s.n), w1(a.s.split ? a.s.n - a.s.split : 1),
          rows((int)min((int64_t)16, a.s.rows - row0_)), row0(row0_) {
        inv0 = 65536u / (unsigned)w0 + 1;   // t / w for t < 1024, w <= 32
        inv1 = 65536u / (unsigned)w1 + 1;
        if (!a.s.split) w1 = 0;
    }
    __device__ __forceinline__ float value(int e) const {
        if (e < rows * w0) return load_param(g0, dtype, row0 * w0 + e);
        e -= rows * w0;
        return e < rows * w1 ? load_param(g1, dtype, row0 * w1 + e) : 0.f;
    }
    // offset in the staged rows, -1 behind the end
    __device__ __forceinline__ int place(int e) const {
        if (e < rows * w0) {
            const int r = (int)((e * inv0) >> 16);
            return r * kNarrowPitch + e - r * w0;
        }
        e -= rows * w0;
        if (e >= rows * w1) return -1;
        const int r = (int)((e * inv1) >> 16);
        return r * kNarrowPitch + w0 + e - r * w1;
    }
};

// kXT: the type of x (and, for 16-bit ones, of everything); kParts: 3 with
// float32 weights; kNF: output channels / 8.
template <int kXT, int kParts, int kNF>
__global__ void __launch_bounds__(32 * kGradWarps, kParts == 3 ? 2 : 3) k_narrow_grad(const SmallGradArgs a) {
    typedef NarrowGradShape<kXT, kParts> Shape;
    constexpr int kPX = Shape::kPX, kKS = kNF > 2 ? 2 : 1;   // steps of 16 output channels in grad_x's sum
    constexpr bool kHalf = kXT == kXHalf;
    extern __shared__ __align__(16) char smem_raw[];
    uint2* frag = reinterpret_cast<uint2*>(smem_raw);   // [kParts][kKS][8][32]
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    char* mine = smem_raw + Shape::kFragBytes + warp * Shape::kWarpBytes;
    float* st = reinterpret_cast<float*>(mine);                                       // gz, 16 x 33
    uint16_t* tile = reinterpret_cast<uint16_t*>(mine + 16 * kNarrowPitch * 4);       // x, [kPX][16][72]
    float* gather = reinterpret_cast<float*>(smem_raw + Shape::kFragBytes + kGradWarps * Shape::kWarpBytes);
    const int ch0 = blockIdx.y * 64, n = a.s.n, k = a.s.k;
    const int cols_per_lane = kKS * 4;   // output channels of lane t in grad_x's sum: t cols_per_lane..

    // fragment f, column c of the weights is channel (c >> 1) 16 + 2 f + (c & 1)
    // of the slice, so that a lane ends up with 16 neighbouring channels
    if (a.need_x) {
        for (int i = threadIdx.x; i < kKS * 8 * 32; i += blockDim.x) {
            const int l = i & 31, f = (i >> 5) & 7, s = i >> 8;
            const int ch = ch0 + (l >> 3) * 16 + 2 * f + ((l >> 2) & 1), o = (l & 3) * cols_per_lane + s * 4;
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                v[j] = o + j < n && ch < k ? load_param(a.s.w, a.s.w_dtype, (int64_t)(o + j) * k + ch) : 0.f;
            uint32_t lo[kParts], hi[kParts];
            to_parts<kParts>(v[0], v[1], kHalf, lo);
            to_parts<kParts>(v[2], v[3], kHalf, hi);
#pragma unroll
            for (int p = 0; p < kParts; ++p) frag[p * kKS * 256 + i] = make_uint2(lo[p], hi[p]);
        }
    }
    for (int i = lane; i < 16 * kNarrowPitch; i += 32) st[i] = 0.f;   // columns behind n stay 0
    __syncthreads();

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
    constexpr int kRun = kNF * 4;   // 16 rows x 8 kNF columns / 32 lanes
    float gn[kRun];                 // the next rows' gradients, x and z, loaded ahead
    uint4 xn[2][NarrowShape<kXT>::kRaw];
    uint8_t xs[2];
    uint4 zn = make_uint4(0, 0, 0, 0);
    uint8_t zs = 127;
    auto load_rows = [&](int64_t b) {
        const GradRun run(a, b * 16);
#pragma unroll
        for (int i = 0; i < kRun; ++i) gn[i] = run.value(i * 32 + lane);
        if (a.s.z_scale) {   // a lane per half row
            const int64_t row = b * 16 + (lane >> 1);
            const bool live = row < a.s.rows;
            zn = live ? reinterpret_cast<const uint4*>(a.s.z)[row * 2 + (lane & 1)] : make_uint4(0, 0, 0, 0);
            zs = live ? a.s.z_scale[row] : 127;
        }
        if (!a.need_w) return;
        NarrowRaw<kXT> r;
        narrow_load<kXT, 1>(r, a.s, b * 16, blockIdx.y, lane);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < NarrowShape<kXT>::kRaw; ++i) xn[h][i] = r.v[0][h][i];
            if (kXT == kX8) xs[h] = r.scale[0][h];
        }
    };
    if (block < blocks) load_rows(block);
    for (; block < blocks; block += stride) {
        const int64_t row0 = block * 16;
        const int rows = (int)min((int64_t)16, a.s.rows - row0);
        __syncwarp();
        {
            const GradRun run(a, row0);
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const int at = run.place(i * 32 + lane);
                if (at >= 0) st[at] = gn[i];
            }
        }
        if (rows < 16)
            for (int i = rows * kNarrowPitch + lane; i < 16 * kNarrowPitch; i += 32) st[i] = 0.f;
        if (a.need_w) {   // x, widened, into the tile
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint16_t* row = tile + (g + 8 * h) * kTilePitch + t * 16;
                if (kXT == kX8) {
                    float v[16];
                    const float sc = scale_of(xs[h]);
                    values4(v, xn[h][0].x, sc);
                    values4(v + 4, xn[h][0].y, sc);
                    values4(v + 8, xn[h][0].z, sc);
                    values4(v + 12, xn[h][0].w, sc);
                    union { uint4 u[2]; __nv_bfloat162 b[8]; } o;   // exact
#pragma unroll
                    for (int i = 0; i < 8; ++i) o.b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                    reinterpret_cast<uint4*>(row)[0] = o.u[0];
                    reinterpret_cast<uint4*>(row)[1] = o.u[1];
                } else if (kXT == kXFloat) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4& q = xn[h][i % NarrowShape<kXT>::kRaw];
                        uint32_t lo[3], hi[3];
                        split3_pair(__uint_as_float(q.x), __uint_as_float(q.y), lo);
                        split3_pair(__uint_as_float(q.z), __uint_as_float(q.w), hi);
#pragma unroll
                        for (int p = 0; p < 3; ++p)
                            *reinterpret_cast<uint2*>(row + (p % kPX) * 16 * kTilePitch + i * 4) = make_uint2(lo[p], hi[p]);
                    }
                } else {
                    reinterpret_cast<uint4*>(row)[0] = xn[h][0];
                    reinterpret_cast<uint4*>(row)[1] = xn[h][1 % NarrowShape<kXT>::kRaw];
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
        if (a.need_b) {
#pragma unroll
            for (int r = 0; r < 16; ++r) db += st[r * kNarrowPitch + lane];
        }
        if (a.need_x) {
            uint32_t o[kKS][kParts][4];
#pragma unroll
            for (int s = 0; s < kKS; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float* p = st + (g + 8 * h) * kNarrowPitch + t * cols_per_lane + s * 4;
                    uint32_t lo[kParts], hi[kParts];
                    to_parts<kParts>(p[0], p[1], kHalf, lo);
                    to_parts<kParts>(p[2], p[3], kHalf, hi);
#pragma unroll
                    for (int q = 0; q < kParts; ++q) {
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
                for (int sum = 2; sum >= 0; --sum)   // small products first
#pragma unroll
                    for (int pa = 0; pa < kParts; ++pa) {
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
            uint32_t b[kParts][kNF][2];
#pragma unroll
            for (int f = 0; f < kNF; ++f)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float* p = st + (2 * t + 8 * h) * kNarrowPitch + f * 8 + g;
                    uint32_t o[kParts];
                    to_parts<kParts>(p[0], p[kNarrowPitch], kHalf, o);
#pragma unroll
                    for (int q = 0; q < kParts; ++q) b[q][f][h] = o[q];
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
#pragma unroll
                for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                    for (int px = 0; px < kPX; ++px) {
                        const int pb = sum - px;
                        if (pb < 0 || pb >= kParts) continue;
#pragma unroll
                        for (int f = 0; f < kNF; ++f)
                            mma16816<kHalf>(dw[m][f], x[px][0], x[px][1], x[px][2], x[px][3],
                                            make_uint2(b[pb][f][0], b[pb][f][1]));
                    }
            }
        }
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
// One warp per output channel reads its weights once, 16 bytes a lane, against
// the rows in shared memory (float32, in pieces of 1024 channels); a CTA takes
// 32 channels, the block of a kept 8-bit pre-activation.  Bound by the read of
// w: 2.x us for 1024 -> 4096 in bfloat16 (8.4 MB).

constexpr int kFewWarps = 32, kFewPiece = 1024;

template <typename TW, int kRows>
__global__ void __launch_bounds__(32 * kFewWarps) k_few(const SmallArgs a) {
    __shared__ __align__(16) float sx[kRows][kFewPiece];
    __shared__ float sz[kRows][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int col = blockIdx.x * 32 + warp;
    const TW* w = static_cast<const TW*>(a.w) + (int64_t)min(col, a.n - 1) * a.k;
    const int width = (a.k + 31) / 32 * 32;
    float acc[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) acc[r] = 0.f;
    for (int base = 0; base < a.k; base += kFewPiece) {
        Raw8<TW> raw[kFewPiece / 256];   // in flight while the rows are staged
#pragma unroll
        for (int j = 0; j < kFewPiece / 256; ++j) {
            const int c = base + j * 256 + lane * 8, left = a.k - c;
            raw[j].load(w + (left > 0 ? c : 0), a.vec_w && left >= 8, left);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < kRows * kFewPiece; i += 32 * kFewWarps) {
            const int r = i / kFewPiece, c = i % kFewPiece;
            float v = 0.f;
            if (r < a.rows && base + c < a.k) {
                if (a.x_scale) {
                    const int64_t at = (int64_t)r * width + base + c;
                    float q[4];
                    values4(q, static_cast<const uint8_t*>(a.x)[at], scale_of(a.x_scale[at >> 5]));
                    v = q[0];
                } else {
                    v = to_f32(static_cast<const TW*>(a.x)[(int64_t)r * a.k + base + c]);
                }
            }
            // a lane's 8 channels as two float4 of separate halves: no bank conflicts
            sx[r][(c & ~255) + ((c >> 2) & 1) * 128 + ((c & 255) >> 3) * 4 + (c & 3)] = v;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kFewPiece / 256; ++j) {
            if (base + j * 256 >= a.k) break;
            float v[8];
            raw[j].widen(v);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                const float4 p = *reinterpret_cast<const float4*>(&sx[r][j * 256 + lane * 4]);
                const float4 q = *reinterpret_cast<const float4*>(&sx[r][j * 256 + 128 + lane * 4]);
                acc[r] = fmaf(v[0], p.x, fmaf(v[1], p.y, fmaf(v[2], p.z, fmaf(v[3], p.w, acc[r]))));
                acc[r] = fmaf(v[4], q.x, fmaf(v[5], q.y, fmaf(v[6], q.z, fmaf(v[7], q.w, acc[r]))));
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[r] += __shfl_xor_sync(0xffffffffu, acc[r], o);
        if (lane == 0) sz[r][warp] = col < a.n ? acc[r] + (a.bias ? load_param(a.bias, a.bias_dtype, col) : 0.f) : 0.f;
    }
    __syncthreads();
    if (warp >= kRows || warp >= a.rows) return;
    // a warp per row, a lane per channel
    const int c = blockIdx.x * 32 + lane;
    float z = sz[warp][lane];
    if (a.z_scale) {
        float amax = is_infinite(fabsf(z)) ? 0.f : fabsf(z);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int e = block_exponent(amax);
        const float v[8] = {z, 0, 0, 0, 0, 0, 0, 0};
        const int64_t at = (int64_t)warp * ((a.n + 31) / 32) + blockIdx.x;
        static_cast<uint8_t*>(a.z)[at * 32 + lane] = (uint8_t)codes8_of(v, pow2(-e), is_infinite(fabsf(z))).x;
        if (lane == 0) a.z_scale[at] = (uint8_t)(e + 127);
    } else if (a.z && c < a.n) {
        store_param(a.z, a.out_dtype, (int64_t)warp * a.n + c, z);
    }
    if (c >= a.n) return;
    float y[2] = {z, 0.f};
    activate(y, a.act);
    if (a.residual) y[0] += load_param(a.residual, a.out_dtype, (int64_t)warp * a.n + c);
    if (c < a.split) store_param(a.y0, a.out_dtype, (int64_t)warp * a.split + c, y[0]);
    else if (a.split) store_param(a.y1, a.out_dtype, (int64_t)warp * (a.n - a.split) + c - a.split, y[0]);
    else store_param(a.y0, a.out_dtype, (int64_t)warp * a.n + c, y[0]);
}

}  // namespace plr
