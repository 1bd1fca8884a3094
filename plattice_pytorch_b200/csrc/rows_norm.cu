// rows_norm.cu -- 8-bit rows (pack, unpack) and the root-mean-square norm of
// rows with the residual's addition, forward and backward.  Formats and
// element access: rows_common.cuh; C ABI: include/plattice.h.
#include <limits.h>

#include "plattice_runtime.h"
#include "rows_common.cuh"
#include "rows_host.h"

namespace plr {

// ------------------------------------------------------------ pack / unpack
//
// A thread takes 8 channels, 4 neighbouring lanes a block of 32.  Both kernels
// move each byte once and are bound by HBM: 262144 x 256 in bfloat16 (203 MB,
// 31.1 us at the copy rate) takes 35.5 us to pack and 33.4 to unpack.  A CTA
// takes kUnits x 256 such groups of 8, so that each thread has kUnits
// independent loads in flight.

constexpr int kUnits = 4;

// Rows without padding and aligned (c a multiple of 32): group g is elements
// 8 g.. whatever its row.
template <typename T>
__global__ void __launch_bounds__(256) k_pack8(uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                                               const T* __restrict__ x, int64_t all) {
    const int64_t base = (int64_t)blockIdx.x * (256 * kUnits);
    float v[kUnits][8];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = base + threadIdx.x + 256 * u;
        load8(v[u], x + (at < all ? at : 0) * 8, true, 8);
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t at = base + threadIdx.x + 256 * u;
        float amax = finite_amax(v[u]);
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int s = block_exponent(amax);
        if (at >= all) continue;
        reinterpret_cast<uint2*>(q)[at] = codes8(v[u], pow2(-s));
        if ((threadIdx.x & 3) == 0) scale[at >> 2] = (uint8_t)(s + 127);
    }
}

// Other rows: a warp takes kBlocks blocks of 32, a lane per channel, so that
// its loads are whole lines wherever the rows begin.
constexpr int kBlocks = 8;

__device__ __forceinline__ uint8_t code1(float v, float inv) {
    if (largest_scale(inv) && !is_infinite(fabsf(v))) v = held8(v);
    return (uint8_t)__nv_cvt_float_to_fp8(is_infinite(fabsf(v)) ? __int_as_float(0x7fffffff) : v * inv, __NV_SATFINITE,
                                          __NV_E4M3);
}

__device__ __forceinline__ float lane_magnitude(float v) { return is_infinite(fabsf(v)) ? 0.f : fmaxf(fabsf(v), 0.f); }

template <typename T>
__global__ void __launch_bounds__(256) k_pack8_any(uint8_t* __restrict__ q, uint8_t* __restrict__ scale,
                                                   const T* __restrict__ x, int64_t rows, int c, unsigned blocks) {
    const int lane = threadIdx.x & 31;
    const GroupAt where(((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * kBlocks, blocks);
    float v[kBlocks];
    int64_t row[kBlocks];
    unsigned b[kBlocks];
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
        where.at(u, row[u], b[u]);
        const int col = (int)b[u] * 32 + lane;
        v[u] = row[u] < rows && col < c ? to_f32(x[row[u] * c + col]) : 0.f;
    }
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
        if (row[u] >= rows) return;   // the same for all lanes
        float amax = lane_magnitude(v[u]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int s = block_exponent(amax);
        const int64_t at = row[u] * blocks + b[u];
        q[at * 32 + lane] = code1(v[u], pow2(-s));
        if (lane == 0) scale[at] = (uint8_t)(s + 127);
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_unpack8(T* __restrict__ y, int64_t pitch, const uint8_t* __restrict__ q,
                                                 const uint8_t* __restrict__ scale, int64_t rows, int c,
                                                 unsigned groups, bool vec) {
    const int64_t base = (int64_t)blockIdx.x * (256 * kUnits);
    const GroupAt where(base, groups);
    uint2 w[kUnits];
    float sc[kUnits];
    int64_t row[kUnits];
    unsigned g[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        where.at(threadIdx.x + 256 * u, row[u], g[u]);
        const int64_t at = row[u] < rows ? row[u] * groups + g[u] : 0;
        w[u] = reinterpret_cast<const uint2*>(q)[at];
        sc[u] = scale_of(scale[at >> 2]);
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if (row[u] >= rows) continue;
        float v[8];
        values8(v, w[u], sc[u]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = within<T>(v[i]);
        const int left = c - (int)g[u] * 8;
        if (left > 0) store8(y + row[u] * pitch + (int64_t)g[u] * 8, v, vec && left >= 8, left);
    }
}

// Rows that lie on no 16-byte boundaries: a warp takes kBlocks blocks of 32, a
// lane per channel.
template <typename T>
__global__ void __launch_bounds__(256) k_unpack8_any(T* __restrict__ y, int64_t pitch, const uint8_t* __restrict__ q,
                                                     const uint8_t* __restrict__ scale, int64_t rows, int c,
                                                     unsigned blocks) {
    const int lane = threadIdx.x & 31;
    const int64_t first = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * kBlocks;
    const GroupAt where(first, blocks);
    uint8_t code[kBlocks], byte[kBlocks];
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
        const int64_t at = min(first + u, rows * blocks - 1);
        code[u] = q[at * 32 + lane];
        byte[u] = scale[at];
    }
#pragma unroll
    for (int u = 0; u < kBlocks; ++u) {
        int64_t row;
        unsigned b;
        where.at(u, row, b);
        const int col = (int)b * 32 + lane;
        if (row < rows && col < c) y[row * pitch + col] = from_f32<T>(within<T>(value1(code[u], scale_of(byte[u]))));
    }
}

// --------------------------------------------------------------- the norm
//
// L threads share a row (L <= 32: several rows per warp; L = 256 or 512: a CTA
// per row); a thread holds kChunks groups of 8 channels in registers, so a row
// is read once whatever its statistics need.  Bound by HBM: 262144 x 256 in
// bfloat16 with residual and 8-bit result (472 MB, 72 us at the copy rate) takes
// 80 us, 65536 x 1024 86, 1048576 x 64 85 (each 82 at the copy rate), 262144 x
// 250 112.  The mean of squares is summed in float32.  h is rounded to the rows' type where it is stored; y is computed
// from the unrounded sum, one rounding from its definition.

// Sum over the threads of a row.  `turn` alternates from call to call: sums of
// one call are still read while the next one's are written elsewhere, so that a
// barrier a call is enough.
template <int L>
__device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
    constexpr int kWarp = L < 32 ? L : 32, kWarps = (L > 256 ? L : 256) / 32;
#pragma unroll
    for (int o = kWarp / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (L > 32) {
        red += turn * kWarps;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int i = 0; i < L / 32; ++i) v += red[threadIdx.x / L * (L / 32) + i];
    }
    return v;
}

// Channel i of a thread's group k, for accesses of kWide neighbouring channels
// (8 where rows lie on 16-byte boundaries, 2 where they have an even number of
// channels, else 1): a warp's lanes take neighbouring pieces of kWide, 8 / kWide
// times, so that each of its accesses is one run wherever the row begins.
template <int L, int kWide> __device__ __forceinline__ int channel_of(int lane, int k, int i) {
    constexpr int kW = L < 32 ? L : 32;
    return (k * L + lane / kW * kW) * 8 + i / kWide * (kW * kWide) + lane % kW * kWide + i % kWide;
}

template <typename T> struct Two;
template <> struct Two<float> { typedef float2 type; };
template <> struct Two<__nv_bfloat16> { typedef __nv_bfloat162 type; };
template <> struct Two<__half> { typedef __half2 type; };
__device__ __forceinline__ float2 pair_f32(float2 v) { return v; }
__device__ __forceinline__ void pair_from(float2& o, float a, float b) { o = make_float2(a, b); }

template <typename T, int L, int kWide>
__device__ __forceinline__ void load_group(float (&v)[8], const T* row, int lane, int k, int c) {
    if constexpr (kWide == 8) {
        const int col = channel_of<L, 8>(lane, k, 0);
        load8(v, row + (col < c ? col : 0), col < c, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += kWide) {
            const int col = channel_of<L, kWide>(lane, k, i);
            if constexpr (kWide == 2) {
                typename Two<T>::type t;
                pair_from(t, 0.f, 0.f);
                if (col < c) t = *reinterpret_cast<const typename Two<T>::type*>(row + col);
                const float2 f = pair_f32(t);
                v[i] = f.x;
                v[i + 1] = f.y;
            } else {
                v[i] = col < c ? to_f32(row[col]) : 0.f;
            }
        }
    }
}

template <typename T, int L, int kWide>
__device__ __forceinline__ void store_group(T* row, const float (&v)[8], int lane, int k, int c) {
    if constexpr (kWide == 8) {
        const int col = channel_of<L, 8>(lane, k, 0);
        if (col < c) store8(row + col, v, true, 8);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i += kWide) {
            const int col = channel_of<L, kWide>(lane, k, i);
            if (col >= c) continue;
            if constexpr (kWide == 2) pair_from(*reinterpret_cast<typename Two<T>::type*>(row + col), v[i], v[i + 1]);
            else row[col] = from_f32<T>(v[i]);
        }
    }
}

// Group k of a row as 8-bit rows; q and scale are the row's.  All lanes call.
// A block of 32 channels is kTimes pieces of each of kLanes neighbouring lanes.
template <int L, int kWide>
__device__ __forceinline__ void store_group8(uint8_t* q, uint8_t* scale, float (&y)[8], int lane, int k, int width,
                                             bool live) {
    constexpr int kW = L < 32 ? L : 32, kLanes = kW < 32 / kWide ? kW : 32 / kWide, kTimes = 32 / (kLanes * kWide);
#pragma unroll
    for (int first = 0; first < 8; first += kTimes * kWide) {
        float amax = 0.f;
#pragma unroll
        for (int i = first; i < first + kTimes * kWide; ++i) {
            if (is_infinite(fabsf(y[i]))) y[i] = __int_as_float(0x7fffffff);   // its code, and passed over here
            amax = fmaxf(amax, fabsf(y[i]));
        }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const int s = block_exponent(amax);
        const float inv = pow2(-s);
        if (kWide < 8 && largest_scale(inv)) {
#pragma unroll
            for (int i = first; i < first + kTimes * kWide; ++i) y[i] = held8(y[i]);
        }
#pragma unroll
        for (int i = first; i < first + kTimes * kWide; i += kWide) {
            const int col = channel_of<L, kWide>(lane, k, i);
            if (!live || col >= width) continue;
            if constexpr (kWide == 8)
                *reinterpret_cast<uint2*>(q + col) = codes8(y, inv);
            else if constexpr (kWide == 2)
                *reinterpret_cast<__nv_fp8x2_storage_t*>(q + col) =
                    __nv_cvt_float2_to_fp8x2(make_float2(y[i] * inv, y[i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
            else
                q[col] = (uint8_t)__nv_cvt_float_to_fp8(y[i] * inv, __NV_SATFINITE, __NV_E4M3);
            if ((col & 31) == 0) scale[col >> 5] = (uint8_t)(s + 127);
        }
    }
}

struct NormArgs {
    void* y;
    uint8_t* yscale;   // non-null: y is 8-bit rows
    void* h;           // null: not stored
    float* rstd;
    const void* x;
    const void* residual;   // null: none
    const void* gain;
    int gain_dtype;
    float eps;
    int64_t rows;
    int c;
    int wide;   // channels of an access: 8, 2 or 1
};

template <typename T, int L, int kChunks, int kWide>
__global__ void __launch_bounds__(L > 256 ? L : 256) k_rms_norm(const NormArgs a) {
    constexpr int kThreads = L > 256 ? L : 256;
    constexpr int kRows = kThreads / L;
    __shared__ float red[L > 32 ? kThreads / 16 : 1];
    int turn = 0;
    const int lane = threadIdx.x % L;
    const int width = (int)width8(a.c);
    float gain[kChunks][8];
#pragma unroll
    for (int k = 0; k < kChunks; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = channel_of<L, kWide>(lane, k, i);
            gain[k][i] = col < a.c ? load_param(a.gain, a.gain_dtype, col) : 0.f;
        }
    const float inv_c = 1.f / (float)a.c;
    const int64_t stride = (int64_t)gridDim.x * kRows;
    Raw8<T> x[kChunks], r[kChunks];   // aligned rows: the next row's, loaded while this one is worked on
    auto load_row = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            const int col = channel_of<L, 8>(lane, k, 0);
            const bool have = row < a.rows && col < a.c;
            const int64_t at = have ? row * a.c + col : 0;
            x[k].load(static_cast<const T*>(a.x) + at, have, 0);
            if (a.residual) r[k].load(static_cast<const T*>(a.residual) + at, have, 0);
        }
    };
    if (kWide == 8) load_row((int64_t)blockIdx.x * kRows + threadIdx.x / L);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.rows; row0 += stride) {
        const int64_t row = row0 + threadIdx.x / L;
        const bool live = row < a.rows;
        const int64_t at = live ? row * a.c : 0;
        float v[kChunks][8];
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            float t[8];
            if (kWide == 8) {
                x[k].widen(v[k]);
                if (a.residual) r[k].widen(t);
            } else {
                load_group<T, L, kWide>(v[k], static_cast<const T*>(a.x) + at, lane, k, live ? a.c : 0);
                if (a.residual) load_group<T, L, kWide>(t, static_cast<const T*>(a.residual) + at, lane, k, live ? a.c : 0);
            }
            if (a.residual) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[k][i] += t[i];
            }
        }
        if (kWide == 8) load_row(row + stride);
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(v[k][i], v[k][i], ss);
        const float rstd = rsqrtf(row_sum<L>(ss, red, turn) * inv_c + a.eps);
        if (live && lane == 0) a.rstd[row] = rstd;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            if (a.h && live) store_group<T, L, kWide>(static_cast<T*>(a.h) + at, v[k], lane, k, a.c);
            float y[8];   // the gain is 0 behind the last channel
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = v[k][i] * rstd * gain[k][i];
            if (a.yscale && !(rstd < INFINITY)) {   // rare: zeros there all the same
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (channel_of<L, kWide>(lane, k, i) >= a.c) y[i] = 0.f;
            }
            if (a.yscale)
                store_group8<L, kWide>(static_cast<uint8_t*>(a.y) + row * width, a.yscale + row * (width / 32), y, lane, k,
                                      width, live);
            else if (live)
                store_group<T, L, kWide>(static_cast<T*>(a.y) + at, y, lane, k, a.c);
        }
    }
}

// CTAs that share an SM: as many as the registers reach for without spilling.
__host__ __device__ constexpr int norm_grad_ctas(int size, int lanes, int chunks) {
    if (chunks > 1) return lanes == 32 ? 2 : 1;
    return (size == 2 ? 4 : 3) / (lanes > 256 ? 2 : 1);
}

struct NormGradArgs {
    void* grad_x;
    float* partial;   // [gridDim.x][c]: each CTA's sum of grad_y * n
    const void* grad_y;
    const void* h;
    const float* rstd;
    const void* gain;
    int gain_dtype;
    const void* grad_h;   // null: none
    int64_t rows;
    int c;
    int wide;
};

// With n = h rstd and gn = grad_y gain:  grad_x = rstd (gn - n mean(gn n)) + grad_h.
// A thread keeps its channels from row to row, so the gain's gradient is
// summed in registers, then over the CTA's rows in shared memory, and one row
// of sums per CTA goes to `partial`; k_column_sums adds those in a fixed order
// (no atomics: the same input gives the same bits).  262144 x 256 in bfloat16
// with grad_h (537 MB, 82 us at the copy rate) takes 87 us and 3.6 for the sums;
// rows of more than 512 channels wait for their CTA's barrier (65536 x 1024: 114).
template <typename T, int L, int kChunks, int kWide>
__global__ void __launch_bounds__(L > 256 ? L : 256, norm_grad_ctas(sizeof(T), L, kChunks)) k_rms_norm_grad(const NormGradArgs a) {
    constexpr int kThreads = L > 256 ? L : 256;
    constexpr int kRows = kThreads / L;
    __shared__ float red[L > 32 ? kThreads / 16 : 1];
    int turn = 0;
    __shared__ float sums[kRows > 1 ? kThreads * 8 : 1];
    const int lane = threadIdx.x % L;
    float gain[kChunks][8], acc[kChunks][8];
#pragma unroll
    for (int k = 0; k < kChunks; ++k)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = channel_of<L, kWide>(lane, k, i);
            gain[k][i] = col < a.c ? load_param(a.gain, a.gain_dtype, col) : 0.f;
            acc[k][i] = 0.f;
        }
    const float inv_c = 1.f / (float)a.c;
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.rows; row0 += (int64_t)gridDim.x * kRows) {
        const int64_t row = row0 + threadIdx.x / L;
        const bool live = row < a.rows;
        const int c = live ? a.c : 0;
        const int64_t at = live ? row * a.c : 0;
        const float rstd = live ? a.rstd[row] : 0.f;
        float n[kChunks][8], g[kChunks][8];
        Raw8<T> gh[kChunks];   // asked for with the others, used after the row's sum
        float dot = 0.f;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            load_group<T, L, kWide>(n[k], static_cast<const T*>(a.h) + at, lane, k, c);
            load_group<T, L, kWide>(g[k], static_cast<const T*>(a.grad_y) + at, lane, k, c);
            if (kWide == 8 && a.grad_h) {
                const int col = channel_of<L, 8>(lane, k, 0);
                gh[k].load(static_cast<const T*>(a.grad_h) + at + (col < c ? col : 0), col < c, 0);
            }
        }
#pragma unroll
        for (int k = 0; k < kChunks; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                n[k][i] *= rstd;
                acc[k][i] = fmaf(g[k][i], n[k][i], acc[k][i]);
                g[k][i] *= gain[k][i];
                dot = fmaf(g[k][i], n[k][i], dot);
            }
        const float m = row_sum<L>(dot, red, turn) * inv_c;
        if (!live) continue;
#pragma unroll
        for (int k = 0; k < kChunks; ++k) {
            float o[8];
            if (kWide == 8 && a.grad_h) gh[k].widen(o);
            else if (a.grad_h) load_group<T, L, kWide>(o, static_cast<const T*>(a.grad_h) + at, lane, k, c);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float d = rstd * (g[k][i] - n[k][i] * m);
                o[i] = a.grad_h ? o[i] + d : d;
            }
            store_group<T, L, kWide>(static_cast<T*>(a.grad_x) + at, o, lane, k, a.c);
        }
    }
#pragma unroll
    for (int k = 0; k < kChunks; ++k) {
        if (kRows == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int col = channel_of<L, kWide>(lane, k, i);
                if (col < a.c) a.partial[(int64_t)blockIdx.x * a.c + col] = acc[k][i];
            }
            continue;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) sums[i * kThreads + threadIdx.x] = acc[k][i];
        __syncthreads();
        for (int t = threadIdx.x; t < L * 8; t += kThreads) {
            const int i = t / L, l = t % L, col = channel_of<L, kWide>(l, k, i);
            float s = 0.f;
            for (int r = 0; r < kRows; ++r) s += sums[i * kThreads + r * L + l];
            if (col < a.c) a.partial[(int64_t)blockIdx.x * a.c + col] = s;
        }
    }
}

// out[col] = sum over the parts of partial[part][col]: a CTA takes 32 columns,
// its 32 warps every 32nd part each.
__global__ void __launch_bounds__(1024) k_column_sums(void* out, int dtype, const float* __restrict__ partial,
                                                      int parts, int64_t c) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t col = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.f;
    if (col < c)
        for (int p = w; p < parts; p += 32) v += partial[(int64_t)p * c + col];
    s[w][lane] = v;
    __syncthreads();
    v = s[lane][w];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int64_t mine = (int64_t)blockIdx.x * 32 + w;
    if (lane == 0 && mine < c) store_param(out, dtype, mine, v);
}

cudaError_t column_sums(void* out, int dtype, const float* partial, int parts, int64_t c, cudaStream_t s) {
    k_column_sums<<<(unsigned)((c + 31) / 32), 1024, 0, s>>>(out, dtype, partial, parts, c);
    return cudaGetLastError();
}

// ------------------------------------------------------------------ launches

template <typename T>
cudaError_t launch_pack(uint8_t* q, uint8_t* scale, const void* x, int64_t rows, int c, cudaStream_t s) {
    const int64_t blocks = width8(c) / kBlock8;
    const bool flat = c % kBlock8 == 0 && aligned16(x);
    const int64_t per = flat ? 256 * kUnits / 4 : 8 * kBlocks, ctas = (rows * blocks + per - 1) / per;
    if (ctas > INT_MAX) return cudaErrorInvalidValue;
    if (flat) k_pack8<T><<<(unsigned)ctas, 256, 0, s>>>(q, scale, static_cast<const T*>(x), rows * blocks * 4);
    else k_pack8_any<T><<<(unsigned)ctas, 256, 0, s>>>(q, scale, static_cast<const T*>(x), rows, c, (unsigned)blocks);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_unpack(void* y, int64_t pitch, const uint8_t* q, const uint8_t* scale, int64_t rows, int c,
                          cudaStream_t s) {
    const unsigned groups = (unsigned)(width8(c) / 8);
    const int64_t ctas = (rows * groups + 256 * kUnits - 1) / (256 * kUnits);
    if (ctas > INT_MAX) return cudaErrorInvalidValue;
    const bool vec = pitch % 8 == 0 && aligned16(y);
    if (!vec && c >= 8) {
        const int64_t n = (rows * (groups / 4) + 8 * kBlocks - 1) / (8 * kBlocks);
        if (n > INT_MAX) return cudaErrorInvalidValue;
        k_unpack8_any<T><<<(unsigned)n, 256, 0, s>>>(static_cast<T*>(y), pitch, q, scale, rows, c, groups / 4);
        return cudaGetLastError();
    }
    k_unpack8<T><<<(unsigned)ctas, 256, 0, s>>>(static_cast<T*>(y), pitch, q, scale, rows, c, groups, vec);
    return cudaGetLastError();
}

cudaError_t unpack_rows(void* y, int dtype, int64_t pitch, const uint8_t* q, const uint8_t* scale, int64_t rows,
                        int c, cudaStream_t s) {
    if (dtype == PLATTICE_F32) return launch_unpack<float>(y, pitch, q, scale, rows, c, s);
    if (dtype == PLATTICE_BF16) return launch_unpack<__nv_bfloat16>(y, pitch, q, scale, rows, c, s);
    return launch_unpack<__half>(y, pitch, q, scale, rows, c, s);
}

// CTAs of a grid-stride launch: what the rows need, at most 8 per SM of the
// current device (each then walks many rows and its loads of the gain and its
// partial sums are paid once).
constexpr int kNormCtas = 8;
static int norm_ctas(int64_t rows, int rows_per_cta) {
    const int64_t need = (rows + rows_per_cta - 1) / rows_per_cta;
    const int64_t most = kNormCtas * (int64_t)sm_count();
    return (int)(need < most ? need : most);
}

// Calls f<L, kChunks>() for the row width: L * 8 * kChunks >= channels.
#define PLR_NORM_SHAPE(CHANNELS, F)                      \
    do {                                                 \
        const int n_ = (int)(((CHANNELS) + 7) / 8);      \
        if (n_ <= 4) return F(4, 1);                     \
        if (n_ <= 8) return F(8, 1);                     \
        if (n_ <= 16) return F(16, 1);                   \
        if (n_ <= 32) return F(32, 1);                   \
        if (n_ <= 64) return F(32, 2);                   \
        if (n_ <= 128) return F(128, 1);                 \
        if (n_ <= 256) return F(256, 1);                 \
        if (n_ <= 512) return F(512, 1);                 \
        if (n_ <= 1024) return F(512, 2);                \
        return F(512, 4);                                \
    } while (0)

template <typename T, int kWide>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s) {
#define PLR_F(L, K)                                                                                            \
    (k_rms_norm<T, L, K, kWide><<<norm_ctas(a.rows, (L > 256 ? L : 256) / L), L > 256 ? L : 256, 0, s>>>(a),    \
     cudaGetLastError())
    PLR_NORM_SHAPE(a.c, PLR_F);
#undef PLR_F
}

template <typename T>
cudaError_t launch_norm(const NormArgs& a, cudaStream_t s) {
    return a.wide == 8 ? launch_norm<T, 8>(a, s) : a.wide == 2 ? launch_norm<T, 2>(a, s) : launch_norm<T, 1>(a, s);
}

static int norm_rows_per_cta(int c) {
#define PLR_F(L, K) ((L > 256 ? L : 256) / L)
    PLR_NORM_SHAPE(c, PLR_F);
#undef PLR_F
}

static int norm_resident(int c, int size) {
#define PLR_F(L, K) norm_grad_ctas(size, L, K)
    PLR_NORM_SHAPE(c, PLR_F);
#undef PLR_F
}

template <typename T, int kWide>
cudaError_t launch_norm_grad(const NormGradArgs& a, int ctas, cudaStream_t s) {
#define PLR_F(L, K) (k_rms_norm_grad<T, L, K, kWide><<<ctas, L > 256 ? L : 256, 0, s>>>(a), cudaGetLastError())
    PLR_NORM_SHAPE(a.c, PLR_F);
#undef PLR_F
}

template <typename T>
cudaError_t launch_norm_grad(const NormGradArgs& a, int ctas, cudaStream_t s) {
    return a.wide == 8   ? launch_norm_grad<T, 8>(a, ctas, s)
           : a.wide == 2 ? launch_norm_grad<T, 2>(a, ctas, s)
                         : launch_norm_grad<T, 1>(a, ctas, s);
}

// Channels that one access may take: rows and pointers on 16-byte boundaries,
// or an even number of channels and pointers on boundaries of two.
static int access_width(int c, int dtype, const void* const* p, int count) {
    uintptr_t bits = 0;
    for (int i = 0; i < count; ++i) bits |= (uintptr_t)p[i];   // null: no constraint
    if (c % 8 == 0 && (bits & 15) == 0) return 8;
    return c % 2 == 0 && (bits & (2 * dtype_size(dtype) - 1)) == 0 ? 2 : 1;
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_rows_pack8(uint8_t* q, uint8_t* scale, const void* x, int dtype, long long rows, int c, void* stream) {
    if (!dtype_ok(dtype) || rows < 0 || c < 1) return PLATTICE_ERR_INVALID;
    if (rows == 0) return PLATTICE_OK;
    if (!q || !scale || !x || !aligned16(q) || !fits(rows, width8(c))) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == PLATTICE_F32    ? launch_pack<float>(q, scale, x, rows, c, s)
                          : dtype == PLATTICE_BF16 ? launch_pack<__nv_bfloat16>(q, scale, x, rows, c, s)
                                                   : launch_pack<__half>(q, scale, x, rows, c, s);
    return rows_status(e, "plattice_rows_pack8");
}

int plattice_rows_unpack8(void* y, int dtype, const uint8_t* q, const uint8_t* scale, long long rows, int c,
                          void* stream) {
    if (!dtype_ok(dtype) || rows < 0 || c < 1) return PLATTICE_ERR_INVALID;
    if (rows == 0) return PLATTICE_OK;
    if (!q || !scale || !y || !aligned16(q) || !fits(rows, width8(c))) return PLATTICE_ERR_INVALID;
    return rows_status(unpack_rows(y, dtype, c, q, scale, rows, c, static_cast<cudaStream_t>(stream)),
                       "plattice_rows_unpack8");
}

int plattice_rms_norm(void* y, uint8_t* yscale, void* h, float* rstd, const void* x, const void* residual,
                      const void* gain, int dtype, int gain_dtype, float eps, long long rows, int c, void* stream) {
    if (!dtype_ok(dtype) || !dtype_ok(gain_dtype) || rows < 0 || c < 1 || c > PLATTICE_NORM_MAX_CHANNELS)
        return PLATTICE_ERR_INVALID;
    if (rows == 0) return PLATTICE_OK;
    if (!y || !rstd || !x || !gain || !fits(rows, width8(c))) return PLATTICE_ERR_INVALID;
    // 8-bit rows always allow whole accesses of their own
    const void* const used[4] = {x, residual, h, yscale ? nullptr : y};
    if (yscale && ((uintptr_t)y & 15)) return PLATTICE_ERR_INVALID;
    const NormArgs a{y, yscale, h, rstd, x, residual, gain, gain_dtype, eps, rows, c, access_width(c, dtype, used, 4)};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = dtype == PLATTICE_F32    ? launch_norm<float>(a, s)
                          : dtype == PLATTICE_BF16 ? launch_norm<__nv_bfloat16>(a, s)
                                                   : launch_norm<__half>(a, s);
    return rows_status(e, "plattice_rms_norm");
}

int plattice_rms_norm_backward_workspace_size(long long rows, int c, size_t* bytes) {
    if (!bytes || rows < 0 || c < 1 || c > PLATTICE_NORM_MAX_CHANNELS) return PLATTICE_ERR_INVALID;
    // one row of partial sums per CTA, whatever the device's SM count (<= 256)
    const int64_t per = norm_rows_per_cta(c);
    const int64_t need = (rows + per - 1) / per;
    *bytes = (size_t)(need < 2048 ? (need < 1 ? 1 : need) : 2048) * c * sizeof(float);
    return PLATTICE_OK;
}

int plattice_rms_norm_backward(void* grad_x, void* grad_gain, const void* grad_y, const void* h, const float* rstd,
                               const void* gain, const void* grad_h, void* workspace, size_t workspace_bytes,
                               int dtype, int gain_dtype, long long rows, int c, void* stream) {
    if (!dtype_ok(dtype) || !dtype_ok(gain_dtype) || rows < 0 || c < 1 || c > PLATTICE_NORM_MAX_CHANNELS)
        return PLATTICE_ERR_INVALID;
    if (!grad_gain || !fits(rows, width8(c))) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (rows == 0)   // the sum over no rows
        return rows_status(cudaMemsetAsync(grad_gain, 0, (size_t)c * dtype_size(gain_dtype), s),
                           "plattice_rms_norm_backward");
    if (!grad_x || !grad_y || !h || !rstd || !gain || !workspace) return PLATTICE_ERR_INVALID;
    size_t need = 0;
    plattice_rms_norm_backward_workspace_size(rows, c, &need);
    if (workspace_bytes < need) return PLATTICE_ERR_WORKSPACE;
    // one round of CTAs: as many as are resident at a time
    const int64_t per = norm_rows_per_cta(c), lines = (rows + per - 1) / per;
    const int64_t most = (int64_t)sm_count() * norm_resident(c, (int)dtype_size(dtype));
    const int ctas = (int)(lines < most ? lines : most < 2048 ? most : 2048);
    const void* const used[4] = {grad_x, grad_y, h, grad_h};
    const NormGradArgs a{grad_x, static_cast<float*>(workspace), grad_y, h,    rstd, gain, gain_dtype,
                         grad_h, rows, c, access_width(c, dtype, used, 4)};
    cudaError_t e = dtype == PLATTICE_F32    ? launch_norm_grad<float>(a, ctas, s)
                    : dtype == PLATTICE_BF16 ? launch_norm_grad<__nv_bfloat16>(a, ctas, s)
                                             : launch_norm_grad<__half>(a, ctas, s);
    if (e == cudaSuccess) e = column_sums(grad_gain, gain_dtype, a.partial, ctas, c, s);
    return rows_status(e, "plattice_rms_norm_backward");
}

}  // extern "C"
