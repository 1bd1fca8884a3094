// rows_linear.cu -- linear map of rows with bias, activation and residual,
// and its backward pass, x plain or in 8-bit rows.  C ABI: include/plattice.h.
#include <limits.h>
#include <string.h>

#include <type_traits>

#include "plattice_runtime.h"
#include "rows_common.cuh"
#include "rows_host.h"
#include "rows_narrow.h"
#include "rows_split.cuh"

namespace plr {

// ----------------------------------------------------- operands for the MMAs

// How a value is stored: N bfloat16 parts, one tensor of them after the other;
// kLone: for products with operands of a single part.
template <int N, bool kLone = false> struct Parts {
    static constexpr int kParts = N;
    static constexpr bool lone = kLone;
};

template <int N, bool kLone>
__device__ __forceinline__ void store_parts(__nv_bfloat16* p, int64_t stride, const float (&v)[8], bool vec, int n) {
    union { uint4 u; uint32_t w[4]; __nv_bfloat16 h[8]; } o[N];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t t[N];
        if constexpr (kLone) split_one_sign<true>(v[2 * i], v[2 * i + 1], t);
        else split_any(v[2 * i], v[2 * i + 1], t);
#pragma unroll
        for (int j = 0; j < N; ++j) o[j].w[i] = t[j];
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
        if (vec) *reinterpret_cast<uint4*>(p + j * stride) = o[j].u;
        else
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) p[j * stride + i] = o[j].h[i];
    }
}

// 8 values as a T (a type, or Parts) from element `at` of a tensor of `size`.
template <typename T>
__device__ __forceinline__ void store8_as(void* p, int64_t at, int64_t size, const float (&v)[8], bool vec, int n) {
    if constexpr (std::is_empty_v<T>) store_parts<T::kParts, T::lone>(static_cast<__nv_bfloat16*>(p) + at, size, v, vec, n);
    else store8(static_cast<T*>(p) + at, v, vec, n);
}

// Rows of c elements copied to rows of `pitch` (a multiple of 8) as TO: what TMA
// needs when the rows do not lie on 16-byte boundaries, and values as parts.
// Costs one read and one (float32: 1.5, float16 as parts: 2) write of the operand.
template <typename T, typename TO>
__global__ void __launch_bounds__(256) k_repack(void* __restrict__ out, const T* __restrict__ x, int64_t rows, int c,
                                                unsigned groups, bool vec) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = t / groups;
    if (row >= rows) return;
    const int col = (int)(t - row * groups) * 8, left = c - col;
    float v[8];
    load8(v, x + row * c + col, vec && left >= 8, left);
    store8_as<TO>(out, t * 8, rows * groups * 8, v, true, 8);
}

// ------------------------------------------------- backward: gz and its sums

struct GradArgs {
    const void* g0;
    const void* g1;
    const void* z;
    const uint8_t* z_scale;
    void* gz;           // [rows][pitch] in the operands' type or as bfloat16 parts; null: not stored
    int64_t pitch;
    float* partial;     // [gridDim.y][n]; null: no bias gradient
    int64_t rows;
    int n, split, act;
    int shift;          // log2 of the threads that share a row
    bool vec;           // rows of grad_y and z allow 16-byte accesses
};

// g *= slope(z); what lies behind the last column is 0 in both
template <int kAct>
__device__ __forceinline__ void times_slope(float (&g)[8], float (&z)[8]) {
    slopes<kAct>(z);
#pragma unroll
    for (int i = 0; i < 8; i += 2) mul2(g[i], g[i + 1], z[i], z[i + 1]);
}

constexpr int kTogether = 2;

// gz = grad_y act'(z) as the two products take it, and the sums of the unrounded
// gz over a CTA's rows.  Behind 16-bit gradients gz is rounded to their type (a
// tensor core takes no wider operand; one rounding, as a stored gradient has, also
// past float16's largest); behind float32 ones it is two bfloat16 parts beside 16-bit operands,
// three beside float32 ones (gz_parts).  2^shift threads of 8 columns share a row;
// gridDim.x strips of columns, gridDim.y parts of rows.
template <typename TG, typename T, bool kFast>
__global__ void __launch_bounds__(256, 4) k_grad_z(const GradArgs a) {
    __shared__ float sums[8 * 256];
    const int lane = threadIdx.x & ((1 << a.shift) - 1), rows = 256 >> a.shift;
    const int col = ((int)blockIdx.x << (a.shift + 3)) + lane * 8;
    const int left = a.n - col, wide = (int)min(a.pitch - col, (int64_t)8);
    const int zgroups = (a.n + 31) / 32 * 4;
    float acc[8] = {};
    auto finish = [&](float (&g)[8], float (&z)[8], int64_t row) {
        if (a.act == PLATTICE_ACT_RELU) times_slope<PLATTICE_ACT_RELU>(g, z);
        else if (a.act == PLATTICE_ACT_GELU) times_slope<PLATTICE_ACT_GELU>(g, z);
        else if (a.act == PLATTICE_ACT_SILU) times_slope<PLATTICE_ACT_SILU>(g, z);
#pragma unroll
        for (int i = 0; i < 8; i += 2) add2(acc[i], acc[i + 1], g[i], g[i + 1]);
        if (!a.gz) return;
        const int64_t at = row * a.pitch + col;   // zeros up to the pitch
        store8_as<T>(a.gz, at, a.rows * a.pitch, g, kFast || (a.pitch % 8 == 0 && wide == 8), wide);
    };
    const int64_t stride = (int64_t)gridDim.y * rows;
    int64_t row = (int64_t)blockIdx.y * rows + (threadIdx.x >> a.shift);
    if (kFast) {
        // whole groups of 8 on 16-byte boundaries, gradient in one tensor:
        // kTogether rows' loads are issued before the first is used
        if (left > 0) {
            const TG* g0 = static_cast<const TG*>(a.g0) + col;
            for (; row < a.rows; row += stride * kTogether) {
                Raw8<TG> g[kTogether], z[kTogether];
                uint2 codes[kTogether];
                uint8_t scale[kTogether];
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    const int64_t r = min(row + u * stride, a.rows - 1);
                    g[u].load(g0 + r * a.n, true, 8);
                    if (a.z_scale) {
                        const int64_t at = r * zgroups + (col >> 3);
                        codes[u] = reinterpret_cast<const uint2*>(a.z)[at];
                        scale[u] = a.z_scale[at >> 2];
                    } else if (a.z) {
                        z[u].load(static_cast<const TG*>(a.z) + r * a.n + col, true, 8);
                    }
                }
#pragma unroll
                for (int u = 0; u < kTogether; ++u) {
                    if (row + u * stride >= a.rows) break;
                    float gv[8], zv[8];
                    g[u].widen(gv);
                    if (a.z_scale) values8(zv, codes[u], scale_of(scale[u]));
                    else if (a.z) z[u].widen(zv);
                    finish(gv, zv, row + u * stride);
                }
            }
        }
    } else if (left > 0) {
        const bool vec = a.vec && left >= 8;
        for (; row < a.rows; row += stride) {
            float g[8], z[8];
            if (a.split == 0) {
                load8(g, static_cast<const TG*>(a.g0) + row * a.n + col, vec, left);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int c = col + i;
                    g[i] = i >= left ? 0.f
                           : c < a.split ? to_f32(static_cast<const TG*>(a.g0)[row * a.split + c])
                                         : to_f32(static_cast<const TG*>(a.g1)[row * (a.n - a.split) + c - a.split]);
                }
            }
            if (a.z_scale) {
                const int64_t at = row * zgroups + col / 8;
                values8(z, reinterpret_cast<const uint2*>(a.z)[at], scale_of(a.z_scale[at >> 2]));
            } else if (a.z) {
                load8(z, static_cast<const TG*>(a.z) + row * a.n + col, vec, left);
            }
            finish(g, z, row);
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[i * 256 + threadIdx.x] = acc[i];
    __syncthreads();
    if (threadIdx.x >> (a.shift + 3)) return;
    const int l = threadIdx.x & ((1 << a.shift) - 1), i = threadIdx.x >> a.shift;
    const int c = ((int)blockIdx.x << (a.shift + 3)) + l * 8 + i;
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += sums[i * 256 + (r << a.shift) + l];
    if (c < a.n) a.partial[(int64_t)blockIdx.y * a.n + c] = s;
}

// The same for gelu and silu of 8-bit z, many values, rows on 16-byte
// boundaries and the gradient in one tensor: a block's scale and a code are all
// that z is, so its slopes are looked up in a table of the 256 codes for each of
// 16 exponents (largest values of 0.1 to 3584; other blocks are computed).  The
// lookups conflict over the banks about three ways, and still take a third of
// the exponentials and reciprocals they replace: 32768 x 4096, gelu, bfloat16:
// 165 -> 120 us, of which moving 675 MB is 103.
constexpr int kTableLow = 127 - 12, kTableScales = 16;

template <typename TG, typename T, int kAct>
__global__ void __launch_bounds__(256, 4) k_grad_z_table(const GradArgs a) {
    __shared__ float table[kTableScales * 256];
    __shared__ float sums[8 * 256];
    for (int i = threadIdx.x; i < kTableScales * 256; i += 256) {
        float v = value1((uint8_t)i, scale_of((uint8_t)(kTableLow + (i >> 8)))), unused = 0.f;
        slope2<kAct>(v, unused);
        table[i] = v;
    }
    __syncthreads();
    const int lane = threadIdx.x & ((1 << a.shift) - 1), rows = 256 >> a.shift;
    const int col = ((int)blockIdx.x << (a.shift + 3)) + lane * 8;
    const int zgroups = (a.n + 31) / 32 * 4;
    const int64_t stride = (int64_t)gridDim.y * rows;
    float acc[8] = {};
    if (col < a.n) {
        const TG* g0 = static_cast<const TG*>(a.g0) + col;
        const uint2* z0 = reinterpret_cast<const uint2*>(a.z) + (col >> 3);
        for (int64_t row = (int64_t)blockIdx.y * rows + (threadIdx.x >> a.shift); row < a.rows; row += stride * kTogether) {
            Raw8<TG> g[kTogether];
            uint2 codes[kTogether];
            uint8_t scale[kTogether];
#pragma unroll
            for (int u = 0; u < kTogether; ++u) {
                const int64_t r = min(row + u * stride, a.rows - 1), at = r * zgroups;
                g[u].load(g0 + r * a.n, true, 8);
                codes[u] = z0[at];
                scale[u] = a.z_scale[(at + (col >> 3)) >> 2];
            }
#pragma unroll
            for (int u = 0; u < kTogether; ++u) {
                if (row + u * stride >= a.rows) break;
                float v[8], m[8];
                g[u].widen(v);
                const int place = scale[u] - kTableLow;
                if ((unsigned)place < (unsigned)kTableScales) {
                    const float* t = table + place * 256;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        m[i] = t[(codes[u].x >> (8 * i)) & 255];
                        m[4 + i] = t[(codes[u].y >> (8 * i)) & 255];
                    }
                } else {
                    values8(m, codes[u], scale_of(scale[u]));
                    slopes<kAct>(m);
                }
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    mul2(v[i], v[i + 1], m[i], m[i + 1]);
                    add2(acc[i], acc[i + 1], v[i], v[i + 1]);
                }
                if (!a.gz) continue;
                const int64_t at = (row + u * stride) * a.pitch + col;
                store8_as<T>(a.gz, at, a.rows * a.pitch, v, true, 8);
            }
        }
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[i * 256 + threadIdx.x] = acc[i];
    __syncthreads();
    if (threadIdx.x >> (a.shift + 3)) return;
    const int l = threadIdx.x & ((1 << a.shift) - 1), i = threadIdx.x >> a.shift;
    const int c = ((int)blockIdx.x << (a.shift + 3)) + l * 8 + i;
    float s = 0.f;
    for (int r = 0; r < rows; ++r) s += sums[i * 256 + (r << a.shift) + l];
    if (c < a.n) a.partial[(int64_t)blockIdx.y * a.n + c] = s;
}

// Lines of nw + nb sums added in order into two tensors (either may be null);
// a CTA takes 32 columns, its 32 warps every 32nd line each.
__global__ void __launch_bounds__(1024) k_sum_lines(void* out_w, int dtype_w, int64_t nw, void* out_b, int dtype_b, int nb,
                                                    const float* __restrict__ partial, int lines) {
    __shared__ float s[32][33];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t all = nw + nb, col = (int64_t)blockIdx.x * 32 + lane;
    float v = 0.f;
    if (col < all && (col < nw ? out_w != nullptr : out_b != nullptr))
        for (int p = w; p < lines; p += 32) v += partial[(int64_t)p * all + col];
    s[w][lane] = v;
    __syncthreads();
    v = s[lane][w];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    const int64_t mine = (int64_t)blockIdx.x * 32 + w;
    if (lane != 0 || mine >= all) return;
    if (mine < nw) {
        if (out_w) store_param(out_w, dtype_w, mine, v);
    } else if (out_b) {
        store_param(out_b, dtype_b, mine - nw, v);
    }
}

// out[e] = sum over the parts of partial[part][e], in order.
template <typename T>
__global__ void __launch_bounds__(256) k_add_parts(T* __restrict__ out, const float* __restrict__ partial, int parts,
                                                   int64_t n) {
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= n) return;
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += partial[(int64_t)p * n + e];
    out[e] = from_f32<T>(s);
}

// ------------------------------------------------------------------ host side

static int64_t up256(int64_t n) { return (n + 255) & ~255ll; }
static int64_t up8(int64_t n) { return (n + 7) & ~7ll; }

// Buffers of a call, one after the other in its workspace.
struct Carve {
    int64_t at = 0;
    int64_t take(int64_t bytes) {
        const int64_t p = at;
        at += up256(bytes);
        return p;
    }
};

static bool linear_shape_ok(const plattice_linear_args* a) {
    if (!a || a->rows < 0 || a->k < 1 || a->n < 1 || a->split < 0 || a->split >= a->n) return false;
    if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype) || !dtype_ok(a->bias_dtype)) return false;
    if (a->out_dtype != a->dtype && a->out_dtype != PLATTICE_F32) return false;
    if (a->x_scale && a->dtype == PLATTICE_F16) return false;
    if (a->act < PLATTICE_ACT_NONE || a->act > PLATTICE_ACT_SILU) return false;
    if (a->split && a->act != PLATTICE_ACT_NONE) return false;
    // TMA coordinates and tile numbers are 32-bit
    if (a->rows > INT_MAX - 256 || a->k > (1 << 30) || a->n > (1 << 30)) return false;
    return fits(a->rows, width8(a->k)) && fits(a->rows, width8(a->n)) && fits(a->k, a->n);
}

static bool workspace_ok(const plattice_linear_args* a, int64_t bytes) {
    return a->workspace && ((uintptr_t)a->workspace & 255) == 0 && a->workspace_bytes >= (size_t)bytes;
}

// Parts summed: few results over the warps of a CTA (a thread each would add
// hundreds of parts one after the other: 7.8 against 3.5 us for 64 x 64 and
// 296 parts), many by a thread each.
template <typename T>
static cudaError_t add_parts(void* out, const float* partial, int parts, int64_t n, cudaStream_t s) {
    k_add_parts<T><<<(unsigned)ceil_div(n, 256), 256, 0, s>>>(static_cast<T*>(out), partial, parts, n);
    return cudaGetLastError();
}

static cudaError_t add_parts_to(void* out, int dtype, const float* partial, int parts, int64_t n, cudaStream_t s) {
    if (parts > 8 && n <= 8192) {
        k_sum_lines<<<(unsigned)ceil_div(n, 32), 1024, 0, s>>>(out, dtype, n, nullptr, dtype, 0, partial, parts);
        return cudaGetLastError();
    }
    if (dtype == PLATTICE_F32) return add_parts<float>(out, partial, parts, n, s);
    if (dtype == PLATTICE_BF16) return add_parts<__nv_bfloat16>(out, partial, parts, n, s);
    return add_parts<__half>(out, partial, parts, n, s);
}

// ---- products on the tensor cores

// Whether TMA can read the rows where they are.
static bool tma_ready(const void* p, int dtype, int64_t width) {
    return dtype != PLATTICE_F32 && width % 8 == 0 && aligned16(p);
}

// Parts that the tiled backward's gz is made of: three beside float32 operands;
// behind float32 gradients, whose 16 leading bits stay and which can be far smaller
// and far larger than float16 holds, two bfloat16 (float16 operands have two then,
// too); else one.
static int gz_parts(const plattice_linear_args* a) {
    return a->dtype == PLATTICE_F32 ? 3 : a->out_dtype == PLATTICE_F32 ? 2 : 1;
}

// Parts of w, and of an x that is not in 8 bits.
static int forward_parts(const plattice_linear_args* a) { return a->dtype == PLATTICE_F32 ? 3 : 1; }
static int backward_parts(const plattice_linear_args* a) { return a->dtype == PLATTICE_BF16 ? 1 : gz_parts(a); }

static int64_t repack_bytes(int parts, int64_t rows, int64_t width) { return rows * up8(width) * 2 * parts; }

template <typename T, typename TO>
static void repack(void* ws, const void* p, int64_t rows, int64_t width, cudaStream_t s) {
    const unsigned groups = (unsigned)(up8(width) / 8);
    k_repack<T, TO><<<(unsigned)ceil_div(rows * groups, 256), 256, 0, s>>>(ws, static_cast<const T*>(p), rows, (int)width,
                                                                         groups, width % 8 == 0 && aligned16(p));
}

// The operand where it is, or repacked into `ws`.
static cudaError_t operand(Operand* o, const void* p, int dtype, int parts, int64_t rows, int64_t width, void* ws,
                           cudaStream_t s) {
    *o = Operand{p, rows, width, width, 1};
    if (parts == 1 && tma_ready(p, dtype, width)) return cudaSuccess;
    o->p = ws;
    o->pitch = up8(width);
    o->parts = parts;
    if (ceil_div(rows * (o->pitch / 8), 256) > INT_MAX) return cudaErrorInvalidValue;
    if (dtype == PLATTICE_F32) repack<float, Parts<3>>(ws, p, rows, width, s);
    else if (dtype == PLATTICE_BF16) repack<__nv_bfloat16, __nv_bfloat16>(ws, p, rows, width, s);
    else if (parts == 2) repack<__half, Parts<2>>(ws, p, rows, width, s);
    else repack<__half, __half>(ws, p, rows, width, s);
    return cudaGetLastError();
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
    static EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return (EncodeTiled) nullptr;
        }
        return (EncodeTiled)p;
    }();
    return f;
}

cudaError_t make_map(CUtensorMap* m, const Operand& o, int box_rows) {
    const EncodeTiled enc = encode_tiled();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {(cuuint64_t)o.width, (cuuint64_t)o.rows, (cuuint64_t)o.parts};
    const cuuint64_t strides[2] = {(cuuint64_t)o.pitch * 2, (cuuint64_t)(o.pitch * o.rows) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1}, unit[3] = {1, 1, 1};
    const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.p), dims, strides, box, unit,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// Cycles of a 64-deep slice of a 128 x bn tile: the MMA itself (512 at 256
// columns), or below that what staging the operands' slices takes.
static double slice_cost(int bn) { return bn == 256 ? 512 : bn == 128 ? 300 : bn == 64 ? 220 : 200; }

// Columns of a tile: the cheapest number of rounds over the device's SMs
// (wide tiles do more per byte staged, narrow ones fill the device when D is
// small and waste less when it is narrow).
static int choose_bn(int64_t ni, int64_t nj, int least, bool deep) {
    int best = least;
    double cost = 1e300;
    for (int bn = deep ? 128 : 256; bn >= least; bn /= 2) {
        const double c = (double)ceil_div(mma_tiles(ni, nj, bn), sm_count()) * slice_cost(bn);
        if (c < cost) cost = c, best = bn;
    }
    return best;
}

// Parts of kGradW's sum: the cheapest of rounds over the SMs, where a part
// costs its slices and some 6 more for filling and emptying the accumulator,
// plus writing and adding the partial results (8 bytes an element, about
// 3 bytes a cycle and SM).  `deepest`: rows that a part may have.
static int choose_parts(int64_t ni, int64_t nj, int bn, int64_t steps, int64_t deepest) {
    const int64_t tiles = mma_tiles(ni, nj, bn);
    const int least = (int)ceil_div(steps * kBK, deepest), most = least > 256 ? least : 256;
    int best = least;
    double cost = 1e300;
    for (int p = least; p <= most && p <= steps; ++p) {
        const double rounds = (double)ceil_div(tiles * p, sm_count());
        double c = rounds * (double)(ceil_div(steps, p) + 6) * slice_cost(bn);
        if (p > 1) c += (double)p * ni * nj * 8 / (3.0 * 8 * sm_count());
        if (c < cost) cost = c, best = p;
    }
    return best;
}

// The products of parts that make up one of values, small ones first: those down
// to 2^-16 of the largest of float32's three parts, to 2^-9 of float16's two (the
// other is within 2^-18, and the result has 11 bits).
template <typename F> static void for_products(int parts_a, int parts_b, F f) {
    static const unsigned char all[6][2] = {{0, 2}, {1, 1}, {2, 0}, {0, 1}, {1, 0}, {0, 0}};
    for (const auto& c : all)
        if (c[0] < parts_a && c[1] < parts_b && !(parts_a == 2 && parts_b == 2 && c[0] + c[1] == 2)) f(c[0], c[1]);
}
static int product_count(int parts_a, int parts_b) {
    int n = 0;
    for_products(parts_a, parts_b, [&](int, int) { ++n; });
    return n;
}

// Columns of a tile of kGradW: as wide as the result and the mode allow, but
// where the sum is short (at most 16 slices, products of parts counted) the
// narrowest whose tiles run in one round, since emptying an accumulator is then
// most of the time (bfloat16, 64 / 256 wide: 100 rows, 1024 x 1024 4.4 / 6.4 us;
// 1000 rows, 256 x 256 4.9 / 6.4; 5000 rows, 512 x 512 9.5 / 8.8).
static int choose_bn_w(const plattice_linear_args* a) {
    const bool deep = a->dtype == PLATTICE_F32 && a->rows > 8 * kBK;   // chunks, or parts no deeper than one
    const int widest = a->n > 128 && !deep ? 256 : a->n > 64 ? 128 : 64;
    if (ceil_div(a->rows, kBK) * product_count(a->x_scale ? 1 : backward_parts(a), gz_parts(a)) > 16) return widest;
    int bn = 64;
    while (bn < widest && mma_tiles(a->k, a->n, bn) > sm_count()) bn *= 2;
    return bn;
}

// The sum's side of the arguments: slices of r and the products of parts.
static void sum_args(MmaArgs* p, int64_t nr, int parts, int parts_a, int parts_b) {
    p->steps = (int)ceil_div(nr, kBK);
    p->part_steps = (int)ceil_div(p->steps, parts);
    p->parts = (int)ceil_div(p->steps, p->part_steps);   // none is empty
    p->pairs = 0;
    p->pairs_a = p->pairs_b = 0;
    for_products(parts_a, parts_b, [&](int i, int j) {
        p->pairs_a |= (unsigned)i << (2 * p->pairs);
        p->pairs_b |= (unsigned)j << (2 * p->pairs);
        ++p->pairs;
    });
    // a slice takes 200 to 500 cycles, bound by memory up to some 2000
    p->patience = 4000000000ll + 4096ll * p->part_steps * p->pairs;
}

// The 8-bit x as a bfloat16 operand in `ws`.
static cudaError_t unpacked(Operand* o, const plattice_linear_args* a, void* ws, cudaStream_t s) {
    *o = Operand{ws, a->rows, a->k, up8(a->k), 1};
    return unpack_rows(ws, PLATTICE_BF16, o->pitch, static_cast<const uint8_t*>(a->x), a->x_scale, a->rows, a->k, s);
}

// How a forward runs.  k_few where its CTAs of 16 rows x 32 channels fit on the
// device at a time (with float32 weights, whose parts the tiles need written
// first, up to twice that); k_narrow with at most 32 output channels; else
// tiles.  Of 16-bit types the tiles take, too, rows that TMA can read once n k is
// above 1536, and deep sums of a few thousand rows (narrow_shares).  Measured (us;
// bfloat16 unless noted):
//   k_few / tiles   1024 -> 4096, 16 rows 4.7 / 9.3, 32 rows (1.7 rounds) 8.5 / 8.7;
//     256 -> 256, 256 rows 3.3 / 4.2, 512 rows 5.7 / 4.3; float32, 512 -> 512, 128
//     rows 6.3 / 16.6, 256 rows 11.5 / 16.8, 512 rows (3.5 rounds) 21.6 / 17.1
//   k_few / k_narrow   64 -> 24, 2300 rows 3.1 / 3.2, 4700 rows 5.3 / 3.3; float32,
//     256 -> 24, 2300 rows 4.3 / 6.2, 9400 rows 14.1 / 9.6
//   k_narrow / tiles   262144 rows, n 8: k 64 9.6 / 13.7, k 192 21.5 / 22.0, k 1024
//     106 / 88; n 24: k 64 14.0 / 15.5, k 128 19.9 / 17.1; k 100 (no 16-byte rows)
//     33.4 / 52.3; 65536 rows, n 24, from 8 bits: k 64 7.0 / 10.3, k 1024 38 / 62;
//     float32: k 64 9.4 / 18.2, k 1024 94 / 206; 9400 rows, n 24: from 8 bits, k 1024
//     18.2 / 12.2, float32, k 768 23.0 / 29.9
enum Way { kWayFew, kWayNarrow, kWayTiles };

static Way forward_way(const plattice_linear_args* a) {
    const int64_t few = ceil_div(a->rows, 16) * ceil_div(a->n, 32);
    if (few <= sm_count()) return kWayFew;
    const int parts = a->dtype == PLATTICE_F32 ? 3 : 1;
    const bool tiles_read = !a->x_scale && tma_ready(a->x, a->dtype, a->k);
    // k_narrow stages its results in the split's order: a z kept whole beside them goes through tiles
    const bool order = a->split && a->z && !a->z_scale;
    if (a->n <= 32 && !order && (!tiles_read || (int64_t)a->n * a->k <= 1536) &&
        !(parts == 1 && narrow_shares(ceil_div(a->rows, a->x_scale ? 32 : 16), a->k)) &&
        narrow_fragments(a->k, (int)ceil_div(a->n, 8), parts) <= kNarrowMost)
        return kWayNarrow;
    return parts == 3 && few <= 2 * (int64_t)sm_count() ? kWayFew : kWayTiles;
}

struct ForwardPlan {
    Way way;
    int bn;
    int64_t x, w, bytes;
};

static ForwardPlan forward_plan(const plattice_linear_args* a) {
    ForwardPlan p{};
    Carve c;
    p.way = forward_way(a);
    if (p.way == kWayTiles) {
        p.bn = choose_bn(a->rows, a->n, 32, chunked((int)ceil_div(a->k, kBK), a->out_dtype, true));
        if (a->x_scale) p.x = c.take(a->rows * up8(a->k) * 2);
        else if (!tma_ready(a->x, a->dtype, a->k)) p.x = c.take(repack_bytes(forward_parts(a), a->rows, a->k));
        p.w = tma_ready(a->w, a->dtype, a->k) ? 0 : c.take(repack_bytes(forward_parts(a), a->n, a->k));
    }
    p.bytes = c.at;
    return p;
}

struct BackwardPlan {
    bool narrow;
    int lines;       // narrow: CTAs along the rows
    bool gz_needed;
    int shift, strips;
    int bn_x, bn_w, parts_b, parts_w;
    int64_t gz, x, w, partial_b, partial_w, pitch, bytes;
};

// Whether the backward runs in one pass over slices of 64 input channels
// (k_narrow_grad), each of which makes gz anew, or as tiled products.  Measured
// (us, one pass / tiles), bfloat16, 65536 rows: n 16, k 512 43 / 53, k 768 80 / 70;
// n 24, k 256 35.5 / 36.6, k 512 85 / 55; 100 rows, n 16, k 512 8.7 / 14.0; from 8
// bits: 34559 rows, n 16, k 1896 102 / 126, 262144 rows, n 32, k 256 103 / 118;
// float32, 8192 rows, n 8, k 2048 69 / 112.  Rows on no 16-byte boundaries, whose
// channels the pass loads and stores one by one: bfloat16, k 50, n 24, 262144 rows
// 71 / 83; k 95, n 8, 20000 rows 26 / 29; k 95, n 4, 848040 rows 587 / 267.  Float32
// gradients beside 16-bit operands, whose parts cost the tiles more: bfloat16, 65536
// rows: n 16, k 768 84 / 92, k 1024 78 / 111; n 24, k 512 84 / 71; float16: n 16, k
// 1024 100 / 196; n 24, k 512 113 / 126; n 32, k 512 130 / 113.
static bool backward_is_narrow(const plattice_linear_args* a) {
    if (a->n > 32 || a->k > kNarrowGradMost) return false;
    if (a->dtype == PLATTICE_F32) return true;
    if (a->k % 8 && a->k > 64 && a->rows > 24000) return false;
    const bool two = a->out_dtype == PLATTICE_F32 && a->n <= (a->dtype == PLATTICE_F16 ? 24 : 16);
    if ((int64_t)a->n * a->k <= (two ? 16384 : 8192)) return true;
    return a->x_scale && a->n <= 24;
}

static BackwardPlan backward_plan(const plattice_linear_args* a) {
    BackwardPlan p{};
    Carve c;
    p.narrow = backward_is_narrow(a);
    if (p.narrow) {
        // one round of CTAs over the slices of 64 channels
        const int64_t slices = ceil_div(a->k, 64), need = ceil_div(ceil_div(a->rows, 16), kGradWarps);
        const int64_t most = ceil_div(narrow_grad_ctas(backward_parts(a), (a->n + 7) / 8) * (int64_t)sm_count(), slices);
        p.lines = (int)(need < most ? (need < 1 ? 1 : need) : most);
        p.partial_w = c.take((int64_t)p.lines * ((int64_t)a->n * a->k + a->n) * 4);
        p.bytes = c.at;
        return p;
    }
    while (p.shift < 5 && (8 << p.shift) < a->n) ++p.shift;   // a row's columns / 8, at most a warp
    p.strips = (int)ceil_div(a->n, 8 << p.shift);
    const int64_t need = ceil_div(a->rows, 256 >> p.shift), most = ceil_div(4 * (int64_t)sm_count(), p.strips);   // one round
    p.parts_b = (int)(need < most ? need : most);
    if (p.parts_b < 1) p.parts_b = 1;
    p.partial_b = c.take((int64_t)p.parts_b * a->n * 4);
    // the incoming gradient itself serves where it is already what TMA reads
    p.gz_needed = !(a->act == PLATTICE_ACT_NONE && !a->split && a->out_dtype == a->dtype &&
                    tma_ready(a->grad0, a->dtype, a->n));
    p.pitch = up8(a->n);
    if (p.gz_needed) p.gz = c.take(repack_bytes(gz_parts(a), a->rows, a->n));
    p.bn_x = choose_bn(a->rows, a->k, 64, chunked((int)ceil_div(a->n, kBK), a->dtype, true));
    p.bn_w = choose_bn_w(a);
    p.parts_w = choose_parts(a->k, a->n, p.bn_w, ceil_div(a->rows, kBK),
                             a->dtype == PLATTICE_F32 ? INT_MAX : deepest_sum(a->dtype));   // float32: in chunks
    const int parts = backward_parts(a);
    if (a->grad_x && (parts > 1 || !tma_ready(a->w, a->dtype, a->k))) p.w = c.take(repack_bytes(parts, a->n, a->k));
    if (a->grad_w && a->x_scale) p.x = c.take(a->rows * up8(a->k) * 2);
    if (a->grad_w && !a->x_scale && (parts > 1 || !tma_ready(a->x, a->dtype, a->k)))
        p.x = c.take(repack_bytes(parts, a->rows, a->k));
    if (a->grad_w && p.parts_w > 1) p.partial_w = c.take((int64_t)p.parts_w * a->n * a->k * 4);
    p.bytes = c.at;
    return p;
}

template <typename TG, typename T>
static cudaError_t launch_grad_z(const GradArgs& g, const BackwardPlan& p, cudaStream_t s) {
    const dim3 ctas(p.strips, p.parts_b);
    const bool fast = g.vec && !g.split && g.pitch % 8 == 0;
    // below 8 M values filling the tables takes what they save (us, 256 columns,
    // bfloat16, gelu, table / computed: 4096 rows 6.2 / 3.9, 16384 8.1 / 7.5, 32768
    // 12.1 / 13.6, 131072 32.3 / 44.6)
    const bool table = fast && g.z_scale && g.rows * g.n >= (1 << 23);
    if (table && g.act == PLATTICE_ACT_GELU) k_grad_z_table<TG, T, PLATTICE_ACT_GELU><<<ctas, 256, 0, s>>>(g);
    else if (table && g.act == PLATTICE_ACT_SILU) k_grad_z_table<TG, T, PLATTICE_ACT_SILU><<<ctas, 256, 0, s>>>(g);
    else if (fast) k_grad_z<TG, T, true><<<ctas, 256, 0, s>>>(g);
    else k_grad_z<TG, T, false><<<ctas, 256, 0, s>>>(g);
    return cudaGetLastError();
}

static cudaError_t forward_small(const plattice_linear_args* a, Way way, cudaStream_t s) {
    const int e = a->dtype == PLATTICE_F32 ? 4 : 8;   // elements of 16 bytes
    const SmallArgs p{a->x, a->x_scale, a->w, a->bias, a->residual, a->y0, a->y1, a->z, a->z_scale, a->rows,
                      a->k, a->n, a->split, a->act, a->out_dtype, a->bias_dtype,
                      a->k % e == 0 && aligned16(a->x), a->k % 8 == 0 && aligned16(a->w),
                      aligned16(a->y0) && (!a->y1 || aligned16(a->y1)) && (!a->residual || aligned16(a->residual)) &&
                          (!a->z || aligned16(a->z))};
    return way == kWayFew ? run_few_rows(p, a->dtype, s) : run_narrow(p, a->dtype, s);
}

static cudaError_t forward_mma(const plattice_linear_args* a, const ForwardPlan& p, cudaStream_t s) {
    char* ws = static_cast<char*>(a->workspace);
    Operand x, w;
    cudaError_t e = cudaSuccess;
    if (a->x_scale) e = unpacked(&x, a, ws + p.x, s);
    else e = operand(&x, a->x, a->dtype, forward_parts(a), a->rows, a->k, ws + p.x, s);
    if (e == cudaSuccess) e = operand(&w, a->w, a->dtype, forward_parts(a), a->n, a->k, ws + p.w, s);
    if (e != cudaSuccess) return e;
    MmaArgs m{};
    m.y0 = a->y0;
    m.y1 = a->y1;
    m.bias = a->bias;
    m.residual = a->residual;
    m.z = a->z;
    m.z_scale = a->z_scale;
    m.ni = a->rows;
    m.nj = a->n;
    m.bias_dtype = a->bias_dtype;
    m.out_dtype = a->out_dtype;
    m.act = a->act;
    m.split = a->split;
    const bool aligned = a->n % 8 == 0 && aligned16(a->y0) && (!a->residual || aligned16(a->residual)) &&
                         (!a->z || a->z_scale || aligned16(a->z));
    m.half = a->dtype == PLATTICE_F16;
    m.fault = pl::fault_word();
    m.precise = true;
    sum_args(&m, a->k, 1, x.parts, w.parts);
    return mma_forward(p.bn, aligned, x, w, m, s);
}

static cudaError_t backward_narrow(const plattice_linear_args* a, const BackwardPlan& p, cudaStream_t s) {
    const bool slope = a->act != PLATTICE_ACT_NONE;
    float* partial = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + p.partial_w);
    const int per = a->dtype == PLATTICE_F32 ? 4 : 8;   // elements of 16 bytes
    SmallGradArgs g{};
    g.s.x = a->x;
    g.s.x_scale = a->x_scale;
    g.s.w = a->w;
    g.s.z = slope ? a->z : nullptr;
    g.s.z_scale = slope ? a->z_scale : nullptr;
    g.s.rows = a->rows;
    g.s.k = a->k;
    g.s.n = a->n;
    g.s.split = a->split;
    g.s.act = a->act;
    g.s.out_dtype = a->out_dtype;
    g.s.vec_x = a->k % per == 0 && aligned16(a->x);
    g.g0 = a->grad0;
    g.g1 = a->grad1;
    g.grad_x = a->grad_x;
    g.partial = partial;
    g.need_x = a->grad_x != nullptr;
    g.need_w = a->grad_w != nullptr;
    g.need_b = a->grad_bias != nullptr;
    g.vec_gx = a->k % 8 == 0 && aligned16(a->grad_x);
    g.vec_g = aligned16(a->grad0) && (!a->split || aligned16(a->grad1));
    const cudaError_t e = run_narrow_grad(g, a->dtype, backward_parts(a), p.lines, s);
    if (e != cudaSuccess || !(a->grad_w || a->grad_bias)) return e;
    const int64_t nw = (int64_t)a->n * a->k, columns = nw + a->n;
    k_sum_lines<<<(unsigned)ceil_div(columns, 32), 1024, 0, s>>>(a->grad_w, a->dtype, nw, a->grad_bias, a->bias_dtype, a->n,
                                                               partial, p.lines);
    return cudaGetLastError();
}

static cudaError_t grad_z(const plattice_linear_args* a, const BackwardPlan& p, cudaStream_t s) {
    char* ws = static_cast<char*>(a->workspace);
    const bool slope = a->act != PLATTICE_ACT_NONE;
    const bool store = p.gz_needed && (a->grad_x || a->grad_w);
    if (!store && !a->grad_bias) return cudaSuccess;
    const GradArgs g{a->grad0, a->grad1, slope ? a->z : nullptr, slope ? a->z_scale : nullptr, store ? ws + p.gz : nullptr, p.pitch,
                     a->grad_bias ? reinterpret_cast<float*>(ws + p.partial_b) : nullptr, a->rows, a->n, a->split,
                     a->act, p.shift,
                     a->n % 8 == 0 && aligned16(a->grad0) && (!slope || a->z_scale || aligned16(a->z))};
    cudaError_t e;
    if (a->out_dtype == PLATTICE_F32)
        e = a->dtype == PLATTICE_F32    ? launch_grad_z<float, Parts<3>>(g, p, s)
            : a->dtype == PLATTICE_BF16 ? launch_grad_z<float, Parts<2, true>>(g, p, s)
                                        : launch_grad_z<float, Parts<2>>(g, p, s);
    else
        e = a->dtype == PLATTICE_BF16 ? launch_grad_z<__nv_bfloat16, __nv_bfloat16>(g, p, s)
                                      : launch_grad_z<__half, __half>(g, p, s);
    if (e == cudaSuccess && a->grad_bias) e = column_sums(a->grad_bias, a->bias_dtype, g.partial, p.parts_b, a->n, s);
    return e;
}

static cudaError_t backward_mma(const plattice_linear_args* a, const BackwardPlan& p, cudaStream_t s) {
    char* ws = static_cast<char*>(a->workspace);
    const Operand gz{p.gz_needed ? ws + p.gz : a->grad0, a->rows, a->n, p.gz_needed ? p.pitch : a->n, gz_parts(a)};
    const int parts = backward_parts(a);
    cudaError_t e = cudaSuccess;
    MmaArgs m{};
    m.half = a->dtype == PLATTICE_F16 && parts == 1;
    m.fault = pl::fault_word();
    if (a->grad_x) {
        Operand w;
        e = operand(&w, a->w, a->dtype, parts, a->n, a->k, ws + p.w, s);
        if (e != cudaSuccess) return e;
        m.y0 = a->grad_x;
        m.ni = a->rows;
        m.nj = a->k;
        m.out_dtype = a->dtype;
        m.precise = true;
        sum_args(&m, a->n, 1, gz.parts, w.parts);
        e = mma_grad_x(p.bn_x, a->k % 8 == 0 && aligned16(a->grad_x), gz, w, m, s);
        if (e != cudaSuccess) return e;
    }
    if (a->grad_w) {
        Operand x;
        if (a->x_scale) e = unpacked(&x, a, ws + p.x, s);
        else e = operand(&x, a->x, a->dtype, parts, a->rows, a->k, ws + p.x, s);
        if (e != cudaSuccess) return e;
        m.ni = a->k;
        m.nj = a->n;
        sum_args(&m, a->rows, p.parts_w, x.parts, gz.parts);
        const bool direct = p.parts_w == 1;
        m.y0 = direct ? a->grad_w : ws + p.partial_w;
        m.out_dtype = direct ? a->dtype : PLATTICE_F32;
        m.precise = a->dtype == PLATTICE_F32;
        e = mma_grad_w(p.bn_w, x, gz, m, s);
        if (e == cudaSuccess && !direct)
            e = add_parts_to(a->grad_w, a->dtype, reinterpret_cast<const float*>(ws + p.partial_w), m.parts,
                             (int64_t)a->n * a->k, s);
    }
    return e;
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_linear_workspace_size(const plattice_linear_args* a, size_t* bytes) {
    if (!bytes || !linear_shape_ok(a)) return PLATTICE_ERR_INVALID;
    *bytes = (size_t)forward_plan(a).bytes;
    return PLATTICE_OK;
}

int plattice_linear(const plattice_linear_args* a, void* stream) {
    if (!linear_shape_ok(a)) return PLATTICE_ERR_INVALID;
    if (a->rows == 0) return PLATTICE_OK;
    if (!a->x || !a->w || !a->y0 || (a->split && !a->y1) || (a->z_scale && !a->z)) return PLATTICE_ERR_INVALID;
    if (a->split && a->residual) return PLATTICE_ERR_INVALID;
    if (a->z_scale && ((uintptr_t)a->z & 31)) return PLATTICE_ERR_INVALID;   // codes leave 32 bytes at a time
    if (a->x_scale && !aligned16(a->x)) return PLATTICE_ERR_INVALID;
    const ForwardPlan p = forward_plan(a);
    if (p.bytes && !workspace_ok(a, p.bytes)) return PLATTICE_ERR_WORKSPACE;
    const int rc = rows_poll("plattice_linear");
    if (rc != PLATTICE_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return rows_status(p.way == kWayTiles ? forward_mma(a, p, s) : forward_small(a, p.way, s), "plattice_linear");
}

int plattice_linear_backward_workspace_size(const plattice_linear_args* a, size_t* bytes) {
    if (!bytes || !linear_shape_ok(a)) return PLATTICE_ERR_INVALID;
    *bytes = (size_t)backward_plan(a).bytes;
    return PLATTICE_OK;
}

int plattice_linear_backward(const plattice_linear_args* a, void* stream) {
    if (!linear_shape_ok(a)) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaSuccess;
    if (a->rows == 0) {   // sums over no rows
        if (a->grad_w) e = cudaMemsetAsync(a->grad_w, 0, (size_t)a->n * a->k * dtype_size(a->dtype), s);
        if (e == cudaSuccess && a->grad_bias)
            e = cudaMemsetAsync(a->grad_bias, 0, (size_t)a->n * dtype_size(a->bias_dtype), s);
        return rows_status(e, "plattice_linear_backward");
    }
    if (!a->grad_x && !a->grad_w && !a->grad_bias) return PLATTICE_OK;
    if (!a->grad0 || (a->split && !a->grad1) || (a->grad_x && !a->w) || (a->grad_w && !a->x) ||
        (a->act != PLATTICE_ACT_NONE && !a->z))
        return PLATTICE_ERR_INVALID;
    if (a->x_scale && !aligned16(a->x)) return PLATTICE_ERR_INVALID;
    if (a->act != PLATTICE_ACT_NONE && a->z_scale && !aligned16(a->z)) return PLATTICE_ERR_INVALID;
    const BackwardPlan p = backward_plan(a);
    if (!workspace_ok(a, p.bytes)) return PLATTICE_ERR_WORKSPACE;
    const int rc = rows_poll("plattice_linear_backward");
    if (rc != PLATTICE_OK) return rc;
    if (p.narrow) return rows_status(backward_narrow(a, p, s), "plattice_linear_backward");
    e = grad_z(a, p, s);
    if (e == cudaSuccess) e = backward_mma(a, p, s);
    return rows_status(e, "plattice_linear_backward");
}

}  // extern "C"
