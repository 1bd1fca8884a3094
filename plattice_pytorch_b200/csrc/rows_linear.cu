// rows_linear.cu -- linear map of rows with bias, activation and residual,
// and its backward pass, x plain or in 8-bit rows.  C ABI: include/plattice.h.
#include <limits.h>

#include "rows_common.cuh"
#include "rows_host.h"

namespace plr {

// ------------------------------------------------------------------- operands

// An operand of the products, seen as element (i, r): i along the result, r
// along the sum.  One of the two strides is 1.  8-bit rows: `scale` non-null;
// their pitch is a multiple of 32, so element e of the buffer has scale e / 32.
struct View {
    const void* p;
    const uint8_t* scale;
    int64_t si, sr;
    int dtype;
};

__device__ __forceinline__ float view_at(const View& v, int64_t i, int64_t r) {
    const int64_t e = i * v.si + r * v.sr;
    if (v.scale) {
        float t[4];
        values4(t, static_cast<const uint8_t*>(v.p)[e], scale_of(v.scale[e >> 5]));
        return t[0];
    }
    return load_param(v.p, v.dtype, e);
}

// ------------------------------------------------- product on the CUDA cores

// out[z][i][j] = sum over r in part z of a(i, r) b(j, r), float32.
constexpr int kTile = 64, kStep = 16;

__global__ void __launch_bounds__(256) k_product(float* __restrict__ out, const View a, const View b, int64_t ni,
                                                 int64_t nj, int64_t nr, int64_t part) {
    __shared__ float sa[kStep][kTile + 4], sb[kStep][kTile + 4];
    const int64_t i0 = (int64_t)blockIdx.x * kTile, j0 = (int64_t)blockIdx.y * kTile;
    const int64_t r0 = (int64_t)blockIdx.z * part, r1 = min(nr, r0 + part);
    const int ti = threadIdx.x & 15, tj = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t rb = r0; rb < r1; rb += kStep) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int t = threadIdx.x + 256 * u;
            // neighbouring threads along the contiguous direction
            const int ia = a.sr == 1 ? t / kStep : t % kTile, ra = a.sr == 1 ? t % kStep : t / kTile;
            const int jb = b.sr == 1 ? t / kStep : t % kTile, rr = b.sr == 1 ? t % kStep : t / kTile;
            sa[ra][ia] = i0 + ia < ni && rb + ra < r1 ? view_at(a, i0 + ia, rb + ra) : 0.f;
            sb[rr][jb] = j0 + jb < nj && rb + rr < r1 ? view_at(b, j0 + jb, rb + rr) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kStep; ++r) {
            const float4 x = *reinterpret_cast<const float4*>(&sa[r][ti * 4]);
            const float4 y = *reinterpret_cast<const float4*>(&sb[r][tj * 4]);
            const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < 4; ++n) acc[m][n] = fmaf(xs[m], ys[n], acc[m][n]);
        }
        __syncthreads();
    }
    float* o = out + (int64_t)blockIdx.z * ni * nj;
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int64_t i = i0 + ti * 4 + m, j = j0 + tj * 4 + n;
            if (i < ni && j < nj) o[i * nj + j] = acc[m][n];
        }
}

// ------------------------------------------------------------------ epilogue

struct FinishArgs {
    const float* acc;   // [rows][n]
    const void* bias;
    int bias_dtype;
    const void* residual;
    void* y0;
    void* y1;
    void* z;
    uint8_t* z_scale;
    int64_t rows;
    int n, split, act, out_dtype;
};

// A thread takes 8 columns of a row, 4 neighbouring lanes a block of 32 (the
// blocks of the kept 8-bit pre-activation).
template <typename T>
__global__ void __launch_bounds__(256) k_finish(const FinishArgs a, unsigned groups) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row = t / groups;
    const int col = (int)(t - row * groups) * 8;
    const int left = row < a.rows ? a.n - col : 0;
    float z[8], y[8];
    load8(z, a.acc + (left > 0 ? row * a.n + col : 0), false, left);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (a.bias && i < left) z[i] += load_param(a.bias, a.bias_dtype, col + i);
        y[i] = act_value(z[i], a.act);
    }
    if (a.residual) {
        float r[8];
        load8(r, static_cast<const T*>(a.residual) + (left > 0 ? row * a.n + col : 0), false, left);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] += r[i];
    }
    if (a.z_scale) {
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) amax = fmaxf(amax, finite_abs(z[i]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const int s = block_exponent(amax);
        if (row < a.rows) {
            reinterpret_cast<uint2*>(a.z)[t] = codes8(z, pow2(-s));
            if ((threadIdx.x & 3) == 0) a.z_scale[t >> 2] = (uint8_t)(s + 127);
        }
    } else if (a.z) {
        store8(static_cast<T*>(a.z) + (left > 0 ? row * a.n + col : 0), z, false, left);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        if (i >= left) continue;
        const int c = col + i;
        if (c < a.split) static_cast<T*>(a.y0)[row * a.split + c] = from_f32<T>(y[i]);
        else if (a.split) static_cast<T*>(a.y1)[row * (a.n - a.split) + c - a.split] = from_f32<T>(y[i]);
        else static_cast<T*>(a.y0)[row * a.n + c] = from_f32<T>(y[i]);
    }
}

// ------------------------------------------------- backward: gz and its sums

struct GradArgs {
    const void* g0;
    const void* g1;
    const void* z;
    const uint8_t* z_scale;
    void* gz;           // [rows][pitch] in the operands' type; null: not stored
    int64_t pitch;
    float* partial;     // [gridDim.y][n]; null: no bias gradient
    int64_t rows;
    int n, split, act;
};

// gz = grad_y act'(z), rounded to the operands' type for the two products (a
// tensor core takes no wider operand; one rounding, as a stored gradient has),
// and the sums of the unrounded gz over a CTA's rows.  32 lanes of 8 columns,
// 8 rows at a time; gridDim.x strips of 256 columns, gridDim.y parts of rows.
template <typename TG, typename T>
__global__ void __launch_bounds__(256) k_grad_z(const GradArgs a) {
    __shared__ float sums[8][256];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int col = blockIdx.x * 256 + lane * 8;
    float acc[8] = {};
    for (int64_t row = (int64_t)blockIdx.y * 8 + w; row < a.rows; row += (int64_t)gridDim.y * 8) {
        const int left = a.n - col;
        float g[8], z[8];
        if (a.split == 0) {
            load8(g, static_cast<const TG*>(a.g0) + (left > 0 ? row * a.n + col : 0), false, left);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int c = col + i;
                g[i] = i >= left ? 0.f
                       : c < a.split ? to_f32(static_cast<const TG*>(a.g0)[row * a.split + c])
                                     : to_f32(static_cast<const TG*>(a.g1)[row * (a.n - a.split) + c - a.split]);
            }
        }
        if (a.act != PLATTICE_ACT_NONE) {
            if (a.z_scale) {
                if (left > 0) {
                    const int64_t at = row * (width8(a.n) / 8) + col / 8;
                    values8(z, reinterpret_cast<const uint2*>(a.z)[at], scale_of(a.z_scale[at >> 2]));
                }
            } else {
                load8(z, static_cast<const TG*>(a.z) + (left > 0 ? row * a.n + col : 0), false, left);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < left) g[i] *= act_slope(z[i], a.act);
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += g[i];
        const int64_t wide = a.pitch - col;   // zeros up to the pitch
        if (a.gz && wide > 0) store8(static_cast<T*>(a.gz) + row * a.pitch + col, g, false, (int)min(wide, (int64_t)8));
    }
    if (!a.partial) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[w][lane * 8 + i] = acc[i];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    float s = 0.f;
#pragma unroll
    for (int r = 0; r < 8; ++r) s += sums[r][threadIdx.x];
    if (c < a.n) a.partial[(int64_t)blockIdx.y * a.n + c] = s;
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

// Parts of a sum over `len` terms whose result has `tiles` tiles: enough CTAs
// for the device, none shorter than 512 terms.
static int parts_of(int64_t tiles, int64_t len) {
    const int64_t want = (2 * (int64_t)sm_count() + tiles - 1) / tiles;
    const int64_t most = (len + 511) / 512;
    int64_t p = want < most ? want : most;
    if (p < 1) p = 1;
    if (p > 512) p = 512;
    return (int)p;
}

static int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

static int grad_rows_parts(int64_t rows, int n) {
    const int64_t strips = (n + 255) / 256, need = (rows + 7) / 8;
    const int64_t most = (4 * (int64_t)sm_count() + strips - 1) / strips;
    return (int)(need < most ? need : most);
}

static View view_rows(const void* p, const uint8_t* scale, int64_t pitch, int dtype, bool along_rows) {
    if (scale) pitch = width8(pitch);
    return along_rows ? View{p, scale, 1, pitch, dtype} : View{p, scale, pitch, 1, dtype};
}

static cudaError_t product(float* out, const View& a, const View& b, int64_t ni, int64_t nj, int64_t nr, int parts,
                           cudaStream_t s) {
    if (tiles_of(ni) > INT_MAX || tiles_of(nj) > 65535) return cudaErrorInvalidValue;
    const int64_t part = (nr + parts - 1) / parts;
    k_product<<<dim3((unsigned)tiles_of(ni), (unsigned)tiles_of(nj), parts), 256, 0, s>>>(out, a, b, ni, nj, nr, part);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t add_parts(void* out, const float* partial, int parts, int64_t n, cudaStream_t s) {
    k_add_parts<T><<<(unsigned)((n + 255) / 256), 256, 0, s>>>(static_cast<T*>(out), partial, parts, n);
    return cudaGetLastError();
}

static cudaError_t add_parts_to(void* out, int dtype, const float* partial, int parts, int64_t n, cudaStream_t s) {
    if (dtype == PLATTICE_F32) return add_parts<float>(out, partial, parts, n, s);
    if (dtype == PLATTICE_BF16) return add_parts<__nv_bfloat16>(out, partial, parts, n, s);
    return add_parts<__half>(out, partial, parts, n, s);
}

static bool linear_shape_ok(const plattice_linear_args* a) {
    if (!a || a->rows < 0 || a->k < 1 || a->n < 1 || a->split < 0 || a->split >= a->n) return false;
    if (!dtype_ok(a->dtype) || !dtype_ok(a->out_dtype) || !dtype_ok(a->bias_dtype)) return false;
    if (a->out_dtype != a->dtype && a->out_dtype != PLATTICE_F32) return false;
    if (a->x_scale && a->dtype == PLATTICE_F16) return false;
    if (a->act < PLATTICE_ACT_NONE || a->act > PLATTICE_ACT_SILU) return false;
    if (a->split && a->act != PLATTICE_ACT_NONE) return false;
    return fits(a->rows, width8(a->k)) && fits(a->rows, width8(a->n)) && fits(a->k, a->n);
}

struct BackwardPlan {
    int64_t gz, partial_b, partial_w, acc_x, bytes;
    int parts_b, parts_w;
    int64_t pitch;
};

static BackwardPlan backward_plan(const plattice_linear_args* a) {
    BackwardPlan p{};
    p.pitch = a->n;
    p.parts_b = grad_rows_parts(a->rows, a->n);
    p.parts_w = parts_of(tiles_of(a->n) * tiles_of(a->k), a->rows);
    int64_t at = 0;
    p.gz = at; at += up256(a->rows * p.pitch * (int64_t)dtype_size(a->dtype));
    p.partial_b = at; at += up256((int64_t)p.parts_b * a->n * 4);
    p.partial_w = at; at += up256((int64_t)p.parts_w * a->n * a->k * 4);
    p.acc_x = at; at += up256(a->rows * a->k * 4);
    p.bytes = at;
    return p;
}

template <typename TG, typename T>
static cudaError_t launch_grad_z(const GradArgs& g, int parts, cudaStream_t s) {
    k_grad_z<TG, T><<<dim3((g.n + 255) / 256, parts), 256, 0, s>>>(g);
    return cudaGetLastError();
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_linear_workspace_size(const plattice_linear_args* a, size_t* bytes) {
    if (!bytes || !linear_shape_ok(a)) return PLATTICE_ERR_INVALID;
    *bytes = (size_t)up256(a->rows * a->n * 4);
    return PLATTICE_OK;
}

int plattice_linear(const plattice_linear_args* a, void* stream) {
    if (!linear_shape_ok(a)) return PLATTICE_ERR_INVALID;
    if (a->rows == 0) return PLATTICE_OK;
    if (!a->x || !a->w || !a->y0 || (a->split && !a->y1) || (a->z_scale && !a->z)) return PLATTICE_ERR_INVALID;
    if (a->split && a->residual) return PLATTICE_ERR_INVALID;
    size_t need = 0;
    plattice_linear_workspace_size(a, &need);
    if (!a->workspace || a->workspace_bytes < need) return PLATTICE_ERR_WORKSPACE;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    float* acc = static_cast<float*>(a->workspace);
    cudaError_t e = product(acc, view_rows(a->x, a->x_scale, a->k, a->dtype, false),
                            view_rows(a->w, nullptr, a->k, a->dtype, false), a->rows, a->n, a->k, 1, s);
    if (e == cudaSuccess) {
        const FinishArgs f{acc, a->bias, a->bias_dtype, a->residual, a->y0, a->y1, a->z, a->z_scale, a->rows,
                           a->n, a->split, a->act, a->out_dtype};
        const unsigned groups = (unsigned)(width8(a->n) / 8);
        const int64_t ctas = (a->rows * groups + 255) / 256;
        if (ctas > INT_MAX) return PLATTICE_ERR_INVALID;
        if (a->out_dtype == PLATTICE_F32) k_finish<float><<<(unsigned)ctas, 256, 0, s>>>(f, groups);
        else if (a->out_dtype == PLATTICE_BF16) k_finish<__nv_bfloat16><<<(unsigned)ctas, 256, 0, s>>>(f, groups);
        else k_finish<__half><<<(unsigned)ctas, 256, 0, s>>>(f, groups);
        e = cudaGetLastError();
    }
    return rows_status(e, "plattice_linear");
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
    if (!a->grad0 || (a->split && !a->grad1) || (a->grad_x && !a->w) || (a->grad_w && !a->x) ||
        (a->act != PLATTICE_ACT_NONE && !a->z))
        return PLATTICE_ERR_INVALID;
    const BackwardPlan p = backward_plan(a);
    if (!a->workspace || a->workspace_bytes < (size_t)p.bytes) return PLATTICE_ERR_WORKSPACE;
    char* ws = static_cast<char*>(a->workspace);
    GradArgs g{a->grad0, a->grad1, a->z, a->z_scale, ws + p.gz, p.pitch,
               a->grad_bias ? reinterpret_cast<float*>(ws + p.partial_b) : nullptr, a->rows, a->n, a->split, a->act};
    if (a->out_dtype == PLATTICE_F32) {
        e = a->dtype == PLATTICE_F32    ? launch_grad_z<float, float>(g, p.parts_b, s)
            : a->dtype == PLATTICE_BF16 ? launch_grad_z<float, __nv_bfloat16>(g, p.parts_b, s)
                                        : launch_grad_z<float, __half>(g, p.parts_b, s);
    } else {
        e = a->dtype == PLATTICE_BF16 ? launch_grad_z<__nv_bfloat16, __nv_bfloat16>(g, p.parts_b, s)
                                      : launch_grad_z<__half, __half>(g, p.parts_b, s);
    }
    if (e == cudaSuccess && a->grad_bias) e = column_sums(a->grad_bias, a->bias_dtype, g.partial, p.parts_b, a->n, s);
    if (e == cudaSuccess && a->grad_x) {
        float* acc = reinterpret_cast<float*>(ws + p.acc_x);
        e = product(acc, view_rows(g.gz, nullptr, p.pitch, a->dtype, false),
                    view_rows(a->w, nullptr, a->k, a->dtype, true), a->rows, a->k, a->n, 1, s);
        if (e == cudaSuccess) e = add_parts_to(a->grad_x, a->dtype, acc, 1, a->rows * a->k, s);
    }
    if (e == cudaSuccess && a->grad_w) {
        float* part = reinterpret_cast<float*>(ws + p.partial_w);
        e = product(part, view_rows(g.gz, nullptr, p.pitch, a->dtype, true),
                    view_rows(a->x, a->x_scale, a->k, a->dtype, true), a->n, a->k, a->rows, p.parts_w, s);
        if (e == cudaSuccess) e = add_parts_to(a->grad_w, a->dtype, part, p.parts_w, (int64_t)a->n * a->k, s);
    }
    return rows_status(e, "plattice_linear_backward");
}

}  // extern "C"
