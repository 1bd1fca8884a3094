// rows_clip.cu -- the norm of many gradients together, and the gradients scaled
// down to a largest norm.
//
//   norm = sqrt(sum g^2),   out = g min(1, max_norm / (norm + eps))
//
// The tensors are cut into pieces of kPiece values; the table of tensors goes
// with the launch (kernel arguments, no copy to the device), and a CTA finds a
// piece's tensor by a search of it.  CTAs add their pieces' squares, the second
// kernel's CTAs each add the CTAs' sums, in the same order, and scale.
#include <stdlib.h>

#include <algorithm>

#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

constexpr int kPiece = 8192;
constexpr int kTensors = 256;   // of one launch

struct Grads {
    const void* g[kTensors];
    void* out[kTensors];
    long long size[kTensors];
    long long end[kTensors];      // pieces up to the tensor's last
    uint8_t type[kTensors];       // dtype | out_dtype << 2 | aligned << 4
    int count;
};

// The tensor of a piece: the first whose end is above it.
__device__ __forceinline__ int tensor_of(const Grads& t, long long piece) {
    int lo = 0, hi = t.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (t.end[mid] > piece) hi = mid;
        else lo = mid + 1;
    }
    return lo;
}

// Squares of 8 values: in float32 where the sum is far from both ends of its
// range, else in float64.
__device__ __forceinline__ double squares(const float (&v)[8]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s = fmaf(v[i], v[i], s);
    if (s > 1e-36f && s < 1e38f) return (double)s;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) amax = max_nan(amax, fabsf(v[i]));
    if (amax == 0.f) return 0.0;
    double d = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) d += (double)v[i] * (double)v[i];
    return d;
}

template <typename T>
__device__ __forceinline__ double piece_squares(const T* g, long long n, bool aligned) {
    double sum = 0.0;
    for (int i = threadIdx.x * 8; i < n; i += 2048) {
        float v[8];
        const int left = (int)(n - i);
        load8(v, g + i, aligned && left >= 8, left);
        sum += squares(v);
    }
    return sum;
}

__device__ __forceinline__ double cta_sum(double v) {
    __shared__ double s[8];
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += s[k];
    return v;
}

__global__ void __launch_bounds__(256) k_square_sums(const __grid_constant__ Grads t, double* __restrict__ sums) {
    double sum = 0.0;
    const long long pieces = t.end[t.count - 1];
    for (long long p = blockIdx.x; p < pieces; p += gridDim.x) {
        const int k = tensor_of(t, p);
        const long long at = (p - (k ? t.end[k - 1] : 0)) * kPiece, left = t.size[k] - at;
        const long long n = left < kPiece ? left : kPiece;
        const bool aligned = t.type[k] >> 4;
        const int dtype = t.type[k] & 3;
        if (dtype == PLATTICE_F32) sum += piece_squares(static_cast<const float*>(t.g[k]) + at, n, aligned);
        else if (dtype == PLATTICE_BF16) sum += piece_squares(static_cast<const __nv_bfloat16*>(t.g[k]) + at, n, aligned);
        else sum += piece_squares(static_cast<const __half*>(t.g[k]) + at, n, aligned);
    }
    sum = cta_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

struct Norm {
    const double* sums;      // null: *in is the norm
    int count;
    const float* in;
    float* out;              // null: not wanted
    float most, eps;
};

// In float64, so that a norm past float32's range still scales.
__device__ __forceinline__ double norm_of(const Norm& q) {
    if (!q.sums) return *q.in;
    double s = 0.0;
    for (int i = threadIdx.x; i < q.count; i += 256) s += q.sums[i];
    return sqrt(cta_sum(s));
}

__global__ void __launch_bounds__(256) k_norm_only(Norm q) {
    const double norm = norm_of(q);
    if (threadIdx.x == 0) *q.out = (float)norm;
}

template <typename T, typename O>
__device__ __forceinline__ void piece_scale(O* out, const T* g, long long n, bool aligned, float f) {
    for (int i = threadIdx.x * 8; i < n; i += 2048) {
        float v[8];
        const int left = (int)(n - i);
        const bool vec = aligned && left >= 8;
        load8(v, g + i, vec, left);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= f;
        store8(out + i, v, vec, left);
    }
}

__global__ void __launch_bounds__(256) k_clip(const __grid_constant__ Grads t, Norm q) {
    const double norm = norm_of(q);
    if (blockIdx.x == 0 && threadIdx.x == 0 && q.out) *q.out = (float)norm;
    const double f64 = (double)q.most / (norm + (double)q.eps);
    const float f = q.most == INFINITY || norm + (double)q.eps == 0.0 ? 1.f : f64 > 1.0 ? 1.f : (float)f64;   // NaN stays
    const long long pieces = t.end[t.count - 1];
    for (long long p = blockIdx.x; p < pieces; p += gridDim.x) {
        const int k = tensor_of(t, p);
        if (f == 1.f && t.g[k] == t.out[k]) continue;   // in place, as it is
        const long long at = (p - (k ? t.end[k - 1] : 0)) * kPiece, left = t.size[k] - at;
        const long long n = left < kPiece ? left : kPiece;
        const bool aligned = t.type[k] >> 4;
        const int dtype = t.type[k] & 3;
        const bool wide = ((t.type[k] >> 2) & 3) == PLATTICE_F32;
        if (dtype == PLATTICE_F32)
            piece_scale(static_cast<float*>(t.out[k]) + at, static_cast<const float*>(t.g[k]) + at, n, aligned, f);
        else if (dtype == PLATTICE_BF16 && wide)
            piece_scale(static_cast<float*>(t.out[k]) + at, static_cast<const __nv_bfloat16*>(t.g[k]) + at, n, aligned, f);
        else if (dtype == PLATTICE_BF16)
            piece_scale(static_cast<__nv_bfloat16*>(t.out[k]) + at, static_cast<const __nv_bfloat16*>(t.g[k]) + at, n, aligned, f);
        else if (wide)
            piece_scale(static_cast<float*>(t.out[k]) + at, static_cast<const __half*>(t.g[k]) + at, n, aligned, f);
        else
            piece_scale(static_cast<__half*>(t.out[k]) + at, static_cast<const __half*>(t.g[k]) + at, n, aligned, f);
    }
}

// ------------------------------------------------------------------ host side

static int most_ctas() { return 8 * sm_count(); }

// Fills a launch's table from grads[first..]; gives the first that did not fit.
static int fill(Grads& t, const plattice_grad* grads, int first, int count, long long* pieces) {
    t.count = 0;
    *pieces = 0;
    for (; first < count && t.count < kTensors; ++first) {
        const plattice_grad& g = grads[first];
        if (g.size == 0) continue;
        const int k = t.count++;
        t.g[k] = g.g;
        t.out[k] = g.out;
        t.size[k] = g.size;
        *pieces += ceil_div(g.size, kPiece);
        t.end[k] = *pieces;
        t.type[k] = (uint8_t)(g.dtype | g.out_dtype << 2 | (aligned16(g.g) && aligned16(g.out) ? 16 : 0));
    }
    return first;
}

static int ctas_of(long long pieces) { return (int)(pieces < most_ctas() ? pieces : most_ctas()); }

struct Span {
    uintptr_t lo, hi;
    int owner;
    bool out;
};

// Whether some `out` shares memory with another tensor's g or out (a tensor's
// own out may lie on it).  The spans in order of their starts: two that overlap
// meet where the later one starts, so that the furthest end of the outs so far
// (disjoint, or this has returned), and of the inputs of another owner, decide.
static bool overlaps(const plattice_grad* grads, Span* v, int count) {
    std::sort(v, v + count, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    const auto own = [&](int i, int j) { return i == j && grads[i].g == grads[i].out; };
    Span out = {0, 0, -1, true}, in = {0, 0, -1, false}, next = in;   // next: of other owners than in's
    for (int i = 0; i < count; ++i) {
        const Span& s = v[i];
        if (s.lo < out.hi && (s.out || !own(s.owner, out.owner))) return true;
        if (s.out) {
            if (s.lo < in.hi && !own(s.owner, in.owner)) return true;
            if (s.lo < next.hi && !own(s.owner, next.owner)) return true;
            if (s.hi > out.hi) out = s;
        } else if (s.hi > in.hi) {
            next = in;
            in = s;
        } else if (s.hi > next.hi) {
            next = s;
        }
    }
    return false;
}

static bool grads_ok(const plattice_grad* grads, int count) {
    if (count < 0 || (count && !grads)) return false;
    for (int i = 0; i < count; ++i) {
        const plattice_grad& g = grads[i];
        if (!dtype_ok(g.dtype) || g.size < 0 || g.size > (1ll << 40) || (g.size && !g.g)) return false;
        if ((uintptr_t)g.g % dtype_size(g.dtype)) return false;
    }
    return true;
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_clip_grads_workspace_size(const plattice_grad* grads, int count, size_t* bytes) {
    if (!bytes || !grads_ok(grads, count)) return PLATTICE_ERR_INVALID;
    // a sum for each CTA of each launch, whatever the device's SM count (<= 256)
    *bytes = (size_t)(ceil_div(count, kTensors) + 1) * 2048 * sizeof(double);
    return PLATTICE_OK;
}

int plattice_clip_grads(const plattice_grad* grads, int count, float max_norm, float eps, const float* norm_in,
                        float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!grads_ok(grads, count)) return PLATTICE_ERR_INVALID;
    int outs = 0, tensors = 0;
    for (int i = 0; i < count; ++i)
        if (grads[i].size) {
            ++tensors;
            outs += grads[i].out != nullptr;
        }
    if (outs && outs != tensors) return PLATTICE_ERR_INVALID;
    if (!outs && !norm_out) return tensors ? PLATTICE_ERR_INVALID : PLATTICE_OK;
    if (outs) {
        if (!(max_norm >= 0.f) || !(eps >= 0.f)) return PLATTICE_ERR_INVALID;
        for (int i = 0; i < count; ++i) {
            const plattice_grad& g = grads[i];
            if (!dtype_ok(g.out_dtype) || (g.out_dtype != g.dtype && g.out_dtype != PLATTICE_F32)) return PLATTICE_ERR_INVALID;
            if (g.size && ((uintptr_t)g.out % dtype_size(g.out_dtype) || (g.out == g.g && g.out_dtype != g.dtype)))
                return PLATTICE_ERR_INVALID;
        }
        Span* v = static_cast<Span*>(malloc(2 * (size_t)tensors * sizeof(Span)));
        if (!v) return PLATTICE_ERR_WORKSPACE;
        int n = 0;
        for (int i = 0; i < count; ++i) {
            const plattice_grad& g = grads[i];
            if (!g.size) continue;
            v[n++] = {(uintptr_t)g.g, (uintptr_t)g.g + g.size * dtype_size(g.dtype), i, false};
            v[n++] = {(uintptr_t)g.out, (uintptr_t)g.out + g.size * dtype_size(g.out_dtype), i, true};
        }
        const bool bad = overlaps(grads, v, n);
        free(v);
        if (bad) return PLATTICE_ERR_INVALID;
    }
    size_t need = 0;
    plattice_clip_grads_workspace_size(grads, count, &need);
    if (!norm_in && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need)) return PLATTICE_ERR_WORKSPACE;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    static thread_local Grads t;
    double* sums = static_cast<double*>(workspace);
    int used = 0;
    long long pieces = 0;
    cudaError_t e = cudaSuccess;
    if (!norm_in) {
        for (int first = 0; first < count && e == cudaSuccess;) {
            first = fill(t, grads, first, count, &pieces);
            if (!t.count) break;
            const int ctas = ctas_of(pieces);
            k_square_sums<<<ctas, 256, 0, s>>>(t, sums + used);
            used += ctas;
            e = cudaGetLastError();
        }
    }
    Norm q{norm_in ? nullptr : sums, used, norm_in, norm_out, max_norm, eps};
    if (e == cudaSuccess && outs) {
        for (int first = 0; first < count && e == cudaSuccess;) {
            first = fill(t, grads, first, count, &pieces);
            if (!t.count) break;
            k_clip<<<ctas_of(pieces), 256, 0, s>>>(t, q);
            q.out = nullptr;   // written by the first launch
            e = cudaGetLastError();
        }
    } else if (e == cudaSuccess) {
        k_norm_only<<<1, 256, 0, s>>>(q);
        e = cudaGetLastError();
    }
    return rows_status(e, "plattice_clip_grads");
}

}  // extern "C"
