// rows_clip.cu -- the norm of many gradients together, and the gradients scaled
// down to a largest norm.
//
//   norm = sqrt(sum g^2),   out = g min(1, max_norm / (norm + eps))
//
// The tensors are cut into pieces of kPiece values; the table of tensors goes
// with the launch (kernel arguments, no copy to the device), and a CTA finds a
// piece's tensor by a search of it.  CTAs add their pieces' squares, the second
// kernel's CTAs each add the CTAs' sums, in the same order, and scale.  Both are
// bound by HBM: the gradients are read twice, as far as the L2 does not hold them.
#include <cooperative_groups.h>
#include <stdlib.h>

#include <algorithm>

#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

namespace cg = cooperative_groups;

constexpr int kPiece = 8192, kUnroll = 4;   // values of a piece: 4 accesses of 8 by each of 256 threads

template <int kTensors> struct Grads {
    const void* g[kTensors];
    void* out[kTensors];
    long long size[kTensors];
    long long end[kTensors];      // pieces up to the tensor's last
    uint8_t type[kTensors];       // dtype | out_dtype << 2 | g and out aligned << 4 | g aligned << 5
    int count;
};
constexpr int kMost = 256, kSome = 64;   // tensors of one launch; of a small one's table
constexpr int kResident = 6;             // CTAs of an SM: one round

// The tensor of a piece: the first whose end is above it.
template <int N> __device__ __forceinline__ int tensor_of(const Grads<N>& t, long long piece) {
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
__device__ __forceinline__ double piece_squares(const T* g, int n, bool aligned) {
    double sum = 0.0;
    float v[8];
    if (aligned && n == kPiece) {   // all accesses under way before the first sum
        Raw8<T> r[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) r[k].load(g + (k * 256 + threadIdx.x) * 8, true, 8);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            r[k].widen(v);
            sum += squares(v);
        }
    } else if (aligned) {
        for (int i = threadIdx.x * 8; i < n; i += 2048) {
            load8(v, g + i, n - i >= 8, n - i);
            sum += squares(v);
        }
    } else {   // neighbouring threads on neighbouring values
        for (int i = threadIdx.x; i < n; i += 2048) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = i + k * 256 < n ? to_f32(g[i + k * 256]) : 0.f;
            sum += squares(v);
        }
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

// Where a piece of kSize values lies; `tensor` where it is known.
template <int kSize = kPiece> struct At {
    int tensor, n, dtype;
    long long first;
    bool aligned, aligned_g, wide;   // aligned_g: all that the squares' order goes by
    template <int N> __device__ __forceinline__ At(const Grads<N>& t, long long piece) : At(t, piece, tensor_of(t, piece)) {}
    template <int N> __device__ __forceinline__ At(const Grads<N>& t, long long piece, int tensor_) : tensor(tensor_) {
        first = (piece - (tensor ? t.end[tensor - 1] : 0)) * kSize;
        const long long left = t.size[tensor] - first;
        n = left < kSize ? (int)left : kSize;
        const int type = t.type[tensor];
        dtype = type & 3;
        wide = ((type >> 2) & 3) == PLATTICE_F32;
        aligned = type >> 4 & 1;
        aligned_g = type >> 5;
    }
};

// The pieces of a CTA: neighbouring ones, so that it searches for a tensor once.
struct Share {
    long long first, end;
    template <int N> __device__ __forceinline__ explicit Share(const Grads<N>& t) {
        const long long pieces = t.end[t.count - 1], each = pieces / gridDim.x, more = pieces - each * gridDim.x;
        first = blockIdx.x * each + (blockIdx.x < more ? blockIdx.x : more);
        end = first + each + (blockIdx.x < more);
    }
};

template <int N> __device__ __forceinline__ double squares_at(const Grads<N>& t, const At<>& p) {
    const void* g = t.g[p.tensor];
    if (p.dtype == PLATTICE_F32) return piece_squares(static_cast<const float*>(g) + p.first, p.n, p.aligned_g);
    if (p.dtype == PLATTICE_BF16) return piece_squares(static_cast<const __nv_bfloat16*>(g) + p.first, p.n, p.aligned_g);
    return piece_squares(static_cast<const __half*>(g) + p.first, p.n, p.aligned_g);
}

template <int N>
__global__ void __launch_bounds__(256, kResident) k_square_sums(const __grid_constant__ Grads<N> t, double* __restrict__ sums) {
    double sum = 0.0;
    const Share s(t);
    int tensor = s.first < s.end ? tensor_of(t, s.first) : 0;
    for (long long p = s.first; p < s.end; ++p) {
        while (t.end[tensor] <= p) ++tensor;
        sum += squares_at(t, At<>(t, p, tensor));
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
__device__ __forceinline__ void piece_scale(O* out, const T* g, int n, bool aligned, float f) {
    // 16 bytes of the wider type a thread: whole sectors of neighbouring threads
    constexpr int V = 16 / (int)(sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O)), kPasses = kPiece / (256 * V);
    float v[V];
    if (aligned && n == kPiece) {
#pragma unroll
        for (int half = 0; half < kPasses; half += 4) {
            Vec<T, V> r[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) r[k].load(g + ((half + k) * 256 + threadIdx.x) * V);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = r[k].at(j) * f;
                Vec<O, V> o;
                o.from(v);
                o.store(out + ((half + k) * 256 + threadIdx.x) * V);
            }
        }
    } else if (aligned) {
        for (int i = threadIdx.x * V; i < n; i += 256 * V) {
            if (n - i >= V) {
                Vec<T, V> r;
                r.load(g + i);
#pragma unroll
                for (int j = 0; j < V; ++j) v[j] = r.at(j) * f;
                Vec<O, V> o;
                o.from(v);
                o.store(out + i);
            } else {
                for (int j = i; j < n; ++j) out[j] = from_f32<O>(to_f32(g[j]) * f);
            }
        }
    } else {
        for (int i = threadIdx.x; i < n; i += 2048) {
            float w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = i + k * 256 < n ? to_f32(g[i + k * 256]) : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (i + k * 256 < n) out[i + k * 256] = from_f32<O>(w[k] * f);
        }
    }
}

template <int N> __device__ __forceinline__ void scale_at(const Grads<N>& t, const At<>& p, float f) {
    const void* g = t.g[p.tensor];
    void* out = t.out[p.tensor];
    if (f == 1.f && g == out) return;   // in place, as it is
    if (p.dtype == PLATTICE_F32)
        piece_scale(static_cast<float*>(out) + p.first, static_cast<const float*>(g) + p.first, p.n, p.aligned, f);
    else if (p.dtype == PLATTICE_BF16 && p.wide)
        piece_scale(static_cast<float*>(out) + p.first, static_cast<const __nv_bfloat16*>(g) + p.first, p.n, p.aligned, f);
    else if (p.dtype == PLATTICE_BF16)
        piece_scale(static_cast<__nv_bfloat16*>(out) + p.first, static_cast<const __nv_bfloat16*>(g) + p.first, p.n, p.aligned, f);
    else if (p.wide)
        piece_scale(static_cast<float*>(out) + p.first, static_cast<const __half*>(g) + p.first, p.n, p.aligned, f);
    else
        piece_scale(static_cast<__half*>(out) + p.first, static_cast<const __half*>(g) + p.first, p.n, p.aligned, f);
}

__device__ __forceinline__ float factor_of(const Norm& q, double norm) {
    const double f = (double)q.most / (norm + (double)q.eps);
    return q.most == INFINITY || norm + (double)q.eps == 0.0 ? 1.f : f > 1.0 ? 1.f : (float)f;   // NaN stays
}

// The pieces that a CTA read last are scaled first: some are still in the L2.
template <int N>
__global__ void __launch_bounds__(256, kResident) k_clip(const __grid_constant__ Grads<N> t, Norm q) {
    const double norm = norm_of(q);
    if (blockIdx.x == 0 && threadIdx.x == 0 && q.out) *q.out = (float)norm;
    const float f = factor_of(q, norm);
    const Share s(t);
    int tensor = s.first < s.end ? tensor_of(t, s.end - 1) : 0;
    for (long long p = s.end - 1; p >= s.first; --p) {
        while (tensor && t.end[tensor - 1] > p) --tensor;
        scale_at(t, At<>(t, p, tensor), f);
    }
}

// Few values: one cluster of kFew CTAs does both, without a second launch, a warp for
// each piece of kSmallPiece values.
constexpr int kFew = 8, kSmallPiece = 1024, kFewPieces = 192;

template <typename T>
__device__ __forceinline__ double warp_squares(const T* g, int n) {
    double sum = 0.0;
    for (int i = threadIdx.x & 31; i < n; i += 256) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = i + k * 32 < n ? to_f32(g[i + k * 32]) : 0.f;
        sum += squares(v);
    }
    return sum;
}
template <typename T, typename O>
__device__ __forceinline__ void warp_scale(O* out, const T* g, int n, float f) {
    for (int i = threadIdx.x & 31; i < n; i += 256) {
        float v[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = i + k * 32 < n ? to_f32(g[i + k * 32]) : 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (i + k * 32 < n) out[i + k * 32] = from_f32<O>(v[k] * f);
    }
}

__global__ void __cluster_dims__(kFew) __launch_bounds__(256) k_clip_few(const __grid_constant__ Grads<kSome> t, Norm q) {
    __shared__ double own;
    const cg::cluster_group cluster = cg::this_cluster();
    const int pieces = t.count ? (int)t.end[t.count - 1] : 0, first = blockIdx.x + kFew * (threadIdx.x >> 5), step = kFew * 8;
    double sum = 0.0;
    for (int p = first; p < pieces; p += step) {
        const At<kSmallPiece> at(t, p);
        const void* g = t.g[at.tensor];
        if (at.dtype == PLATTICE_F32) sum += warp_squares(static_cast<const float*>(g) + at.first, at.n);
        else if (at.dtype == PLATTICE_BF16) sum += warp_squares(static_cast<const __nv_bfloat16*>(g) + at.first, at.n);
        else sum += warp_squares(static_cast<const __half*>(g) + at.first, at.n);
    }
    sum = cta_sum(sum);
    if (threadIdx.x == 0) own = sum;
    cluster.sync();
    sum = 0.0;
#pragma unroll
    for (int c = 0; c < kFew; ++c) sum += *cluster.map_shared_rank(&own, c);
    cluster.sync();   // the others' sums have been read
    const double norm = sqrt(sum);
    if (blockIdx.x == 0 && threadIdx.x == 0 && q.out) *q.out = (float)norm;
    const float f = factor_of(q, norm);
    if (!t.count || !t.out[0]) return;
    for (int p = first; p < pieces; p += step) {
        const At<kSmallPiece> at(t, p);
        const void* g = t.g[at.tensor];
        void* out = t.out[at.tensor];
        if (f == 1.f && g == out) continue;   // in place, as it is
        if (at.dtype == PLATTICE_F32) warp_scale(static_cast<float*>(out) + at.first, static_cast<const float*>(g) + at.first, at.n, f);
        else if (at.dtype == PLATTICE_BF16 && at.wide)
            warp_scale(static_cast<float*>(out) + at.first, static_cast<const __nv_bfloat16*>(g) + at.first, at.n, f);
        else if (at.dtype == PLATTICE_BF16)
            warp_scale(static_cast<__nv_bfloat16*>(out) + at.first, static_cast<const __nv_bfloat16*>(g) + at.first, at.n, f);
        else if (at.wide) warp_scale(static_cast<float*>(out) + at.first, static_cast<const __half*>(g) + at.first, at.n, f);
        else warp_scale(static_cast<__half*>(out) + at.first, static_cast<const __half*>(g) + at.first, at.n, f);
    }
}

// ------------------------------------------------------------------ host side

static int most_ctas() { return kResident * sm_count(); }

// Fills a launch's table from grads[first..]; gives the first that did not fit.
template <int N> static int fill(Grads<N>& t, const plattice_grad* grads, int first, int count, long long* pieces, int size = kPiece) {
    t.count = 0;
    *pieces = 0;
    for (; first < count && t.count < N; ++first) {
        const plattice_grad& g = grads[first];
        if (g.size == 0) continue;
        const int k = t.count++;
        t.g[k] = g.g;
        t.out[k] = g.out;
        t.size[k] = g.size;
        *pieces += ceil_div(g.size, size);
        t.end[k] = *pieces;
        t.type[k] = (uint8_t)(g.dtype | g.out_dtype << 2 | (aligned16(g.g) ? aligned16(g.out) ? 48 : 32 : 0));
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
    *bytes = (size_t)(ceil_div(count, kMost) + 1) * 2048 * sizeof(double);
    return PLATTICE_OK;
}

int plattice_clip_grads(const plattice_grad* grads, int count, float max_norm, float eps, const float* norm_in,
                        float* norm_out, void* workspace, size_t workspace_bytes, void* stream) {
    if (!grads_ok(grads, count) || !on_elements(sizeof(float), norm_in, norm_out)) return PLATTICE_ERR_INVALID;
    int outs = 0, tensors = 0;
    for (int i = 0; i < count; ++i)
        if (grads[i].size) {
            ++tensors;
            outs += grads[i].out != nullptr;
        }
    if (outs && outs != tensors) return PLATTICE_ERR_INVALID;
    if (!outs && !norm_out) return tensors ? PLATTICE_ERR_INVALID : PLATTICE_OK;
    if (outs) {
        if (!(max_norm >= 0.f) || !(eps >= 0.f && eps < INFINITY)) return PLATTICE_ERR_INVALID;
        for (int i = 0; i < count; ++i) {
            const plattice_grad& g = grads[i];
            if (!dtype_ok(g.out_dtype) || (g.out_dtype != g.dtype && g.out_dtype != PLATTICE_F32)) return PLATTICE_ERR_INVALID;
            if (g.size && ((uintptr_t)g.out % dtype_size(g.out_dtype) || (g.out == g.g && g.out_dtype != g.dtype)))
                return PLATTICE_ERR_INVALID;
        }
        Span* v = static_cast<Span*>(malloc((2 * (size_t)tensors + 2) * sizeof(Span)));
        if (!v) return PLATTICE_ERR_WORKSPACE;
        int n = 0;
        for (int i = 0; i < count; ++i) {
            const plattice_grad& g = grads[i];
            if (!g.size) continue;
            v[n++] = {(uintptr_t)g.g, (uintptr_t)g.g + g.size * dtype_size(g.dtype), i, false};
            v[n++] = {(uintptr_t)g.out, (uintptr_t)g.out + g.size * dtype_size(g.out_dtype), i, true};
        }
        // every CTA reads the norm given, some while others write
        if (norm_in && norm_in != norm_out) v[n++] = {(uintptr_t)norm_in, (uintptr_t)norm_in + sizeof(float), count, false};
        if (norm_out) v[n++] = {(uintptr_t)norm_out, (uintptr_t)norm_out + sizeof(float), count + 1, true};
        const bool bad = overlaps(grads, v, n);
        free(v);
        if (bad) return PLATTICE_ERR_INVALID;
    }
    size_t need = 0;
    plattice_clip_grads_workspace_size(grads, count, &need);
    if (!norm_in && (!workspace || ((uintptr_t)workspace & 255) || workspace_bytes < need)) return PLATTICE_ERR_WORKSPACE;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    long long pieces = 0;
    for (int i = 0; i < count; ++i) pieces += ceil_div(grads[i].size, kSmallPiece);
    Norm q{norm_in ? nullptr : static_cast<double*>(workspace), 0, norm_in, norm_out, max_norm, eps};
    cudaError_t e = cudaSuccess;
    if (!norm_in && pieces <= kFewPieces && tensors <= kSome) {
        Grads<kSome> t;
        fill(t, grads, 0, count, &pieces, kSmallPiece);
        k_clip_few<<<kFew, 256, 0, s>>>(t, q);
        return rows_status(cudaGetLastError(), "plattice_clip_grads");
    }
    static thread_local Grads<kMost> t;
    if (!norm_in) {
        for (int first = 0; first < count && e == cudaSuccess;) {
            first = fill(t, grads, first, count, &pieces);
            if (!t.count) break;
            const int ctas = ctas_of(pieces);
            k_square_sums<<<ctas, 256, 0, s>>>(t, static_cast<double*>(workspace) + q.count);
            q.count += ctas;
            e = cudaGetLastError();
        }
    }
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
