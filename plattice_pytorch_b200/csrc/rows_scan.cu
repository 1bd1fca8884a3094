// rows_scan.cu -- gated linear recurrence along lines of rows, and its gradients.
//
//   h[t] = a[t] h[t-1] + u[t],    u = x or (1 - a) x
//   G[t] = g[t] + a[t+1] G[t+1];  grad_x = G or (1 - a) G,
//   grad_a[t] = G[t] (h[t-1] or h[t-1] - x[t])
//
// A thread walks the steps of V neighbouring channels of a line in blocks of 16
// (PLATTICE_SCAN_KEEP), whose loads are in flight together.  The forward keeps
// the float32 state before each block (4 bytes per 16 steps: 3 % of what a pass
// over 16-bit rows moves), from which the backward computes h again: in float32
// and without reading h.
#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

constexpr int kSteps = PLATTICE_SCAN_KEEP;

struct ScanArgs {
    const void *x, *a;
    const float* state;
    void* h;
    float *last, *states;
    const void* g;
    const float* grad_last;
    void *gx, *ga;
    float* gs;
    int64_t lines, steps;
    int c, reverse;
};

// Where a thread's channels lie: element of step s of its line, and of a state.
struct At {
    int64_t first, stride;   // of the step taken first, to the next
    int64_t state;           // in [lines][c]
    __device__ __forceinline__ At(const ScanArgs& p, int64_t index, int units, int v) {
        const int64_t line = index / units, col = (index - line * units) * v;
        first = (line * p.steps + (p.reverse ? p.steps - 1 : 0)) * p.c + col;
        stride = p.reverse ? -(int64_t)p.c : p.c;
        state = line * p.c + col;
    }
};

template <typename T, int V, bool kBlend>
__global__ void __launch_bounds__(128) k_scan(ScanArgs p) {
    const int units = p.c / V;
    const int64_t index = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (index >= p.lines * units) return;
    const At at(p, index, units, V);
    const int64_t blocks = (p.steps + kSteps - 1) / kSteps, line = index / units;
    float h[V];
#pragma unroll
    for (int j = 0; j < V; ++j) h[j] = p.state ? p.state[at.state + j] : 0.f;
    for (int64_t b = 0; b < blocks; ++b) {
        const int64_t t0 = b * kSteps;
        const int n = p.steps - t0 < kSteps ? (int)(p.steps - t0) : kSteps;
        const int64_t o = at.first + t0 * at.stride;
        Vec<T, V> x[kSteps], a[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (i < n) {
                x[i].load(static_cast<const T*>(p.x) + o + i * at.stride);
                a[i].load(static_cast<const T*>(p.a) + o + i * at.stride);
            }
        if (p.states) {
            float* s = p.states + (line * blocks + b) * p.c + (at.state - line * p.c);
#pragma unroll
            for (int j = 0; j < V; ++j) s[j] = h[j];
        }
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (i < n) {
                Vec<T, V> y;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float g = a[i].at(j), u = kBlend ? (1.f - g) * x[i].at(j) : x[i].at(j);
                    h[j] = fmaf(g, h[j], u);
                    y.set(j, h[j]);
                }
                y.store(static_cast<T*>(p.h) + o + i * at.stride);
            }
    }
    if (p.last)
#pragma unroll
        for (int j = 0; j < V; ++j) p.last[at.state + j] = h[j];
}

template <typename T, int V, bool kBlend>
__global__ void __launch_bounds__(128) k_scan_grad(ScanArgs p) {
    const int units = p.c / V;
    const int64_t index = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (index >= p.lines * units) return;
    const At at(p, index, units, V);
    const int64_t blocks = (p.steps + kSteps - 1) / kSteps, line = index / units;
    float r[V];   // what reaches h from later steps
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = p.grad_last ? p.grad_last[at.state + j] : 0.f;
    for (int64_t b = blocks - 1; b >= 0; --b) {
        const int64_t t0 = b * kSteps;
        const int n = p.steps - t0 < kSteps ? (int)(p.steps - t0) : kSteps;
        const int64_t o = at.first + t0 * at.stride;
        Vec<T, V> x[kSteps], a[kSteps], g[kSteps];
        float h[V], d[kSteps][V];   // d: h[t-1], or h[t-1] - x[t]
        const float* s = p.states + (line * blocks + b) * p.c + (at.state - line * p.c);
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (i < n) {
                x[i].load(static_cast<const T*>(p.x) + o + i * at.stride);
                a[i].load(static_cast<const T*>(p.a) + o + i * at.stride);
                g[i].load(static_cast<const T*>(p.g) + o + i * at.stride);
            }
#pragma unroll
        for (int j = 0; j < V; ++j) h[j] = s[j];
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            if (i < n) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float ga = a[i].at(j), xv = x[i].at(j);
                    d[i][j] = kBlend ? h[j] - xv : h[j];
                    h[j] = fmaf(ga, h[j], kBlend ? (1.f - ga) * xv : xv);
                }
            }
#pragma unroll
        for (int i = kSteps - 1; i >= 0; --i)
            if (i < n) {
                Vec<T, V> gx, ga;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float gate = a[i].at(j), whole = g[i].at(j) + r[j];
                    gx.set(j, kBlend ? (1.f - gate) * whole : whole);
                    ga.set(j, whole * d[i][j]);
                    r[j] = gate * whole;
                }
                gx.store(static_cast<T*>(p.gx) + o + i * at.stride);
                ga.store(static_cast<T*>(p.ga) + o + i * at.stride);
            }
    }
    if (p.gs)
#pragma unroll
        for (int j = 0; j < V; ++j) p.gs[at.state + j] = r[j];
}

// ------------------------------------------------------------------ host side

template <typename T, int V, bool kBlend>
static cudaError_t launch(const ScanArgs& p, bool grad, cudaStream_t s) {
    const int64_t ctas = ceil_div(p.lines * (p.c / V), 128);
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    if (grad) k_scan_grad<T, V, kBlend><<<(unsigned)ctas, 128, 0, s>>>(p);
    else k_scan<T, V, kBlend><<<(unsigned)ctas, 128, 0, s>>>(p);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t launch(const ScanArgs& p, bool blend, bool grad, int v, cudaStream_t s) {
    constexpr int kPair = sizeof(T) == 2 ? 2 : 1;
    if (v >= kPair) return blend ? launch<T, kPair, true>(p, grad, s) : launch<T, kPair, false>(p, grad, s);
    return blend ? launch<T, 1, true>(p, grad, s) : launch<T, 1, false>(p, grad, s);
}

static int run(const plattice_scan_args* q, bool grad, cudaStream_t s, const char* call) {
    const ScanArgs p{q->x, q->gate, q->state, q->h, q->last, q->states, q->grad_h, q->grad_last, q->grad_x, q->grad_gate,
                     q->grad_state, q->lines, q->steps, q->c, q->reverse};
    uintptr_t bits = (uintptr_t)p.x | (uintptr_t)p.a;
    bits |= grad ? (uintptr_t)p.g | (uintptr_t)p.gx | (uintptr_t)p.ga : (uintptr_t)p.h;
    const int v = widest(p.c, dtype_size(q->dtype), bits);
    const cudaError_t e = q->dtype == PLATTICE_F32    ? launch<float>(p, q->blend, grad, v, s)
                          : q->dtype == PLATTICE_BF16 ? launch<__nv_bfloat16>(p, q->blend, grad, v, s)
                                                      : launch<__half>(p, q->blend, grad, v, s);
    return rows_status(e, call);
}

static bool shape_ok(const plattice_scan_args* q) {
    return q && dtype_ok(q->dtype) && q->lines >= 0 && q->steps >= 0 && q->c >= 1 && q->c <= (1 << 30) &&
           fits(q->lines, q->c) && fits(q->steps, q->c) && fits(q->lines, q->steps * q->c);
}

}  // namespace plr

using namespace plr;

extern "C" {

int plattice_scan_workspace_size(const plattice_scan_args* q, size_t* bytes) {
    if (!bytes || !shape_ok(q)) return PLATTICE_ERR_INVALID;
    *bytes = 0;
    return PLATTICE_OK;
}

int plattice_scan(const plattice_scan_args* q, void* stream) {
    if (!shape_ok(q)) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (q->lines == 0) return PLATTICE_OK;
    if (q->steps == 0) {   // the state as it came
        if (!q->last) return PLATTICE_OK;
        const size_t b = (size_t)q->lines * q->c * sizeof(float);
        return rows_status(q->state ? cudaMemcpyAsync(q->last, q->state, b, cudaMemcpyDeviceToDevice, s)
                                    : cudaMemsetAsync(q->last, 0, b, s),
                           "plattice_scan");
    }
    if (!q->x || !q->gate || !q->h) return PLATTICE_ERR_INVALID;
    return run(q, false, s, "plattice_scan");
}

int plattice_scan_backward_workspace_size(const plattice_scan_args* q, size_t* bytes) {
    return plattice_scan_workspace_size(q, bytes);
}

int plattice_scan_backward(const plattice_scan_args* q, void* stream) {
    if (!shape_ok(q)) return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (q->lines == 0) return PLATTICE_OK;
    if (q->steps == 0) {
        if (!q->grad_state) return PLATTICE_OK;
        const size_t b = (size_t)q->lines * q->c * sizeof(float);
        return rows_status(q->grad_last ? cudaMemcpyAsync(q->grad_state, q->grad_last, b, cudaMemcpyDeviceToDevice, s)
                                        : cudaMemsetAsync(q->grad_state, 0, b, s),
                           "plattice_scan_backward");
    }
    if (!q->x || !q->gate || !q->states || !q->grad_h || !q->grad_x || !q->grad_gate) return PLATTICE_ERR_INVALID;
    return run(q, true, s, "plattice_scan_backward");
}

}  // extern "C"
