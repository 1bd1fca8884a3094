// rows_logp.cu -- log probabilities of given labels, entropy and the best
// alternatives of rows of scores, and the scores' gradient.
//
//   m = max x, s = log sum exp(x - m);  log p_j = (x_j - m) - s
//   entropy = -sum p log p = s - sum exp(x - m) (x - m) / sum exp(x - m)
//   grad_j = g_l ([j = label] - p_j) - g_e p_j (log p_j + entropy) + g_z p_j
//
// m and s are kept apart: their sum would lose s beside a large m (rows whose
// scores are all the type's lowest value, say).  The sum leaves the largest
// score's own 1 out, so that s = log1p(rest) and the log probability of a
// confident answer keep their precision.
#include "plattice_runtime.h"
#include "rows_host.h"
#include "rows_vec.cuh"

namespace plr {

struct LogpArgs {
    const void* x;
    Labels labels;         // p null: none
    float *logp, *entropy;
    float2* stats;
    float* lse;
    float* top_logp;
    long long* top_ids;
    const float *gl, *ge, *gz;
    void* gx;
    int64_t rows;
    int n, top;
};

// Scores in order as unsigned numbers (-0 as 0, NaN below all), the class behind
// them so that of equal scores the lowest class is the greatest.
__device__ __forceinline__ uint64_t ranked(float v, int j) {
    const unsigned b = __float_as_uint(v + 0.f);
    const unsigned u = v != v ? 0u : (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return (uint64_t)u << 32 | (unsigned)~j;
}
__device__ __forceinline__ int class_of(uint64_t key) { return (int)~(unsigned)key; }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, d));
    return v;
}
__device__ __forceinline__ uint64_t warp_best(uint64_t v) {
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const uint64_t o = __shfl_xor_sync(0xffffffffu, v, d);
        v = o > v ? o : v;
    }
    return v;
}

// A row by a CTA of 256.
template <typename T>
__global__ void __launch_bounds__(256) k_logp(LogpArgs p) {
    __shared__ float sa[8], sb[8];
    __shared__ int sc[8];
    __shared__ uint64_t best[8];
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.n;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float m = -INFINITY;
    for (int j = threadIdx.x; j < p.n; j += 256) m = max_nan(m, to_f32(x[j]));
    m = warp_max(m);
    if (lane == 0) sa[warp] = m;
    __syncthreads();
    m = sa[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) m = max_nan(m, sa[k]);
    __syncthreads();
    const bool empty = m == -INFINITY;
    float sum = 0.f, weighted = 0.f;   // of the scores below m (each score equal to m is a 1 more)
    int equal = 0;
    if (!empty)
        for (int j = threadIdx.x; j < p.n; j += 256) {
            const float d = to_f32(x[j]) - m;
            if (d == 0.f) {
                ++equal;
            } else {
                const float e = expf(d);
                sum += e;
                if (e != 0.f) weighted += e * d;
            }
        }
    sum = warp_sum(sum);
    weighted = warp_sum(weighted);
    equal = (int)__reduce_add_sync(0xffffffffu, (unsigned)equal);
    if (lane == 0) {
        sa[warp] = sum;
        sb[warp] = weighted;
        sc[warp] = equal;
    }
    __syncthreads();
    sum = weighted = 0.f;
    equal = -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        sum += sa[k];
        weighted += sb[k];
        equal += sc[k];
    }
    sum += (float)equal;   // beside the 1 of one largest score
    const float s = empty ? 0.f : log1pf(sum);
    if (threadIdx.x == 0) {
        p.stats[row] = make_float2(m, s);
        if (p.lse) p.lse[row] = m + s;
        if (p.entropy) p.entropy[row] = empty ? 0.f : s - weighted / (1.f + sum);
        if (p.logp) {
            const int l = p.labels.at(row, p.n);
            p.logp[row] = l < 0 ? 0.f : empty ? -INFINITY : to_f32(x[l]) - m - s;
        }
    }
    uint64_t before = ~0ull;
    for (int k = 0; k < p.top; ++k) {
        uint64_t b = 0;
        for (int j = threadIdx.x; j < p.n; j += 256) {
            const uint64_t r = ranked(to_f32(x[j]), j);
            if (r < before && r > b) b = r;
        }
        b = warp_best(b);
        __syncthreads();
        if (lane == 0) best[warp] = b;
        __syncthreads();
        b = best[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) b = best[i] > b ? best[i] : b;
        before = b;
        if (threadIdx.x == 0) {
            const int j = class_of(b);
            p.top_ids[row * p.top + k] = j;
            p.top_logp[row * p.top + k] = empty ? -INFINITY : to_f32(x[j]) - m - s;
        }
    }
    __syncthreads();
    }
}

template <typename T>
__global__ void __launch_bounds__(256) k_logp_grad(LogpArgs p) {
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.n;
    T* gx = static_cast<T*>(p.gx) + row * p.n;
    const float2 st = p.stats[row];
    const int l = p.gl ? p.labels.at(row, p.n) : -1;
    const float gl = l >= 0 ? p.gl[row] : 0.f, ge = p.ge ? p.ge[row] : 0.f, gz = p.gz ? p.gz[row] : 0.f;
    const float entropy = p.ge ? p.entropy[row] : 0.f;
    for (int j = threadIdx.x; j < p.n; j += 256) {
        float v = 0.f;
        if (st.x != -INFINITY) {
            const float lp = to_f32(x[j]) - st.x - st.y, q = expf(lp);
            const float own = j == l ? -gl * expm1f(lp) : -gl * q;   // 1 - p of the label itself
            v = own + gz * q;
            if (q != 0.f) v -= ge * q * (lp + entropy);
        }
        gx[j] = from_f32<T>(v);
    }
    }
}

}  // namespace plr

using namespace plr;

extern "C" {

static bool logp_ok(const plattice_log_probs_args* q) {
    return q && dtype_ok(q->dtype) && q->rows >= 0 && q->n >= 1 && q->n <= (1 << 30) && q->top >= 0 &&
           q->top <= PLATTICE_MAX_TOP && q->top <= q->n && fits(q->rows, q->n) &&
           (!q->labels || (uintptr_t)q->labels % (q->labels_wide ? 8 : 4) == 0);
}

static LogpArgs logp_args(const plattice_log_probs_args* q) {
    return {q->logits, {q->labels, q->labels_wide}, q->logp, q->entropy, reinterpret_cast<float2*>(q->stats), q->lse, q->top_logp,
            q->top_ids, q->grad_logp, q->grad_entropy, q->grad_lse, q->grad_logits, q->rows, q->n, q->top};
}

int plattice_log_probs(const plattice_log_probs_args* q, void* stream) {
    if (!logp_ok(q)) return PLATTICE_ERR_INVALID;
    if (q->rows == 0) return PLATTICE_OK;
    if (!q->logits || !q->stats || (uintptr_t)q->stats % 8 || (q->logp && !q->labels) ||
        (q->top && (!q->top_logp || !q->top_ids)))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const LogpArgs a = logp_args(q);
    if (q->dtype == PLATTICE_F32) k_logp<float><<<(unsigned)(q->rows < (1 << 20) ? q->rows : 1 << 20), 256, 0, s>>>(a);
    else if (q->dtype == PLATTICE_BF16) k_logp<__nv_bfloat16><<<(unsigned)(q->rows < (1 << 20) ? q->rows : 1 << 20), 256, 0, s>>>(a);
    else k_logp<__half><<<(unsigned)(q->rows < (1 << 20) ? q->rows : 1 << 20), 256, 0, s>>>(a);
    return rows_status(cudaGetLastError(), "plattice_log_probs");
}

int plattice_log_probs_backward(const plattice_log_probs_args* q, void* stream) {
    if (!logp_ok(q)) return PLATTICE_ERR_INVALID;
    if (q->rows == 0) return PLATTICE_OK;
    if (!q->logits || !q->stats || (uintptr_t)q->stats % 8 || !q->grad_logits || (q->grad_logp && !q->labels) ||
        (q->grad_entropy && !q->entropy))
        return PLATTICE_ERR_INVALID;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const LogpArgs a = logp_args(q);
    if (q->dtype == PLATTICE_F32) k_logp_grad<float><<<(unsigned)(q->rows < (1 << 20) ? q->rows : 1 << 20), 256, 0, s>>>(a);
    else if (q->dtype == PLATTICE_BF16) k_logp_grad<__nv_bfloat16><<<(unsigned)(q->rows < (1 << 20) ? q->rows : 1 << 20), 256, 0, s>>>(a);
    else k_logp_grad<__half><<<(unsigned)(q->rows < (1 << 20) ? q->rows : 1 << 20), 256, 0, s>>>(a);
    return rows_status(cudaGetLastError(), "plattice_log_probs_backward");
}

}  // extern "C"
