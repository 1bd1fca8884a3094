// rows_logp.h -- arguments of the log probabilities' kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/plattice.h"

namespace plr {

struct LogpArgs {
    const void* x;
    const void* labels;    // null: none
    int labels_wide;
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

template <typename T> cudaError_t logp_forward(const LogpArgs& a, cudaStream_t s);
template <typename T> cudaError_t logp_backward(const LogpArgs& a, cudaStream_t s);

}  // namespace plr
