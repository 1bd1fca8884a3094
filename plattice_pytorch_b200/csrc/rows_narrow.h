// rows_narrow.h -- arguments and launches of the linear map where one side is
// small (rows_narrow.cuh).
#pragma once
#include "rows_host.h"

namespace plr {

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
    int out_dtype, bias_dtype;
    bool vec_x;    // 16-byte accesses to x's rows
    bool vec_w;    // the same for w's
    bool vec_y;    // the outputs and the residual begin on 16-byte boundaries
};

struct SmallGradArgs {
    SmallArgs s;          // x, x_scale, w, z, z_scale, rows, k, n, split, act, types, alignments
    const void* g0;
    const void* g1;
    void* grad_x;
    float* partial;       // [gridDim.x][n k + n]: grad_w [n][k], then grad_bias [n]
    bool need_x, need_w, need_b;
    bool vec_gx;          // 16-byte accesses to grad_x's rows
    bool vec_g;           // g0 and g1 begin on 16-byte boundaries
};

__host__ __device__ inline int narrow_steps(int k) { return (k + 63) / 64 * 4; }   // of 16 channels
__host__ inline int64_t narrow_fragments(int k, int nf, int parts) { return (int64_t)parts * narrow_steps(k) * nf * 256; }
// Bytes of weights that k_narrow takes: what fits beside its staging (even one
// CTA an SM beats the tiles, which write float32's parts first: 65536 rows,
// 1024 -> 24, float32: 94 against 206 us).
constexpr int64_t kNarrowMost = 190 * 1024;
constexpr int kGradWarps = 4;
constexpr int kNarrowGradMost = 65535 * 64;      // input channels of the narrow backward: slices are gridDim.y
// CTAs of the narrow backward that share an SM
__host__ __device__ constexpr int narrow_grad_ctas(int parts, int nf) { return parts == 3 ? 2 : nf > 2 ? 3 : 4; }

// Few blocks of rows and many channels: the warps of a CTA of k_narrow then share
// a block (float32 weights; the tiles take the others).  us, n 24, 4700 rows,
// float32, shared / a block a warp: k 128 6.8 / 6.2, k 256 8.9 / 9.5, k 768 15.4 /
// 21.6.
inline bool narrow_shares(int64_t blocks, int k) { return blocks * 256 <= (int64_t)sm_count() * k; }

cudaError_t run_narrow(const SmallArgs& a, int dtype, cudaStream_t s);
cudaError_t run_few_rows(const SmallArgs& a, int dtype, cudaStream_t s);
// parts: of the weights (NarrowGradShape).
cudaError_t run_narrow_grad(const SmallGradArgs& a, int dtype, int parts, int lines, cudaStream_t s);

}  // namespace plr
