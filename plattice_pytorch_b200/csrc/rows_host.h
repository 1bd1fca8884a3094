// rows_host.h -- host-side helpers of the row operators.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <cuda.h>

#include "../../include/plattice.h"

namespace plr {

// ------------------------------------------------- products on the tensor cores
// (rows_mma.cuh has the kernel and what the kinds and their operands are)

enum Kind { kForward = 0, kGradX = 1, kGradW = 2 };

constexpr int kBM = 128, kBK = 64;   // rows of a tile, depth of a slice of the sum

// A 16-bit operand [parts][rows][pitch] of `width` columns.
struct Operand {
    const void* p = nullptr;
    int64_t rows = 0, width = 0, pitch = 0;
    int parts = 1;
};

struct MmaArgs {
    // result
    void* y0;
    void* y1;             // split: columns split.. of D
    const void* bias;     // null: none
    const void* residual;
    void* z;              // kept pre-activation (null: none)
    uint8_t* z_scale;
    int64_t ni, nj;       // D is ni x nj
    int bias_dtype, out_dtype, act, split;
    // sum
    int steps;            // 64-deep slices of r
    int part_steps;       // of a part (kGradW); parts are numbered tile-slowest
    int parts;
    unsigned pairs_a, pairs_b;   // parts of A and B of each product, 2 bits each
    int pairs;
    bool half;            // operands are float16 (else bfloat16)
    bool precise;         // the result ends in float32 (not in 16 bits after a float32 sum of parts)
    long long patience;   // cycles that a wait may take
    unsigned* fault;      // host-mapped word that reports a wait that gave up (may be null)
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t mma_tiles(int64_t ni, int64_t nj, int bn) { return ceil_div(ni, kBM) * ceil_div(nj, bn); }

// The deepest sum that an accumulator takes for a 16-bit result.  The MMA cuts
// where an addition rounds: sums of like terms drift by up to 2^-23 with each 16
// (float16, whose products have 22 bits, 1.0e-4 at a depth of 16384 and 8.7e-4 at a
// million; bfloat16's of 16 bits drift from some thousand on).  Held to a quarter of
// half a step of the type.
inline int64_t deepest_sum(int dtype) { return dtype == PLATTICE_F16 ? 16384 : 131072; }

// Whether a sum of `steps` slices goes in chunks (rows_mma.cuh, kChunk).
inline bool chunked(int steps, int out_dtype, bool precise) {
    return precise && (out_dtype == PLATTICE_F32 ? steps > 8 : (int64_t)steps * kBK > deepest_sum(out_dtype));
}

// TMA map of an operand: boxes of 64 columns x box_rows rows, zeros outside.
cudaError_t make_map(CUtensorMap* m, const Operand& o, int box_rows);

// Products with tiles of bn columns (256, 128, 64; the forward also 32).
// aligned: rows of the result (the forward: of y0, residual and z) allow
// 16-byte accesses.
cudaError_t mma_forward(int bn, bool aligned, const Operand& x, const Operand& w, const MmaArgs& p, cudaStream_t s);
cudaError_t mma_grad_x(int bn, bool aligned, const Operand& gz, const Operand& w, const MmaArgs& p, cudaStream_t s);
cudaError_t mma_grad_w(int bn, const Operand& x, const Operand& gz, const MmaArgs& p, cudaStream_t s);

// Status code of a CUDA result; an error is noted for
// plattice_last_error_detail under the call's name.
int rows_status(cudaError_t e, const char* call);

// PLATTICE_ERR_DEVICE when an earlier call's kernels reported a failure, else
// PLATTICE_OK (plattice_poll_status's check).
int rows_poll(const char* call);

// SMs of the current device (148 when it cannot be asked).
int sm_count();

constexpr int kMaxSmem = 232448;   // shared memory a CTA can have

inline bool dtype_ok(int d) { return d == PLATTICE_F32 || d == PLATTICE_BF16 || d == PLATTICE_F16; }
inline size_t dtype_size(int d) { return d == PLATTICE_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Element counts stay below 2^40, far from overflowing the 64-bit offsets.
inline bool fits(long long rows, long long width) { return rows <= ((1ll << 40) / (width > 0 ? width : 1)); }

// out[col] = sum of partial[part][col] over the parts, in a fixed order.
cudaError_t column_sums(void* out, int dtype, const float* partial, int parts, int64_t c, cudaStream_t s);

// Values of 8-bit rows as rows of `pitch` elements.
cudaError_t unpack_rows(void* y, int dtype, int64_t pitch, const uint8_t* q, const uint8_t* scale, int64_t rows,
                        int c, cudaStream_t s);

}  // namespace plr
