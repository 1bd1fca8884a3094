// rows_host.h -- host-side helpers of the row operators.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/plattice.h"

namespace plr {

// Status code of a CUDA result; an error is noted for
// plattice_last_error_detail under the call's name.
int rows_status(cudaError_t e, const char* call);

// PLATTICE_ERR_DEVICE when an earlier call's kernels reported a failure, else
// PLATTICE_OK (plattice_poll_status's check).
int rows_poll(const char* call);

// SMs of the current device (148 when it cannot be asked).
int sm_count();

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
