// Host functions shared by the expert products' translation units.
#pragma once

#include "common.cuh"

namespace lfb {

// out[r] = x[rows[r]] for R rows of `width` 16-bit values (a multiple of 8), zeros for an index
// outside [0, x_rows); strides in 16-bit values (grouped_gemm.cu).
int gather_rows(const void* x, int64_t x_stride, int64_t x_rows, const int32_t* rows, int64_t R, int64_t width,
                void* out, void* stream, const char* what);

// Expired bounded waits counted by the two units (synchronous).
int grouped_wait_timeouts(unsigned int* value, int reset);
int mx_wait_timeouts(unsigned int* value, int reset);

}  // namespace lfb
