// dimn_rowops.h -- what the row operators (dimn_rowops.hip: layer normalisation, linear softmax cross entropy) and the rest of libdimn share.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/dimn.h"

typedef unsigned short bf16_t;

#define DIMN_HIDDEN __attribute__((visibility("hidden")))

// sets the calling thread's error message (dimn_last_error) and returns `code`
DIMN_HIDDEN int dimn_fail(int code, const char* fmt, ...);

// One layer normalisation: planes of [groups][rows] rows of `width` elements (strides in elements), float32 parameters [groups][width].
struct NormP {
    const void* x; const void* dy;            // dy: backward only
    void* out;                                // y / dx
    int64_t x_group, x_row, dy_group, dy_row, out_group, out_row;
    const float* gamma; const float* beta;    // NULL: 1 / 0
    float* mean; float* rstd;                 // [groups][rows]: written forward, read backward
    const float* gate;                        // NULL, or a float32 plane laid out like `out` that multiplies the result (dropout, activation gates)
    float* part;                              // backward: [groups][parts][2][width] partial sums of dgamma, dbeta (NULL: neither is wanted)
    int64_t rows;
    int32_t width;
    float eps;
};
// Both on the current device; type: DIMN_TYPE_*.  The backward pass's workspace holds norm_workspace_floats() floats.
DIMN_HIDDEN int norm_forward(hipStream_t stream, int32_t type, int64_t groups, const NormP& p);
DIMN_HIDDEN int norm_backward(hipStream_t stream, int32_t type, int64_t groups, NormP p, float* dgamma, float* dbeta, float* workspace);
DIMN_HIDDEN int64_t norm_workspace_floats(int32_t type, int64_t groups, int64_t rows, int32_t width);
