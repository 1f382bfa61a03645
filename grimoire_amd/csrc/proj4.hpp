// proj4.hpp -- host interface of the dense 4-bit projections.
#pragma once

#include "common.hpp"

namespace grim {

// y_t = base_t + W x_t, W [N][K] INT4, INT4_F16 or MXFP4; with glu, N = 2I
// and y_t [I] = silu(v[i]) * v[I + i] of v = W x_t.
struct Proj4Args {
    WView w;
    int fmt, N, K;
    const void* x;            // [T] rows, x_stride elements apart
    const void* base;         // or null
    void* y;
    int64_t x_stride, base_stride, y_stride;
    int x_bf16, base_bf16, y_bf16;
    int T, glu;
};

hipError_t proj4_launch(hipStream_t st, const Proj4Args& a);

}  // namespace grim
