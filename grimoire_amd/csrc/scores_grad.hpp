// scores_grad.hpp -- host interface of the router scores' gradient.
#pragma once

#include "common.hpp"

namespace grim {

struct ScoresGradArgs {
    const void* logits;       // [T] rows of row_stride elements, fp32 or bf16
    const int32_t* expert;    // [T][K] picks; outside [0, E): no pick
    const float* dw;          // [T][K] gradient of the picks' weights
    void* dlogits;            // [T] rows of d_stride elements, the logits' type
    int64_t row_stride, d_stride;
    int bf16;
    int T, E, K;
    int sigmoid, normalize;
    float scaling;
};

constexpr int kScoresGradMaxTokens = 1 << 24;   // a wavefront a token, 2^32 threads a launch

hipError_t scores_grad_launch(hipStream_t st, const ScoresGradArgs& a);

}  // namespace grim
