// scores.hpp -- host interface of the router scores kernel.
#pragma once

#include "common.hpp"

namespace grim {

struct ScoresArgs {
    const void* logits;       // [T] rows of row_stride elements, fp32 or bf16
    int64_t row_stride;
    int bf16;
    int T, E, K;
    int sigmoid;              // 0: softmax over the E logits
    const float* bias;        // [E] added for the choice only, or null
    int n_group, topk_group;  // n_group 1: no group limit
    int top2;                 // group score: sum of its two best (else its best)
    int normalize;
    float scaling;
    int32_t* out_e;           // [T][K]
    float* out_w;
    // the split-K router's second partial sum (fp32 logits), laid out as the
    // logits: the row is logits + part1
    const float* part1 = nullptr;
};

constexpr int kScoresMaxE = 512, kScoresMaxK = 16, kScoresMaxGroups = 64;

hipError_t scores_launch(hipStream_t st, const ScoresArgs& a);

}  // namespace grim
