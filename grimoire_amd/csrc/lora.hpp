// lora.hpp -- host interface of the low-rank adapter kernels.
#pragma once

#include "common.hpp"
#include "lora_layout.hpp"

namespace grim {

// y_t = base_t + scale_a B_a (A_a x_t), a = row_slot[t]; with glu, N = 2I and
// y_t [I] = silu(v[i]) * v[I + i] of v = that sum.
struct LoraArgs {
    const uint16_t* a;        // bf16 [slots][R][K]
    const uint16_t* b;        // bf16 [slots][N][R]
    const int32_t* rank;      // [slots]
    const float* scale;       // [slots]
    int slots, R, K, N;
    const int32_t* row_slot;  // [T], outside [0, slots) = no adapter
    const void* x;            // [T] rows, x_stride elements apart
    const void* base;
    void* y;
    int64_t x_stride, base_stride, y_stride;
    int x_bf16, base_bf16, y_bf16;
    int T, glu;
    float* part;              // workspace: partials of A x by K split
};

constexpr int kLoraMaxRank = 256;
constexpr int64_t kLoraMaxStride = int64_t(1) << 24;

hipError_t lora_launch(hipStream_t st, const LoraArgs& a);

}  // namespace grim
