// block_norm.hpp -- host interface of the norms around a block.
#pragma once

#include "common.hpp"

namespace grim {

// h_out = rs * h + bs * gate * norm_post(f); out = norm_pre(h_out), where f
// is a dense row x[t] or, with routed, the combine of the token's experts.
struct BlockNormArgs {
    const float* h;           // [T][H]
    const void* x;            // dense: [T] rows of x_stride elements, fp32 or bf16
    int64_t x_stride;
    int x_bf16;
    const uint16_t* routed;   // bf16 [R][H] expert outputs, dispatch order (K > 0)
    const int32_t* inverse;   // [T*K], outside [0, routed_rows) = no row here
    const float* rw;          // [T*K]
    const float* shared;      // [T][H] or null
    const uint16_t* post_w;   // [H] bf16 or null: f is not normed
    const uint16_t* pre_w;    // [H] bf16 (null only without out / out_bf)
    float offset;             // added to every norm weight
    float eps;
    float rs, bs;             // residual and block scale
    const void* gate;         // by gate_kind, fp32 or bf16
    int gate_kind;            // enum grim_gate_kind
    int gate_bf16, gate_sigmoid;
    float* h_out;             // [T][H] or null; may be h
    float* out;               // [T][H] or null
    uint16_t* out_bf;         // [T][H] or null
    int T, H, K;
    int routed_rows;
};

constexpr int kBlockNormMaxHidden = 32768;   // 1024 threads of 8 four-column chunks

hipError_t block_norm_launch(hipStream_t st, const BlockNormArgs& a);

}  // namespace grim
