// proj4_out.hpp -- the last step of a dense 4-bit projection.
#pragma once

#include "proj4.hpp"

namespace grim {

// An output o (of a gate and up) on its way to y.
__device__ __forceinline__ void proj4_out(const Proj4Args& a, int64_t row, int n, float o, float up) {
    if (a.glu) o = silu(o) * up;
    if (a.base) {
        const int64_t at = row * a.base_stride + n;
        o += a.base_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.base)[at]) : static_cast<const float*>(a.base)[at];
    }
    const int64_t at = row * a.y_stride + n;
    if (a.y_bf16) static_cast<uint16_t*>(a.y)[at] = f32_to_bf16(o);
    else static_cast<float*>(a.y)[at] = o;
}

}  // namespace grim
