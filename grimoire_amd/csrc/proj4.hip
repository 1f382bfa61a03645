// proj4.hip -- a dense projection with 4-bit weights for a few rows:
//   y_t[n] = base_t[n] + sum_g s[n,g] sum_{k in g} (q[n,k] - z[n,g]) x_t[k]
// (MXFP4: sum_g 2^(e[n,g] - 127) sum_k e2m1[n,k] x_t[k]), optionally with the
// SwiGLU of a gate|up projection.
//
// The weights are read once, 4.06 (groups of 256) to 4.75 bits an element (of 32,
// with zeros), and bound a few rows: 7168 x 32768 is 123 MB, 24 us at a copy's
// 5.1 TB/s.  Products go to the matrix cores with x as rows and
// the decoded weights as columns: x's 16 rows (bf16) cost what one does.  fp32 x
// is cut into three bf16 pieces whose sum it is, so every product is exact and
// 4 rows take the tile's 16.  INT4: the code's bf16 is 16 + q, two
// operations for two codes (bf16's 8 bits hold 16 + q exactly), and the 16 and
// the zero point come off a group's sum with the sum of x, which a product
// with ones gives; the scale is applied to that sum in fp32.  MXFP4: the
// conversion instruction gives w s in bf16, exact.  Sums are fp32.
//
// What bounds it now: one row of 7168 x 32768 INT4, weights in no cache, 29 us,
// 4.2 TB/s, 83 % of a copy's rate; its loads alone take as long, the decoding alone
// (51 to 84 vector operations for 1 KiB of codes and 64 lanes) three quarters,
// x and the launch 4 of either.  Small ones are chains: 768 x 2048 5 us, 2880 x 5760
// with SwiGLU for 8 rows 7 (fetch x, LDS, the first weights, the sum over the
// waves).  32 rows of 7168 x 4096 with SwiGLU 14 us: 58 KB of x a part of K in each
// work-group, and the second launch that sums (of bf16 x; of fp32, 8 rows a
// work-group, 26).
#include "proj4_out.hpp"

namespace grim {

// The sums over the parts of K, in order, and the last step.
__global__ __launch_bounds__(256) void proj4_sum_kernel(Proj4Dev p) {
    const Proj4Args& a = p.a;
    const int PT = a.glu ? 8 : 16;
    const int64_t u = int64_t(blockIdx.x) * 256 + threadIdx.x, per = int64_t(p.tiles) * PT;
    if (u >= per * a.T) return;
    const int64_t t = u / per;
    const int n = int(u - t * per);
    if (n >= p.half) return;
    const float* at = p.part + (t * p.tiles + n / PT) * 16 + n % PT;
    const int64_t step = int64_t(a.T) * p.tiles * 16;
    const int gu = a.glu ? 8 : 0;
    float o = 0.0f, up = 0.0f;
    float e[kProj4Parts], f[kProj4Parts];              // all asked for together (a missing one is not used)
#pragma unroll
    for (int k = 0; k < kProj4Parts; ++k) {
        const float* from = at + (k < p.kw ? k : 0) * step;
        e[k] = from[0];
        f[k] = from[gu];
    }
#pragma unroll
    for (int k = 0; k < kProj4Parts; ++k) {
        o += k < p.kw ? e[k] : 0.0f;
        up += k < p.kw ? f[k] : 0.0f;
    }
    proj4_out(a, t, n, o, up);
}

hipError_t proj4_sum_launch(hipStream_t st, const Proj4Dev& p) {
    const int64_t n = int64_t(p.tiles) * (p.a.glu ? 8 : 16) * p.a.T;
    hipLaunchKernelGGL(proj4_sum_kernel, dim3(unsigned((n + 255) / 256)), dim3(256), 0, st, p);
    return hipGetLastError();
}

hipError_t proj4_launch(hipStream_t st, const Proj4Args& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.fmt == GRIM_FMT_MXFP4) return proj4_launch_g0(st, a);
    switch (a.w.gshift) {
        case 5: return proj4_launch_g32(st, a);
        case 6: return proj4_launch_g64(st, a);
        case 7:
        case 8: return proj4_launch_g128(st, a);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace grim
