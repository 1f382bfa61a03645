// scores_grad.hip -- the gradient of the router scores' weights to the logits,
// one wavefront a token.  With s the scores, u_k = s of pick k, g its weight's
// gradient times the scaling:
//   kept as they are:  du_k = g_k
//   renormalised:      du_k = (g_k - sum_j p_j g_j) / Z,  p = u / Z, Z = sum u
//   softmax:  dl_e = s_e ([e picked] du_e - sum_k u_k du_k);  renormalised the
//             sum is 0 and dl_k = p_k (g_k - sum_j p_j g_j), p the softmax of
//             the picks alone: the other logits are not read
//   sigmoid:  dl_e = s_e (1 - s_e) [e picked] du_e;  renormalised
//             dl_k = p_k (1 - s_k) (g_k - sum_j p_j g_j), p by the differences of
//             the scores' exponents: Z, which may be any small number, is not
//             divided by (scores of logits below -84 have a 1 / Z near fp32's largest)
// The choice, and with it a selection bias and groups, has no gradient.  An
// expert picked twice gets the sum, picks in order.  An expert that is out
// (logit NaN or -inf) has score and gradient 0; +inf counts as the largest
// finite logit, as in the scores.  All is fp32; an exponential is off by 2 ulp.
//
// Bound by latency (4096 x 128 fp32, softmax kept, 4.5 MB, 0.9 us at a large copy's
// 5.1 TB/s: 4.1 in a graph, 6.2 a call, the host's; 64 x 256 sigmoid 3.0 in a graph,
// 4096 x 512 softmax kept, 17 MB, 6 to 8; one token 2.4).  A wave holds a token's logits in
// registers, 1 to 8 a lane as E needs, so that each is read once and every sum
// is one of lanes; the picks lie one a lane.  Renormalised softmax reads the
// picks' logits alone.  The picks' values go to their experts' places through a
// row of the LDS, which no other wave reads: no barrier of the work-group.
#include "scores_grad.hpp"

#include "scores.hpp"
#include "topk.hpp"

namespace grim {

namespace {

constexpr int kWaves = 4;     // tokens a work-group

template <bool BF16>
__device__ __forceinline__ float logit(const void* p, int64_t at) {
    float v;
    if constexpr (BF16) v = bf16_to_f32(static_cast<const uint16_t*>(p)[at]);
    else v = static_cast<const float*>(p)[at];
    return fminf(fmaxf(v, -__builtin_inff()), 3.402823466e+38f);       // fmaxf drops a NaN
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, kWave));
    return v;
}

// The largest of a row of 16 lanes, on each of them.
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, dpp_f<kDppXor1>(v));
    v = fmaxf(v, dpp_f<kDppXor2>(v));
    v = fmaxf(v, dpp_f<kDppHalfMirror>(v));
    return fmaxf(v, dpp_f<kDppMirror>(v));
}
static_assert(kScoresMaxK == 16, "a token's picks are one row");

// Where every pick's logit is at or below this, their sigmoids are 0 in the 64 bits
// of the forward pass (e^709.783 > 2^1024), whose weights are 0 then.
constexpr float kNoScores = -709.7827f;

// exp(x), x <= 0: 2^(hi + lo) of x log2(e) in two parts, 1 - 2 ulp
__device__ __forceinline__ float exp_neg(float x) {
    const float L = 1.44269504088896341f, Ll = 1.92596299112661746887e-8f;   // log2(e) = L + Ll
    const float h = x * L, l = __builtin_fmaf(x, Ll, __builtin_fmaf(x, L, -h));
    const float e = __builtin_amdgcn_exp2f(h);
    return x > -87.0f ? __builtin_fmaf(e, l * 0.693147180559945f, e) : e;
}

template <bool BF16, int NV>     // NV: logits a lane
__global__ __launch_bounds__(kWaves * kWave) void scores_grad_kernel(ScoresGradArgs a) {
    __shared__ float row[kWaves][kScoresMaxE];       // du (softmax kept as it is) or dl of the picks
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t t = int64_t(blockIdx.x) * kWaves + wave;
    if (t >= a.T) return;
    const int E = a.E;
    const float ninf = -__builtin_inff();
    const bool full = !a.sigmoid && !a.normalize;    // the softmax over all experts counts
    float* mine = row[wave];
    float lv[NV];
    if (full)                                        // on their way while the picks are read
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int e = j * kWave + lane;
            lv[j] = logit<BF16>(a.logits, t * a.row_stride + (e < E ? e : E - 1));
        }
#pragma unroll
    for (int j = 0; j < NV; ++j) mine[j * kWave + lane] = 0.0f;

    // pick k on lane k
    int id = lane < a.K ? a.expert[t * a.K + lane] : -1;
    id = id >= 0 && id < E ? id : -1;
    const float pl = id >= 0 ? logit<BF16>(a.logits, t * a.row_stride + id) : ninf;
    const float g = id >= 0 ? a.dw[t * a.K + lane] * a.scaling : 0.0f;

    float m = 0.0f, iz = 0.0f, u, sum = 0.0f, d;
    if (full) {
        float top = ninf;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            lv[j] = j * kWave + lane < E ? lv[j] : ninf;
            top = fmaxf(top, lv[j]);
        }
        top = wave_max(top);
        m = top > ninf ? top : 0.0f;
        float z = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            lv[j] = exp_neg(lv[j] - m);
            z += lv[j];
        }
        z = group_sum<kWave>(z);
        iz = z > 0.0f ? 1.0f / z : 0.0f;
        u = id >= 0 ? exp_neg(pl - m) * iz : 0.0f;
        sum = group_sum<kWave>(u * g);
        d = g;
    } else if (!a.sigmoid) {
        const float top = wave_max(pl);
        const float e = id >= 0 && top > ninf ? exp_neg(pl - top) : 0.0f;
        const float z = group_sum<kWave>(e);
        const float p = z > 0.0f ? e / z : 0.0f;
        d = p * (g - group_sum<kWave>(p * g));
    } else {
        // s = e^min(l, 0) / (1 + e^-|l|), 1 - s = e^min(-l, 0) / (1 + e^-|l|)
        const float e = exp_neg(-__builtin_fabsf(pl)), q = 1.0f / (1.0f + e);
        if (a.normalize) {
            // the picks lie in the first 16 lanes: nothing comes from the others
            const float low = fminf(pl, 0.0f), top = row_max(low);
            u = id >= 0 && top > kNoScores ? exp_neg(low - top) * q : 0.0f;
            const float z = group_sum<kScoresMaxK>(u);
            const float p = z > 0.0f ? u / z : 0.0f;
            d = p * (pl >= 0.0f ? e * q : q) * (g - group_sum<kScoresMaxK>(p * g));
        } else {
            d = e * q * q * g;
        }
    }
    // an expert's picks summed by the first of them
    float tot = 0.0f;
    bool first = id >= 0;
    for (int k = 0; k < a.K; ++k) {
        const int o = __builtin_amdgcn_readlane(id, k);
        const float v = lane_f(d, k);
        if (o == id) {
            tot += v;
            first = first && k >= lane;
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (first) mine[id] = tot;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int e = j * kWave + lane;
        if (e >= E) continue;
        float v = mine[e];
        if (full) v = lv[j] * iz * (v - sum);
        if constexpr (BF16) static_cast<uint16_t*>(a.dlogits)[t * a.d_stride + e] = f32_to_bf16(v);
        else static_cast<float*>(a.dlogits)[t * a.d_stride + e] = v;
    }
}

template <bool BF16>
void launch_nv(hipStream_t st, const ScoresGradArgs& a) {
    const dim3 grid((a.T + kWaves - 1) / kWaves), block(kWaves * kWave);
#define GRIM_SG(NV) hipLaunchKernelGGL((scores_grad_kernel<BF16, NV>), grid, block, 0, st, a)
    if (a.E <= 64) GRIM_SG(1);
    else if (a.E <= 128) GRIM_SG(2);
    else if (a.E <= 256) GRIM_SG(4);
    else GRIM_SG(8);
#undef GRIM_SG
}

}  // namespace

hipError_t scores_grad_launch(hipStream_t st, const ScoresGradArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.E <= 0 || a.E > kScoresMaxE || a.K <= 0 || a.K > kScoresMaxK) return hipErrorInvalidValue;
    if (a.bf16) launch_nv<true>(st, a);
    else launch_nv<false>(st, a);
    return hipGetLastError();
}

}  // namespace grim
