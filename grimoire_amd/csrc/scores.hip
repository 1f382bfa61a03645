// scores.hip -- router scores to experts, one wavefront a token:
//   s = softmax_E(l) or 1 / (1 + exp(-l)); s' = s + bias
//   groups: score = the best s' (or the sum of the two best) of the group,
//   the topk_group best groups stay (lower index first among equals)
//   picks: the K largest s' (lower index first among equals)
//   w = s of the picks (/ their sum) * scaling
// An expert whose logit is NaN or -inf, or whose s' is NaN or -inf, is out;
// slots nothing is left for get expert -1 and weight 0.
//
// The scores are formed in fp64.  A choice is a border: in fp32 two scores
// closer than their rounding (an exp and a sum over E) swap places with the
// order of the sum, about once in 10^5 picks at E = 512; in fp64 the choice
// is that of the exact scores.  It costs E exps of the fp64 pipe a token.
//
// Lanes: each group owns lpg = 2^floor(log2(64 / n_group)) lanes of V =
// ceil(group / lpg) <= 16 consecutive experts, so a group's reductions are
// butterflies inside its lanes and the lowest lane (then its lowest slot)
// holding a value is the lowest expert.
#include "scores.hpp"
#include "topk.hpp"

namespace grim {

namespace {

constexpr int kScWaves = 4;   // tokens a work-group

__device__ __forceinline__ double shfl_xor_d(double v, int o) {
    const int lo = __shfl_xor(__double2loint(v), o, kWave);
    const int hi = __shfl_xor(__double2hiint(v), o, kWave);
    return __hiloint2double(hi, lo);
}

__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) v += shfl_xor_d(v, o);
    return v;
}

// The order of doubles as that of their bits: key(a) < key(b) iff a < b.
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));   // -0 -> +0
    return (u >> 63) ? ~u : (u | (uint64_t(1) << 63));
}

constexpr double kOut = -__builtin_huge_val();   // an expert that cannot be picked

template <int NV, bool BF16>
__global__ __launch_bounds__(kScWaves * kWave) void scores_kernel(ScoresArgs a, int lpg, int V) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t t = int64_t(blockIdx.x) * kScWaves + threadIdx.x / kWave;
    if (t >= a.T) return;
    const int E = a.E, gsz = E / a.n_group;
    const int gi = lane / lpg, sub = lane - gi * lpg;
    const int e0 = gi * gsz + sub * V;
    int nv = gi < a.n_group ? min(V, gsz - sub * V) : 0;   // experts of this lane (may be <= 0)

    auto logit = [&](int e) {
        if constexpr (BF16) {
            return bf16_to_f32(static_cast<const uint16_t*>(a.logits)[t * a.row_stride + e]);
        } else {
            const int64_t o = t * a.row_stride + e;
            float l = static_cast<const float*>(a.logits)[o];
            if (a.part1) l = (l + a.part1[o]) + (a.lbias ? a.lbias[e] : 0.0f);
            return l;
        }
    };
    // an expert that is out: -inf; +inf is the largest finite logit
    auto clean = [](float l) { return l == l ? fminf(l, 3.402823466e+38f) : -__builtin_inff(); };

    float lv[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) lv[j] = j < nv ? clean(logit(e0 + j)) : -__builtin_inff();

    double m = 0.0, iz = 1.0;   // softmax: the largest logit, 1 / sum exp(l - m)
    double v[NV];
    if (!a.sigmoid) {
        float lm = lv[0];
#pragma unroll
        for (int j = 1; j < NV; ++j) lm = fmaxf(lm, lv[j]);
        m = double(bits_f(0));
        const uint32_t k = wave_max_u32(score_key(lm));
        lm = (k & 0x80000000u) ? bits_f(k & 0x7FFFFFFFu) : bits_f(~k);
        m = lm > -__builtin_inff() ? double(lm) : 0.0;
        double z = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] = j < V ? exp(double(lv[j]) - m) : 0.0;
            z += v[j];
        }
        z = wave_sum_d(z);
        iz = z > 0.0 ? 1.0 / z : 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] *= iz;
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = j < V ? 1.0 / (1.0 + exp(-double(lv[j]))) : 0.0;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if (a.bias && j < nv) v[j] += double(a.bias[e0 + j]);
        if (!(lv[j] > -__builtin_inff()) || v[j] != v[j]) v[j] = kOut;
    }

    if (a.n_group > 1) {
        double b1 = kOut, b2 = kOut;   // the two best of the lane, then of its group
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            b2 = fmax(b2, fmin(b1, v[j]));
            b1 = fmax(b1, v[j]);
        }
        for (int o = 1; o < lpg; o <<= 1) {
            const double c1 = shfl_xor_d(b1, o), c2 = shfl_xor_d(b2, o);
            b2 = fmax(fmin(b1, c1), fmax(b2, c2));
            b1 = fmax(b1, c1);
        }
        const double gs = a.top2 && b2 > kOut ? b1 + b2 : b1;
        int rank = 0;
        for (int g = 0; g < a.n_group; ++g) {
            const double o = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(gs), g * lpg),
                                              __builtin_amdgcn_readlane(__double2loint(gs), g * lpg));
            rank += (o > gs || (o == gs && g < gi)) ? 1 : 0;
        }
        if (rank >= a.topk_group) {
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = kOut;
        }
    }

    int my = -1;
    for (int s = 0; s < a.K; ++s) {
        double best = v[0];
#pragma unroll
        for (int j = 1; j < NV; ++j) best = fmax(best, v[j]);
        const uint64_t key = order_key(best);
        const uint32_t hi = uint32_t(key >> 32), lo = uint32_t(key);
        const uint32_t whi = wave_max_u32(hi);
        bool mine = hi == whi;
        uint64_t bal = __ballot(mine);
        if (bal & (bal - 1)) {                 // equal to 20 bits of mantissa: the low words decide
            const uint32_t wlo = wave_max_u32(mine ? lo : 0u);
            mine = mine && lo == wlo;
            bal = __ballot(mine);
        }
        const int owner = int(__builtin_ctzll(bal));
        int slot = NV;
#pragma unroll
        for (int j = NV - 1; j >= 0; --j)
            if (v[j] == best) slot = j;
        const int jw = __builtin_amdgcn_readlane(slot, owner);
        const int ew = __builtin_amdgcn_readlane(e0, owner) + jw;
        const bool none = __builtin_amdgcn_readlane(int(best == kOut), owner);
        if (none) break;                       // nothing is left
        if (lane == owner) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (j == jw) v[j] = kOut;
        }
        if (lane == s) my = ew;
    }

    // the picks' scores again, one a lane
    double w = 0.0;
    if (my >= 0) {
        const double l = double(clean(logit(my)));
        w = a.sigmoid ? 1.0 / (1.0 + exp(-l)) : exp(l - m) * iz;
    }
    if (a.normalize) {
        const double z = wave_sum_d(w);
        w = z > 0.0 ? w / z : 0.0;
    }
    if (lane < a.K) {
        a.out_e[t * a.K + lane] = my;
        a.out_w[t * a.K + lane] = float(w * double(a.scaling));
    }
}

template <bool BF16>
void launch_nv(hipStream_t st, const ScoresArgs& a, int lpg, int V) {
    const dim3 grid((a.T + kScWaves - 1) / kScWaves), block(kScWaves * kWave);
#define GRIM_SC(NV) hipLaunchKernelGGL((scores_kernel<NV, BF16>), grid, block, 0, st, a, lpg, V)
    if (V <= 1) GRIM_SC(1);
    else if (V <= 2) GRIM_SC(2);
    else if (V <= 4) GRIM_SC(4);
    else if (V <= 8) GRIM_SC(8);
    else GRIM_SC(16);
#undef GRIM_SC
}

}  // namespace

hipError_t scores_launch(hipStream_t st, const ScoresArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.E <= 0 || a.E > kScoresMaxE || a.K <= 0 || a.K > kScoresMaxK || a.n_group <= 0 ||
        a.n_group > kScoresMaxGroups || a.E % a.n_group)
        return hipErrorInvalidValue;
    int lpg = kWave;
    while (lpg * a.n_group > kWave) lpg >>= 1;
    const int gsz = a.E / a.n_group, V = (gsz + lpg - 1) / lpg;   // V <= 2 * 512 / 64
    if (a.bf16) launch_nv<true>(st, a, lpg, V);
    else launch_nv<false>(st, a, lpg, V);
    return hipGetLastError();
}

}  // namespace grim
