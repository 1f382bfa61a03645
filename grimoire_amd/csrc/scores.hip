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
// closer than their rounding (an exp, a sum over E, a bias) swap places with
// the order of the sum (Gaussian logits, a balance bias of 0.3 / E: 3 of
// 4.9 million picks at E = 512, 6 of 3.9 million at E = 256), and scores that
// saturate are equal (sigmoids of logits above 18 all round to 1); in fp64 the
// choice is that of the exact scores.  It costs E exps of the fp64 pipe a
// token, also where no bias and no sum of two makes the order another than the
// logits' own.
//
// Lanes: without groups expert e is lane e % 64's, so a load of a lane's j-th
// expert is one run of memory.  With groups each owns lpg =
// 2^floor(log2(64 / n_group)) lanes of V = ceil(group / lpg) <= 16
// consecutive experts: a group's reductions are butterflies in its lanes.
//
// The choice: a search over the lanes' best values, rounded to fp32, gives a
// bound that at least K experts reach (rounding keeps the order); the few
// experts that reach it are gathered, one a lane, and ranked against each
// other in fp64.  More than 64 of them (ties) take K rounds over all values.
//
// 4096 tokens, 512 experts, top 10, bias: 8.1 us (the logits' bytes take 1.8
// at the rate of a large copy): vector issue bounds this form of it, 726
// instructions a token, 210 of them the exps (K rounds of wave maxima in place of the search
// and the ranking: 925 and 10.2 us; over the fp64 values: 16.0).  One token
// of 128 experts: 3 us.
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

__device__ __forceinline__ double lane_d(double v, int lane) {
    return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), lane),
                            __builtin_amdgcn_readlane(__double2loint(v), lane));
}

template <int CTRL>
__device__ __forceinline__ double dpp_d(double v) {
    return __hiloint2double(int(dpp_u<CTRL>(uint32_t(__double2hiint(v)))),
                            int(dpp_u<CTRL>(uint32_t(__double2loint(v)))));
}

// Sum over the wave, the same on every lane.
__device__ __forceinline__ double wave_sum_d(double v) {
    v += dpp_d<kDppXor1>(v);
    v += dpp_d<kDppXor2>(v);
    v += dpp_d<kDppHalfMirror>(v);
    v += dpp_d<kDppMirror>(v);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}

// exp(x) = 2^k e^r, k = round(x / ln 2), |r| <= ln(2) / 2, ln 2 in two parts
// (the first its top 30 bits: k * it is exact), e^r by its Taylor polynomial of
// degree 13 (what is left out is below 5e-18).  Clamped to where the result
// is 0 or infinite.
template <bool NEG>      // x <= 0
__device__ __forceinline__ double exp64(double x) {
    x = fmax(x, -1000.0);
    if constexpr (!NEG) x = fmin(x, 1000.0);
    const double k = __builtin_rint(x * 1.4426950408889634);
    double r = __builtin_fma(k, -0x1.62e42fe800000p-1, x);
    r = __builtin_fma(k, -0x1.e8e7bcd5e4f1ep-31, r);
    double p = 1.0 / 6227020800.0;
    p = __builtin_fma(p, r, 1.0 / 479001600.0);
    p = __builtin_fma(p, r, 1.0 / 39916800.0);
    p = __builtin_fma(p, r, 1.0 / 3628800.0);
    p = __builtin_fma(p, r, 1.0 / 362880.0);
    p = __builtin_fma(p, r, 1.0 / 40320.0);
    p = __builtin_fma(p, r, 1.0 / 5040.0);
    p = __builtin_fma(p, r, 1.0 / 720.0);
    p = __builtin_fma(p, r, 1.0 / 120.0);
    p = __builtin_fma(p, r, 1.0 / 24.0);
    p = __builtin_fma(p, r, 1.0 / 6.0);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    p = __builtin_fma(p, r, 1.0);
    return __builtin_amdgcn_ldexp(p, int(k));
}

// The order of doubles as that of their bits: key(a) < key(b) iff a < b.
__device__ __forceinline__ uint64_t order_key(double v) {
    const uint64_t u = uint64_t(__double_as_longlong(v + 0.0));   // -0 -> +0
    return (u >> 63) ? ~u : (u | (uint64_t(1) << 63));
}

constexpr double kOut = -__builtin_huge_val();   // an expert that cannot be picked

__device__ __forceinline__ void wave_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// lpg: lanes of a group (64 without groups); V: experts of a lane.
template <int NV, bool BF16>
__global__ __launch_bounds__(kScWaves * kWave) void scores_kernel(ScoresArgs a, int lpg, int V) {
    __shared__ double c_v[kScWaves][kWave];      // the gathered candidates
    __shared__ int c_e[kScWaves][kWave];
    __shared__ float c_l[kScWaves][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int64_t t = int64_t(blockIdx.x) * kScWaves + wave;
    if (t >= a.T) return;
    const int E = a.E, gsz = E / a.n_group;
    const bool groups = a.n_group > 1;
    const int gi = lane / lpg, sub = lane - gi * lpg;
    // expert j of this lane is e0 + j * es, j < nv (nv may be <= 0)
    const int e0 = groups ? gi * gsz + sub * V : lane, es = groups ? 1 : kWave;
    const int nv = !groups ? (E - lane + kWave - 1) / kWave : gi < a.n_group ? min(V, gsz - sub * V) : 0;

    // all loads first, without a branch between them
    float lv[NV], bv[NV];
    int at[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) at[j] = j < nv ? e0 + j * es : 0;
    const int64_t row = t * a.row_stride;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        if constexpr (BF16) lv[j] = bf16_to_f32(static_cast<const uint16_t*>(a.logits)[row + at[j]]);
        else lv[j] = static_cast<const float*>(a.logits)[row + at[j]];
    }
    if (a.bias) {
#pragma unroll
        for (int j = 0; j < NV; ++j) bv[j] = a.bias[at[j]];
    }
    if (a.part1) {
#pragma unroll
        for (int j = 0; j < NV; ++j) lv[j] += a.part1[row + at[j]];
    }
    // an expert that is out (NaN too, which fmaxf drops): -inf; +inf is the
    // largest finite logit
#pragma unroll
    for (int j = 0; j < NV; ++j)
        lv[j] = j < nv ? fminf(fmaxf(lv[j], -__builtin_inff()), 3.402823466e+38f) : -__builtin_inff();

    double m = 0.0, iz = 1.0;   // softmax: the largest logit, 1 / sum exp(l - m)
    double v[NV];
    if (!a.sigmoid) {
        float lm = lv[0];
#pragma unroll
        for (int j = 1; j < NV; ++j) lm = fmaxf(lm, lv[j]);
        const uint32_t k = wave_max_u32(score_key(lm));
        lm = (k & 0x80000000u) ? bits_f(k & 0x7FFFFFFFu) : bits_f(~k);
        m = lm > -__builtin_inff() ? double(lm) : 0.0;
        double z = 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] = exp64<true>(double(lv[j]) - m);      // -inf: 0
            z += v[j];
        }
        z = wave_sum_d(z);
        iz = z > 0.0 ? 1.0 / z : 0.0;
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] *= iz;
    } else {
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = 1.0 / (1.0 + exp64<false>(-double(lv[j])));
    }
    if (a.bias) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            v[j] += double(bv[j]);
            v[j] = v[j] == v[j] ? v[j] : kOut;
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) v[j] = lv[j] > -__builtin_inff() ? v[j] : kOut;

    if (groups) {
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
            const double o = lane_d(gs, g * lpg);
            rank += (o > gs || (o == gs && g < gi)) ? 1 : 0;
        }
        if (rank >= a.topk_group) {
#pragma unroll
            for (int j = 0; j < NV; ++j) v[j] = kOut;
        }
    }

    // a bound that at least K lanes' best (rounded to fp32) reach, or all that
    // are left: the highest by its top 20 bits, a bit and a ballot each
    uint32_t key[NV], top = 0, bound = 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint32_t u = f_bits(float(v[j]) + 0.0f);         // -0 -> +0
        key[j] = v[j] > kOut ? u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u) : 0;
        top = max(top, key[j]);
    }
    for (uint32_t bit = 0x80000000u; bit >= 0x1000u; bit >>= 1) {
        const int c = __popcll(__ballot(top >= (bound | bit)));
        bound = c >= a.K ? bound | bit : bound;
        if (c == a.K) break;
    }
    bound = max(bound, 1u);
    int n = 0;                          // candidates
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const uint64_t bal = __ballot(key[j] >= bound);
        if (bal) {
            const int pos = n + __builtin_amdgcn_mbcnt_hi(uint32_t(bal >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(bal), 0));
            if (key[j] >= bound && pos < kWave) {
                c_v[wave][pos] = v[j];
                c_e[wave][pos] = e0 + j * es;
                c_l[wave][pos] = lv[j];
            }
            n += __popcll(bal);
        }
    }

    int my = -1, slot = lane;           // this lane's pick and its place in the row
    float ml = 0.0f;                    // its logit
    if (n <= kWave) {
        wave_sync_lds();
        const bool live = lane < n;
        const double cv = live ? c_v[wave][lane] : kOut;
        const int ce = live ? c_e[wave][lane] : 0x7FFFFFFF;
        int rank = 0;
        for (int i = 0; i < n; ++i) {
            const double ov = lane_d(cv, i);
            const int oe = __builtin_amdgcn_readlane(ce, i);
            rank += (ov > cv || (ov == cv && oe < ce)) ? 1 : 0;
        }
        slot = live ? rank : lane;      // lanes past the candidates: slots nothing is left for
        if (live && rank < a.K) {
            my = ce;
            ml = c_l[wave][lane];
        }
    } else {
        for (int s = 0; s < a.K; ++s) {
            double best = v[0];
#pragma unroll
            for (int j = 1; j < NV; ++j) best = fmax(best, v[j]);
            int jl = 0;                 // its first slot: the lane's lowest expert of that value
#pragma unroll
            for (int j = NV - 1; j >= 0; --j)
                if (v[j] == best) jl = j;
            const int e = e0 + jl * es;
            const uint64_t k = order_key(best);
            const uint32_t hi = uint32_t(k >> 32), lo = uint32_t(k);
            // each maximum over all lanes, outside of any condition
            const uint32_t whi = wave_max_u32(best > kOut ? hi : 0u);
            if (whi == 0) break;                      // nothing is left
            bool mine = best > kOut && hi == whi;
            const uint32_t wlo = wave_max_u32(mine ? lo : 0u);
            mine = mine && lo == wlo;
            const uint32_t wne = wave_max_u32(mine ? ~uint32_t(e) : 0u);
            mine = mine && ~uint32_t(e) == wne;
            const int owner = int(__builtin_ctzll(__ballot(mine)));
            const int we = __builtin_amdgcn_readlane(e, owner);
            float wl = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (mine && j == jl) {
                    v[j] = kOut;
                    wl = lv[j];
                }
            wl = lane_f(wl, owner);
            if (lane == s) {
                my = we;
                ml = wl;
            }
        }
    }

    double w = 0.0;
    if (my >= 0) w = a.sigmoid ? 1.0 / (1.0 + exp64<false>(-double(ml))) : exp64<true>(double(ml) - m) * iz;
    if (a.normalize) {
        const double z = wave_sum_d(w);
        w = z > 0.0 ? w / z : 0.0;
    }
    if (slot < a.K) {
        a.out_e[t * a.K + slot] = my;
        a.out_w[t * a.K + slot] = float(w * double(a.scaling));
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
