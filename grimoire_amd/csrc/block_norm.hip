// block_norm.hip -- the norms around a block in one pass over the row:
//   f  = x[t], or sum_s rw[t,s] * routed[inverse[t,s]] (+ shared[t])
//   p  = f * rsqrt(sum(f^2)/H + eps) * (offset + post_w)      (or f)
//   h' = rs * h + bs * gate * p
//   o  = h' * rsqrt(sum(h'^2)/H + eps) * (offset + pre_w)
// Two dependent sums over a row, so the row stays in registers: thread i of
// a work-group holds the 4-column chunks i, i + NT, ...  Memory bound: h and
// f are read once, h', o written once.  Everything the row needs (h, gate,
// weights, expert rows) is requested before the first barrier and without a
// branch in between, so one memory latency is paid a row and not three.  Sums
// are fp32 over at most 32 squares a thread, then a tree.
//
// 4096 x 7168, bf16 block output, bf16 gate an element: 98.6 us, 5.4 TB/s
// (a large copy: 4.94); 3001 x 2048 behind ten experts and a shared one: 48.2
// us, 4.9 TB/s.  One to 32 rows: 4 to 8 us, two barriers and a chain of loads.
// Above 8192 columns a row takes 1024 threads of 92 registers and more, one
// work-group a CU: 2048 x 16384, bf16 block output 96 us, 4.2 TB/s.  Above
// 16384 a thread's eight chunks leave no registers for the norm weights ahead,
// and 2 to 8 are spilled (24 with 16 routes): 1024 x 32768 112 us, 3.6 TB/s;
// 512 x 32768 behind ten experts 122 us, 4.1 TB/s.
#include "block_norm.hpp"

namespace grim {

namespace {

struct F4 {
    float v[4];
};

__device__ __forceinline__ F4 load_f32(const float* p) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    return {{u.x, u.y, u.z, u.w}};
}
__device__ __forceinline__ F4 widen(uint2 u) {
    return {{bits_f(u.x << 16), bits_f(u.x & 0xFFFF0000u), bits_f(u.y << 16), bits_f(u.y & 0xFFFF0000u)}};
}
__device__ __forceinline__ F4 load_b16(const uint16_t* p) { return widen(*reinterpret_cast<const uint2*>(p)); }

// 1 / (1 + exp(-g)) by the hardware exp2 and reciprocal (about 1 ulp each,
// plus the rounding of the exponent, up to |g| 2^-23 relative): the gate scales
// an fp32 sum that is compared to a tolerance.
__device__ __forceinline__ float gate_act(float g, int sigmoid) {
    return sigmoid ? __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896341f)) : g;
}

// Sum over the work-group; every thread gets it.  part: NT / 64 floats of
// LDS, not written again before another barrier.
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* part) {
    v = group_sum<kWave>(v);
    if constexpr (NT == kWave) return v;
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < NT / kWave; ++i) t += part[i];
    return t;
}

enum { kSrcF32 = 0, kSrcBf16 = 1 };   // SRC of a dense block; 2 + KT: KT routes

template <int NT, int VPT, int SRC>
__global__ __launch_bounds__(NT) void block_norm_kernel(BlockNormArgs a) {
    constexpr int KT = SRC >= 2 ? SRC - 2 : 0;
    const int64_t t = blockIdx.x;
    const int H = a.H;
    const int64_t base = t * H;
    __shared__ float part[2][NT / kWave];

    // No load below waits for a branch: columns past H read the row's last
    // four, routes without a row here and absent weights read the row of h,
    // and what was read for nothing is left out of the arithmetic.
    const float* hrow = a.h + base;
    const uint16_t* dummy = reinterpret_cast<const uint16_t*>(hrow);
    const uint16_t* rrow[KT > 0 ? KT : 1];
    float rw[KT > 0 ? KT : 1];
    bool on[KT > 0 ? KT : 1];
    if constexpr (KT > 0) {
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            const int64_t r = t * a.K + (s < a.K ? s : a.K - 1);
            const int p = a.inverse[r];
            on[s] = s < a.K && p >= 0 && p < a.routed_rows;
            rrow[s] = on[s] ? a.routed + int64_t(p) * H : dummy;
            rw[s] = a.rw[r];
        }
    }
    int d[VPT];
    bool in[VPT];
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const int o = (int(threadIdx.x) + c * NT) * 4;
        in[c] = o < H;
        d[c] = in[c] ? o : H - 4;
    }

    constexpr bool kAhead = VPT <= 4;      // weights too, where the registers hold them
    F4 f[VPT], h[VPT], g[VPT];
    uint2 wp[kAhead ? VPT : 1], wn[kAhead ? VPT : 1];
    const uint16_t* post = a.post_w ? a.post_w : dummy;
    const uint16_t* pre = a.pre_w ? a.pre_w : dummy;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        h[c] = load_f32(hrow + d[c]);
        if constexpr (kAhead) {
            wp[c] = *reinterpret_cast<const uint2*>(post + d[c]);
            wn[c] = *reinterpret_cast<const uint2*>(pre + d[c]);
        }
        if constexpr (SRC == kSrcF32) f[c] = load_f32(static_cast<const float*>(a.x) + t * a.x_stride + d[c]);
        if constexpr (SRC == kSrcBf16) f[c] = load_b16(static_cast<const uint16_t*>(a.x) + t * a.x_stride + d[c]);
    }
    if (a.gate_kind == GRIM_GATE_CHANNEL || a.gate_kind == GRIM_GATE_FULL) {
        const int64_t o = a.gate_kind == GRIM_GATE_FULL ? base : 0;
        if (a.gate_bf16) {
#pragma unroll
            for (int c = 0; c < VPT; ++c) g[c] = load_b16(static_cast<const uint16_t*>(a.gate) + o + d[c]);
        } else {
#pragma unroll
            for (int c = 0; c < VPT; ++c) g[c] = load_f32(static_cast<const float*>(a.gate) + o + d[c]);
        }
    } else {
        float row_gate = 1.0f;
        if (a.gate_kind == GRIM_GATE_ROW)
            row_gate = a.gate_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.gate)[t])
                                   : static_cast<const float*>(a.gate)[t];
#pragma unroll
        for (int c = 0; c < VPT; ++c) g[c] = F4{{row_gate, row_gate, row_gate, row_gate}};
    }
    if constexpr (KT > 0) {
#pragma unroll
        for (int c = 0; c < VPT; ++c) f[c] = F4{{0.0f, 0.0f, 0.0f, 0.0f}};
        if (a.shared) {
#pragma unroll
            for (int c = 0; c < VPT; ++c) f[c] = load_f32(a.shared + base + d[c]);
        }
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            uint2 u[KT];
#pragma unroll
            for (int s = 0; s < KT; ++s) u[s] = *reinterpret_cast<const uint2*>(rrow[s] + d[c]);
#pragma unroll
            for (int s = 0; s < KT; ++s) {
                const F4 e = widen(u[s]);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[c].v[i] = on[s] ? __builtin_fmaf(rw[s], e.v[i], f[c].v[i]) : f[c].v[i];
            }
        }
    }

    float fs = 1.0f;
    if (a.post_w) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            float q = ss;
#pragma unroll
            for (int i = 0; i < 4; ++i) q = __builtin_fmaf(f[c].v[i], f[c].v[i], q);
            ss = in[c] ? q : ss;
        }
        fs = rsqrtf(block_sum<NT>(ss, part[0]) / float(H) + a.eps);
    }
    const bool act = a.gate_kind != GRIM_GATE_NONE && a.gate_sigmoid;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const F4 w = kAhead ? widen(wp[kAhead ? c : 0]) : load_b16(post + d[c]);
        float s = ss;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float p = f[c].v[i];
            if (a.post_w) p = p * fs * (a.offset + w.v[i]);
            p *= gate_act(g[c].v[i], act);
            h[c].v[i] = __builtin_fmaf(a.bs, p, a.rs * h[c].v[i]);
            s = __builtin_fmaf(h[c].v[i], h[c].v[i], s);
        }
        ss = in[c] ? s : ss;
        if (a.h_out && in[c])
            *reinterpret_cast<float4*>(a.h_out + base + d[c]) = make_float4(h[c].v[0], h[c].v[1], h[c].v[2], h[c].v[3]);
    }
    if (!a.out && !a.out_bf) return;
    const float hs = rsqrtf(block_sum<NT>(ss, part[1]) / float(H) + a.eps);
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        if (!in[c]) continue;
        const F4 w = kAhead ? widen(wn[kAhead ? c : 0]) : load_b16(pre + d[c]);
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = h[c].v[i] * hs * (a.offset + w.v[i]);
        if (a.out) *reinterpret_cast<float4*>(a.out + base + d[c]) = make_float4(o[0], o[1], o[2], o[3]);
        if (a.out_bf) {
            uint2 b;
            b.x = uint32_t(f32_to_bf16(o[0])) | (uint32_t(f32_to_bf16(o[1])) << 16);
            b.y = uint32_t(f32_to_bf16(o[2])) | (uint32_t(f32_to_bf16(o[3])) << 16);
            *reinterpret_cast<uint2*>(a.out_bf + base + d[c]) = b;
        }
    }
}

template <int NT, int VPT>
void launch_src(hipStream_t st, const BlockNormArgs& a) {
#define GRIM_BN(SRC) hipLaunchKernelGGL((block_norm_kernel<NT, VPT, SRC>), dim3(a.T), dim3(NT), 0, st, a)
    if (a.K == 0) {
        if (a.x_bf16) GRIM_BN(kSrcBf16);
        else GRIM_BN(kSrcF32);
    } else if (a.K <= 2) GRIM_BN(2 + 2);
    else if (a.K <= 4) GRIM_BN(2 + 4);
    else if (a.K <= 6) GRIM_BN(2 + 6);
    else if (a.K <= 8) GRIM_BN(2 + 8);
    else if (a.K <= 10) GRIM_BN(2 + 10);
    else GRIM_BN(2 + 16);
#undef GRIM_BN
}

}  // namespace

// Up to this many rows (one a CU) a row is spread over 1024 threads rather
// than 256 or 512 with more columns each: 8 rows of 2880, 3.50 against 3.82
// us; 32 of 2048 behind ten experts, 4.28 against 4.45; 512 of 7168 behind
// eight, 30.6 against 28.3.
constexpr int kFewRows = 256;

hipError_t block_norm_launch(hipStream_t st, const BlockNormArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.H <= 0 || a.H % 4 || a.H > kBlockNormMaxHidden || a.K < 0 || a.K > 16) return hipErrorInvalidValue;
    const int chunks = a.H / 4;
    // few rows: a row's loads over as many waves as a CU holds
    const bool few = a.T <= kFewRows;
    if (chunks <= 64) launch_src<64, 1>(st, a);
    else if (chunks <= 256) launch_src<256, 1>(st, a);
    else if (few && chunks <= 512) launch_src<512, 1>(st, a);
    else if (few && chunks <= 1024) launch_src<1024, 1>(st, a);
    else if (few && chunks <= 2048) launch_src<1024, 2>(st, a);
    else if (chunks <= 512) launch_src<256, 2>(st, a);
    else if (chunks <= 1024) launch_src<256, 4>(st, a);
    else if (chunks <= 2048) launch_src<512, 4>(st, a);
    else if (chunks <= 4096) launch_src<1024, 4>(st, a);
    else launch_src<1024, 8>(st, a);
    return hipGetLastError();
}

}  // namespace grim
