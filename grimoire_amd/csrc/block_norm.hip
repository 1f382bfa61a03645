// block_norm.hip -- the norms around a block in one pass over the row:
//   f  = x[t], or sum_s rw[t,s] * routed[inverse[t,s]] (+ shared[t])
//   p  = f * rsqrt(sum(f^2)/H + eps) * (offset + post_w)      (or f)
//   h' = rs * h + bs * gate * p
//   o  = h' * rsqrt(sum(h'^2)/H + eps) * (offset + pre_w)
// Two dependent sums over a row, so the row stays in registers: thread i of
// a work-group holds the 4-column chunks i, i + NT, ...  Memory bound: h and
// f are read once, h', o written once.  Everything the row needs (h, gate,
// weights) is requested before the first barrier, so one memory latency is
// paid a row and not three.  Sums are fp32 over at most 32 squares a thread,
// then a tree.
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

// 1 / (1 + exp(-g)) by the hardware exp2 and reciprocal (about 1 ulp each):
// the gate scales an fp32 sum that is compared to a tolerance.
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

    const uint16_t* rrow[KT > 0 ? KT : 1];
    float rw[KT > 0 ? KT : 1];
    if constexpr (KT > 0) {
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            int p = s < a.K ? a.inverse[t * a.K + s] : -1;
            p = p < a.routed_rows ? p : -1;
            rrow[s] = p < 0 ? nullptr : a.routed + int64_t(p) * H;
            rw[s] = p < 0 ? 0.0f : a.rw[t * a.K + s];
        }
    }
    float row_gate = 1.0f;
    if (a.gate_kind == GRIM_GATE_ROW)
        row_gate = a.gate_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.gate)[t])
                               : static_cast<const float*>(a.gate)[t];

    F4 f[VPT], h[VPT], g[VPT];
    uint2 wp[VPT], wn[VPT];
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const int d = (int(threadIdx.x) + c * NT) * 4;
        if (d >= H) continue;
        if constexpr (SRC == kSrcF32) {
            f[c] = load_f32(static_cast<const float*>(a.x) + t * a.x_stride + d);
        } else if constexpr (SRC == kSrcBf16) {
            f[c] = load_b16(static_cast<const uint16_t*>(a.x) + t * a.x_stride + d);
        } else {
            // a route without a row here adds nothing (its row is not read)
            f[c] = a.shared ? load_f32(a.shared + base + d) : F4{{0.0f, 0.0f, 0.0f, 0.0f}};
            uint2 u[KT > 0 ? KT : 1];
#pragma unroll
            for (int s = 0; s < KT; ++s)
                u[s] = rrow[s] ? *reinterpret_cast<const uint2*>(rrow[s] + d) : make_uint2(0u, 0u);
#pragma unroll
            for (int s = 0; s < KT; ++s) {
                const F4 e = widen(u[s]);
#pragma unroll
                for (int i = 0; i < 4; ++i) f[c].v[i] = __builtin_fmaf(rw[s], e.v[i], f[c].v[i]);
            }
        }
        h[c] = load_f32(a.h + base + d);
        if (a.gate_kind >= GRIM_GATE_CHANNEL && a.gate_kind != GRIM_GATE_ROW) {
            const int64_t o = (a.gate_kind == GRIM_GATE_FULL ? base : 0) + d;
            g[c] = a.gate_bf16 ? load_b16(static_cast<const uint16_t*>(a.gate) + o)
                               : load_f32(static_cast<const float*>(a.gate) + o);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) g[c].v[i] = row_gate;
        }
        wp[c] = a.post_w ? *reinterpret_cast<const uint2*>(a.post_w + d) : make_uint2(0u, 0u);
        wn[c] = a.pre_w ? *reinterpret_cast<const uint2*>(a.pre_w + d) : make_uint2(0u, 0u);
    }

    float fs = 1.0f;
    if (a.post_w) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < VPT; ++c) {
            if ((int(threadIdx.x) + c * NT) * 4 >= H) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) ss = __builtin_fmaf(f[c].v[i], f[c].v[i], ss);
        }
        fs = rsqrtf(block_sum<NT>(ss, part[0]) / float(H) + a.eps);
    }
    const bool act = a.gate_kind != GRIM_GATE_NONE && a.gate_sigmoid;
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const int d = (int(threadIdx.x) + c * NT) * 4;
        if (d >= H) continue;
        const F4 w = widen(wp[c]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float p = f[c].v[i];
            if (a.post_w) p = p * fs * (a.offset + w.v[i]);
            p *= gate_act(g[c].v[i], act);
            h[c].v[i] = __builtin_fmaf(a.bs, p, a.rs * h[c].v[i]);
            ss = __builtin_fmaf(h[c].v[i], h[c].v[i], ss);
        }
        if (a.h_out)
            *reinterpret_cast<float4*>(a.h_out + base + d) = make_float4(h[c].v[0], h[c].v[1], h[c].v[2], h[c].v[3]);
    }
    if (!a.out && !a.out_bf) return;
    const float hs = rsqrtf(block_sum<NT>(ss, part[1]) / float(H) + a.eps);
#pragma unroll
    for (int c = 0; c < VPT; ++c) {
        const int d = (int(threadIdx.x) + c * NT) * 4;
        if (d >= H) continue;
        const F4 w = widen(wn[c]);
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = h[c].v[i] * hs * (a.offset + w.v[i]);
        if (a.out) *reinterpret_cast<float4*>(a.out + base + d) = make_float4(o[0], o[1], o[2], o[3]);
        if (a.out_bf) {
            uint2 b;
            b.x = uint32_t(f32_to_bf16(o[0])) | (uint32_t(f32_to_bf16(o[1])) << 16);
            b.y = uint32_t(f32_to_bf16(o[2])) | (uint32_t(f32_to_bf16(o[3])) << 16);
            *reinterpret_cast<uint2*>(a.out_bf + base + d) = b;
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
    else if (a.K <= 8) GRIM_BN(2 + 8);
    else if (a.K <= 10) GRIM_BN(2 + 10);
    else GRIM_BN(2 + 16);
#undef GRIM_BN
}

}  // namespace

hipError_t block_norm_launch(hipStream_t st, const BlockNormArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.H <= 0 || a.H % 4 || a.H > kBlockNormMaxHidden || a.K < 0 || a.K > 16) return hipErrorInvalidValue;
    const int chunks = a.H / 4;
    if (chunks <= 64) launch_src<64, 1>(st, a);
    else if (chunks <= 256) launch_src<256, 1>(st, a);
    else if (chunks <= 512) launch_src<256, 2>(st, a);
    else if (chunks <= 1024) launch_src<256, 4>(st, a);
    else if (chunks <= 2048) launch_src<512, 4>(st, a);
    else if (chunks <= 4096) launch_src<1024, 4>(st, a);
    else launch_src<1024, 8>(st, a);
    return hipGetLastError();
}

}  // namespace grim
