// sort_rows.hip -- tokens to rows in expert order, weighted, and the gradients
// of the ways there and back:
//   sort          rows[p] = w[t,s] x[t],                p = inverse[t,s]
//   sort_grad     dx[t] = sum_s w[t,s] drows[p],        dw[t,s] = <drows[p], x[t]>
//   combine_grad  drows[p] = w[t,s] dy[t],              dw[t,s] = <dy[t], rows[p]>,
//                 dshared[t] = gate[t] dy[t],           dgate[t] = <dy[t], shared[t]>
#include "sort_rows.hpp"

#include "dispatch.hpp"

namespace grim {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxSlots = 16;

typedef float f32x4 __attribute__((ext_vector_type(4)));

// V elements at p + at (p's element type) as fp32.
template <bool B16, int V>
__device__ __forceinline__ void load_v(const void* p, int64_t at, float (&f)[V]) {
    if constexpr (B16) {
        uint32_t u[V / 2];
        __builtin_memcpy(u, __builtin_assume_aligned(static_cast<const uint16_t*>(p) + at, V * 2), V * 2);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            f[2 * i] = bits_f(u[i] << 16);
            f[2 * i + 1] = bits_f(u[i] & 0xFFFF0000u);
        }
    } else {
        __builtin_memcpy(f, __builtin_assume_aligned(static_cast<const float*>(p) + at, 16), V * 4);
    }
}

template <bool B16, int V>
__device__ __forceinline__ void store_v(void* p, int64_t at, const float (&f)[V]) {
    if constexpr (B16) {
        uint32_t u[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) u[i] = uint32_t(f32_to_bf16(f[2 * i])) | (uint32_t(f32_to_bf16(f[2 * i + 1])) << 16);
        __builtin_memcpy(__builtin_assume_aligned(static_cast<uint16_t*>(p) + at, V * 2), u, V * 2);
    } else {
        __builtin_memcpy(__builtin_assume_aligned(static_cast<float*>(p) + at, 16), f, V * 4);
    }
}

// The sums over the work-group of N values a thread, in part [waves][N];
// thread i < N gets value i's (waves in order).
template <int N>
__device__ __forceinline__ float group_sums(const float (&v)[N], float* part) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float s = group_sum<kWave>(v[i]);
        if (lane == 0) part[wave * N + i] = s;
    }
    __syncthreads();
    float s = 0.0f;
    if (threadIdx.x < N)
        for (int w = 0; w < int(blockDim.x / kWave); ++w) s += part[w * N + threadIdx.x];
    return s;
}

// no tokens: no routes
__global__ void sort_none_kernel(int32_t* counts, int32_t* offsets, int E) {
    const int e = blockIdx.x * kThreads + threadIdx.x;
    if (e < E) counts[e] = offsets[e] = 0;
}

template <bool XB, bool RB, int V>
__global__ __launch_bounds__(kThreads) void sort_rows_kernel(SortRowsArgs a) {
    const int64_t t = blockIdx.x;
    int64_t p[kMaxSlots];
    float w[kMaxSlots];
#pragma unroll
    for (int s = 0; s < kMaxSlots; ++s) {
        const int64_t at = t * a.K + (s < a.K ? s : 0);
        p[s] = s < a.K ? a.inverse[at] : -1;
        w[s] = a.w ? a.w[at] : 1.0f;
    }
    for (int d = threadIdx.x * V; d < a.H; d += kThreads * V) {
        float f[V], o[V];
        load_v<XB, V>(a.x, t * a.x_stride + d, f);
#pragma unroll
        for (int s = 0; s < kMaxSlots; ++s) {
            if (p[s] < 0) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = a.w ? w[s] * f[i] : f[i];
            store_v<RB, V>(a.rows, p[s] * a.H + d, o);
        }
    }
}

template <bool RB, bool XB, int KT, int V>
__global__ __launch_bounds__(1024) void sort_grad_kernel(SortGradArgs a) {
    __shared__ float part[1024 / kWave * KT];
    const int64_t t = blockIdx.x;
    int64_t p[KT];
    float w[KT], dot[KT];
#pragma unroll
    for (int s = 0; s < KT; ++s) {
        const int64_t at = t * a.K + (s < a.K ? s : 0);
        const int64_t q = s < a.K ? a.inverse[at] : -1;
        p[s] = q < a.R ? q : -1;
        w[s] = a.w ? a.w[at] : 1.0f;
        dot[s] = 0.0f;
    }
    for (int d = threadIdx.x * V; d < a.H; d += blockDim.x * V) {
        float f[KT][V], x[V], o[V];
        if (a.R > 0) {      // a route without a row reads row 0, which is left out below
#pragma unroll
            for (int s = 0; s < KT; ++s) load_v<RB, V>(a.drows, (p[s] < 0 ? 0 : p[s]) * a.H + d, f[s]);
        }
        if (a.dw) load_v<XB, V>(a.x, t * a.x_stride + d, x);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float v = 0.0f;
#pragma unroll
            for (int s = 0; s < KT; ++s) v = p[s] >= 0 ? __builtin_fmaf(w[s], f[s][i], v) : v;
            o[i] = v;
            if (a.dw) {
#pragma unroll
                for (int s = 0; s < KT; ++s) dot[s] = p[s] >= 0 ? __builtin_fmaf(x[i], f[s][i], dot[s]) : dot[s];
            }
        }
        if (a.dx_bf16) store_v<true, V>(a.dx, t * a.dx_stride + d, o);
        else store_v<false, V>(a.dx, t * a.dx_stride + d, o);
    }
    if (a.dw) {
        const float s = group_sums<KT>(dot, part);
        if (int(threadIdx.x) < KT && int(threadIdx.x) < a.K) a.dw[t * a.K + threadIdx.x] = s;
    }
}

// slots blockIdx.y * KT ...; the first of them does the shared expert too
template <bool YB, bool RB, int KT, int V>
__global__ __launch_bounds__(kThreads) void combine_grad_kernel(CombineGradArgs a) {
    __shared__ float part[kThreads / kWave * (KT + 1)];
    const int64_t t = blockIdx.x;
    const int s0 = blockIdx.y * KT;
    const bool sh = a.shared && blockIdx.y == 0;
    int64_t p[KT];
    float w[KT], dot[KT + 1];
#pragma unroll
    for (int s = 0; s < KT; ++s) {
        const int64_t at = t * a.K + (s0 + s < a.K ? s0 + s : 0);
        const int64_t q = s0 + s < a.K ? a.inverse[at] : -1;
        p[s] = q < a.R ? q : -1;
        w[s] = a.w[at];
        dot[s] = 0.0f;
    }
    dot[KT] = 0.0f;
    const float gate = a.gate ? a.gate[t] : 1.0f;
    for (int d = threadIdx.x * V; d < a.H; d += kThreads * V) {
        float g[V], f[KT][V], o[V];
        load_v<YB, V>(a.dy, t * a.dy_stride + d, g);
        if (a.R > 0) {
#pragma unroll
            for (int s = 0; s < KT; ++s) load_v<RB, V>(a.rows, (p[s] < 0 ? 0 : p[s]) * a.H + d, f[s]);
        }
        if (sh) {
            const int64_t at = t * a.H + d;
            if (a.dgate) {
                float e[V];
                if (a.shared_bf16) load_v<true, V>(a.shared, at, e);
                else load_v<false, V>(a.shared, at, e);
#pragma unroll
                for (int i = 0; i < V; ++i) dot[KT] = __builtin_fmaf(g[i], e[i], dot[KT]);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = a.gate ? gate * g[i] : g[i];
            if (a.shared_bf16) store_v<true, V>(a.dshared, at, o);
            else store_v<false, V>(a.dshared, at, o);
        }
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            if (p[s] < 0) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                dot[s] = __builtin_fmaf(g[i], f[s][i], dot[s]);
                o[i] = w[s] * g[i];
            }
            store_v<RB, V>(a.drows, p[s] * a.H + d, o);
        }
    }
    const float s = group_sums<KT + 1>(dot, part);
    const int i = threadIdx.x;
    if (i < KT && s0 + i < a.K) a.dw[t * a.K + s0 + i] = s;
    if (i == KT && sh && a.dgate) a.dgate[t] = s;
}

// 16-byte accesses of bf16 need rows of a multiple of 8 elements and such distances
bool by8(const void* p, int64_t stride, bool b16) { return !b16 || (stride % 8 == 0 && reinterpret_cast<uintptr_t>(p) % 16 == 0); }

}  // namespace

hipError_t sort_rows_launch(hipStream_t st, const SortRowsArgs& a) {
    if (a.T <= 0) {
        hipLaunchKernelGGL(sort_none_kernel, dim3((a.E + kThreads - 1) / kThreads), dim3(kThreads), 0, st, a.counts,
                           a.offsets, a.E);
        return hipGetLastError();
    }
    if (a.K <= 0 || a.K > kMaxSlots || a.H % 4) return hipErrorInvalidValue;
    DispatchArgs d{};
    d.ids = a.ids;
    d.T = a.T; d.K = a.K; d.E = a.E; d.H = a.H;
    d.counts = a.counts; d.offsets = a.offsets; d.inverse = a.inverse; d.perm_token = a.perm_token;
    d.workspace = a.workspace;
    const hipError_t e = dispatch_launch(st, d);
    if (e != hipSuccess) return e;
    const bool v8 = a.H % 8 == 0 && by8(a.x, a.x_stride, a.x_bf16) && by8(a.rows, a.H, a.rows_bf16);
#define GRIM_SORT(XB, RB) \
    if (v8) hipLaunchKernelGGL((sort_rows_kernel<XB, RB, 8>), dim3(a.T), dim3(kThreads), 0, st, a); \
    else hipLaunchKernelGGL((sort_rows_kernel<XB, RB, 4>), dim3(a.T), dim3(kThreads), 0, st, a)
    if (a.x_bf16) { if (a.rows_bf16) { GRIM_SORT(true, true); } else { GRIM_SORT(true, false); } }
    else { if (a.rows_bf16) { GRIM_SORT(false, true); } else { GRIM_SORT(false, false); } }
#undef GRIM_SORT
    return hipGetLastError();
}

namespace {

template <bool RB, bool XB, int V>
void sort_grad_k(hipStream_t st, const SortGradArgs& a) {
    const int threads = a.T < 256 && a.H > kThreads * V ? 1024 : kThreads;
#define GRIM_GRAD(KT) hipLaunchKernelGGL((sort_grad_kernel<RB, XB, KT, V>), dim3(a.T), dim3(threads), 0, st, a)
    if (a.K <= 1) GRIM_GRAD(1);
    else if (a.K <= 2) GRIM_GRAD(2);
    else if (a.K <= 4) GRIM_GRAD(4);
    else if (a.K <= 8) GRIM_GRAD(8);
    else GRIM_GRAD(16);
#undef GRIM_GRAD
}

template <bool YB, bool RB, int V>
void combine_grad_k(hipStream_t st, const CombineGradArgs& a) {
#define GRIM_GRAD(KT) \
    hipLaunchKernelGGL((combine_grad_kernel<YB, RB, KT, V>), dim3(a.T, (a.K + KT - 1) / KT), dim3(kThreads), 0, st, a)
    if (a.K <= 1 || a.T <= 64) GRIM_GRAD(1);
    else if (a.K <= 2) GRIM_GRAD(2);
    else if (a.K <= 4) GRIM_GRAD(4);
    else if (a.K <= 8) GRIM_GRAD(8);
    else GRIM_GRAD(16);
#undef GRIM_GRAD
}

}  // namespace

hipError_t sort_grad_launch(hipStream_t st, const SortGradArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.K <= 0 || a.K > kMaxSlots || a.H % 4) return hipErrorInvalidValue;
    const bool v8 = a.H % 8 == 0 && by8(a.drows, a.H, a.rows_bf16) && by8(a.dx, a.dx_stride, a.dx_bf16) &&
                    (!a.w || by8(a.x, a.x_stride, a.x_bf16));
#define GRIM_BY(RB, XB) v8 ? sort_grad_k<RB, XB, 8>(st, a) : sort_grad_k<RB, XB, 4>(st, a)
    if (a.rows_bf16) a.x_bf16 ? (GRIM_BY(true, true)) : (GRIM_BY(true, false));
    else a.x_bf16 ? (GRIM_BY(false, true)) : (GRIM_BY(false, false));
#undef GRIM_BY
    return hipGetLastError();
}

hipError_t combine_grad_launch(hipStream_t st, const CombineGradArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.K <= 0 || a.K > kMaxSlots || a.H % 4) return hipErrorInvalidValue;
    const bool v8 = a.H % 8 == 0 && by8(a.dy, a.dy_stride, a.dy_bf16) && by8(a.rows, a.H, a.rows_bf16) &&
                    by8(a.drows, a.H, a.rows_bf16) &&
                    (!a.shared || (by8(a.shared, a.H, a.shared_bf16) && by8(a.dshared, a.H, a.shared_bf16)));
#define GRIM_BY(YB, RB) v8 ? combine_grad_k<YB, RB, 8>(st, a) : combine_grad_k<YB, RB, 4>(st, a)
    if (a.dy_bf16) a.rows_bf16 ? (GRIM_BY(true, true)) : (GRIM_BY(true, false));
    else a.rows_bf16 ? (GRIM_BY(false, true)) : (GRIM_BY(false, false));
#undef GRIM_BY
    return hipGetLastError();
}

}  // namespace grim
