// sort_rows.hip -- tokens to rows in expert order, weighted, and the gradients
// of the ways there and back:
//   sort          rows[p] = w[t,s] x[t],                p = inverse[t,s]
//   sort_grad     dx[t] = sum_s w[t,s] drows[p],        dw[t,s] = <drows[p], x[t]>
//   combine_grad  drows[p] = w[t,s] dy[t],              dw[t,s] = <dy[t], rows[p]>,
//                 dshared[t] = gate[t] dy[t],           dgate[t] = <dy[t], shared[t]>
// All are bound by the memory: each row is read or written once, past the
// caches (a batch's rows are larger than they, and 4096 x 10 rows of 2048 bf16
// took 5 - 40 % longer through them).  A token's work-group has its element of
// x or dy in registers for all of its slots, and unrolled for their number,
// so that the slots' rows are asked for together (a loop with an exit in it
// took 10 us more at 4096 x 10).  Products are fp32, rounded once to bf16;
// dots are an fp32 chain a thread, then lanes, then waves in order: the same
// bits every time.
#include "sort_rows.hpp"

#include "dispatch.hpp"

namespace grim {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxSlots = 16;
constexpr int kCus = 256;

typedef float f32x4 __attribute__((ext_vector_type(4)));

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// V elements at p + at (p's element type) as fp32.  NT: not kept in the caches.
template <bool B16, int V, bool NT = false>
__device__ __forceinline__ void load_v(const void* p, int64_t at, float (&f)[V]) {
    if constexpr (B16) {
        uint32_t u[V / 2];
        if constexpr (V == 8) {
            const u32x4* from = reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p) + at);
            const u32x4 v = NT ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
            for (int i = 0; i < 4; ++i) u[i] = v[i];
        } else {
            const u32x2* from = reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(p) + at);
            const u32x2 v = NT ? __builtin_nontemporal_load(from) : *from;
            u[0] = v[0];
            u[1] = v[1];
        }
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            f[2 * i] = bits_f(u[i] << 16);
            f[2 * i + 1] = bits_f(u[i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) {
            const f32x4* from = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at + i);
            const f32x4 v = NT ? __builtin_nontemporal_load(from) : *from;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[i + j] = v[j];
        }
    }
}

template <bool B16, int V>
__device__ __forceinline__ void store_v(void* p, int64_t at, const float (&f)[V]) {
    if constexpr (B16) {
        uint32_t u[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) u[i] = uint32_t(f32_to_bf16(f[2 * i])) | (uint32_t(f32_to_bf16(f[2 * i + 1])) << 16);
        if constexpr (V == 8) __builtin_nontemporal_store(u32x4{u[0], u[1], u[2], u[3]}, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(p) + at));
        else __builtin_nontemporal_store(u32x2{u[0], u[1]}, reinterpret_cast<u32x2*>(static_cast<uint16_t*>(p) + at));
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4)
            __builtin_nontemporal_store(f32x4{f[i], f[i + 1], f[i + 2], f[i + 3]}, reinterpret_cast<f32x4*>(static_cast<float*>(p) + at + i));
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

// What lanes 0 ... KT - 1 hold, the same on every lane (one load for all slots
// of a token: loads behind conditions would wait for each other).
template <int KT>
__device__ __forceinline__ void from_lanes(int v, int (&out)[KT]) {
#pragma unroll
    for (int s = 0; s < KT; ++s) out[s] = __builtin_amdgcn_readlane(v, s);
}

// Token t's columns [d0, d1) to the rows p[s] of its slots (< 0: none).
template <bool XB, bool RB, int KT, int V>
__device__ __forceinline__ void copy_rows(const SortRowsArgs& a, int64_t t, const int (&p)[KT], int d0, int d1) {
    const int lane = threadIdx.x & (kWave - 1);
    int w[KT];
    from_lanes<KT>(a.w ? __float_as_int(a.w[t * a.K + (lane < a.K ? lane : 0)]) : 0, w);
    for (int d = d0 + threadIdx.x * V; d < d1; d += kThreads * V) {
        float f[V], o[V];
        load_v<XB, V>(a.x, t * a.x_stride + d, f);
#pragma unroll
        for (int s = 0; s < KT; ++s) {
            if (p[s] < 0) continue;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = a.w ? __int_as_float(w[s]) * f[i] : f[i];
            store_v<RB, V>(a.rows, int64_t(p[s]) * a.H + d, o);
        }
    }
}

// The experts' counts and offsets of a batch of R routes, by one work-group.
__device__ __forceinline__ void count_experts(const SortRowsArgs& a, int32_t* hist, int32_t* wsum) {
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave, R = a.T * a.K, E = a.E;
    for (int e = tid; e < E; e += kThreads) hist[e] = 0;
    __syncthreads();
    constexpr int B = 8;
    for (int r0 = tid; r0 < R; r0 += B * kThreads) {
        int v[B];
#pragma unroll
        for (int j = 0; j < B; ++j) v[j] = a.ids[min(r0 + j * kThreads, R - 1)];
#pragma unroll
        for (int j = 0; j < B; ++j)
            if (r0 + j * kThreads < R && v[j] >= 0 && v[j] < E) atomicAdd(&hist[v[j]], 1);
    }
    __syncthreads();
    const int per = (E + kThreads - 1) / kThreads, e0 = min(tid * per, E), e1 = min(e0 + per, E);
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += hist[e];
    int base = sum;
    for (int o = 1; o < kWave; o <<= 1) {
        const int v = __shfl_up(base, o, kWave);
        if (lane >= o) base += v;
    }
    if (lane == kWave - 1) wsum[wave] = base;
    __syncthreads();
    base -= sum;
    for (int w = 0; w < wave; ++w) base += wsum[w];
    for (int e = e0; e < e1; ++e) {
        a.counts[e] = hist[e];
        a.offsets[e] = base;
        base += hist[e];
    }
}

// Small batches.  The whole sort of at most kBruteRoutes routes in one launch: a
// work-group takes a token and counts, for each of its routes, the routes
// before it in expert order (keys expert * 2^12 + route, each lane a share of
// them).  One more work-group writes the experts' counts and offsets.
// blockIdx.y: part of the columns.  What it costs is the chain of its waits (the
// ids, a barrier, x) and of a launch: 2 tokens x 8 4.7 us, 64 x 8 of 2048 5.2 us.
constexpr int kBruteRoutes = 4096, kBruteE = 2048;
constexpr uint32_t kNoKey = 0xFFFFFFFFu;
template <bool XB, bool RB, int KT, int V>
__global__ __launch_bounds__(kThreads) void sort_brute_kernel(SortRowsArgs a, int cols) {
    __shared__ int32_t part[kThreads / kWave][KT];
    __shared__ int32_t hist[kBruteE];
    __shared__ int32_t wsum[kThreads / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int t = blockIdx.x, R = a.T * a.K, E = a.E;
    if (t == a.T) {
        if (blockIdx.y == 0) count_experts(a, hist, wsum);
        return;
    }
    auto key_of = [&](int r, int e) {
        return r < R && e >= 0 && e < E ? uint32_t(e) << 12 | uint32_t(r) : kNoKey;
    };
    // lane s: this token's route s
    const bool slot = lane < a.K;
    const int own = t * a.K + (slot ? lane : 0);
    const uint32_t my_key = slot ? key_of(own, a.ids[own]) : kNoKey;
    int key[KT], before[KT];                           // the same on every lane
    from_lanes<KT>(int(my_key), key);
#pragma unroll
    for (int s = 0; s < KT; ++s) before[s] = 0;
    constexpr int B = 8;                               // loads in flight
    for (int r0 = wave * kWave; r0 < R; r0 += B * kThreads) {
        int e[B];
#pragma unroll
        for (int j = 0; j < B; ++j) e[j] = a.ids[min(r0 + j * kThreads + lane, R - 1)];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            if (r0 + j * kThreads >= R) break;
            const uint32_t k = key_of(r0 + j * kThreads + lane, e[j]);
#pragma unroll
            for (int s = 0; s < KT; ++s) before[s] += __popcll(__ballot(k < uint32_t(key[s])));
        }
    }
#pragma unroll
    for (int s = 0; s < KT; ++s)
        if (lane == s) part[wave][s] = before[s];
    __syncthreads();
    int row = 0;
#pragma unroll
    for (int w = 0; w < kThreads / kWave; ++w) row += part[w][lane < KT ? lane : 0];
    row = my_key != kNoKey ? row : -1;
    if (wave == 0 && slot && blockIdx.y == 0) {
        a.inverse[own] = row;
        if (a.perm_token && row >= 0) a.perm_token[row] = t;
    }
    int p[KT];
    from_lanes<KT>(row, p);
    const int d0 = blockIdx.y * cols;
    copy_rows<XB, RB, KT, V>(a, t, p, d0, min(a.H, d0 + cols));
}

// The table of a batch of at most kTableRoutes routes in one launch: each
// work-group counts all routes by expert, those before its own apart, and
// ranks its own kThreads routes behind them.  No counts pass through memory;
// what each reads again, the ids, lies in the L2: 4096 x 10 routes over 512
// experts with their rows of 2048 bf16 take 41.4 us (rows written at 5.2 TB/s),
// with the four launches of dispatch.hip 51; 2048 x 8 of 1024 14.5 and 23.3.
// Reading them once per 256 costs more than those past about 100000 routes (96000
// with rows of 1024: 61.8 us and 65.4, 131072 91.2 and 85.1).
constexpr int kTableRoutes = 98304, kTableThreads = 1024;
__global__ __launch_bounds__(kTableThreads) void sort_table_kernel(SortRowsArgs a) {
    __shared__ int32_t before[kBruteE], behind[kBruteE];   // routes of an expert before the block, and from it on
    __shared__ int32_t wsum[kTableThreads / kWave];
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int E = a.E, R = a.T * a.K, r0 = blockIdx.x * kThreads;
    for (int e = tid; e < E; e += kTableThreads) before[e] = behind[e] = 0;
    // this thread's route: four waves have one
    int my = tid < kThreads && r0 + tid < R ? a.ids[r0 + tid] : -1;
    my = my >= 0 && my < E ? my : -1;
    __syncthreads();
    constexpr int B = 8;                               // loads in flight
    for (int r = tid; r < R; r += B * kTableThreads) {
        int e[B];
#pragma unroll
        for (int j = 0; j < B; ++j) e[j] = a.ids[min(r + j * kTableThreads, R - 1)];
#pragma unroll
        for (int j = 0; j < B; ++j) {
            const int at = r + j * kTableThreads;      // a wave's are all before the block or all behind
            int32_t* to = __builtin_amdgcn_readfirstlane(at) < r0 ? before : behind;
            if (at < R && uint32_t(e[j]) < uint32_t(E)) atomicAdd(&to[e[j]], 1);
        }
    }
    // the lanes of this wave with the same expert, by the bits of its number
    uint64_t same = __ballot(my >= 0);
    for (int b = 0; (E - 1) >> b; ++b) {
        const bool bit = my >> b & 1;
        const uint64_t m = __ballot(bit);
        same &= bit ? m : ~m;
    }
    const int rank = __popcll(same & ((uint64_t(1) << lane) - 1)), count = __popcll(same);
    __syncthreads();
    // exclusive offsets of the experts: this thread's are [e0, e1)
    const int pe = (E + kTableThreads - 1) / kTableThreads, e0 = min(tid * pe, E), e1 = min(e0 + pe, E);
    int sum = 0;
    for (int e = e0; e < e1; ++e) sum += before[e] + behind[e];
    int base = sum;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int v = __shfl_up(base, o, kWave);
        if (lane >= o) base += v;
    }
    if (lane == kWave - 1) wsum[wave] = base;
    __syncthreads();
    base -= sum;
#pragma unroll
    for (int w = 0; w < kTableThreads / kWave; ++w) base += w < wave ? wsum[w] : 0;
    for (int e = e0; e < e1; ++e) {
        const int c = before[e] + behind[e];
        if (blockIdx.x == 0) {
            a.counts[e] = c;
            a.offsets[e] = base;
        }
        before[e] += base;                             // the row of the block's first route of e
        base += c;
    }
    // the block's waves in turn, each moving its experts' rows on
    int row = -1;
    for (int w = 0; w < kThreads / kWave; ++w) {
        __syncthreads();
        if (wave == w && my >= 0) {
            const int first = before[my];
            row = first + rank;
            if (rank == count - 1) before[my] = first + count;
        }
    }
    if (tid < kThreads && r0 + tid < R) {
        if (row >= 0 && a.perm_token) a.perm_token[row] = (r0 + tid) / a.K;
        a.inverse[r0 + tid] = row;
    }
}

// rows of a table that is there
template <bool XB, bool RB, int KT, int V>
__global__ __launch_bounds__(kThreads) void sort_rows_kernel(SortRowsArgs a) {
    const int64_t t = blockIdx.x;
    const int lane = threadIdx.x & (kWave - 1);
    int p[KT];
    from_lanes<KT>(lane < a.K ? a.inverse[t * a.K + lane] : -1, p);
    copy_rows<XB, RB, KT, V>(a, t, p, 0, a.H);
}

// dx and the weights' gradients: a work-group a token, or without the weights'
// a token's columns blockIdx.y * cols ....  3001 x 4 rows of 2880
// bf16 with weights 21.2 us, 4.9 TB/s; 4096 x 10 of 2048 40.5, 5.0 TB/s.
template <bool RB, bool XB, int KT, int V>
__global__ __launch_bounds__(1024) void sort_grad_kernel(SortGradArgs a, int cols) {
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
    const int d0 = blockIdx.y * cols, d1 = min(a.H, d0 + cols);
    for (int d = d0 + threadIdx.x * V; d < d1; d += blockDim.x * V) {
        float f[KT][V], x[V], o[V];
        if (a.R > 0) {      // a route without a row reads row 0, which is left out below
#pragma unroll
            for (int s = 0; s < KT; ++s) load_v<RB, V, true>(a.drows, (p[s] < 0 ? 0 : p[s]) * a.H + d, f[s]);
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

// The gradient of the combine, a work-group a token and KT slots, blockIdx.y *
// KT ...; the first of them does the shared expert too.  Reads and writes as
// many rows: 4096 x 10 of 2048 bf16 with a gated shared expert 79.5 us, 4.86 TB/s (a
// large copy reaches 5.09).
template <bool YB, bool RB, int KT, int V>
__global__ __launch_bounds__(KT == 1 ? 1024 : kThreads) void combine_grad_kernel(CombineGradArgs a) {
    __shared__ float part[(KT == 1 ? 1024 : kThreads) / kWave * (KT + 1)];
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
    for (int d = threadIdx.x * V; d < a.H; d += blockDim.x * V) {
        float g[V], f[KT][V], o[V];
        load_v<YB, V>(a.dy, t * a.dy_stride + d, g);
        if (a.R > 0) {
#pragma unroll
            for (int s = 0; s < KT; ++s) load_v<RB, V, true>(a.rows, (p[s] < 0 ? 0 : p[s]) * a.H + d, f[s]);
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

template <bool XB, bool RB, int KT, int V>
hipError_t sort_k(hipStream_t st, const SortRowsArgs& a) {
    const int64_t R = int64_t(a.T) * a.K;
    // One launch while the counting costs less than a second launch: every
    // token's work-group reads all routes, (8 + 3 KT) / 64 operations a route
    // (rows of 2048 bf16, one launch and two: 64 tokens x 8 5.3 and 8.0 us, 400 x 8
    // 9.5 and 10.0, 2000 x 1 7.9 and 9.0; 512 x 8 10.4 and 10.2, 300 x 10 12.9 and 11.2)
    if (R <= kBruteRoutes && a.E <= kBruteE && R * a.T * (8 + 3 * KT) <= 45'000'000) {
        // columns shared out until there are two work-groups a CU (8 tokens x 8
        // of 7168: 4.8 us, undivided 9.9; 64: 6.6 and 10.7)
        const int most = (a.H + kThreads * V - 1) / (kThreads * V);
        const int parts = a.T >= 512 ? 1 : most < 512 / a.T ? most : 512 / a.T;
        const int cols = ((a.H + parts - 1) / parts + V - 1) / V * V;
        hipLaunchKernelGGL((sort_brute_kernel<XB, RB, KT, V>), dim3(a.T + 1, (a.H + cols - 1) / cols), dim3(kThreads), 0,
                           st, a, cols);
        return hipGetLastError();
    }
    if (R <= kTableRoutes && a.E <= kBruteE) {
        hipLaunchKernelGGL(sort_table_kernel, dim3(unsigned((R + kThreads - 1) / kThreads)), dim3(kTableThreads), 0, st, a);
    } else {
        DispatchArgs d{};
        d.ids = a.ids;
        d.T = a.T; d.K = a.K; d.E = a.E; d.H = a.H;
        d.counts = a.counts; d.offsets = a.offsets; d.inverse = a.inverse; d.perm_token = a.perm_token;
        d.workspace = a.workspace;
        const hipError_t e = dispatch_launch(st, d);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((sort_rows_kernel<XB, RB, KT, V>), dim3(a.T), dim3(kThreads), 0, st, a);
    return hipGetLastError();
}

// the number of slots that loops are unrolled for
template <bool XB, bool RB, int V>
hipError_t sort_slots(hipStream_t st, const SortRowsArgs& a) {
    if (a.K <= 1) return sort_k<XB, RB, 1, V>(st, a);
    if (a.K <= 2) return sort_k<XB, RB, 2, V>(st, a);
    if (a.K <= 4) return sort_k<XB, RB, 4, V>(st, a);
    if (a.K <= 8) return sort_k<XB, RB, 8, V>(st, a);
    return sort_k<XB, RB, 16, V>(st, a);
}

}  // namespace

size_t sort_rows_workspace_bytes(int T, int K, int E) { return dispatch_workspace_bytes(T, K, E); }

hipError_t sort_rows_launch(hipStream_t st, const SortRowsArgs& a) {
    if (a.T <= 0) {
        hipLaunchKernelGGL(sort_none_kernel, dim3((a.E + kThreads - 1) / kThreads), dim3(kThreads), 0, st, a.counts,
                           a.offsets, a.E);
        return hipGetLastError();
    }
    if (a.K <= 0 || a.K > kMaxSlots || a.H % 4) return hipErrorInvalidValue;
    // 16 bytes of a bf16 row a lane where they are aligned (4096 x 10 of 2048: 42.6
    // us, by 8 bytes 46.0); of an fp32 row too, so that a wave's are side by side
    const bool v8 = a.H % 8 == 0 && by8(a.x, a.x_stride, a.x_bf16) && by8(a.rows, a.H, a.rows_bf16);
#define GRIM_SORT(XB, RB) RB && v8 ? sort_slots<XB, RB, RB ? 8 : 4>(st, a) : sort_slots<XB, RB, 4>(st, a)
    if (a.x_bf16) return a.rows_bf16 ? (GRIM_SORT(true, true)) : (GRIM_SORT(true, false));
    return a.rows_bf16 ? (GRIM_SORT(false, true)) : (GRIM_SORT(false, false));
#undef GRIM_SORT
}

namespace {

template <bool RB, bool XB, int V>
void sort_grad_k(hipStream_t st, const SortGradArgs& a) {
    // less than a work-group a CU: larger ones (8 slots of 7168: 32 tokens 11.5 ->
    // 8.0 us, 255 15.1 -> 11.8; 512 21.1 -> 22.4)
    const int threads = a.w && a.T < kCus && a.H > kThreads * V ? 1024 : kThreads;
    // without sums over the columns these are shared out until there are two
    // work-groups a CU (32 tokens x 8 of 7168 in one work-group each 6.1 us, in
    // four 4.8; 128: 7.3 and 6.4)
    const int most = (a.H + kThreads * V - 1) / (kThreads * V);
    const int parts = a.w || a.T >= 2 * kCus ? 1 : most < 2 * kCus / a.T ? most : 2 * kCus / a.T;
    const int cols = ((a.H + parts - 1) / parts + V - 1) / V * V;
    const dim3 grid(a.T, (a.H + cols - 1) / cols);
#define GRIM_GRAD(KT) hipLaunchKernelGGL((sort_grad_kernel<RB, XB, KT, V>), grid, dim3(threads), 0, st, a, cols)
    if (a.K <= 1) GRIM_GRAD(1);
    else if (a.K <= 2) GRIM_GRAD(2);
    else if (a.K <= 4) GRIM_GRAD(4);
    else if (a.K <= 6) GRIM_GRAD(6);
    else if (a.K <= 8) GRIM_GRAD(8);
    else if (a.K <= 10) GRIM_GRAD(10);
    else GRIM_GRAD(16);
#undef GRIM_GRAD
}

template <bool YB, bool RB, int V>
void combine_grad_k(hipStream_t st, const CombineGradArgs& a) {
    // Few tokens: a larger work-group a slot, which reads dy again (8 slots of 7168:
    // 32 tokens 20.4 -> 5.7 us, 256 24.8 -> 20.7, 1024 61 -> 74; 4 of 2880: 256 8.3
    // and 8.3, 512 12.3 -> 14.1).
    const bool few = a.T <= kCus;
    const int threads = few && a.H > kThreads * V ? 1024 : kThreads;
#define GRIM_GRAD(KT) \
    hipLaunchKernelGGL((combine_grad_kernel<YB, RB, KT, V>), dim3(a.T, (a.K + KT - 1) / KT), dim3(threads), 0, st, a)
    if (a.K <= 1 || few) GRIM_GRAD(1);
    else if (a.K <= 2) GRIM_GRAD(2);
    else if (a.K <= 4) GRIM_GRAD(4);
    else if (a.K <= 6) GRIM_GRAD(6);
    else if (a.K <= 8) GRIM_GRAD(8);
    else if (a.K <= 10) GRIM_GRAD(10);
    else GRIM_GRAD(16);
#undef GRIM_GRAD
}

}  // namespace

hipError_t sort_grad_launch(hipStream_t st, const SortGradArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.K <= 0 || a.K > kMaxSlots || a.H % 4) return hipErrorInvalidValue;
    const bool v8 = a.H % 8 == 0 && by8(a.drows, a.H, a.rows_bf16) && by8(a.dx, a.dx_stride, a.dx_bf16) &&
                    (!a.w || by8(a.x, a.x_stride, a.x_bf16));
#define GRIM_BY(RB, XB) RB && v8 ? sort_grad_k<RB, XB, RB ? 8 : 4>(st, a) : sort_grad_k<RB, XB, 4>(st, a)
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
#define GRIM_BY(YB, RB) RB && v8 ? combine_grad_k<YB, RB, RB ? 8 : 4>(st, a) : combine_grad_k<YB, RB, 4>(st, a)
    if (a.dy_bf16) a.rows_bf16 ? (GRIM_BY(true, true)) : (GRIM_BY(true, false));
    else a.rows_bf16 ? (GRIM_BY(false, true)) : (GRIM_BY(false, false));
#undef GRIM_BY
    return hipGetLastError();
}

}  // namespace grim
