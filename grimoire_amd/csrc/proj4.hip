// proj4.hip -- a dense projection with 4-bit weights for a few rows:
//   y_t[n] = base_t[n] + sum_g s[n,g] sum_{k in g} (q[n,k] - z[n,g]) x_t[k]
// (MXFP4: sum_g 2^(e[n,g] - 127) sum_k e2m1[n,k] x_t[k]), optionally with the
// SwiGLU of a gate|up projection.
#include "proj4.hpp"

#include <algorithm>

namespace grim {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlk = 128;                 // k of a block: 16 bytes a lane, 4 lanes a weight row
constexpr int kChunks = kBlk / 8;         // its chunks of 8 k

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    bf16x8 av, bv;
    __builtin_memcpy(&av, &a, 16);
    __builtin_memcpy(&bv, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, c, 0, 0, 0);
}

// v minus its top 16 bits: the rest of a cut to bf16 (exact; NaN for an infinity)
__device__ __forceinline__ float rest(float v) { return v - bits_f(f_bits(v) & 0xFFFF0000u); }
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
    return (f_bits(lo) >> 16) | (f_bits(hi) & 0xFFFF0000u);
}

// Eight 4-bit codes of a word as bf16 16 + q, pairs (k, k + 4).
__device__ __forceinline__ u32x4 codes16(uint32_t w) {
    uint32_t m = 0x00780078u, e = 0x41804180u;
    asm("" : "+v"(m), "+v"(e));           // both in vector registers: one v_bfi_b32 a word
    u32x4 o;
    o[0] = (m & (w << 3)) | (~m & e);
    o[1] = (m & (w >> 1)) | (~m & e);
    o[2] = (m & (w >> 5)) | (~m & e);
    o[3] = (m & (w >> 9)) | (~m & e);
    return o;
}

__device__ __forceinline__ u32x4 mx8(uint32_t w, float s) {
    const bf16x2 v[4] = {__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2),
                         __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3)};
    u32x4 r;
    __builtin_memcpy(&r, v, 16);
    return r;
}

struct Proj4Dev {
    Proj4Args a;
    int limbs;          // columns of a row of x: 1 (bf16) or 3 (fp32)
    int tile_rows;      // rows of x a work-group takes
    int row_tiles;      // work-groups along N
    int col_tiles;      // ... along the rows of x
    int nb;             // blocks of kBlk along K
    int slab;           // blocks whose x is in the LDS together, a multiple of waves * DEPTH
    int half;           // outputs: N, or N / 2 with glu
};

// GS: group size of INT4 (32, 64, 128; 256 reads each scale twice), 0: MXFP4.
// RT: 16-row weight tiles of a work-group (glu: half of them gate rows, half
// up rows), CT: 16-column tiles of x; DEPTH: blocks of weights in flight.
template <int GS, bool F16, bool GLU, int RT, int CT, int DEPTH>
__global__ __launch_bounds__(512) void proj4_kernel(Proj4Dev p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Proj4Args& a = p.a;
    constexpr int R = RT * 16;
    constexpr int PG = GS == 0 ? 4 : kBlk / GS;        // scales of a row and block
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), W = blockDim.x >> 6;
    // work-groups of the same weight rows lie on one XCD, one after the other
    const int id = blockIdx.x, xcd = id & 7, seq = id >> 3;
    const int rtile = (seq / p.col_tiles) * 8 + xcd, ctile = seq % p.col_tiles;
    if (rtile >= p.row_tiles) return;
    const int t0 = ctile * p.tile_rows, nt = min(p.tile_rows, a.T - t0), L = p.limbs, NC = nt * L;
    constexpr int OUT = GLU ? RT / 2 : RT;             // output tiles
    const int n0 = rtile * OUT * 16;

    // weight rows of this lane; past the last one that row again
    const uint8_t* wrow[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int up = GLU && i >= OUT, n = n0 + (i - (up ? OUT : 0)) * 16 + r;
        wrow[i] = a.w.payload + (int64_t(min(n, p.half - 1)) + (up ? p.half : 0)) * a.w.row_bytes;
    }
    u32x4 ring[DEPTH][RT];
    auto load = [&](int slot, int b) {
        // a lane past the row's end (x is 0 there) reads its start
        const int k = b * kBlk + q * 32;
        const int64_t at = k < a.K ? k >> 1 : 0;
#pragma unroll
        for (int i = 0; i < RT; ++i) ring[slot][i] = *reinterpret_cast<const u32x4*>(wrow[i] + at);
    };
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) load(d, wave + d * W);

    const int xs = (NC + 1) * 16;                      // bytes of a chunk's columns, padded against bank conflicts
    uint8_t* lx = lds;
    float* ls = reinterpret_cast<float*>(lds + p.slab * kChunks * xs);     // [group][R] scales
    float* lz = ls + p.slab * PG * R;                                      // [group][R] 16 + zero (< 0: signed codes)

    f32x4 acc[RT][CT];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};

    // LDS column of this lane in each tile (past the last: the first, not used)
    int col[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) col[c] = (c * 16 + r < NC ? c * 16 + r : 0) * 16;

    for (int s0 = 0; s0 < p.nb; s0 += p.slab) {
        const int sb = min(p.slab, p.nb - s0);
        if (s0) __syncthreads();
        // x of the slab: bf16, in the order the codes come in
        const int chunks = sb * kChunks, c0 = s0 * kChunks, cK = a.K >> 3;
        for (int u = tid; u < chunks * nt; u += blockDim.x) {
            const int t = u / chunks, c = u - t * chunks;
            uint32_t v[3][4] = {};
            if (c0 + c < cK) {
                const int64_t at = int64_t(t0 + t) * a.x_stride + int64_t(c0 + c) * 8;
                if (a.x_bf16) {
                    const u32x4 w = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.x) + at);
                    if constexpr (GS == 0) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[0][j] = w[j];
                    } else {        // (0, 4), (1, 5), (2, 6), (3, 7)
                        v[0][0] = (w[0] & 0xFFFFu) | (w[2] << 16);
                        v[0][1] = (w[0] >> 16) | (w[2] & 0xFFFF0000u);
                        v[0][2] = (w[1] & 0xFFFFu) | (w[3] << 16);
                        v[0][3] = (w[1] >> 16) | (w[3] & 0xFFFF0000u);
                    }
                } else {
                    const float* px = static_cast<const float*>(a.x) + at;
                    const f32x4 f0 = *reinterpret_cast<const f32x4*>(px), f1 = *reinterpret_cast<const f32x4*>(px + 4);
                    float f[8] = {f0[0], f0[1], f0[2], f0[3], f1[0], f1[1], f1[2], f1[3]};
#pragma unroll
                    for (int l = 0; l < 3; ++l) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            v[l][j] = GS == 0 ? cut2(f[2 * j], f[2 * j + 1]) : cut2(f[j], f[j + 4]);
#pragma unroll
                        for (int j = 0; j < 8; ++j) f[j] = rest(f[j]);
                    }
                }
            }
#pragma unroll
            for (int l = 0; l < 3; ++l)
                if (l < L)
                    *reinterpret_cast<u32x4*>(lx + c * xs + (t * L + l) * 16) = u32x4{v[l][0], v[l][1], v[l][2], v[l][3]};
        }
        // scales of the slab's groups
        const int groups = sb * PG;
        for (int u = tid; u < groups * R; u += blockDim.x) {
            const int i = u / groups, g = u - i * groups;
            const int up = GLU && i >= OUT * 16, n = n0 + i - (up ? OUT * 16 : 0);
            const int64_t row = int64_t(min(n, p.half - 1)) + (up ? p.half : 0);
            const int k = (s0 * PG + g) * (GS == 0 ? 32 : GS);
            float s = 0.0f, z = 0.0f;
            if (k < a.K) {
                if constexpr (GS == 0) {
                    s = e8m0_to_f32(static_cast<const uint8_t*>(a.w.scales)[row * a.w.row_scales + (k >> 5)]);
                } else {
                    const int64_t at = row * a.w.row_scales + (k >> a.w.gshift);
                    const uint16_t raw = static_cast<const uint16_t*>(a.w.scales)[at];
                    s = F16 ? f16_to_f32(raw) : bf16_to_f32(raw);
                    const int zero = a.w.zeros ? int(a.w.zeros[at]) : a.w.default_zero;
                    z = zero == 0xFF ? -24.0f : 16.0f + float(zero);
                }
            }
            ls[g * R + i] = s;
            if constexpr (GS != 0) lz[g * R + i] = z;
        }
        __syncthreads();

        for (int j0 = 0; j0 < sb; j0 += W * DEPTH) {
#pragma unroll
            for (int d = 0; d < DEPTH; ++d) {
                const int j = j0 + d * W + wave;       // the block inside the slab
                if (j < sb) {
                    const uint8_t* xb = lx + j * kChunks * xs;
                    if constexpr (GS == 0) {
                        float s[RT];
#pragma unroll
                        for (int i = 0; i < RT; ++i) s[i] = ls[(j * 4 + q) * R + i * 16 + r];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            u32x4 xf[CT];
#pragma unroll
                            for (int c = 0; c < CT; ++c)
                                xf[c] = *reinterpret_cast<const u32x4*>(xb + (q * 4 + k) * xs + col[c]);
#pragma unroll
                            for (int i = 0; i < RT; ++i) {
                                const u32x4 wf = mx8(ring[d][i][k], s[i]);
#pragma unroll
                                for (int c = 0; c < CT; ++c) acc[i][c] = mfma(xf[c], wf, acc[i][c]);
                            }
                        }
                    } else {
                        constexpr int KG = 4 / PG;     // steps of a group
                        u32x4 raw[RT];
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            raw[i] = ring[d][i];
                            if constexpr (GS <= 64) {
                                // words to steps: a step's four lanes of a row hold codes of one group
                                const auto e = __builtin_amdgcn_permlane32_swap(raw[i][0], raw[i][2], false, false);
                                const auto o = __builtin_amdgcn_permlane32_swap(raw[i][1], raw[i][3], false, false);
                                raw[i] = u32x4{e[0], o[0], e[1], o[1]};
                            }
                            if constexpr (GS == 32) {
                                const auto e = __builtin_amdgcn_permlane16_swap(raw[i][0], raw[i][1], false, false);
                                const auto o = __builtin_amdgcn_permlane16_swap(raw[i][2], raw[i][3], false, false);
                                raw[i] = u32x4{e[0], e[1], o[0], o[1]};
                            }
                        }
#pragma unroll
                        for (int g = 0; g < PG; ++g) {
                            f32x4 D[RT][CT], X[CT];
#pragma unroll
                            for (int c = 0; c < CT; ++c) X[c] = f32x4{0.f, 0.f, 0.f, 0.f};
                            float s[RT], z[RT];
                            uint32_t sg[RT];
#pragma unroll
                            for (int i = 0; i < RT; ++i) {
                                s[i] = ls[(j * PG + g) * R + i * 16 + r];
                                z[i] = lz[(j * PG + g) * R + i * 16 + r];
                                sg[i] = z[i] < 0.0f ? 0x88888888u : 0u;
                                z[i] = __builtin_fabsf(z[i]);
#pragma unroll
                                for (int c = 0; c < CT; ++c) D[i][c] = f32x4{0.f, 0.f, 0.f, 0.f};
                            }
#pragma unroll
                            for (int k0 = 0; k0 < KG; ++k0) {
                                const int k = g * KG + k0;
                                // the chunk that word k of this lane belongs to
                                const int ch = GS == 128 ? q * 4 + k
                                             : GS == 64  ? ((k >> 1) * 2 + (q & 1)) * 4 + (k & 1) + 2 * (q >> 1)
                                                         : k * 4 + q;
                                u32x4 xf[CT];
#pragma unroll
                                for (int c = 0; c < CT; ++c) {
                                    xf[c] = *reinterpret_cast<const u32x4*>(xb + ch * xs + col[c]);
                                    const uint32_t one = 0x3F803F80u;
                                    X[c] = mfma(xf[c], u32x4{one, one, one, one}, X[c]);
                                }
#pragma unroll
                                for (int i = 0; i < RT; ++i) {
                                    const u32x4 wf = codes16(raw[i][k] ^ sg[i]);
#pragma unroll
                                    for (int c = 0; c < CT; ++c) D[i][c] = mfma(xf[c], wf, D[i][c]);
                                }
                            }
#pragma unroll
                            for (int i = 0; i < RT; ++i)
#pragma unroll
                                for (int c = 0; c < CT; ++c)
#pragma unroll
                                    for (int m = 0; m < 4; ++m)
                                        acc[i][c][m] = __builtin_fmaf(s[i], __builtin_fmaf(-z[i], X[c][m], D[i][c][m]),
                                                                      acc[i][c][m]);
                        }
                    }
                }
                load(d, s0 + j + DEPTH * W);
            }
        }
    }

    // partial sums: over waves, then over a row's pieces
    constexpr int TILE = RT * CT * 256;
    float* red = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int m = 0; m < 4; ++m)
                red[wave * TILE + ((i * CT + c) * 16 + q * 4 + m) * 16 + r] = acc[i][c][m];
    __syncthreads();
    for (int u = tid; u < TILE; u += blockDim.x) {
        if (((u / 256) % CT) * 16 + (u & 255) / 16 >= NC) continue;
        float v = red[u];
        for (int w = 1; w < W; ++w) v += red[w * TILE + u];
        red[u] = v;
    }
    __syncthreads();
    for (int u = tid; u < nt * OUT * 16; u += blockDim.x) {
        const int t = u / (OUT * 16), i = u - t * (OUT * 16), n = n0 + i;
        if (n >= p.half) continue;
        float v[2];
#pragma unroll
        for (int h = 0; h < (GLU ? 2 : 1); ++h) {
            v[h] = 0.0f;
            for (int l = L - 1; l >= 0; --l) {         // the small pieces first
                const int c = t * L + l;
                v[h] += red[((h * OUT + i / 16) * CT + c / 16) * 256 + (c & 15) * 16 + (i & 15)];
            }
        }
        const int64_t row = t0 + t;
        float o = v[0];
        if constexpr (GLU) {
            o = silu(v[0]) * v[1];
        } else if (a.base) {
            const int64_t at = row * a.base_stride + n;
            o += a.base_bf16 ? bf16_to_f32(static_cast<const uint16_t*>(a.base)[at])
                             : static_cast<const float*>(a.base)[at];
        }
        const int64_t at = row * a.y_stride + n;
        if (a.y_bf16) static_cast<uint16_t*>(a.y)[at] = f32_to_bf16(o);
        else static_cast<float*>(a.y)[at] = o;
    }
}

constexpr size_t kLdsMost = 160 * 1024;

template <int GS, bool F16, bool GLU, int RT, int CT, int DEPTH>
hipError_t go(hipStream_t st, Proj4Dev& p) {
    const Proj4Args& a = p.a;
    constexpr int PG = GS == 0 ? 4 : kBlk / GS, R = RT * 16;
    p.limbs = a.x_bf16 ? 1 : 3;
    p.tile_rows = std::min(a.T, CT * 16 / p.limbs);
    p.half = GLU ? a.N / 2 : a.N;
    const int per = (GLU ? RT / 2 : RT) * 16;
    p.row_tiles = (p.half + per - 1) / per;
    p.col_tiles = (a.T + p.tile_rows - 1) / p.tile_rows;
    p.nb = (a.K + kBlk - 1) / kBlk;
    // x and scales of as many blocks as half a CU's LDS holds
    const size_t per_blk = size_t(kChunks) * (p.tile_rows * p.limbs + 1) * 16 + size_t(PG) * R * (GS == 0 ? 4 : 8);
    int W = p.nb >= 16 ? 8 : 4;
    while (W > 1 && per_blk * W * DEPTH > kLdsMost / 2) W /= 2;
    const int step = W * DEPTH;
    int steps = std::max<int>(1, int(kLdsMost / 2 / (per_blk * step)));
    steps = std::min(steps, (p.nb + step - 1) / step);
    p.slab = steps * step;
    const size_t lds = std::max(per_blk * p.slab, size_t(W) * RT * CT * 1024);
    if (lds > kLdsMost) return hipErrorInvalidValue;
    const int64_t grid = int64_t((p.row_tiles + 7) / 8 * 8) * p.col_tiles;
    if (grid > 0x7FFFFFFF) return hipErrorInvalidValue;
    auto k = proj4_kernel<GS, F16, GLU, RT, CT, DEPTH>;
    hipLaunchKernelGGL(k, dim3(unsigned(grid)), dim3(W * 64), lds, st, p);
    return hipGetLastError();
}

template <int GS, bool F16>
hipError_t pick(hipStream_t st, const Proj4Args& a) {
    Proj4Dev p{};
    p.a = a;
    const bool wide = a.T * (a.x_bf16 ? 1 : 3) > 16;
    if (a.glu) return wide ? go<GS, F16, true, 2, 2, 2>(st, p) : go<GS, F16, true, 2, 1, 2>(st, p);
    return wide ? go<GS, F16, false, 1, 2, 4>(st, p) : go<GS, F16, false, 1, 1, 4>(st, p);
}

}  // namespace

hipError_t proj4_launch(hipStream_t st, const Proj4Args& a) {
    if (a.T <= 0) return hipSuccess;
    if (a.fmt == GRIM_FMT_MXFP4) return pick<0, false>(st, a);
    const bool f16 = a.fmt == GRIM_FMT_INT4_F16;
    switch (a.w.gshift) {
        case 5: return f16 ? pick<32, true>(st, a) : pick<32, false>(st, a);
        case 6: return f16 ? pick<64, true>(st, a) : pick<64, false>(st, a);
        case 7:
        case 8: return f16 ? pick<128, true>(st, a) : pick<128, false>(st, a);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace grim
