// proj4_impl.hpp -- the kernel of the dense 4-bit projections (proj4.hip).
//
// A wave takes tiles of 16 weight rows (8 gate rows and their up rows) and a
// part of K, in blocks of 128: 16 bytes a lane, straight to registers, four
// blocks in flight (through the LDS, with whole lines a wave, was no faster; past
// the caches slower, as a block is half a line of its rows: 31 -> 34 us at 7168 x
// 32768).
// The words of a lane are one matrix step's operand each; groups of 64
// and 32 exchange them between lanes so that a step has one group a column.  x
// lies in the LDS, in operand order, for all of the work-group's tiles; its
// scales a wave takes through its own part of the LDS, where a load a lane
// becomes a value a column.  A kernel with many more tiles than work-groups
// keeps x and goes on with the next weights, whose loads are on their way
// by then.  Two column tiles of x a work-group at most: four needed 230
// registers, and 64 rows of 4096 x 8192 took 30.8 us where twos take 21.7.
#pragma once

#include "bf16_mfma.hpp"
#include "proj4_out.hpp"

#include <algorithm>

namespace grim {

namespace {

constexpr int kBlk = 128;                 // k of a block: 16 bytes a lane, 4 lanes a weight row
constexpr int kChunks = kBlk / 8;         // its chunks of 8 k
constexpr int kSeg = 4;                   // blocks in flight
constexpr int kWaves = 8;                 // of a work-group

// v, finite, minus its top 16 bits: the rest of a cut to bf16, exact (an
// infinity's is NaN, which INT4 products come to anyway)
__device__ __forceinline__ float rest_of_finite(float v) { return v - bits_f(f_bits(v) & 0xFFFF0000u); }
// the top / bottom halves of two words: {hi, lo}
__device__ __forceinline__ uint32_t tops(uint32_t hi, uint32_t lo) { return __builtin_amdgcn_perm(hi, lo, 0x07060302u); }
__device__ __forceinline__ uint32_t bottoms(uint32_t hi, uint32_t lo) { return __builtin_amdgcn_perm(hi, lo, 0x05040100u); }

// Eight 4-bit codes of a word as bf16 16 + q, pairs (k, k + 4); flip is kCodes,
// or kSigned where the codes are signed (q xor 8: zero point 8).  The mask in a
// vector register: each pair is a shift and one three-input operation.
constexpr uint32_t kCodes = 0x41804180u, kSigned = kCodes ^ 0x00400040u;
__device__ __forceinline__ u32x4 codes16(uint32_t w, uint32_t flip) {
    uint32_t m = 0x00780078u;
    asm("" : "+v"(m));
    return u32x4{((w << 3) & m) ^ flip, ((w >> 1) & m) ^ flip, ((w >> 5) & m) ^ flip, ((w >> 9) & m) ^ flip};
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

// v, but what is computed of it is computed here: addresses that a loop does not
// change would be kept in the registers of weights in flight.
__device__ __forceinline__ int here(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Between LDS writes and reads of one wave (its LDS operations run in order):
// keeps the compiler from exchanging them.
__device__ __forceinline__ void wave_lds_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// A chunk of 8 elements of x as matrix-core operands, one per piece, in the
// order its weights are decoded in: 16 bytes at to, to + 16, ...
template <int GS, bool XB>
__device__ __forceinline__ void put_chunk(uint8_t* to, u32x4 lo, u32x4 hi, bool on) {
    if constexpr (XB) {
        u32x4 v = lo;
        if constexpr (GS != 0)                         // (0, 4), (1, 5), (2, 6), (3, 7)
            v = u32x4{bottoms(lo[2], lo[0]), tops(lo[2], lo[0]), bottoms(lo[3], lo[1]), tops(lo[3], lo[1])};
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = on ? v[k] : 0u;
        *reinterpret_cast<u32x4*>(to) = v;
    } else {
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] = on ? bits_f(k < 4 ? lo[k & 3] : hi[k & 3]) : 0.0f;
#pragma unroll
        for (int l = 0; l < 3; ++l) {
            u32x4 v;
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = GS == 0 ? tops(f_bits(f[2 * k + 1]), f_bits(f[2 * k])) : tops(f_bits(f[k + 4]), f_bits(f[k]));
            *reinterpret_cast<u32x4*>(to + l * 16) = v;
            if constexpr (GS == 0) {
                // MXFP4 products keep an infinity: its other pieces are 0.  One
                // test of a chunk (of each element: 32 rows of 2880 x 5760 17.7 ->
                // 18.7 us)
                float most = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) most = fmaxf(most, __builtin_fabsf(f[k]));
                if (l == 0 && __builtin_expect(most == __builtin_inff(), 0)) {
#pragma unroll
                    for (int k = 0; k < 8; ++k) f[k] = __builtin_fabsf(f[k]) == __builtin_inff() ? 0.0f : f[k];
                }
            }
            if (l < 2)
#pragma unroll
                for (int k = 0; k < 8; ++k) f[k] = rest_of_finite(f[k]);
        }
    }
}

template <bool XB>
__device__ __forceinline__ void get_chunk(const uint8_t* at, u32x4& lo, u32x4& hi) {
    lo = reinterpret_cast<const u32x4*>(at)[0];
    if constexpr (!XB) hi = reinterpret_cast<const u32x4*>(at)[1];
}

// GS: group size of INT4 (32, 64, 128; 256 reads each scale twice), 0: MXFP4.
// XB: x is bf16.  CT: 16-column tiles of x.
template <int GS, bool XB, int CT>
__global__ __launch_bounds__(kWaves * 64, 4) void proj4_kernel(Proj4Dev p) {
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const Proj4Args& a = p.a;
    constexpr int PG = GS == 0 ? 4 : kBlk / GS;        // scales of a row and block
    constexpr int L = XB ? 1 : 3;                      // pieces of a row of x
    constexpr int TR = XB ? 16 : 4;                    // its rows in a tile; column 4 t + l is piece l
    constexpr int kFetch = XB ? 8 : 4;                 // a lane's chunks of x in flight
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, q = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int KS = 1 << p.ks, kg = wave & (KS - 1), rg = wave >> p.ks, RG = kWaves >> p.ks;
    // gridDim.x is a multiple of 8: work-groups of the same weights lie on one XCD
    const int set0 = blockIdx.x, kw = blockIdx.y, ctile = blockIdx.z;
    if (set0 >= p.stride) return;
    const int t0 = ctile * p.tile_rows, nt = min(p.tile_rows, a.T - t0), NC = nt * L;
    const int kb0 = kw * p.kw_blocks, KB = min(p.nb - kb0, p.kw_blocks);   // this work-group's blocks (at least one)
    // a tile has 16 outputs' rows, or 8 gate rows and their 8 up rows
    const int PT = a.glu ? 8 : 16;
    auto weight_row = [&](int tile, int row) {         // past the last output the last one's
        const int up = a.glu ? row >> 3 : 0, n = tile * PT + (a.glu ? row & 7 : row);
        return int64_t(min(n, p.half - 1)) + (up ? p.half : 0);
    };
    const int WB = p.wave_blocks, items = (WB + kSeg - 1) / kSeg, cK = a.K >> 3;

    // An item: kSeg blocks of a tile's 16 rows; a lane's word of block u.
    u32x4 ring[kSeg];
    const uint8_t* row_at;
    int64_t s_row;                                     // of the scales this lane loads
    auto tile_rows = [&](int set) {
        row_at = a.w.payload + weight_row(set * RG + rg, here(r)) * a.w.row_bytes;
        s_row = weight_row(set * RG + rg, here(lane) >> 2) * a.w.row_scales;
    };
    auto load_w = [&](int u, int first) {
        // a lane past the row's end (x is 0 there) reads its start
        const int b = min(first + u, p.nb - 1), k = b * kBlk + q * 32;
        ring[u] = *reinterpret_cast<const u32x4*>(row_at + (k < a.K ? k >> 1 : 0));
    };
    // scales of an item: lane (row lane / 4, block lane % 4), PG of them
    uint32_t sr[PG], zr[PG];
    auto load_s = [&](int first) {
        const int64_t base = s_row;
        const int k0 = min(first + (here(lane) & 3), p.nb - 1) * kBlk;
#pragma unroll
        for (int e = 0; e < PG; ++e) {
            if constexpr (GS == 0) {
                sr[e] = static_cast<const uint8_t*>(a.w.scales)[base + (min(k0 + e * 32, a.K - 1) >> 5)];
            } else {
                const int64_t at = base + (min(k0 + e * GS, a.K - 1) >> a.w.gshift);
                sr[e] = static_cast<const uint16_t*>(a.w.scales)[at];
                if (a.w.zeros) zr[e] = a.w.zeros[at];
            }
        }
    };
    float* ls = reinterpret_cast<float*>(lds + p.s_at) + wave * kSeg * PG * 16 * (GS == 0 ? 1 : 2);   // [block][group][row]
    float* lz = ls + kSeg * PG * 16;                   // 16 + zero point (< 0: signed codes)
    auto store_s = [&](int first) {
        const int srow = here(lane) >> 2, sblk = here(lane) & 3;
        const int k0 = (first + sblk) * kBlk;
#pragma unroll
        for (int e = 0; e < PG; ++e) {
            const bool on = k0 + e * (GS == 0 ? 32 : GS) < a.K;
            const int to = (sblk * PG + e) * 16 + srow;
            if constexpr (GS == 0) {
                ls[to] = on ? e8m0_to_f32(uint8_t(sr[e])) : 0.0f;
            } else {
                const float s = a.fmt == GRIM_FMT_INT4_F16 ? f16_to_f32(uint16_t(sr[e])) : bits_f(sr[e] << 16);
                const int zero = a.w.zeros ? int(zr[e]) : a.w.default_zero;
                ls[to] = on ? s : 0.0f;
                lz[to] = zero == 0xFF ? -24.0f : 16.0f + float(zero);
            }
        }
    };

    const int xs = (NC + 1) * 16;                      // bytes of a chunk's columns, padded against bank conflicts
    // LDS column of this lane in each tile (past the last: the first, not used)
    int col[CT];
#pragma unroll
    for (int c = 0; c < CT; ++c) {
        const int t = c * TR + (XB ? r : r >> 2), l = XB ? 0 : min(r & 3, 2);
        col[c] = (t < nt ? t * L + l : 0) * 16;
    }
    // the chunk of a block that word k of this lane belongs to
    auto chunk_of = [&](int k) {
        return GS == 0 || GS == 128 ? q * 4 + k
             : GS == 64             ? ((k >> 1) * 2 + (q & 1)) * 4 + (k & 1) + 2 * (q >> 1)
                                    : k * 4 + q;
    };
    auto x_of = [&](int b, int k, int c) {
        return *reinterpret_cast<const u32x4*>(lds + (b * kChunks + chunk_of(k)) * xs + col[c]);
    };
    // x of blocks [s0, s0 + n) into the LDS: a wave takes 1, 2 or 4 rows of 64,
    // 32 or 16 chunks at a time, kFetch such units in flight; past the end of K
    // zeros
    const int rb = nt >= 3 ? 2 : nt - 1, cb = 6 - rb;
    const int tqb = nt <= 4 ? 0 : 32 - __builtin_clz((nt - 1) >> 2);       // log2 of the units along the rows
    const int size = XB ? 2 : 4;
    const uint8_t* x_at = static_cast<const uint8_t*>(a.x) + int64_t(t0) * a.x_stride * size;
    auto fetch = [&](u32x4 (&xv)[kFetch][2], int s0, int n, int i) {
        const int cl = here(lane) & ((1 << cb) - 1), tl = here(lane) >> cb;
        const uint8_t* lane_at = x_at + (int64_t(tl) * a.x_stride + cl * 8) * size;
#pragma unroll
        for (int j = 0; j < kFetch; ++j) {
            const int u = i + j * kWaves, cu = (u >> tqb) << cb, tu = (u & ((1 << tqb) - 1)) << rb;
            const bool in = cu + cl < n * kChunks && s0 * kChunks + cu + cl < cK && tu + tl < nt;
            const int64_t at = (int64_t(tu) * a.x_stride + (s0 * kChunks + cu) * int64_t(8)) * size;   // of every lane
            get_chunk<XB>(in ? lane_at + at : x_at, xv[j][0], xv[j][1]);       // a lane with none: the first
        }
    };
    auto put = [&](const u32x4 (&xv)[kFetch][2], int s0, int n, int i) {
        const int cl = here(lane) & ((1 << cb) - 1), tl = here(lane) >> cb;
#pragma unroll
        for (int j = 0; j < kFetch; ++j) {
            const int u = i + j * kWaves, c = ((u >> tqb) << cb) + cl, t = ((u & ((1 << tqb) - 1)) << rb) + tl;
            if (c < n * kChunks && t < nt)
                put_chunk<GS, XB>(lds + c * xs + t * L * 16, xv[j][0], xv[j][1], s0 * kChunks + c < cK);
        }
    };
    // ... the units from i on
    auto stage = [&](int s0, int n, int i) {
        const int total = ((n * kChunks + (1 << cb) - 1) >> cb) << tqb;
        for (; i < total; i += kFetch * kWaves) {
            u32x4 xv[kFetch][2];
            fetch(xv, s0, n, i);
            put(xv, s0, n, i);
        }
        __syncthreads();
    };

    {
        const int n = min(p.slab, KB);
        u32x4 xv[kFetch][2];
        fetch(xv, kb0, n, wave);                       // x first: it is waited for first
        tile_rows(set0);
        load_s(kb0 + kg * WB);
#pragma unroll
        for (int u = 0; u < kSeg; ++u) load_w(u, kb0 + kg * WB);
        put(xv, kb0, n, wave);
        stage(kb0, n, wave + kFetch * kWaves);
    }

    // block b of the slab, the u-th of its item
    auto block = [&](f32x4 (&acc)[CT], int b, int u) {
        // x of PRE steps at a time, asked for together
        constexpr int PRE = CT == 1 ? 4 : 2;
        u32x4 xf[PRE][CT];
        auto operands = [&](int k) {
            if (k % PRE == 0)
#pragma unroll
                for (int j = 0; j < PRE; ++j)
#pragma unroll
                    for (int c = 0; c < CT; ++c) xf[j][c] = x_of(b, k + j, c);
        };
        u32x4 raw = ring[u];
        if constexpr (GS == 0) {
            const float s = ls[(u * 4 + q) * 16 + r];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                operands(k);
                const u32x4 wf = mx8(raw[k], s);
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[c] = mfma(xf[k % PRE][c], wf, acc[c]);
            }
        } else {
            constexpr int KG = 4 / PG;                 // steps of a group
            if constexpr (GS <= 64) {
                // words to steps: a step's four lanes of a row hold codes of one group
                const auto e = __builtin_amdgcn_permlane32_swap(raw[0], raw[2], false, false);
                const auto o = __builtin_amdgcn_permlane32_swap(raw[1], raw[3], false, false);
                raw = u32x4{e[0], o[0], e[1], o[1]};
            }
            if constexpr (GS == 32) {
                const auto e = __builtin_amdgcn_permlane16_swap(raw[0], raw[1], false, false);
                const auto o = __builtin_amdgcn_permlane16_swap(raw[2], raw[3], false, false);
                raw = u32x4{e[0], e[1], o[0], o[1]};
            }
#pragma unroll
            for (int g = 0; g < PG; ++g) {
                const float s = ls[(u * PG + g) * 16 + r], z = lz[(u * PG + g) * 16 + r];
                const uint32_t flip = z < 0.0f ? kSigned : kCodes;
                f32x4 D[CT], X1[CT];
#pragma unroll
                for (int c = 0; c < CT; ++c) D[c] = X1[c] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = g * KG; k < (g + 1) * KG; ++k) {
                    operands(k);
                    const u32x4 wf = codes16(raw[k], flip);
                    const uint32_t one = 0x3F803F80u;
#pragma unroll
                    for (int c = 0; c < CT; ++c) {
                        X1[c] = mfma(xf[k % PRE][c], u32x4{one, one, one, one}, X1[c]);
                        D[c] = mfma(xf[k % PRE][c], wf, D[c]);
                    }
                }
#pragma unroll
                for (int c = 0; c < CT; ++c) {
#pragma unroll
                    for (int m = 0; m < 4; ++m)
                        acc[c][m] = __builtin_fmaf(s, __builtin_fmaf(-__builtin_fabsf(z), X1[c][m], D[c][m]), acc[c][m]);
                }
            }
        }
    };

    for (int set = set0; set < p.sets; set += p.stride) {
        f32x4 acc[CT];
#pragma unroll
        for (int c = 0; c < CT; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int s0 = 0; s0 < KB; s0 += p.slab) {
            // (a work-group goes on to other tiles only where all of its x stays)
            if (s0) {
                __syncthreads();                       // x of the slab before is not read any more
                stage(kb0 + s0, min(p.slab, KB - s0), wave);
            }
            const int end = min(KB - s0, p.slab);
            for (int item = 0; item < items; ++item) {
                const int in = kg * WB + item * kSeg;  // its first block inside the slab
                wave_lds_fence();
                store_s(kb0 + s0 + in);
                wave_lds_fence();
                // what comes next; behind the last this set's first item again
                int nset = set, next = kb0 + s0 + in + kSeg;
                if (item + 1 == items) {
                    next = kb0 + s0 + p.slab + kg * WB;
                    if (s0 + p.slab >= KB) {
                        next = kb0 + kg * WB;
                        nset = set + p.stride < p.sets ? set + p.stride : set;
                        if (nset != set) tile_rows(nset);
                    }
                }
                load_s(next);
                // whole items without a branch between their blocks, so that one
                // block's operands are on their way while another's are used
                const int valid = min(min(kSeg, WB - item * kSeg), end - in);
                if (CT == 1 && valid == kSeg) {
#pragma unroll
                    for (int u = 0; u < kSeg; ++u) {
                        block(acc, in + u, u);
                        load_w(u, next);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < kSeg; ++u) {
                        if (u < valid) block(acc, in + u, u);
                        load_w(u, next);
                    }
                }
            }
        }

        // outputs; fp32: the pieces lie in one lane, the small ones first
        constexpr int V = XB ? 4 : 1;                  // rows of x of a lane and tile: (XB ? 4 q + j : q)
        float v[CT][V];
#pragma unroll
        for (int c = 0; c < CT; ++c) {
            if constexpr (XB) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[c][j] = acc[c][j];
            } else {
                v[c][0] = (acc[c][2] + acc[c][1]) + acc[c][0];
            }
        }
        const int oq = here(q);
        if (KS == 1) {
            const int tile = set * RG + rg;
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const int t = c * TR + oq * V + j;
                    if (p.kw > 1) {
                        if (t < nt && tile < p.tiles) p.part[((int64_t(kw) * a.T + t0 + t) * p.tiles + tile) * 16 + r] = v[c][j];
                    } else {
                        const float up = a.glu ? __shfl_xor(v[c][j], 8, kWave) : 0.0f;
                        const int n = tile * PT + r;
                        if (t < nt && r < PT && n < p.half) proj4_out(a, t0 + t, n, v[c][j], up);
                    }
                }
        } else {
            constexpr int TILE = CT * TR * 16;
            float* red = reinterpret_cast<float*>(lds + p.red_at);
            float* mine = red + wave * TILE;
            __syncthreads();                           // of the set before
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int j = 0; j < V; ++j) mine[(c * TR + q * V + j) * 16 + r] = v[c][j];
            __syncthreads();
            const int wide = p.kw > 1 ? 16 : PT, gu = a.glu && p.kw == 1 ? 8 : 0, outs = RG * wide;
            for (int u = tid; u < nt * outs; u += kWaves * 64) {
                const int t = u / outs, i = u - t * outs, g = i / wide, in = i - g * wide, tile = set * RG + g;
                const float* at = red + g * KS * TILE + t * 16 + in;
                float o = 0.0f, up = 0.0f;
                for (int w0 = 0; w0 < KS; w0 += 4) {   // four waves' at a time (a missing one's are not used)
                    float e[4], f[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int s = min(w0 + w, KS - 1) * TILE;
                        e[w] = at[s];
                        f[w] = at[s + gu];
                    }
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        o += w0 + w < KS ? e[w] : 0.0f;
                        up += w0 + w < KS ? f[w] : 0.0f;
                    }
                }
                if (p.kw > 1) {
                    if (tile < p.tiles) p.part[((int64_t(kw) * a.T + t0 + t) * p.tiles + tile) * 16 + in] = o;
                } else if (tile * PT + in < p.half) {
                    proj4_out(a, t0 + t, tile * PT + in, o, up);
                }
            }
        }
    }
}

constexpr size_t kLdsMost = 160 * 1024, kLdsHalf = kLdsMost / 2;
constexpr int kCus = 256;

template <int GS, bool XB, int CT>
hipError_t proj4_go(hipStream_t st, Proj4Dev& p) {
    const Proj4Args& a = p.a;
    constexpr int PG = GS == 0 ? 4 : kBlk / GS, L = XB ? 1 : 3, TR = XB ? 16 : 4;
    p.tile_rows = std::min(a.T, CT * TR);
    p.half = a.glu ? a.N / 2 : a.N;
    p.col_tiles = (a.T + p.tile_rows - 1) / p.tile_rows;
    p.nb = (a.K + kBlk - 1) / kBlk;
    p.tiles = (p.half + (a.glu ? 7 : 15)) / (a.glu ? 8 : 16);
    const auto up = [](int n, int d) { return (n + d - 1) / d; };
    const int x_blk = kChunks * (p.tile_rows * L + 1) * 16;
    const int s_all = kWaves * kSeg * PG * 16 * (GS == 0 ? 4 : 8), red_most = kWaves * CT * TR * 64;
    // blocks whose x fits beside a second work-group (room: with the sums there are)
    const int fit = std::max(1, int(kLdsHalf - s_all - red_most) / x_blk);
    // Tiles are shared out over K, until 4096 waves have one.  Where x would come
    // to the LDS in three turns or more, by work-groups, each with its part of x,
    // and a second launch that sums (4 fp32 rows, 7168 x 16384, 3 turns: 23.7 us in
    // 4 parts, 25.7 by waves; 16 of 2048 x 8192, 2 turns: 12.5 in 4 parts, 9.6 by
    // waves).  More than 8 parts are slower again (16 rows, 7168 x 4096: 14.5 us in
    // 4, 12.1 in 8, 16.7 in 16).
    const int64_t n = int64_t(p.tiles) * p.col_tiles;
    int kw = 1, lks = 0;
    if (p.nb > 2 * fit) kw = int(std::max<int64_t>(1, std::min<int64_t>({kProj4Tiles / n, p.nb / kSeg, kProj4Parts})));
    // By waves of a work-group: past 2048 waves only where each keeps two items
    // (7168 x 32768, one row: 38.5 us by one wave a tile, 31.3 by two; 2048 x 7168:
    // 6.4 by four, 7.7 by eight with two blocks each).
    const auto wide = [&](int to) { return (int64_t(2) << to) * kw; };
    while (lks < 3 && wide(lks) <= p.nb && n * wide(lks) <= (wide(lks) * 2 * kSeg <= p.nb ? kProj4Tiles : kProj4Tiles / 2)) ++lks;
    p.ks = lks;
    const int ks = 1 << p.ks;
    p.sets = up(p.tiles, kWaves / ks);
    p.kw = kw;
    p.part = static_cast<float*>(a.ws);
    p.kw_blocks = up(p.nb, p.kw);
    p.kw = up(p.nb, p.kw_blocks);
    if (p.kw > 1 && n * p.kw > kProj4Tiles) return hipErrorInvalidValue;
    const int red = ks > 1 ? red_most : 0;
    const int room = std::max(1, int(kLdsHalf - s_all - red) / x_blk);
    p.slab = up(p.kw_blocks, up(p.kw_blocks, room));
    p.wave_blocks = up(p.slab, ks);
    p.s_at = p.slab * x_blk;
    p.red_at = p.s_at + s_all;
    const size_t lds = p.red_at + red;
    if (lds > kLdsMost) return hipErrorInvalidValue;
    const bool again = p.slab >= p.kw_blocks && p.col_tiles == 1 && p.kw == 1;   // x stays for the next weights
    p.stride = again ? std::min(p.sets, 2 * kCus) : p.sets;
    if (p.col_tiles > 65535) return hipErrorInvalidValue;
    const dim3 grid(unsigned(up(p.stride, 8)) * 8, p.kw, p.col_tiles);
    hipLaunchKernelGGL((proj4_kernel<GS, XB, CT>), grid, dim3(kWaves * 64), lds, st, p);
    return p.kw > 1 ? proj4_sum_launch(st, p) : hipGetLastError();
}

template <int GS, bool XB>
hipError_t proj4_x(hipStream_t st, const Proj4Args& a) {
    Proj4Dev p{};
    p.a = a;
    constexpr int TR = XB ? 16 : 4;
    if (a.T <= TR) return proj4_go<GS, XB, 1>(st, p);
    return proj4_go<GS, XB, 2>(st, p);
}

}  // namespace

#define GRIM_PROJ4(GS)                                                        \
    hipError_t proj4_launch_g##GS(hipStream_t st, const Proj4Args& a) {       \
        return a.x_bf16 ? proj4_x<GS, true>(st, a) : proj4_x<GS, false>(st, a); \
    }

}  // namespace grim
