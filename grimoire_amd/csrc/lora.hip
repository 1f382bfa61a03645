// lora.hip -- low-rank adapters of many requests beside a shared projection:
//   y_t = base_t + scale_a B_a (A_a x_t),  a = row_slot[t]
// in two launches.  shrink: z_t = A_a x_t, K split over waves and
// work-groups, fp32 partials to the workspace.  expand: the partials are
// summed in a fixed order, scaled, multiplied with B_a and added to base
// (and, for a gate|up projection, SwiGLU'd) on the way to y.
//
// Both are memory bound at every size (2 r operations an element of x and y
// read or written), so the matrix cores are fed straight from memory: a tile
// is 16 rows, and the lane pieces of A, B and x are MFMA operands as they
// lie.  Rows of a tile that name different adapters are done one distinct
// adapter after the other (long batches: runs of one request), or by one
// work-group each (short batches, where rows are mixed).
//
// fp32 values are multiplied exactly: an fp32 x (and z) is the sum of three
// bf16 pieces of 8 significant bits, cut off, not rounded, so each rest is
// exact; with bf16 weights every product is exact in the fp32 accumulator.
#include "lora.hpp"

namespace grim {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
// 16 bytes from an 8-byte aligned row (one load: global accesses need 4)
typedef uint32_t u32x4_a8 __attribute__((ext_vector_type(4), aligned(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = 16;        // rows of a tile
constexpr int kStep = 64;        // shrink: k of one step of a wave, 16 a lane
constexpr int kShrinkWaves = 8;
constexpr int kExpandWaves = 4;
constexpr int kCols = 32;        // expand: columns of one block of a wave
// Batches of up to this many rows give every distinct adapter of a tile its
// own work-groups.
constexpr int kItemRows = 512;
constexpr int kMaxSplits = 8;

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    bf16x8 av, bv;
    __builtin_memcpy(&av, &a, 16);
    __builtin_memcpy(&bv, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, c, 0, 0, 0);
}

// v minus its top 16 bits: the rest of a cut to bf16 (0 for infinities,
// whose first piece holds them; a NaN stays one)
__device__ __forceinline__ float rest(float v) {
    const float r = v - bits_f(f_bits(v) & 0xFFFF0000u);
    return __builtin_fabsf(v) == __builtin_inff() ? 0.0f : r;
}
__device__ __forceinline__ uint32_t cut2(float lo, float hi) {
    return (f_bits(lo) >> 16) | (f_bits(hi) & 0xFFFF0000u);
}
// eight fp32 values as three MFMA operands whose sum they are
__device__ __forceinline__ void pieces(float (&v)[8], u32x4 (&o)[3]) {
#pragma unroll
    for (int l = 0; l < 3; ++l) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[l][i] = cut2(v[2 * i], v[2 * i + 1]);
        if (l < 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = rest(v[i]);
        }
    }
}

// The rows of a tile and the adapters they name: lane l (and l+16, l+32,
// l+48) holds row l's.
struct Tile {
    int row;      // this lane's row, clamped into the batch
    bool in;      // the row exists
    int slot;     // its adapter or -1
};

__device__ __forceinline__ Tile tile_rows(const LoraArgs& p, int tile) {
    const int r = tile * kRows + (threadIdx.x & 15);
    Tile t;
    t.in = r < p.T;
    t.row = t.in ? r : p.T - 1;
    const int s = p.row_slot[t.row];
    t.slot = t.in && s >= 0 && s < p.slots ? s : -1;
    return t;
}

// The next distinct adapter among the rows `todo` (a bit a row), its first
// row's lane in lead; takes its rows out of todo.
__device__ __forceinline__ int next_slot(const Tile& t, uint64_t& todo, int& lead) {
    lead = int(__builtin_ctzll(todo));
    const int s = __builtin_amdgcn_readlane(t.slot, lead);
    todo &= ~__ballot(t.slot == s);
    return s;
}

// ------------------------------------------------------------------ shrink

// A wave's share of z = A x: NF fragments of 16 ranks, the K steps s0, s0 +
// kShrinkWaves, ... < s1, two at a time so that both are in flight.  All
// loads are unconditional: a step past the end and k past K read memory the
// wave reads anyway, under an x of zero; ranks past the slot read its last
// row, and are not stored.
template <bool XB, int NF>
__device__ __forceinline__ void shrink_steps(const void* xrow, const uint16_t* aslot, int64_t K, int rows, int col,
                                             int q, int s0, int s1, f32x4 (&acc)[4]) {
    constexpr int XV = XB ? 2 : 4;
    const uint16_t* ap[NF];
#pragma unroll
    for (int r = 0; r < NF; ++r) ap[r] = aslot + min(r * 16 + col, rows - 1) * K;
    for (int s = s0; s < s1; s += 2 * kShrinkWaves) {
        u32x4 x[2][XV], a[2][NF][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int k = min(s + u * kShrinkWaves, s1 - 1) * kStep + q * 8;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t kk = min(int64_t(k + h * 32), K - 8);
                if constexpr (XB) {
                    x[u][h] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(xrow) + kk);
                } else {
                    const float* xp = static_cast<const float*>(xrow) + kk;
                    x[u][h * 2] = *reinterpret_cast<const u32x4*>(xp);
                    x[u][h * 2 + 1] = *reinterpret_cast<const u32x4*>(xp + 4);
                }
#pragma unroll
                for (int r = 0; r < NF; ++r) a[u][r][h] = *reinterpret_cast<const u32x4*>(ap[r] + kk);
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int k = (s + u * kShrinkWaves) * kStep + q * 8;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool in = s + u * kShrinkWaves < s1 && k + h * 32 < K;
                u32x4 xv[3];
                if constexpr (XB) {
                    xv[0] = in ? x[u][h] : u32x4{0, 0, 0, 0};
                } else {
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[i] = in ? bits_f(x[u][h * 2][i]) : 0.0f;
                        v[4 + i] = in ? bits_f(x[u][h * 2 + 1][i]) : 0.0f;
                    }
                    pieces(v, xv);
                }
#pragma unroll
                for (int l = XB ? 0 : 2; l >= 0; --l)
#pragma unroll
                    for (int r = 0; r < NF; ++r) acc[r] = mfma(a[u][r][h], xv[l], acc[r]);
            }
        }
    }
}

// NR fragments of 16 ranks a work-group (max_rank 16, 32 or more).
template <bool XB, int NR>
__global__ __launch_bounds__(kShrinkWaves * kWave) void lora_shrink_kernel(LoraArgs p, int splits, int ksteps,
                                                                           int chunks, int items) {
    __shared__ f32x4 red[kShrinkWaves][NR][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int q = lane >> 4, col = lane & 15;
    const int tile = blockIdx.x, split = blockIdx.y;
    const int chunk = blockIdx.z % chunks, item = blockIdx.z / chunks;
    const Tile t = tile_rows(p, tile);
    uint64_t todo = __ballot(t.slot >= 0) & 0xFFFFu;
    // the split's steps [s0, s1), dealt to the waves in turn
    const int per = (ksteps + splits - 1) / splits;
    const int s0 = split * per + wave, s1 = min(ksteps, (split + 1) * per);
    const int r0 = chunk * NR * 16;

    for (int it = 0; todo; ++it) {
        int lead;
        const int slot = next_slot(t, todo, lead);
        if (items > 1 && it != item) continue;
        const int rank = min(max(p.rank[slot], 0), p.R);
        const int nr = min(NR, (rank - r0 + 15) / 16);      // fragments with live ranks
        if (nr > 0) {
            f32x4 acc[4] = {};
            // rows of another adapter read the group's first row instead:
            // their column of the product is not used
            const bool mine = t.slot == slot;
            const int64_t xo = int64_t(mine ? t.row : __builtin_amdgcn_readlane(t.row, lead)) * p.x_stride;
            const void* xrow = XB ? static_cast<const void*>(static_cast<const uint16_t*>(p.x) + xo)
                                  : static_cast<const void*>(static_cast<const float*>(p.x) + xo);
            const uint16_t* as = p.a + (int64_t(slot) * p.R + r0) * p.K;
            if (NR == 1 || nr == 1) shrink_steps<XB, 1>(xrow, as, p.K, p.R - r0, col, q, s0, s1, acc);
            else if (NR == 2 || nr == 2) shrink_steps<XB, 2>(xrow, as, p.K, p.R - r0, col, q, s0, s1, acc);
            else shrink_steps<XB, 4>(xrow, as, p.K, p.R - r0, col, q, s0, s1, acc);
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (r < nr) red[wave][r][lane] = acc[r];
            __syncthreads();
            // D of a fragment: lane (q, col) holds ranks 4q .. 4q+3 of row
            // col, and wave r sums fragment r over the waves
            if (wave < nr) {
                f32x4 z = red[0][wave][lane];
#pragma unroll
                for (int w = 1; w < kShrinkWaves; ++w) z += red[w][wave][lane];
                if (mine)
                    *reinterpret_cast<f32x4*>(p.part + (int64_t(split) * p.T + t.row) * p.R + r0 + wave * 16 + q * 4) = z;
            }
            __syncthreads();
        }
        if (items > 1) break;
    }
}

// ------------------------------------------------------------------ expand

// silu(g) * u with the hardware exp2 / rcp (about 1 ulp each, plus the
// rounding of the exponent, |g| 2^-24 relative).
__device__ __forceinline__ float glu(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// Eight columns of a base row: n .. n+7, of which the first four or all
// (whole) exist.
template <bool BB>
struct Base {
    u32x4 v[BB ? 1 : 2];
};

template <bool BB>
__device__ __forceinline__ void load_base(Base<BB>& b, const void* base, int64_t o, bool whole) {
    if constexpr (BB) {
        const uint16_t* p = static_cast<const uint16_t*>(base) + o;
        if (whole) {
            b.v[0] = *reinterpret_cast<const u32x4_a8*>(p);
        } else {
            const uint2 u = *reinterpret_cast<const uint2*>(p);
            b.v[0] = u32x4{u.x, u.y, 0, 0};
        }
    } else {
        const float* p = static_cast<const float*>(base) + o;
        b.v[0] = *reinterpret_cast<const u32x4*>(p);
        b.v[1] = *reinterpret_cast<const u32x4*>(p + (whole ? 4 : 0));
    }
}

template <bool BB>
__device__ __forceinline__ float base_at(const Base<BB>& b, int i) {
    if constexpr (BB)
        return i & 1 ? bits_f(b.v[0][i / 2] & 0xFFFF0000u) : bits_f(b.v[0][i / 2] << 16);
    else
        return bits_f(b.v[i / 4][i & 3]);
}

// two fp32 to bf16, nearest even (the hardware conversion)
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const bf16x2 b = __builtin_convertvector(f32x2{lo, hi}, bf16x2);
    uint32_t u;
    __builtin_memcpy(&u, &b, 4);
    return u;
}

__device__ __forceinline__ void store8(void* y, int64_t o, int bf16, const float (&v)[8], bool whole) {
    if (bf16) {
        uint16_t* p = static_cast<uint16_t*>(y) + o;
        u32x4 u;
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
        if (whole) *reinterpret_cast<u32x4_a8*>(p) = u;
        else *reinterpret_cast<uint2*>(p) = make_uint2(u[0], u[1]);
    } else {
        float* p = static_cast<float*>(y) + o;
        *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
        if (whole) *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
    }
}

// One group of rows of a tile (one adapter, or none) against columns
// [first, last) of y: CC chunks of 32 ranks (HALF: max_rank 16, where an
// instruction's 32 k hold the 16 ranks twice, under two pieces of z; CC 0:
// base alone), G blocks of 32 columns at a time whose base is requested
// together.  A block is two MFMA tiles of 16 columns, tile j's operand row m
// being column 8 (m / 4) + 4 j + m % 4, so that a lane's part of the two
// products is eight columns in a row.
template <bool GLU, int CC, bool HALF, bool BB, int G>
__device__ __forceinline__ void expand_cols(const LoraArgs& p, int splits, int slot, int rank, int row, int lead_row,
                                            bool mine, int q, int col, int first, int last, int width) {
    constexpr int NP = GLU ? 2 : 1, C = CC ? CC : 1;
    // rows of other groups read the first row's z and base, and do not store
    const int64_t src = mine ? row : lead_row;
    // z, scaled and without what lies past the rank, in three pieces
    u32x4 zv[C][3];
    if constexpr (CC > 0) {
        const float scale = p.scale[slot];
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int r = HALF ? (q & 1) * 8 : c * 32 + q * 8;
            const float* zp = p.part + src * p.R + min(r, p.R - 8);
            f32x4 lo = {}, hi = {};
            for (int s = 0; s < splits; s += 4) {
                f32x4 l[4], h[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float* sp = zp + int64_t(min(s + i, splits - 1)) * p.T * p.R;
                    l[i] = *reinterpret_cast<const f32x4*>(sp);
                    h[i] = *reinterpret_cast<const f32x4*>(sp + 4);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (s + i < splits) {
                        lo += l[i];
                        hi += h[i];
                    }
            }
            float z[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = r + i < rank ? (i < 4 ? lo[i & 3] : hi[i & 3]) * scale : 0.0f;
            pieces(z, zv[c]);
            if constexpr (HALF) {
                zv[c][0] = q < 2 ? zv[c][0] : zv[c][1];
                zv[c][1] = q < 2 ? zv[c][2] : u32x4{0, 0, 0, 0};
            }
        }
    }
    const uint16_t* bs = p.b + int64_t(slot) * p.N * p.R;
    const int64_t bo = src * p.base_stride, yo = int64_t(row) * p.y_stride;
    const int ncol = 8 * (col >> 2) + (col & 3);

    for (int n0 = first; n0 < last; n0 += G * kCols) {
        Base<BB> base[G][NP];
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const int n = min(n0 + g * kCols + q * 8, width - 4);
#pragma unroll
            for (int h = 0; h < NP; ++h) load_base<BB>(base[g][h], p.base, bo + n + h * width, n + 8 <= width);
        }
        u32x4 b[2][C][NP][2];
        auto load_b = [&](u32x4 (&d)[C][NP][2], int nb) {
#pragma unroll
            for (int c = 0; c < CC; ++c) {
                const int r = HALF ? (q & 1) * 8 : min(c * 32 + q * 8, p.R - 8);
#pragma unroll
                for (int h = 0; h < NP; ++h)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int n = min(nb + ncol + 4 * j, width - 1) + h * width;
                        d[c][h][j] = *reinterpret_cast<const u32x4*>(bs + int64_t(n) * p.R + r);
                    }
            }
        };
        load_b(b[0], n0);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            if (g + 1 < G) load_b(b[(g + 1) & 1], n0 + (g + 1) * kCols);
            // -0: what adds nothing leaves base's own sign of zero
            f32x4 acc[NP][2];
#pragma unroll
            for (int h = 0; h < NP; ++h)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[h][j] = f32x4{-0.0f, -0.0f, -0.0f, -0.0f};
#pragma unroll
            for (int c = 0; c < CC; ++c) {
                u32x4(&d)[NP][2] = b[g & 1][c];
                if (rank < c * 32 + (HALF ? 16 : 32)) {     // what lies past the rank, whatever it is
                    const int r = HALF ? (q & 1) * 8 : c * 32 + q * 8;
#pragma unroll
                    for (int h = 0; h < NP; ++h)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                uint32_t w = d[h][j][i];
                                w = r + 2 * i + 1 < rank ? w : w & 0xFFFFu;
                                d[h][j][i] = r + 2 * i < rank ? w : 0u;
                            }
                }
#pragma unroll
                for (int l = HALF ? 1 : 2; l >= 0; --l)
#pragma unroll
                    for (int h = 0; h < NP; ++h)
#pragma unroll
                        for (int j = 0; j < 2; ++j) acc[h][j] = mfma(d[h][j], zv[c][l], acc[h][j]);
            }
            // D: lane (q, col) holds columns 8q + 4j .. + 3 of row col
            const int n = n0 + g * kCols + q * 8;
            if (mine && n < width) {
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    v[i] = base_at<BB>(base[g][0], i) + acc[0][i / 4][i & 3];
                    if constexpr (GLU) v[i] = glu(v[i], base_at<BB>(base[g][NP - 1], i) + acc[NP - 1][i / 4][i & 3]);
                }
                store8(p.y, yo + n, p.y_bf16, v, n + 8 <= width);
            }
        }
    }
}

// MC: chunks of 32 ranks of max_rank (0: max_rank 16); a group of rows takes
// the code of its own adapter's rank.
template <bool GLU, int MC, bool BB, int G>
__global__ __launch_bounds__(kExpandWaves * kWave) void lora_expand_kernel(LoraArgs p, int splits, int items,
                                                                           int wave_rows, int cgroups, int ngroups) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int q = lane >> 4, col = lane & 15;
    const int cg = blockIdx.x % cgroups, rg = blockIdx.x / cgroups;
    const int tile = wave_rows ? rg * kExpandWaves + wave : rg;
    const int width = GLU ? p.N / 2 : p.N;                 // columns of y
    const int first = (wave_rows ? cg : cg * kExpandWaves + wave) * ngroups * G * kCols;
    const int last = min(width, first + ngroups * G * kCols);
    const int item = blockIdx.y;
    if (tile * kRows >= p.T || first >= width) return;
    const Tile t = tile_rows(p, tile);
    // rows without an adapter are a group of their own (slot -1): they copy
    // base, which in place is nothing to do
    const bool copy = GLU || p.base != p.y;
    uint64_t todo = (copy ? __ballot(t.in) : __ballot(t.slot >= 0)) & 0xFFFFu;
    for (int it = 0; todo; ++it) {
        int lead;
        const int slot = next_slot(t, todo, lead);
        if (items > 1 && it != item) continue;
        const bool mine = t.in && t.slot == slot;
        const int lead_row = __builtin_amdgcn_readlane(t.row, lead);
        const int rank = slot < 0 ? 0 : min(max(p.rank[slot], 0), p.R);
#define GRIM_COLS(CC, HALF) \
    expand_cols<GLU, CC, HALF, BB, G>(p, splits, slot, rank, t.row, lead_row, mine, q, col, first, last, width)
        if (rank == 0) {
            if (copy) GRIM_COLS(0, false);
        } else if constexpr (MC == 0) {
            GRIM_COLS(1, true);
        } else {
            if (MC == 1 || rank <= 32) GRIM_COLS(1, false);
            else if (MC == 2 || rank <= 64) GRIM_COLS((MC < 2 ? MC : 2), false);
            else if (MC == 4 || rank <= 128) GRIM_COLS((MC < 4 ? MC : 4), false);
            else GRIM_COLS(MC, false);
        }
#undef GRIM_COLS
        if (items > 1) break;
    }
}

// K splits over work-groups: as many as leave each wave two steps, for short
// batches; long ones take as many of these as make two work-groups a CU.
int short_splits(int K) {
    const int ksteps = (K + kStep - 1) / kStep, s = (ksteps + 2 * kShrinkWaves - 1) / (2 * kShrinkWaves);
    return s > kMaxSplits ? kMaxSplits : s;
}
constexpr int kShrinkGroups = 512;
int lora_splits(int K, int T) {
    const int s = short_splits(K);
    if (T <= kItemRows) return s;
    const int tiles = (T + kRows - 1) / kRows, w = (kShrinkGroups + tiles - 1) / tiles;
    return s < w ? s : w;
}

template <bool XB>
void shrink(hipStream_t st, const LoraArgs& a, int splits, int items) {
    const int tiles = (a.T + kRows - 1) / kRows, ksteps = (a.K + kStep - 1) / kStep;
#define GRIM_SHRINK(NR)                                                                            \
    do {                                                                                           \
        const int chunks = (a.R + NR * 16 - 1) / (NR * 16);                                        \
        hipLaunchKernelGGL((lora_shrink_kernel<XB, NR>), dim3(tiles, splits, chunks * items),      \
                           dim3(kShrinkWaves * kWave), 0, st, a, splits, ksteps, chunks, items);   \
    } while (0)
    if (a.R <= 16) GRIM_SHRINK(1);
    else if (a.R <= 32) GRIM_SHRINK(2);
    else GRIM_SHRINK(4);
#undef GRIM_SHRINK
}

constexpr int kExpandWavesBusy = 4096;   // waves that fill the chip: 16 a CU

template <bool GLU, int MC, bool BB, int G>
void expand_g(hipStream_t st, const LoraArgs& a, int splits, int items, int64_t waves) {
    const int tiles = (a.T + kRows - 1) / kRows;
    const int width = GLU ? a.N / 2 : a.N, groups = (width + G * kCols - 1) / (G * kCols);
    // a work-group's waves: four row tiles of the same columns, which share
    // B's rows in the L1 (long batches), or four column ranges of one tile;
    // columns of a wave so that the chip is filled about once
    const int wave_rows = a.T > kItemRows;
    int ng = int(waves / G / kExpandWavesBusy);
    ng = ng < 1 ? 1 : ng > groups ? groups : ng;
    const int per = ng * (wave_rows ? 1 : kExpandWaves), cgroups = (groups + per - 1) / per;
    const int rgroups = wave_rows ? (tiles + kExpandWaves - 1) / kExpandWaves : tiles;
    hipLaunchKernelGGL((lora_expand_kernel<GLU, MC, BB, G>), dim3(unsigned(cgroups) * rgroups, items),
                       dim3(kExpandWaves * kWave), 0, st, a, splits, items, wave_rows, cgroups, ng);
}

template <bool GLU, bool BB>
void expand(hipStream_t st, const LoraArgs& a, int splits, int items) {
    const int width = GLU ? a.N / 2 : a.N;
    constexpr int G = GLU ? 2 : 4;
    // waves of one block each (every row tile with as many adapters as it
    // can name); fewer than fill the chip stay at one block
    const int64_t waves = int64_t((a.T + kRows - 1) / kRows) * items * ((width + kCols - 1) / kCols);
    const bool one = waves < kExpandWavesBusy * G;
#define GRIM_EXPAND(MC)                                                              \
    do {                                                                             \
        if (one) expand_g<GLU, MC, BB, 1>(st, a, splits, items, waves);              \
        else expand_g<GLU, MC, BB, G>(st, a, splits, items, waves);                  \
    } while (0)
    if (a.R <= 16) GRIM_EXPAND(0);
    else if (a.R <= 32) GRIM_EXPAND(1);
    else if (a.R <= 64) GRIM_EXPAND(2);
    else if (a.R <= 128) expand_g<GLU, 4, BB, 1>(st, a, splits, items, waves);
    else expand_g<GLU, 8, BB, 1>(st, a, splits, items, waves);
#undef GRIM_EXPAND
}

}  // namespace

size_t lora_workspace_bytes(int K, int R, int T) {
    if (K <= 0 || R <= 0 || T <= 0) return 0;
    // for up to T rows: splits * rows is at most this for every shorter batch
    const size_t most = size_t(short_splits(K)) * T, lng = size_t(kShrinkGroups) * kRows + T;
    return (most < lng || T <= kItemRows ? most : lng) * R * sizeof(float);
}

hipError_t lora_launch(hipStream_t st, const LoraArgs& a) {
    if (a.T <= 0) return hipSuccess;
    const int splits = lora_splits(a.K, a.T);
    // distinct adapters a tile can name, rows without one among them
    const int items = a.T > kItemRows ? 1 : a.T < kRows ? a.T : kRows;
    if (a.x_bf16) shrink<true>(st, a, splits, items);
    else shrink<false>(st, a, splits, items);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.glu) a.base_bf16 ? expand<true, true>(st, a, splits, items) : expand<true, false>(st, a, splits, items);
    else a.base_bf16 ? expand<false, true>(st, a, splits, items) : expand<false, false>(st, a, splits, items);
    return hipGetLastError();
}

}  // namespace grim
