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
typedef short i16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kRows = 16;        // rows of a tile
constexpr int kStep = 64;        // k of one step of a wave: 16 a lane
// Batches of up to this many rows give every distinct adapter of a tile its
// own work-groups.
constexpr int kItemRows = 512;
constexpr int kMaxSplits = 8;

__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
    bf16x8 av, bv;
    __builtin_memcpy(&av, &a, 16);
    __builtin_memcpy(&bv, &b, 16);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(av, bv, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(uint2 a, uint2 b, f32x4 c) {
    i16x4 av, bv;
    __builtin_memcpy(&av, &a, 8);
    __builtin_memcpy(&bv, &b, 8);
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(av, bv, c, 0, 0, 0);
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

// The rows of a tile and the distinct adapters they name.  Lane l (and l+16,
// l+32, l+48) holds row l's adapter, -1 for none.
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

// Lanes of rows still to do; takes out those of the next distinct adapter
// and returns it.
__device__ __forceinline__ int next_slot(const Tile& t, uint64_t& todo) {
    const int lead = int(__builtin_ctzll(todo));
    const int s = __builtin_amdgcn_readlane(t.slot, lead);
    todo &= ~__ballot(t.slot == s);
    return s;
}

template <bool XB, int NR>
__global__ __launch_bounds__(kWaves * kWave) void lora_shrink_kernel(LoraArgs p, int splits, int ksteps,
                                                                     int chunks, int items) {
    __shared__ f32x4 red[kWaves][NR][kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int q = lane >> 4, col = lane & 15;
    const int tile = blockIdx.x, split = blockIdx.y;
    const int chunk = blockIdx.z % chunks, item = blockIdx.z / chunks;
    const Tile t = tile_rows(p, tile);
    uint64_t todo = __ballot(t.slot >= 0) & 0xFFFFu;
    // split's steps: [s0, s1) of ksteps, dealt to the waves in turn
    const int per = (ksteps + splits - 1) / splits;
    const int s0 = split * per, s1 = min(ksteps, s0 + per);

    for (int it = 0; todo; ++it) {
        const int slot = next_slot(t, todo);
        if (items > 1 && it != item) continue;
        const int rank = min(max(p.rank[slot], 0), p.R);
        const int r0 = chunk * NR * 16;
        const int nr = min(NR, (rank - r0 + 15) / 16);      // fragments with live ranks
        if (nr > 0) {
            f32x4 acc[NR] = {};
            const bool mine = t.slot == slot;
            const uint16_t* arow = p.a + (int64_t(slot) * p.R + r0 + col) * p.K;
            for (int s = s0 + wave; s < s1; s += kWaves) {
                const int k = s * kStep + q * 16;
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int kk = k + half * 8;
                    const bool kin = kk < p.K;               // K % 8 == 0
                    u32x4 xv[XB ? 1 : 3] = {};
                    if (mine && kin) {
                        if constexpr (XB) {
                            xv[0] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(p.x) +
                                                                    t.row * p.x_stride + kk);
                        } else {
                            const float* xp = static_cast<const float*>(p.x) + t.row * p.x_stride + kk;
                            const f32x4 lo = *reinterpret_cast<const f32x4*>(xp);
                            const f32x4 hi = *reinterpret_cast<const f32x4*>(xp + 4);
                            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
#pragma unroll
                            for (int l = 0; l < 3; ++l) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) xv[l][i] = cut2(v[2 * i], v[2 * i + 1]);
#pragma unroll
                                for (int i = 0; i < 8; ++i) v[i] = rest(v[i]);
                            }
                        }
                    }
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        if (r < nr) {
                            u32x4 av = {};
                            if (kin)
                                av = *reinterpret_cast<const u32x4*>(arow + int64_t(r) * 16 * p.K + kk);
#pragma unroll
                            for (int l = (XB ? 1 : 3) - 1; l >= 0; --l) acc[r] = mfma32(av, xv[l], acc[r]);
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < NR; ++r) red[wave][r][lane] = acc[r];
            __syncthreads();
            // D of a fragment: lane (q, col) holds ranks 4q .. 4q+3 of row col
            for (int i = threadIdx.x; i < nr * kWave; i += kWaves * kWave) {
                const int r = i / kWave, l = i % kWave;
                f32x4 z = red[0][r][l];
#pragma unroll
                for (int w = 1; w < kWaves; ++w) z += red[w][r][l];
                const int row = tile * kRows + (l & 15);
                // thread i holds row l & 15 of the tile as its own (i % 64 == lane)
                if (mine)
                    *reinterpret_cast<f32x4*>(p.part + (int64_t(split) * p.T + row) * p.R + r0 + r * 16 +
                                              (l >> 4) * 4) = z;
            }
            __syncthreads();
        }
        if (items > 1) break;
    }
}

__device__ __forceinline__ f32x4 load4(const void* p, int64_t o, int bf16) {
    if (bf16) {
        const uint2 u = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + o);
        return f32x4{bits_f(u.x << 16), bits_f(u.x & 0xFFFF0000u), bits_f(u.y << 16), bits_f(u.y & 0xFFFF0000u)};
    }
    return *reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + o);
}

__device__ __forceinline__ void store4(void* p, int64_t o, int bf16, f32x4 v) {
    if (bf16) {
        uint2 u;
        u.x = uint32_t(f32_to_bf16(v[0])) | (uint32_t(f32_to_bf16(v[1])) << 16);
        u.y = uint32_t(f32_to_bf16(v[2])) | (uint32_t(f32_to_bf16(v[3])) << 16);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + o) = u;
    } else {
        *reinterpret_cast<f32x4*>(static_cast<float*>(p) + o) = v;
    }
}

// silu(g) * u with the hardware exp2 / rcp (about 1 ulp each, plus the
// rounding of the exponent, |g| 2^-24 relative).
__device__ __forceinline__ float glu(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// NTL column tiles of 16 a wave (GLU: NTL of the gate half and the NTL
// beside them of the up half).
template <bool GLU, int NTL>
__global__ __launch_bounds__(kWaves * kWave) void lora_expand_kernel(LoraArgs p, int splits, int items,
                                                                     int wave_rows, int cblocks) {
    constexpr int NP = GLU ? 2 : 1;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int q = lane >> 4, col = lane & 15;
    const int cb = blockIdx.x % cblocks, rb = blockIdx.x / cblocks;
    const int tile = wave_rows ? rb * kWaves + wave : rb;
    const int width = GLU ? p.N / 2 : p.N;                 // columns of y
    const int n0 = (wave_rows ? cb : cb * kWaves + wave) * NTL * 16;
    const int item = blockIdx.y;
    if (tile * kRows >= p.T || n0 >= width) return;
    const Tile t = tile_rows(p, tile);
    // rows without an adapter are a group of their own (slot -1): they copy
    // base, which in place is nothing to do
    const bool copy = GLU || p.base != p.y;
    uint64_t todo = (copy ? __ballot(t.in) : __ballot(t.slot >= 0)) & 0xFFFFu;

    for (int it = 0; todo; ++it) {
        const int slot = next_slot(t, todo);
        if (items > 1 && it != item) continue;
        const bool mine = t.in && t.slot == slot;
        const int rank = slot < 0 ? 0 : min(max(p.rank[slot], 0), p.R);
        const float scale = slot < 0 ? 0.0f : p.scale[slot];
        f32x4 acc[NP][NTL] = {};
        for (int r0 = 0; r0 < rank; r0 += 16) {
            const int r = r0 + q * 4;
            // z of this lane's row, ranks r .. r+3, in three bf16 pieces
            f32x4 z = {};
            if (mine && r < rank) {
                const float* zp = p.part + int64_t(t.row) * p.R + r;
                for (int s = 0; s < splits; ++s)
                    z += *reinterpret_cast<const f32x4*>(zp + int64_t(s) * p.T * p.R);
            }
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = r + i < rank ? z[i] * scale : 0.0f;
            uint2 zv[3];
#pragma unroll
            for (int l = 0; l < 3; ++l) {
                zv[l] = make_uint2(cut2(v[0], v[1]), cut2(v[2], v[3]));
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = rest(v[i]);
            }
#pragma unroll
            for (int h = 0; h < NP; ++h) {
#pragma unroll
                for (int j = 0; j < NTL; ++j) {
                    const int n = min(n0 + j * 16 + col, width - 1) + h * width;
                    uint2 bv = make_uint2(0u, 0u);
                    if (r < rank)
                        bv = *reinterpret_cast<const uint2*>(p.b + (int64_t(slot) * p.N + n) * p.R + r);
                    // what lies past the rank is not part of the adapter
                    if (r + 1 >= rank) bv.x &= 0x0000FFFFu;
                    if (r + 2 >= rank) bv.y = 0u;
                    if (r + 3 >= rank) bv.y &= 0x0000FFFFu;
#pragma unroll
                    for (int l = 2; l >= 0; --l) acc[h][j] = mfma16(bv, zv[l], acc[h][j]);
                }
            }
        }
        // D: lane (q, col) holds columns 4q .. 4q+3 of row col
        if (mine) {
#pragma unroll
            for (int j = 0; j < NTL; ++j) {
                const int n = n0 + j * 16 + q * 4;
                if (n < width) {
                    const int64_t o = t.row * p.base_stride + n;
                    f32x4 y = load4(p.base, o, p.base_bf16) + acc[0][j];
                    if constexpr (GLU) {
                        const f32x4 u = load4(p.base, o + width, p.base_bf16) + acc[1][j];
#pragma unroll
                        for (int i = 0; i < 4; ++i) y[i] = glu(y[i], u[i]);
                    }
                    store4(p.y, t.row * p.y_stride + n, p.y_bf16, y);
                }
            }
        }
        if (items > 1) break;
    }
}

// K splits over work-groups: as many as leave each wave two steps, so that
// short batches still fill the chip; one for long batches, whose row tiles
// fill it by themselves.
int lora_splits(int K, int T) {
    if (T > kItemRows) return 1;
    const int ksteps = (K + kStep - 1) / kStep;
    const int s = (ksteps + 2 * kWaves - 1) / (2 * kWaves);
    return s < 1 ? 1 : s > kMaxSplits ? kMaxSplits : s;
}

template <bool XB>
void shrink(hipStream_t st, const LoraArgs& a, int splits, int items) {
    const int tiles = (a.T + kRows - 1) / kRows, ksteps = (a.K + kStep - 1) / kStep;
#define GRIM_SHRINK(NR)                                                                            \
    do {                                                                                           \
        const int chunks = (a.R + NR * 16 - 1) / (NR * 16);                                        \
        hipLaunchKernelGGL((lora_shrink_kernel<XB, NR>), dim3(tiles, splits, chunks * items),      \
                           dim3(kWaves * kWave), 0, st, a, splits, ksteps, chunks, items);         \
    } while (0)
    if (a.R <= 16) GRIM_SHRINK(1);
    else if (a.R <= 32) GRIM_SHRINK(2);
    else GRIM_SHRINK(4);
#undef GRIM_SHRINK
}

template <bool GLU>
void expand(hipStream_t st, const LoraArgs& a, int splits, int items) {
    constexpr int NTL = GLU ? 2 : 4;
    const int tiles = (a.T + kRows - 1) / kRows;
    const int width = GLU ? a.N / 2 : a.N, cols = (width + NTL * 16 - 1) / (NTL * 16);
    const int wave_rows = a.T > kItemRows;
    // a work-group's waves: four row tiles of one column block, which share
    // B's rows in the L1 (long batches), or four column blocks of one tile
    const int cblocks = wave_rows ? cols : (cols + kWaves - 1) / kWaves;
    const int rblocks = wave_rows ? (tiles + kWaves - 1) / kWaves : tiles;
    hipLaunchKernelGGL((lora_expand_kernel<GLU, NTL>), dim3(unsigned(cblocks) * rblocks, items),
                       dim3(kWaves * kWave), 0, st, a, splits, items, wave_rows, cblocks);
}

}  // namespace

size_t lora_workspace_bytes(int K, int R, int T) {
    if (K <= 0 || R <= 0 || T <= 0) return 0;
    // for up to T rows: the short batches, which split K, can need more
    const int S = T < kItemRows ? T : kItemRows;
    const size_t lng = size_t(lora_splits(K, T)) * T, shrt = size_t(lora_splits(K, S)) * S;
    return (lng > shrt ? lng : shrt) * R * sizeof(float);
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
    if (a.glu) expand<true>(st, a, splits, items);
    else expand<false>(st, a, splits, items);
    return hipGetLastError();
}

}  // namespace grim
