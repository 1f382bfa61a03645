// proj4.hpp -- host interface of the dense 4-bit projections.
#pragma once

#include "common.hpp"

namespace grim {

// y_t = base_t + W x_t, W [N][K] INT4, INT4_F16 or MXFP4; with glu, N = 2I
// and y_t [I] = silu(v[i]) * v[I + i] of v = W x_t.
struct Proj4Args {
    WView w;
    int fmt, N, K;
    const void* x;            // [T] rows, x_stride elements apart
    const void* base;         // or null
    void* y;
    int64_t x_stride, base_stride, y_stride;
    int x_bf16, base_bf16, y_bf16;
    int T, glu;
    void* ws;                 // workspace: sums over parts of K
};

// What a launch tells its kernel.
struct Proj4Dev {
    Proj4Args a;
    float* part;              // [kw][T][tiles][16]
    int tile_rows, col_tiles; // rows of x a work-group takes, and how many such
    int tiles;                // 16-row weight tiles
    int sets, stride;         // ... by the work-group, and the distance of one's
    int kw, kw_blocks;        // parts of K by work-groups, and blocks of 128 of one
    int ks, wave_blocks;      // log2 of the waves that share a tile, and blocks of one in a slab
    int nb, slab;             // blocks along K, and of those whose x is in the LDS together
    int s_at, red_at;         // LDS offsets: scales, partial sums
    int half;                 // outputs: N, or N / 2 with glu
};

constexpr int kProj4MaxRows = 1 << 18;     // parts of 8 rows, 65535 of which a grid takes
// Sums over at most kProj4Parts parts of K are of at most this many (tile of 16 outputs, part of K,
// work-group's rows of x), whose rows are at most kProj4TileRows.
constexpr int kProj4Tiles = 4096, kProj4TileRows = 32, kProj4Parts = 8;
inline size_t proj4_workspace_bytes(int rows) {
    return size_t(kProj4Tiles) * 64 * (rows < kProj4TileRows ? rows : kProj4TileRows);
}

hipError_t proj4_sum_launch(hipStream_t st, const Proj4Dev& p);

// by INT4 group size, 0: MXFP4
hipError_t proj4_launch_g0(hipStream_t st, const Proj4Args& a);
hipError_t proj4_launch_g32(hipStream_t st, const Proj4Args& a);
hipError_t proj4_launch_g64(hipStream_t st, const Proj4Args& a);
hipError_t proj4_launch_g128(hipStream_t st, const Proj4Args& a);
hipError_t proj4_launch(hipStream_t st, const Proj4Args& a);

}  // namespace grim
