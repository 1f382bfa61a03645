// lora_layout.hpp -- where z = A x lies between the adapters' two launches,
// and which of it expand reads.  Integers alone, for the kernels and for host
// code that follows their indexes.
//
// The workspace holds z as expand's operands: per K split, tile of 16 rows
// and chunk of 32 ranks two runs of 64 lanes' four fp32 values, as many chunks
// as expand's code for max_rank reads (max_rank 80 or 96: four).
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define GRIM_HD __host__ __device__
#else
#define GRIM_HD
#endif

namespace grim {

constexpr int kLoraRows = 16;          // rows of a tile
constexpr int kLoraStep = 64;          // shrink: k of one step of a wave
constexpr int kLoraShrinkWaves = 8;
// shrink: batches of up to this many rows give every distinct adapter of a
// tile a work-group of its own.
constexpr int kLoraItemRows = 512;
constexpr int kLoraMaxSplits = 8;
constexpr int kLoraShrinkGroups = 512;
constexpr int kLoraRunBytes = 64 * 16;

// K splits over work-groups: as many as leave each wave one step, for short
// batches; long ones take as many of these as make two work-groups a CU.
constexpr int lora_short_splits(int K) {
    const int ksteps = (K + kLoraStep - 1) / kLoraStep, s = (ksteps + kLoraShrinkWaves - 1) / kLoraShrinkWaves;
    return s > kLoraMaxSplits ? kLoraMaxSplits : s;
}
constexpr int lora_splits(int K, int T) {
    const int s = lora_short_splits(K);
    if (T <= kLoraItemRows) return s;
    const int tiles = (T - 1) / kLoraRows + 1, w = (kLoraShrinkGroups + tiles - 1) / tiles;
    return s < w ? s : w;
}

// expand has code for 1, 2, 4 and 8 chunks of 32 ranks.  mc: the most that
// max_rank's kernel has; an adapter takes the first code that holds its rank,
// which reads all of its chunks of z, live ranks in them or not.
GRIM_HD constexpr int lora_max_chunks(int R) { return R <= 32 ? 1 : R <= 64 ? 2 : R <= 128 ? 4 : 8; }
GRIM_HD constexpr bool lora_code_is(int chunks, int mc, int rank) { return mc <= chunks || rank <= chunks * 32; }

// run `half` of a split's, tile's and chunk's z, counted in runs
GRIM_HD constexpr int64_t lora_z_run(int R, int T, int split, int64_t tile, int chunk, int half) {
    const int64_t tiles = (T + kLoraRows - 1) / kLoraRows;
    return ((split * tiles + tile) * lora_max_chunks(R) + chunk) * 2 + half;
}
constexpr size_t lora_workspace_bytes(int K, int R, int T) {
    if (K <= 0 || R <= 0 || T <= 0) return 0;
    // for up to T rows: splits * rows is at most this for every shorter batch
    const size_t rows = (size_t(T) + kLoraRows - 1) / kLoraRows * kLoraRows, most = lora_short_splits(K) * rows;
    const size_t lng = size_t(kLoraShrinkGroups) * kLoraRows + rows;
    return (most < lng || T <= kLoraItemRows ? most : lng) * (lora_max_chunks(R) * 32) * sizeof(float);
}

}  // namespace grim
