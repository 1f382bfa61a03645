// lora.hip -- low-rank adapters of many requests beside a shared projection:
//   y_t = base_t + scale_a B_a (A_a x_t),  a = row_slot[t]
// in two launches (one for a few rows of small adapters).  shrink: z_t =
// A_a x_t, K split over waves and work-groups, fp32 partials to the
// workspace.  expand: the partials are summed in a fixed order, scaled,
// multiplied with B_a and added to base (and, for a gate|up projection,
// SwiGLU'd) on the way to y.
//
// Both are memory bound at every size (2 r operations an element of x and y
// read or written), and their rows go through the LDS on the way to the
// matrix cores, so that adjacent lanes ask memory for adjacent pieces.  Rows
// of a tile that name different adapters are done one distinct adapter after
// the other, or by work-groups of their own.
//
// Where it stands (us, shrink + expand, and what their bytes take at the 4.94
// TB/s of a large copy): 4096 rows of 9 requests, 2048 -> 7168, rank 64 of
// mixed ranks, bf16: 13 + 37 (28; base copied to y by the same loop 25.5);
// 2001 rows of 5, 2880 -> 2 x 2880, rank 16, fp32: 11 + 19 (19); 48 mixed
// rows of 32 adapters, 2048 -> 7168: 5 + 10 (3.3); one row, 768 -> 2048: 5 in
// one launch, a chain of dependent loads.
//
// Long batches should hold their rows in runs of one adapter: rows are tiled
// in the order they come in, and a tile reads A and B once for every adapter
// it names.  2048 -> 7168, 32 adapters of rank 64, bf16, both launches: 4096
// rows in 9 runs 52 us, in no order 367; 1024 in no order 117, 512 63, 256 40.
//
// fp32 values are multiplied exactly: an fp32 x (and z) is the sum of three
// bf16 pieces of 8 significant bits, cut off, not rounded, so each rest is
// exact; with bf16 weights every product is exact in the fp32 accumulator.
#include "lora.hpp"

namespace grim {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kRows = kLoraRows;
constexpr int kStep = kLoraStep;     // 16 k a lane
constexpr int kShrinkWaves = kLoraShrinkWaves;
constexpr int kExpandWaves = 4;

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

// The rows of a tile of ROWS (16 or 64) and the adapters they name: lane l
// holds row l % ROWS's.
struct Tile {
    int row;      // this lane's row, clamped into the batch
    bool in;      // the row exists
    int slot;     // its adapter or -1
};

template <int ROWS>
__device__ __forceinline__ Tile tile_rows(const LoraArgs& p, int tile) {
    const int64_t r = int64_t(tile) * ROWS + (threadIdx.x & (ROWS - 1));
    Tile t;
    t.in = r < p.T;
    t.row = t.in ? int(r) : p.T - 1;
    const int s = p.row_slot[t.row];
    t.slot = t.in && s >= 0 && s < p.slots ? s : -1;
    return t;
}

// Where this lane's row stands among the distinct adapters that the rows `of`
// name (no adapter counts as one more), in the order of their first rows.
// Equal slots are found by a ballot a bit of their numbers, so that 64
// adapters cost what two do (48 mixed rows of 32 adapters, 2048 -> 7168: 15.4
// us; counted one after the other 17.7).
struct Place {
    uint64_t rows;   // the rows of its adapter, a bit each
    bool first;      // it is the first of them
    int index;       // first: its adapter's place
    int count;       // of distinct adapters
};

__device__ __forceinline__ Place tile_places(const LoraArgs& p, const Tile& t, uint64_t of) {
    const int lane = threadIdx.x & (kWave - 1);
    Place w;
    w.rows = of;
    const uint32_t s = uint32_t(t.slot + 1);
    for (uint32_t bit = 1; bit <= uint32_t(p.slots); bit <<= 1) {   // slots < 2^31: ends at 2^31
        const uint64_t set = __ballot((s & bit) != 0);
        w.rows &= (s & bit) ? set : ~set;
    }
    w.first = ((of >> lane) & 1) && (w.rows & ((uint64_t(1) << lane) - 1)) == 0;
    const uint64_t firsts = __ballot(w.first);
    w.index = __builtin_amdgcn_mbcnt_hi(uint32_t(firsts >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(firsts), 0));
    w.count = __popcll(firsts);
    return w;
}

// The next distinct adapter among the rows `todo`, its first row's lane in
// lead; takes its rows out of todo.
__device__ __forceinline__ int next_slot(const Tile& t, uint64_t& todo, int& lead) {
    lead = int(__builtin_ctzll(todo));
    const int s = __builtin_amdgcn_readlane(t.slot, lead);
    todo &= ~__ballot(t.slot == s);
    return s;
}

// An adapter that a tile names.
struct Group {
    uint64_t rows;   // its rows, a bit each
    int slot;        // -1: the rows without an adapter
    int rank;
    float scale;
};

// The distinct adapters of the rows `of` to the LDS (one entry a row at
// most); returns how many.  Ranks and scales are loaded for all rows at once.
// All waves of the work-group come here with the same rows; a barrier at the
// end.
__device__ __forceinline__ int tile_groups(const LoraArgs& p, const Tile& t, uint64_t of, Group* out) {
    const int at = max(t.slot, 0);
    const int rank = p.rank[at];
    const float scale = p.scale[at];
    const Place w = tile_places(p, t, of);
    if (w.first && threadIdx.x < kWave)
        out[w.index] = Group{w.rows, t.slot, t.slot >= 0 ? min(max(rank, 0), p.R) : 0, scale};
    __syncthreads();
    return w.count;
}
// entry g, the same on every lane
__device__ __forceinline__ Group group_at(const Group* groups, int g) {
    const Group v = groups[g];
    const uint32_t lo = __builtin_amdgcn_readfirstlane(uint32_t(v.rows)), hi = __builtin_amdgcn_readfirstlane(uint32_t(v.rows >> 32));
    return Group{(uint64_t(hi) << 32) | lo, __builtin_amdgcn_readfirstlane(v.slot), __builtin_amdgcn_readfirstlane(v.rank),
                 bits_f(__builtin_amdgcn_readfirstlane(f_bits(v.scale)))};
}

__device__ __forceinline__ void wave_sync_lds() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Of a chunk's two runs of z in the workspace expand's lane (q, col) takes
// ranks 8 q .. 8 q + 3 of row col from the first, the next four from the
// second.  This is where shrink's lane (q, col), with ranks 4 q .. 4 q + 3 of
// fragment f, puts its own.
__device__ __forceinline__ f32x4* z_run(const LoraArgs& p, int split, int64_t tile, int chunk, int half) {
    return reinterpret_cast<f32x4*>(p.part) + lora_z_run(p.R, p.T, split, tile, chunk, half) * kWave;
}
__device__ __forceinline__ f32x4* z_at(const LoraArgs& p, int split, int64_t tile, int f, int q, int col) {
    return z_run(p, split, tile, f >> 1, q & 1) + ((f & 1) * 2 + (q >> 1)) * 16 + col;
}

// ------------------------------------------------------------------ shrink

// A wave's share of z = A x: NF fragments of 16 ranks, the K steps s0, s0 +
// kShrinkWaves, ... < s1, the next one's loads in flight while one is used.
// As in expand, A and x go through the LDS so that adjacent lanes load
// adjacent pieces of a row (as operands every lane would load from a row of
// its own: 64 tag look-ups an instruction; 16.4 against 10.9 us at 4096
// rows of one adapter, K 2048, rank 64).  A row's pieces are permuted by its
// number, so that the 16 rows of an operand lie in different banks.  All
// loads are unconditional: k past K reads the row's end under an x of zero, ranks past
// the slot read its last row and are not stored.
template <bool XB, int NF>
__device__ __forceinline__ void shrink_steps(const LoraArgs& p, int slot, int r0, uint32_t mask, int64_t row0,
                                             int lead, int lane, int s0, int s1, u32x4* lds, f32x4 (&acc)[4]) {
    constexpr int XP = XB ? 8 : 16, XL = XP / 4;          // pieces of an x row, its loads
    const int q = lane >> 4, col = lane & 15;
    u32x4* xl = lds + NF * 16 * 8;
    const char* as = reinterpret_cast<const char*>(p.a + (int64_t(slot) * p.R + r0) * p.K);
    const char* xs = static_cast<const char*>(p.x) + row0 * p.x_stride * (XB ? 2 : 4);
    uint32_t ao[NF * 2], xo[XL];
#pragma unroll
    for (int i = 0; i < NF * 2; ++i) ao[i] = uint32_t(min(i * 8 + (lane >> 3), p.R - r0 - 1)) * p.K * 2u;
#pragma unroll
    for (int i = 0; i < XL; ++i) {
        // rows of another adapter read the group's first row instead: their
        // column of the product is not used
        const int r = i * (kWave / XP) + lane / XP;
        xo[i] = uint32_t((mask >> r) & 1 ? r : lead) * uint32_t(p.x_stride) * (XB ? 2u : 4u);
    }
    u32x4 a[NF * 2], x[XL];
    auto load = [&](int s) {
        const uint32_t ak = min(s * kStep + (lane & 7) * 8, p.K - 8) * 2u;
#pragma unroll
        for (int i = 0; i < NF * 2; ++i) a[i] = *reinterpret_cast<const u32x4*>(as + (ao[i] + ak));
        const uint32_t xk = XB ? ak : min(s * kStep + (lane & 15) * 4, p.K - 4) * 4u;
#pragma unroll
        for (int i = 0; i < XL; ++i) x[i] = *reinterpret_cast<const u32x4*>(xs + (xo[i] + xk));
    };
    if (s0 < s1) load(s0);
#pragma nounroll
    for (int s = s0; s < s1; s += kShrinkWaves) {
        const bool in = s * kStep + (lane % XP) * (XB ? 8 : 4) < p.K;
#pragma unroll
        for (int i = 0; i < NF * 2; ++i) lds[(i * 8 + (lane >> 3)) * 8 + ((lane & 7) ^ (lane >> 3))] = a[i];
#pragma unroll
        for (int i = 0; i < XL; ++i) {
            const int r = i * (kWave / XP) + lane / XP;
            xl[r * XP + ((lane % XP) ^ (r & (XP - 1)))] = in ? x[i] : u32x4{0, 0, 0, 0};
        }
        wave_sync_lds();
        load(min(s + kShrinkWaves, s1 - 1));               // past the end: memory read already
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u32x4 xv[3];
            if constexpr (XB) {
                xv[0] = xl[col * 8 + ((h * 4 + q) ^ (col & 7))];
            } else {
                const u32x4 lo = xl[col * 16 + ((h * 8 + q * 2) ^ col)], hi = xl[col * 16 + ((h * 8 + q * 2 + 1) ^ col)];
                float v[8];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[i] = bits_f(lo[i]);
                    v[4 + i] = bits_f(hi[i]);
                }
                pieces(v, xv);
            }
            u32x4 av[NF];
#pragma unroll
            for (int r = 0; r < NF; ++r) av[r] = lds[(r * 16 + col) * 8 + ((h * 4 + q) ^ (col & 7))];
#pragma unroll
            for (int l = XB ? 0 : 2; l >= 0; --l)
#pragma unroll
                for (int r = 0; r < NF; ++r) acc[r] = mfma(av[r], xv[l], acc[r]);
        }
        wave_sync_lds();
    }
}

// NR fragments of 16 ranks a work-group (max_rank 16, 32 or more).
template <bool XB, int NR>
__global__ __launch_bounds__(kShrinkWaves * kWave) void lora_shrink_kernel(LoraArgs p, int splits, int ksteps,
                                                                           int chunks, int items) {
    // a wave's A and x; at the end its fragments of z, for the sum over waves
    __shared__ u32x4 lds[kShrinkWaves][NR * 16 * 8 + kRows * (XB ? 8 : 16)];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int q = lane >> 4, col = lane & 15;
    const int tile = blockIdx.x, split = blockIdx.y;
    const int chunk = blockIdx.z % chunks, item = blockIdx.z / chunks;
    const Tile t = tile_rows<kRows>(p, tile);
    uint64_t todo = __ballot(t.slot >= 0) & 0xFFFFu;
    if (items > 1) {                                        // one of them, if there are as many
        const Place w = tile_places(p, t, todo);
        const uint64_t is = __ballot(w.first && w.index == item);
        todo = is ? __builtin_amdgcn_readlane(uint32_t(w.rows), int(__builtin_ctzll(is))) : 0;
    }
    // the split's steps [s0, s1), dealt to the waves in turn
    const int per = (ksteps + splits - 1) / splits;
    const int s0 = split * per + wave, s1 = min(ksteps, (split + 1) * per);
    const int r0 = chunk * NR * 16;

    while (todo) {
        int lead;
        const int slot = next_slot(t, todo, lead);
        const int rank = min(max(p.rank[slot], 0), p.R);
        const int nr = min(NR, (rank - r0 + 15) / 16);      // fragments with live ranks
        if (nr > 0) {
            f32x4 acc[4] = {};
            const uint32_t mask = uint32_t(__ballot(t.slot == slot)) & 0xFFFFu;
            int ln = lane;                                  // opaque: see expand_cols
            asm volatile("" : "+v"(ln));
#define GRIM_STEPS(NF) \
    shrink_steps<XB, NF>(p, slot, r0, mask, int64_t(tile) * kRows, lead, ln, s0, s1, lds[wave], acc)
            if (NR == 1 || nr == 1) GRIM_STEPS(1);
            else if (NR == 2 || nr == 2) GRIM_STEPS(2);
            else GRIM_STEPS(4);
#undef GRIM_STEPS
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (r < nr) __builtin_memcpy(&lds[wave][r * kWave + lane], &acc[r], 16);
            __syncthreads();
            // D of a fragment: lane (q, col) holds ranks 4q .. 4q+3 of row
            // col, and wave r sums fragment r over the waves
            if (wave < nr) {
                f32x4 z = {};
#pragma unroll
                for (int w = 0; w < kShrinkWaves; ++w) {
                    f32x4 o;
                    __builtin_memcpy(&o, &lds[w][wave * kWave + lane], 16);
                    z += o;
                }
                if (t.slot == slot) *z_at(p, split, tile, (r0 >> 4) + wave, q, col) = z;
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------ expand

// silu(g) * u with the hardware exp2 / rcp (about 1 ulp each, plus the
// rounding of the exponent, |g| 2^-24 relative).
__device__ __forceinline__ float glu(float g, float u) {
    const float e = __builtin_amdgcn_exp2f(g * -1.44269504088896341f);
    return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

// two fp32 to bf16, nearest even (the hardware conversion)
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    const bf16x2 b = __builtin_convertvector(f32x2{lo, hi}, bf16x2);
    uint32_t u;
    __builtin_memcpy(&u, &b, 4);
    return u;
}

// W columns of a base row as loaded (2 or 4, fp32 or bf16).
template <bool BB, int W>
struct Base {
    uint32_t v[BB ? W / 2 : W];
};

// Memory is addressed as a pointer all lanes share and 32 bits of byte
// offset (the entry points bound strides and adapters so that it fits).
template <bool BB, int W>
__device__ __forceinline__ void load_base(Base<BB, W>& b, const void* base, uint32_t off) {
    __builtin_memcpy(b.v, __builtin_assume_aligned(static_cast<const char*>(base) + off, BB ? 2 * W : 4 * W), sizeof b.v);
}

template <bool BB, int W>
__device__ __forceinline__ float base_at(const Base<BB, W>& b, int i) {
    if constexpr (BB) return i & 1 ? bits_f(b.v[i / 2] & 0xFFFF0000u) : bits_f(b.v[i / 2] << 16);
    else return bits_f(b.v[i]);
}

// columns at element `off` past y
template <int W>
__device__ __forceinline__ void store_cols(void* y, uint32_t off, int bf16, const float (&v)[W]) {
    if (bf16) {
        uint32_t u[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; ++i) u[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
        __builtin_memcpy(__builtin_assume_aligned(static_cast<char*>(y) + off * 2u, 2 * W), u, sizeof u);
    } else {
        __builtin_memcpy(__builtin_assume_aligned(static_cast<char*>(y) + off * 4u, 4 * W), v, sizeof v);
    }
}

// A work-group takes 64 rows, 16 a wave.  A block is 64 rows of B: 64 columns
// of y, or 32 and the 32 beside them of the up half.  Four MFMA tiles of 16;
// tile j's column n is column 4 n + j of the block (gate|up: column 2 n +
// j % 2 of half j / 2), so that a lane's results are adjacent columns and a
// row's base and y are runs of memory over adjacent lanes.
//
// B goes through the LDS, once for the four waves: as operands (lane =
// column, 16 bytes of its ranks) its loads would touch a row a lane, 64 tag
// look-ups an instruction, which bound this kernel; adjacent lanes read
// adjacent pieces instead.  A row of the LDS is 16 bytes longer than its
// ranks, an odd number of pieces: the 16 rows of a tile's read lie in
// different banks.
constexpr int kExpandRows = kExpandWaves * kRows;
template <bool GLU>
__device__ __forceinline__ int block_col(int r) {      // block row -> its column of y (and half)
    return GLU ? (r & 31) : r;
}
template <bool GLU>
__device__ __forceinline__ int lds_row(int r) {        // -> its place: tile by tile
    return GLU ? ((r >> 5) * 2 + (r & 1)) * 16 + ((r & 31) >> 1) : (r & 3) * 16 + (r >> 2);
}

// The wave's rows `mask` of one adapter (of none: slot -1) against columns
// [first, last) of y: CC chunks of 32 ranks (HALF: max_rank 16, where an
// instruction's 32 k hold the 16 ranks twice, under two pieces of z; CC 0:
// base alone).  All NW waves of the work-group come here together, also those
// without such rows (mask 0), which only bring B.  ZL: z of the wave's rows
// lies in the LDS, in the workspace's order.
template <bool GLU, int CC, bool HALF, bool BB, int NW, bool ZL>
__device__ __forceinline__ void expand_cols(const LoraArgs& p, int splits, int slot, int rank, float scale,
                                            uint32_t mask, int64_t row0, int first, int last, int width, u32x4* lds,
                                            const f32x4* zl) {
    constexpr int kThreads = NW * kWave;
    constexpr int W = GLU ? 2 : 4, NP = GLU ? 2 : 1, C = CC ? CC : 1;
    constexpr int PH = C < 2 ? C : 2;                 // chunks of one pass through the LDS
    constexpr int P = HALF ? 2 : PH * 4;              // pieces of a row in a pass
    constexpr int kPitch = P + 1, kBuffer = 64 * kPitch;
    constexpr int L = (64 * P + kThreads - 1) / kThreads;   // loads a thread and pass
    // (opaque: what hangs on the lane is formed here, not kept in registers
    // for every rank's code from before the loop over the adapters)
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));
    const int lane = tid & (kWave - 1), q = lane >> 4, col = lane & 15;

    // the four rows of this lane's results; rows that are not stored read
    // the first stored one's base
    constexpr uint32_t ES = BB ? 2 : 4;
    const char* base0 = static_cast<const char*>(p.base) + row0 * p.base_stride * ES;
    char* y0 = static_cast<char*>(p.y) + row0 * p.y_stride * (p.y_bf16 ? 2 : 4);
    const uint32_t brow = uint32_t(p.base_stride) * ES, yrow = uint32_t(p.y_stride);
    const int lead = mask ? __builtin_ctz(mask) : 0;
    auto mine = [&](int i) { return (mask >> (q * 4 + i)) & 1; };
    auto row = [&](int i) { return uint32_t(mine(i) ? q * 4 + i : lead); };

    // a pass's B: thread reads piece % P of rows tid / P, + 256 / P
    const uint16_t* bs = p.b + int64_t(slot) * p.N * p.R;
    auto load_b = [&](u32x4 (&d)[L], int n0, int c0) {
        const uint32_t pitch = p.R * 2u, r = min((HALF ? 0 : c0 * 32) + (tid % P) * 8, p.R - 8) * 2u;
        const uint32_t end = (width - 1) * pitch + r;      // the last column's
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int br = (i * (kThreads / P) + tid / P) & 63;
            const uint32_t o = min((n0 + block_col<GLU>(br)) * pitch + r, end) + (GLU && br >= 32 ? width * pitch : 0u);
            d[i] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(bs) + o);
        }
    };
    auto load_y = [&](Base<BB, W> (&d)[NP][4], int n0) {
        const uint32_t n = min(n0 + col * W, width - W) * ES;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < NP; ++h) load_base<BB, W>(d[h][i], base0 + h * width * ES, row(i) * brow + n);
    };

    constexpr int kBlock = GLU ? 32 : 64;
    u32x4 b[L];
    Base<BB, W> base[NP][4] = {};
    if (mask) load_y(base, first);
    if constexpr (CC > 0) load_b(b, first, 0);

    // z of row `col`, ranks q * 8 .. + 7 of each chunk, scaled and without
    // what lies past the rank, in three pieces (rows of other adapters hold
    // anything: their rows of the product are not stored)
    u32x4 zv[C][3];
    if constexpr (CC > 0) {
        if (mask) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int r = HALF ? (q & 1) * 8 : c * 32 + q * 8;
                const int at = HALF ? lane & 31 : lane;
                f32x4 lo = {}, hi = {};
                if constexpr (ZL) {
                    lo = zl[c * 2 * kWave + at];
                    hi = zl[(c * 2 + 1) * kWave + at];
                } else {
                    const int64_t apart = z_run(p, 1, 0, 0, 0) - z_run(p, 0, 0, 0, 0);
                    const f32x4* z0 = z_run(p, 0, row0 / kRows, c, 0) + at;
                    for (int s = 0; s < splits; s += 2) {
                        const f32x4* z1 = z0 + s * apart;
                        const f32x4* z2 = z0 + min(s + 1, splits - 1) * apart;
                        const f32x4 l1 = z1[0], h1 = z1[kWave], l2 = z2[0], h2 = z2[kWave];
                        lo += l1;
                        hi += h1;
                        if (s + 1 < splits) {
                            lo += l2;
                            hi += h2;
                        }
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
    }

    int turn = 0;
#pragma nounroll
    for (int n0 = first; n0 < last; n0 += kBlock) {
        const int next = n0 + kBlock < last ? n0 + kBlock : n0;   // past the end: memory read already
        // -0: what adds nothing leaves base's own sign of zero
        f32x4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = f32x4{-0.0f, -0.0f, -0.0f, -0.0f};
        Base<BB, W> cur[NP][4];
#pragma unroll
        for (int h = 0; h < NP; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) cur[h][i] = base[h][i];
        if constexpr (CC > 0) {
#pragma unroll
            for (int c0 = 0; c0 < C; c0 += PH, turn ^= 1) {
                // what lies past the rank is not part of the adapter
                const int r = (HALF ? 0 : c0 * 32) + (tid % P) * 8;
                if (rank < c0 * 32 + P * 8) {
#pragma unroll
                    for (int i = 0; i < L; ++i)
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            uint32_t w = b[i][d];
                            w = r + 2 * d + 1 < rank ? w : w & 0xFFFFu;
                            b[i][d] = r + 2 * d < rank ? w : 0u;
                        }
                }
                // two buffers in turn: who writes one has passed the barrier
                // that every wave reached after its reads of it
                u32x4* buf = lds + turn * kBuffer;
#pragma unroll
                for (int i = 0; i < L; ++i) {
                    const int br = i * (kThreads / P) + tid / P;
                    if (64 * P % kThreads == 0 || br < 64) buf[lds_row<GLU>(br) * kPitch + tid % P] = b[i];
                }
                __syncthreads();
                const bool more = c0 + PH < C;
                load_b(b, more ? n0 : next, more ? c0 + PH : 0);
                if (!mask) continue;
                if (c0 == 0) load_y(base, next);
#pragma unroll
                for (int c = 0; c < PH; ++c) {
                    u32x4 d[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) d[j] = buf[(j * 16 + col) * kPitch + (HALF ? q & 1 : c * 4 + q)];
#pragma unroll
                    for (int l = HALF ? 1 : 2; l >= 0; --l)
#pragma unroll
                        for (int j = 0; j < 4; ++j) acc[j] = mfma(zv[c0 + c][l], d[j], acc[j]);
                }
            }
        } else {
            if (mask) load_y(base, next);
        }
        // D of tile j: lane (q, col) holds rows 4q .. 4q+3 of its column
        const int n = n0 + col * W;
        if (mask && n < width) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v[W];
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    v[w] = base_at<BB, W>(cur[0][i], w) + acc[w][i];
                    if constexpr (GLU) v[w] = glu(v[w], base_at<BB, W>(cur[NP - 1][i], w) + acc[2 + w][i]);
                }
                if (mine(i)) store_cols<W>(y0, row(i) * yrow + n, p.y_bf16, v);
            }
        }
    }
    if constexpr (CC > 0) __syncthreads();             // the next adapter starts at the first buffer
}

// MC: chunks of 32 ranks of max_rank (0: max_rank 16); a group of rows takes
// the code of its own adapter's rank.
//
// A tile's work is its distinct adapters (rows with none, where there is
// something to do for them, count as one more) times the blocks of columns,
// adapter by adapter; `share` work-groups split it evenly into runs of at
// least nblocks.  How many adapters a tile names is known here only: one for
// most tiles of a prompt, dozens for sequences decoding together.
// (Rank 64 in 3 waves a SIMD, without spills: 48 mixed rows 15.4 us, in 4
// 15.7; long batches alike.)
template <bool GLU, int MC, bool BB>
__global__ __launch_bounds__(kExpandWaves* kWave)
    __attribute__((amdgpu_waves_per_eu(MC > 2 ? 2 : 3))) void lora_expand_kernel(
    LoraArgs p, int splits, int share, int nblocks) {
    constexpr int kMaxPitch = (MC == 0 ? 2 : MC == 1 ? 4 : 8) + 1;
    __shared__ u32x4 lds[2 * 64 * kMaxPitch];
    const int wave = threadIdx.x / kWave;
    // part by part over the tiles, the last ones first: those that a tile of
    // one adapter leaves unused end at once, on every XCD alike, and those of
    // tiles of two start before the others
    const int tiles = gridDim.x / share, part = share - 1 - blockIdx.x / tiles, tile = blockIdx.x % tiles;
    constexpr int kBlock = GLU ? 32 : 64;
    const int width = GLU ? p.N / 2 : p.N;                 // columns of y
    const int blocks = (width + kBlock - 1) / kBlock;
    const Tile t = tile_rows<kExpandRows>(p, tile);
    const int64_t row0 = int64_t(tile) * kExpandRows + wave * kRows;
    // rows without an adapter copy base, which in place is nothing to do
    const bool copy = GLU || p.base != p.y;
    __shared__ Group groups[kExpandRows];
    const int count = tile_groups(p, t, copy ? __ballot(t.in) : __ballot(t.slot >= 0), groups);
    const int64_t total = int64_t(count) * blocks;
    const int64_t run = max(int64_t(nblocks), (total + share - 1) / share);
    int64_t at = part * run;
    const int64_t end = min(total, at + run);
    while (at < end) {
        const int g = int(at / blocks), b0 = int(at - int64_t(g) * blocks);
        const int n = int(min(end - at, int64_t(blocks - b0)));
        at += n;
        const int first = b0 * kBlock, last = min(width, first + n * kBlock);
        const Group gr = group_at(groups, g);
        const int rank = gr.rank;
        const uint32_t mask = uint32_t(gr.rows >> (wave * kRows)) & 0xFFFFu;
#define GRIM_COLS(CC, HALF) \
    expand_cols<GLU, CC, HALF, BB, kExpandWaves, false>(p, splits, gr.slot, rank, gr.scale, mask, row0, first, last, width, lds, nullptr)
        if (rank == 0) {
            if (copy) GRIM_COLS(0, false);
        } else if constexpr (MC == 0) {
            GRIM_COLS(1, true);
        } else {
            if (lora_code_is(1, MC, rank)) GRIM_COLS(1, false);
            else if (lora_code_is(2, MC, rank)) GRIM_COLS((MC < 2 ? MC : 2), false);
            else if (lora_code_is(4, MC, rank)) GRIM_COLS((MC < 4 ? MC : 4), false);
            else GRIM_COLS(MC, false);
        }
#undef GRIM_COLS
    }
}

// --------------------------------------------------------- both in one launch

// A few rows (one tile of 16) of small adapters: every work-group forms the z
// that it needs itself, all of K over its eight waves, and goes on to its
// columns.  What it costs is A once a work-group from the L2, what it saves
// is a launch and the trip of z through memory.
template <bool GLU, bool XB, bool BB, int NR>
__global__ __launch_bounds__(kShrinkWaves* kWave) void lora_one_kernel(LoraArgs p, int share) {
    constexpr int MC = NR == 1 ? 0 : NR == 2 ? 1 : 2;
    constexpr int kMaxPitch = (MC == 0 ? 2 : MC == 1 ? 4 : 8) + 1, kRegion = NR * 16 * 8 + kRows * (XB ? 8 : 16);
    // shrink's regions; then expand's two buffers
    __shared__ u32x4 lds[kShrinkWaves][kRegion];
    static_assert(kShrinkWaves * kRegion >= 2 * 64 * kMaxPitch, "expand's buffers lie in shrink's regions");
    __shared__ f32x4 zl[(MC < 2 ? 1 : 2) * 2 * kWave];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int q = lane >> 4, col = lane & 15;
    constexpr int kBlock = GLU ? 32 : 64;
    const int width = GLU ? p.N / 2 : p.N;
    const int blocks = (width + kBlock - 1) / kBlock, ksteps = (p.K + kStep - 1) / kStep;
    const Tile t = tile_rows<kRows>(p, 0);
    const bool copy = GLU || p.base != p.y;
    __shared__ Group groups[kRows];
    const int count = tile_groups(p, t, (copy ? __ballot(t.in) : __ballot(t.slot >= 0)) & 0xFFFFu, groups);
    const int total = count * blocks, run = (total + share - 1) / share;
    int at = int(blockIdx.x) * run;
    const int end = min(total, at + run);
    while (at < end) {
        const int g = at / blocks, b0 = at - g * blocks, n = min(end - at, blocks - b0);
        at += n;
        const int first = b0 * kBlock, last = min(width, first + n * kBlock);
        const Group gr = group_at(groups, g);
        const int rank = gr.rank;
        const uint32_t mask = uint32_t(gr.rows);
        const int nr = min(NR, (rank + 15) / 16);
        if (nr > 0) {
            f32x4 acc[4] = {};
            int ln = lane;                                  // opaque: see expand_cols
            asm volatile("" : "+v"(ln));
#define GRIM_STEPS(NF) shrink_steps<XB, NF>(p, gr.slot, 0, mask, 0, __builtin_ctz(mask), ln, wave, ksteps, lds[wave], acc)
            if (NR == 1 || nr == 1) GRIM_STEPS(1);
            else if (NR == 2 || nr == 2) GRIM_STEPS(2);
            else GRIM_STEPS(4);
#undef GRIM_STEPS
#pragma unroll
            for (int r = 0; r < NR; ++r)
                if (r < nr) __builtin_memcpy(&lds[wave][r * kWave + lane], &acc[r], 16);
            __syncthreads();
            if (wave < nr) {
                f32x4 z = {};
#pragma unroll
                for (int w = 0; w < kShrinkWaves; ++w) {
                    f32x4 o;
                    __builtin_memcpy(&o, &lds[w][wave * kWave + lane], 16);
                    z += o;
                }
                zl[((wave >> 1) * 2 + (q & 1)) * kWave + ((wave & 1) * 2 + (q >> 1)) * 16 + col] = z;
            }
            __syncthreads();
        }
        const uint32_t mine = wave == 0 ? mask : 0;
#define GRIM_COLS(CC, HALF) \
    expand_cols<GLU, CC, HALF, BB, kShrinkWaves, true>(p, 1, gr.slot, rank, gr.scale, mine, 0, first, last, width, lds[0], zl)
        if (rank == 0) {
            if (copy) GRIM_COLS(0, false);
        } else if constexpr (MC == 0) {
            GRIM_COLS(1, true);
        } else {
            if (MC == 1 || rank <= 32) GRIM_COLS(1, false);
            else GRIM_COLS(MC, false);
        }
#undef GRIM_COLS
        __syncthreads();                                    // the next z takes the buffers and zl
    }
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

// expand's work-groups, 3 or 4 a CU at once: runs of blocks of two of them while
// every tile is one adapter's, which leaves room for the tiles of two (4096
// rows of 9 requests, 2048 -> 7168: 34.8 us; runs that fill the chip: 40.4);
// three of them share out tiles of many (48 mixed rows of 32 adapters:
// 15.4 us in all; with two or four 18.4, 17.0).  Measured at rank 64 alone;
// above 64 a CU holds two or three work-groups.
constexpr int kExpandRuns = 512, kExpandGroups = 768;

template <bool GLU, bool BB>
void expand(hipStream_t st, const LoraArgs& a, int splits) {
    const int tiles = (a.T + kExpandRows - 1) / kExpandRows;
    const int width = GLU ? a.N / 2 : a.N, block = GLU ? 32 : 64, blocks = (width + block - 1) / block;
    // twice the work-groups that tiles of one adapter need, so that tiles of
    // two take no longer (the others' second half ends at once)
    const int nb = int((int64_t(tiles) * blocks + kExpandRuns - 1) / kExpandRuns);
    int64_t share = 2 * ((blocks + nb - 1) / nb);
    if (share < kExpandGroups / tiles) share = kExpandGroups / tiles;
    const int64_t most = int64_t(a.T < kExpandRows ? a.T : kExpandRows) * blocks;
    if (share > most) share = most;
    const dim3 grid(unsigned(share) * tiles);
#define GRIM_EXPAND(MC) \
    hipLaunchKernelGGL((lora_expand_kernel<GLU, MC, BB>), grid, dim3(kExpandWaves * kWave), 0, st, a, splits, int(share), nb)
    if (a.R <= 16) GRIM_EXPAND(0);
    else if (lora_max_chunks(a.R) == 1) GRIM_EXPAND(1);
    else if (lora_max_chunks(a.R) == 2) GRIM_EXPAND(2);
    else if (lora_max_chunks(a.R) == 4) GRIM_EXPAND(4);
    else GRIM_EXPAND(8);
#undef GRIM_EXPAND
}

// One launch takes up to 16 rows where a wave has at most four steps of K and
// a work-group (one a CU) at most two blocks of columns, every row an adapter
// of its own.  As a graph, one launch against two: one row, 768 -> 2048, rank
// 16: 5.2, 7.4 us; 2048 -> 2048: 7.3, 7.9 (rank 64: 10.1, 10.4); 4096 ->
// 4096: 10.8, 8.8; 16 rows 2048 -> 2048: 8.1, 9.3; 2048 -> 7168: 11.3, 10.2.
// Called one by one the launch saved counts 3 us more.
constexpr int kOneSteps = 4, kOneGroups = 256, kOneBlocks = 2;
int one_groups(const LoraArgs& a) {
    if (a.T > kRows || a.R > 64 || a.K > kOneSteps * kShrinkWaves * kStep) return 0;
    const int width = a.glu ? a.N / 2 : a.N, block = a.glu ? 32 : 64;
    const int64_t work = int64_t(a.T) * ((width + block - 1) / block);
    return work > kOneGroups * kOneBlocks ? 0 : int(work < kOneGroups ? work : kOneGroups);
}

template <bool GLU, bool XB>
void one(hipStream_t st, const LoraArgs& a, int groups) {
#define GRIM_ONE(BB, NR) \
    hipLaunchKernelGGL((lora_one_kernel<GLU, XB, BB, NR>), dim3(groups), dim3(kShrinkWaves * kWave), 0, st, a, groups)
#define GRIM_ONE_R(BB)               \
    if (a.R <= 16) GRIM_ONE(BB, 1);  \
    else if (a.R <= 32) GRIM_ONE(BB, 2); \
    else GRIM_ONE(BB, 4)
    if (a.base_bf16) {
        GRIM_ONE_R(true);
    } else {
        GRIM_ONE_R(false);
    }
#undef GRIM_ONE_R
#undef GRIM_ONE
}

}  // namespace

hipError_t lora_launch(hipStream_t st, const LoraArgs& a) {
    if (a.T <= 0) return hipSuccess;
    if (const int groups = one_groups(a)) {
        if (a.glu) a.x_bf16 ? one<true, true>(st, a, groups) : one<true, false>(st, a, groups);
        else a.x_bf16 ? one<false, true>(st, a, groups) : one<false, false>(st, a, groups);
        return hipGetLastError();
    }
    const int splits = lora_splits(a.K, a.T);
    // distinct adapters a tile can name, rows without one among them
    const int items = a.T > kLoraItemRows ? 1 : a.T < kRows ? a.T : kRows;
    if (a.x_bf16) shrink<true>(st, a, splits, items);
    else shrink<false>(st, a, splits, items);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (a.glu) a.base_bf16 ? expand<true, true>(st, a, splits) : expand<true, false>(st, a, splits);
    else a.base_bf16 ? expand<false, true>(st, a, splits) : expand<false, false>(st, a, splits);
    return hipGetLastError();
}

}  // namespace grim
