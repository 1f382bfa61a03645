// sort_rows.hpp -- host interface of the weighted rows in expert order and of
// the gradients of the ways there and back.
#pragma once

#include "common.hpp"

namespace grim {

// rows[inverse[t][s]] = w[t][s] * x[t]  (w null: 1)
struct SortRowsArgs {
    const int32_t* ids;      // [T][K]; outside [0, E): no row
    const void* x;           // [T] rows, x_stride elements apart
    int64_t x_stride;
    const float* w;          // [T][K] or null
    void* rows;              // [T * K][H]
    int32_t *counts, *offsets, *inverse, *perm_token;   // perm_token may be null
    int x_bf16, rows_bf16;
    int T, K, E, H;
    void* workspace;         // sort_rows_workspace_bytes
};

// dx[t] = sum_s w[t][s] * drows[inverse[t][s]],  dw[t][s] = <drows[inverse[t][s]], x[t]>
struct SortGradArgs {
    const void* drows;       // [R][H]
    int64_t R;
    const int32_t* inverse;  // [T][K]; outside [0, R): no row
    const float* w;          // [T][K], or null: 1 and no dw
    const void* x;           // [T] rows (with w)
    void* dx;
    float* dw;               // [T][K] (with w)
    int64_t x_stride, dx_stride;
    int rows_bf16, x_bf16, dx_bf16;
    int T, K, H;
};

// y[t] = sum_s w[t][s] * rows[inverse[t][s]] + gate[t] * shared[t]:
// drows[inverse[t][s]] = w[t][s] * dy[t],  dw[t][s] = <dy[t], rows[inverse[t][s]]>,
// dshared[t] = gate[t] * dy[t],  dgate[t] = <dy[t], shared[t]>
struct CombineGradArgs {
    const void* dy;          // [T] rows, dy_stride elements apart
    int64_t dy_stride, R;
    const void* rows;        // [R][H]
    const int32_t* inverse;
    const float* w;          // [T][K]
    void* drows;             // [R][H]; rows no route names are left alone
    float* dw;               // [T][K]
    const void* shared;      // [T][H] or null
    const float* gate;       // [T] or null: 1
    void* dshared;           // with shared
    float* dgate;            // with gate
    int dy_bf16, rows_bf16, shared_bf16;
    int T, K, H;
};

constexpr int kSortMaxTokens = 1 << 23;   // a work-group a token, 2^32 threads a launch
constexpr int kSortMaxE = 16384;     // a count a byte quad in 64 KiB of LDS

size_t sort_rows_workspace_bytes(int T, int K, int E);
hipError_t sort_rows_launch(hipStream_t st, const SortRowsArgs& a);
hipError_t sort_grad_launch(hipStream_t st, const SortGradArgs& a);
hipError_t combine_grad_launch(hipStream_t st, const CombineGradArgs& a);

}  // namespace grim
