// The 16-bit product for a few rows (a token, or one for each of a few sequences)
// by weights contiguous along k: bound by reading them once, so they go from memory
// to registers as they lie, at any alignment and extent, and the multiply-adds run
// on the vector units beside them. One row of 8192 x 8192 bf16: 26 us (5.1 TB/s).
#pragma once

#include "dense_tile.h"

#include "hip_common.h"

namespace chelis {
namespace {

constexpr int kFewRows = 8;

// A workgroup takes eight columns, a thread eight neighbouring k of each.
template <Narrow KIND, int R>
__global__ __launch_bounds__(256) void dense_few_nk_kernel(DenseProblem p) {
    constexpr int THREADS = 256, C = 8;
    __shared__ float lds[THREADS / 64][R * C];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t n0 = (int64_t)blockIdx.x * C;
    float acc[R][C] = {};
    for (int64_t k = 8 * (int64_t)threadIdx.x; k < p.K; k += 8 * THREADS) {
        const int64_t left = p.K - k;
        Vec16<KIND> x[R], w[C];
#pragma unroll
        for (int c = 0; c < C; ++c) w[c] = load8v<KIND>(p.b + (n0 + c < p.N ? n0 + c : n0) * p.sbn + k, left);
#pragma unroll
        for (int r = 0; r < R; ++r) x[r] = load8v<KIND>(p.a + (r < p.M ? r : 0) * p.sam + k, left);
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[r][c] = fmaf(x[r].get(i), w[c].get(i), acc[r][c]);
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const float s = wave_tree_sum(acc[r][c]);
            if (lane == 0) lds[wave][r * C + c] = s;
        }
    __syncthreads();
    const int r = threadIdx.x;
    if (r >= R || r >= p.M) return;
    const int64_t count = p.N - n0;
    float v[8], bias[8];
    load_bias<KIND>(p, n0, count, bias);
    Vec16<KIND> resid;
    if (p.resid) resid = load8v<KIND>(p.resid + r * p.ldr + n0, count);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        v[i] = lds[0][r * C + i];
#pragma unroll
        for (int w = 1; w < THREADS / 64; ++w) v[i] += lds[w][r * C + i];
    }
    finish8<KIND>(p, r * p.ldc + n0, r * p.ldz + n0, count, v, bias, resid);
}

template <Narrow KIND, int R>
int32_t few_rows_of(const DenseProblem &p, hipStream_t st) {
    dense_few_nk_kernel<KIND, R><<<grid_for(p.N, 8), 256, 0, st>>>(p);
    CHELIS_LAUNCH_CHECK();
    return CHELIS_HIP_OK;
}
// p.a [M, K] with rows sam apart, p.b with columns sbn apart; M at most kFewRows.
template <Narrow KIND>
int32_t few_rows(const DenseProblem &p, hipStream_t st) {
    if (p.M == 1) return few_rows_of<KIND, 1>(p, st);
    if (p.M == 2) return few_rows_of<KIND, 2>(p, st);
    if (p.M <= 4) return few_rows_of<KIND, 4>(p, st);
    return few_rows_of<KIND, 8>(p, st);
}

}  // namespace
}  // namespace chelis
