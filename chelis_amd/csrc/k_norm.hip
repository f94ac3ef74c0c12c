// Layer norm for training: 16-bit forward rows with their statistics, and
// the gradients of every float dtype.
//
//   h = (x - mean) * rstd
//   dbeta = sum over rows of g,  dgamma = sum over rows of g * h
//   dx = rstd * (g gamma - mean_n(g gamma) - h * mean_n(g gamma h))
//
// A row lives in the registers of L lanes of a wave or of W waves, so x and
// g are read once for all three gradients. A workgroup walks rows a fixed
// step apart and each lane keeps the partial dgamma and dbeta of its own
// columns in registers; the workgroup's partial sums go to scratch once, and
// a second launch adds them in workgroup order: no atomics, the same bits on
// every run. Sums and statistics are binary32 (binary64 for f64), 16-bit
// results are rounded once.
//
// Bound by HBM: x, g and dx once each. [65536, 1024] bf16 with f32 weights:
// 70-73 us (5.5 TB/s) and 3-4 us for the second launch; [4096, 1024] f32: 12-13
// and 3 us, the partial sums' 2 MB and the second launch's latency showing.
#include "elem.h"

#include <algorithm>
#include <type_traits>

namespace chelis {
namespace {

// A lane's columns of one row: S vectors of V elements. A vector that would
// pass the row's end moves back inside it; its first `dup` elements then
// belong to the lane before (all V where nothing is left for the lane) and
// stay out of sums and stores.
template <int V, int S, int W, int L>
struct Columns {
    int at[S], dup[S];
    __device__ Columns(int n, int tid_in_row) {
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const int want = (s * L * W + tid_in_row) * V;
            at[s] = want < n - V ? want : n - V;
            dup[s] = want < n ? want - at[s] : V;
        }
    }
};

template <int V, typename T>
__device__ inline void store_own(const Pack<T, V> &p, T *row, int at, int dup) {
    if (dup == 0) p.store_streamed(row + at);
    else if constexpr (V > 1) {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i >= dup) row[at + i] = p.q[i];
    }
}

// Sum of one value per lane over the lanes of a row within a wave; every
// lane gets it.
template <int L, typename A>
__device__ inline A lane_sum(A x) {
    x = x + dpp_perm<kDppXor1>(x);
    x = x + dpp_perm<kDppXor2>(x);
    x = x + dpp_perm<kDppHalfMirror>(x);
    x = x + dpp_perm<kDppMirror>(x);
    if constexpr (L == 16) return x;
    else return (read_lane(x, 0) + read_lane(x, 16)) + (read_lane(x, 32) + read_lane(x, 48));
}

// N sums over a row of W waves. `slot` alternates between calls, so one
// barrier a call keeps a call's reads apart from the next one's writes.
template <int W, int L, int N, typename A>
__device__ inline void row_sums(A (&v)[N], A (*lds)[2][W], int slot, int wave) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = lane_sum<L>(v[k]);
    if constexpr (W > 1) {
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < N; ++k) lds[slot][k][wave] = v[k];
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = lds[slot][k][0];
#pragma unroll
            for (int w = 1; w < W; ++w) v[k] += lds[slot][k][w];
        }
    }
}

struct NormArgs {
    const void *x, *gamma, *beta, *g, *mean, *rstd;
    void *y, *dx, *mean_out, *rstd_out, *part;
    int64_t rows, ldx, ldg, ldy;
    int n;
    double eps;
};

// ---------------------------------------------------------------- forward
template <typename T, typename WT, int V, int S, int W, int R, int L>
__global__ __launch_bounds__(64 * W * R) void norm16_kernel(NormArgs a) {
    __shared__ float lds[2][2][W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tid = L == 64 ? (wave % W) * 64 + lane : lane % L;
    int64_t row = (int64_t)blockIdx.x * R + wave / W;
    if (L < 64) row = row * (64 / L) + lane / L;
    const bool live = row < a.rows;
    if (!live) row = a.rows - 1;
    const Columns<V, S, W, L> c(a.n, tid);
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    Pack<T, V> q[S];
    Pack<WT, V> gm[S], bt[S];
#pragma unroll
    for (int s = 0; s < S; ++s) q[s].load_streamed(x + c.at[s]);
#pragma unroll
    for (int s = 0; s < S; ++s) {
        gm[s].load(static_cast<const WT *>(a.gamma) + c.at[s]);
        bt[s].load(static_cast<const WT *>(a.beta) + c.at[s]);
    }
    float sum[1] = {};
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) sum[0] += i >= c.dup[s] ? q[s].get(i) : 0.f;
    row_sums<W, L>(sum, lds, 0, wave % W);
    const float mean = sum[0] / (float)a.n;
    float sq[1] = {};
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = q[s].get(i) - mean;
            sq[0] += i >= c.dup[s] ? d * d : 0.f;
        }
    row_sums<W, L>(sq, lds, 1, wave % W);
    const float rstd = 1.f / sqrtf(sq[0] / (float)a.n + (float)a.eps);
    if (!live) return;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        Pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out.set(i, (q[s].get(i) - mean) * rstd * gm[s].get(i) + bt[s].get(i));
        store_own<V>(out, y, c.at[s], c.dup[s]);
    }
    if (tid == 0) {
        static_cast<float *>(a.mean_out)[row] = canon_bits(mean);
        static_cast<float *>(a.rstd_out)[row] = canon_bits(rstd);
    }
}

// Rows past the register capacity: one workgroup a row, three passes.
constexpr int kLongThreads = 1024;

template <int N, typename A>
__device__ inline void block_sums(A (&v)[N]) {
    __shared__ A lds[2][2][kLongThreads / 64];
    __syncthreads();
    row_sums<kLongThreads / 64, 64>(v, lds, 0, threadIdx.x >> 6);
}

template <typename T, typename WT>
__global__ __launch_bounds__(kLongThreads) void norm16_long_kernel(NormArgs a) {
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx;
        T *y = static_cast<T *>(a.y) + row * a.ldy;
        float sum[1] = {}, sq[1] = {};
        for (int j = threadIdx.x; j < a.n; j += kLongThreads) sum[0] += widen(x[j]);
        block_sums(sum);
        const float mean = sum[0] / (float)a.n;
        for (int j = threadIdx.x; j < a.n; j += kLongThreads) {
            const float d = widen(x[j]) - mean;
            sq[0] += d * d;
        }
        block_sums(sq);
        const float rstd = 1.f / sqrtf(sq[0] / (float)a.n + (float)a.eps);
        for (int j = threadIdx.x; j < a.n; j += kLongThreads)
            y[j] = finalize<T>((widen(x[j]) - mean) * rstd * widen(static_cast<const WT *>(a.gamma)[j]) +
                               widen(static_cast<const WT *>(a.beta)[j]));
        if (threadIdx.x == 0) {
            static_cast<float *>(a.mean_out)[row] = canon_bits(mean);
            static_cast<float *>(a.rstd_out)[row] = canon_bits(rstd);
        }
    }
}

// ---------------------------------------------------------------- backward
// part holds, for workgroup b, its dgamma sums at [(2b) n ..] and its dbeta
// sums at [(2b + 1) n ..].
template <typename T, typename WT, int V, int S, int W, int R, int L>
__global__ __launch_bounds__(64 * W * R) void norm_adjoint_kernel(NormArgs a) {
    using A = typename Wide<T>::type;
    constexpr int G = R * (64 / L);  // rows the workgroup holds at a time
    constexpr int CAP = S * L * W * V;
    __shared__ A lds[2][2][W];
    __shared__ A join[G > 1 ? G * CAP : 1];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tid = L == 64 ? (wave % W) * 64 + lane : lane % L;
    const int group = L == 64 ? wave / W : wave * (64 / L) + lane / L;
    const Columns<V, S, W, L> col(a.n, tid);
    Pack<WT, V> gm[S];
#pragma unroll
    for (int s = 0; s < S; ++s) gm[s].load(static_cast<const WT *>(a.gamma) + col.at[s]);
    A dg[S][V], db[S][V];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) dg[s][i] = db[s][i] = A(0);
    const A inv_n = A(1) / (A)a.n;
    const int64_t step = (int64_t)gridDim.x * G;
    int slot = 0;
    for (int64_t base = (int64_t)blockIdx.x * G; base < a.rows; base += step) {
        const bool live = base + group < a.rows;
        const int64_t row = live ? base + group : a.rows - 1;
        const T *x = static_cast<const T *>(a.x) + row * a.ldx, *g = static_cast<const T *>(a.g) + row * a.ldg;
        Pack<T, V> xq[S], gq[S];
#pragma unroll
        for (int s = 0; s < S; ++s) xq[s].load_streamed(x + col.at[s]);
#pragma unroll
        for (int s = 0; s < S; ++s) gq[s].load_streamed(g + col.at[s]);
        const A mean = static_cast<const A *>(a.mean)[row], rstd = static_cast<const A *>(a.rstd)[row];
        A c[2] = {};
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A h = (xq[s].get(i) - mean) * rstd, gv = gq[s].get(i), w = gv * gm[s].get(i);
                const bool own = i >= col.dup[s];
                c[0] += own ? w : A(0);
                c[1] += own ? w * h : A(0);
                if (live) {
                    dg[s][i] += gv * h;
                    db[s][i] += gv;
                }
            }
        if (a.dx) {
            row_sums<W, L>(c, lds, slot, wave % W);
            slot ^= 1;
            const A c1 = c[0] * inv_n, c2 = c[1] * inv_n;
            T *dx = static_cast<T *>(a.dx) + row * a.ldy;
            if (live) {
#pragma unroll
                for (int s = 0; s < S; ++s) {
                    Pack<T, V> out;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const A h = (xq[s].get(i) - mean) * rstd;
                        out.set(i, rstd * (gq[s].get(i) * gm[s].get(i) - c1 - h * c2));
                    }
                    store_own<V>(out, dx, col.at[s], col.dup[s]);
                }
            }
        }
    }
    if (!a.part) return;
    A *part = static_cast<A *>(a.part) + (int64_t)blockIdx.x * 2 * a.n;
    if constexpr (G == 1) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i >= col.dup[s]) {
                    part[col.at[s] + i] = dg[s][i];
                    part[a.n + col.at[s] + i] = db[s][i];
                }
    } else {
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i >= col.dup[s]) join[group * CAP + col.at[s] + i] = which ? db[s][i] : dg[s][i];
            __syncthreads();
            for (int j = threadIdx.x; j < a.n; j += 64 * W * R) {
                A sum = join[j];
#pragma unroll
                for (int k = 1; k < G; ++k) sum += join[k * CAP + j];
                part[(int64_t)which * a.n + j] = sum;
            }
        }
    }
}

template <typename T, typename WT>
__global__ __launch_bounds__(kLongThreads) void norm_adjoint_long_kernel(NormArgs a) {
    using A = typename Wide<T>::type;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx, *g = static_cast<const T *>(a.g) + row * a.ldg;
        const WT *gamma = static_cast<const WT *>(a.gamma);
        const A mean = static_cast<const A *>(a.mean)[row], rstd = static_cast<const A *>(a.rstd)[row];
        A c[2] = {};
        for (int j = threadIdx.x; j < a.n; j += kLongThreads) {
            const A w = widen(g[j]) * (A)widen(gamma[j]);
            c[0] += w;
            c[1] += w * ((widen(x[j]) - mean) * rstd);
        }
        block_sums(c);
        const A c1 = c[0] / (A)a.n, c2 = c[1] / (A)a.n;
        T *dx = static_cast<T *>(a.dx) + row * a.ldy;
        for (int j = threadIdx.x; j < a.n; j += kLongThreads)
            dx[j] = finalize<T>(rstd * (widen(g[j]) * (A)widen(gamma[j]) - c1 - (widen(x[j]) - mean) * rstd * c2));
    }
}

// Partial column sums of rows blockIdx.y, blockIdx.y + gridDim.y, ..
template <typename T>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormArgs a) {
    using A = typename Wide<T>::type;
    const int64_t j = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (j >= a.n) return;
    A dg = A(0), db = A(0);
    for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const A g = widen(static_cast<const T *>(a.g)[row * a.ldg + j]);
        const A h = (widen(static_cast<const T *>(a.x)[row * a.ldx + j]) - static_cast<const A *>(a.mean)[row]) *
                    static_cast<const A *>(a.rstd)[row];
        dg += g * h;
        db += g;
    }
    A *part = static_cast<A *>(a.part) + (int64_t)blockIdx.y * 2 * a.n;
    part[j] = dg;
    part[a.n + j] = db;
}

// dgamma and dbeta: the sums of `count` partial rows [2][n] each, 32 columns
// a workgroup, 32 threads a column, joined in order.
template <typename A, typename WT>
__global__ __launch_bounds__(1024) void norm_weights_kernel(const A *part, int count, int64_t n, WT *dgamma,
                                                            WT *dbeta) {
    __shared__ A lds[32][33];
    const int col = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + col;
    A sum = A(0);
    if (j < 2 * n) {
#pragma unroll 8
        for (int b = k; b < count; b += 32) sum += part[(int64_t)b * 2 * n + j];
    }
    lds[k][col] = sum;
    __syncthreads();
    if (k == 0 && j < 2 * n) {
#pragma unroll
        for (int i = 1; i < 32; ++i) sum += lds[i][col];
        (j < n ? dgamma[j] : dbeta[j - n]) = finalize<WT>((typename Wide<WT>::type)sum);
    }
}

// ---------------------------------------------------------------- dispatch
// Lanes hold at most 16 binary32 (8 binary64) columns each: x, g, gamma and
// both partial sums stay in registers at full occupancy of a 1024-thread
// workgroup.
template <typename T>
constexpr int kMaxS = sizeof(typename Wide<T>::type) == 8 ? 4 : 16 / (16 / sizeof(T));

template <typename T>
constexpr int64_t kCapacity = (int64_t)(16 / sizeof(T)) * kMaxS<T> * 64 * 16;

// f(V, S, W, R, L) as integral constants for a row of n elements.
template <int X>
using K = std::integral_constant<int, X>;
template <typename T, class F>
int32_t with_shape(int64_t n, F &&f) {
    constexpr int V = 16 / sizeof(T), S = kMaxS<T>;
    if (n < V) return f(K<1>(), K<1>(), K<1>(), K<8>(), K<16>());
    if (n <= 16 * V) return f(K<V>(), K<1>(), K<1>(), K<8>(), K<16>());
    if (n <= 64 * V) return f(K<V>(), K<1>(), K<1>(), K<8>(), K<64>());
    if constexpr (S > 2)
        if (n <= 128 * V) return f(K<V>(), K<2>(), K<1>(), K<8>(), K<64>());
    if (n <= 64 * V * S) return f(K<V>(), K<S>(), K<1>(), K<8>(), K<64>());
    if (n <= 128 * V * S) return f(K<V>(), K<S>(), K<2>(), K<1>(), K<64>());
    if (n <= 256 * V * S) return f(K<V>(), K<S>(), K<4>(), K<1>(), K<64>());
    if (n <= 512 * V * S) return f(K<V>(), K<S>(), K<8>(), K<1>(), K<64>());
    return f(K<V>(), K<S>(), K<16>(), K<1>(), K<64>());
}

template <typename T, typename WT>
int32_t forward16(const NormArgs &a, hipStream_t st) {
    if (a.n > kCapacity<T>) {
        norm16_long_kernel<T, WT><<<(unsigned)std::min<int64_t>(a.rows, 65536), kLongThreads, 0, st>>>(a);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    }
    return with_shape<T>(a.n, [&](auto V, auto S, auto W, auto R, auto L) -> int32_t {
        const unsigned grid = grid_for(a.rows, R * (64 / L));
        if (!grid_fits(grid, 64 * W * R))
            return set_error(CHELIS_HIP_EUNSUPPORTED, "layer_norm_stats: %lld rows exceed one launch",
                             (long long)a.rows);
        norm16_kernel<T, WT, V, S, W, R, L><<<grid, 64 * W * R, 0, st>>>(a);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    });
}

template <typename T, typename WT>
int32_t adjoint(NormArgs a, void *dgamma, void *dbeta, hipStream_t st) {
    using A = typename Wide<T>::type;
    int64_t parts = 0;
    size_t bytes = 0;
    auto partials = [&](int64_t count) -> int32_t {
        parts = count;
        if (!dgamma) return CHELIS_HIP_OK;
        bytes = (size_t)count * 2 * a.n * sizeof(A);
        a.part = scratch_alloc(bytes);
        return a.part ? CHELIS_HIP_OK
                      : set_error(CHELIS_HIP_EHIP, "layer_norm_adjoint: scratch of %zu bytes", bytes);
    };
    int32_t status;
    if (a.n > kCapacity<T>) {
        // at least 32 rows to a partial sum, at most 64 partial sums
        const int64_t chunks = std::max<int64_t>(1, std::min<int64_t>(64, (a.rows + 31) / 32));
        if ((status = partials(chunks))) return status;
        // the columns first: dx may be x or g
        if (dgamma) norm_columns_kernel<T><<<dim3(grid_for(a.n, 256), (unsigned)chunks), 256, 0, st>>>(a);
        if (a.dx && a.rows)
            norm_adjoint_long_kernel<T, WT><<<(unsigned)std::min<int64_t>(a.rows, 65536), kLongThreads, 0, st>>>(a);
    } else {
        status = with_shape<T>(a.n, [&](auto V, auto S, auto W, auto R, auto L) -> int32_t {
            // two waves a SIMD over the whole device: more would only
            // write more partial sums
            const int64_t most = (int64_t)device_cus() * 8 / (W * R);
            const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(most, (a.rows + R * (64 / L) - 1) / (R * (64 / L))));
            if (int32_t s = partials(grid)) return s;
            norm_adjoint_kernel<T, WT, V, S, W, R, L><<<(unsigned)grid, 64 * W * R, 0, st>>>(a);
            return CHELIS_HIP_OK;
        });
    }
    if (status == CHELIS_HIP_OK && dgamma)
        norm_weights_kernel<A, WT><<<grid_for(2 * (int64_t)a.n, 32), 1024, 0, st>>>(
            static_cast<const A *>(a.part), (int)parts, a.n, static_cast<WT *>(dgamma), static_cast<WT *>(dbeta));
    const hipError_t e = hipGetLastError();
    scratch_free(a.part, bytes);
    if (status) return status;
    if (e != hipSuccess) return set_error(CHELIS_HIP_EHIP, "kernel launch: %s", hipGetErrorString(e));
    return CHELIS_HIP_OK;
}

// f(T(), WT()): elements of dt with weights of their type, or f32 weights
// beside 16-bit elements.
template <class F>
int32_t with_types(chelis_dtype dt, chelis_dtype wt, F &&f) {
    return with_elem(dt, [&](auto t) -> int32_t {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2)
            if (wt == CHELIS_DTYPE_F32) return f(t, float());
        return f(t, t);
    });
}

int32_t check_weights(const chelis_gpu_tensor *w, const char *name, const chelis_gpu_tensor *x, int64_t n,
                      const char *what) {
    if (int32_t s = check_tensor(w, name)) return s;
    if (!(w->dtype == x->dtype || (is_narrow16(x->dtype) && w->dtype == CHELIS_DTYPE_F32)))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must have x's dtype, or f32 beside 16-bit rows", what, name);
    if (w->rank != 1 || w->shape[0] != n || (n > 1 && w->strides[0] != 1))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be contiguous [hidden]", what, name);
    return check_device(w, name);
}

// A row statistic: contiguous over x's leading axes, f32 (f64 beside f64).
int32_t check_stat(const chelis_gpu_tensor *t, const char *name, const chelis_gpu_tensor *x, const char *what) {
    if (int32_t s = check_tensor(t, name)) return s;
    if (t->dtype != (x->dtype == CHELIS_DTYPE_F64 ? CHELIS_DTYPE_F64 : CHELIS_DTYPE_F32))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be f32 (f64 beside f64 rows)", what, name);
    bool fits = t->rank == x->rank - 1 && is_contiguous(t);
    for (int32_t i = 0; fits && i < t->rank; ++i) fits = t->shape[i] == x->shape[i];
    if (!fits) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be contiguous over x's leading axes", what, name);
    return check_device(t, name);
}

// Rows of x and of a tensor of x's shape and dtype; `out` tensors may be x
// itself (or g), element for element, but no other view that shares storage.
int32_t check_rows(const chelis_gpu_tensor *t, const char *name, const chelis_gpu_tensor *x, RowView *v,
                   const char *what) {
    if (int32_t s = check_tensor(t, name)) return s;
    if (!(is_float(t->dtype) || is_narrow16(t->dtype)))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be f32, f64, bf16 or f16", what, name);
    if (t->rank < 1) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s needs a last axis", what, name);
    if (t->dtype != x->dtype || !same_shape(t, x))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must match x in shape and dtype", what, name);
    if (!row_view(t, v))
        return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: %s: last axis must be contiguous with uniform row stride", what,
                         name);
    if (v->n == 0) return set_error(CHELIS_HIP_EDOMAIN, "%s: hidden extent must be positive", what);
    if (v->n > INT32_MAX / 2) return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: rows past 2^30 elements", what);
    return check_device(t, name);
}

int32_t check_in_place(const chelis_gpu_tensor *out, const chelis_gpu_tensor *in, const char *name, const char *what) {
    if (!non_overlapping(out)) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s overlaps itself", what, name);
    if (!same_view(out, in) && shares_storage(out, in))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s overlaps an input with other strides or from another element", what,
                         name);
    return CHELIS_HIP_OK;
}

int32_t check_apart(const chelis_gpu_tensor *out, const char *name, std::initializer_list<NamedTensor> others,
                    const char *what) {
    if (const char *other = shared_with(out, others))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s and %s overlap", what, name, other);
    return CHELIS_HIP_OK;
}

}  // namespace
}  // namespace chelis

using namespace chelis;

extern "C" int32_t chelis_hip_layer_norm_stats(const chelis_gpu_tensor *x, const chelis_gpu_tensor *gamma,
                                               const chelis_gpu_tensor *beta, double epsilon,
                                               const chelis_gpu_tensor *y, const chelis_gpu_tensor *mean,
                                               const chelis_gpu_tensor *rstd) {
    const char *what = "layer_norm_stats";
    RowView vx, vy;
    int32_t s;
    if ((s = check_tensor(x, "x")) || (s = check_rows(x, "x", x, &vx, what)) || (s = check_rows(y, "y", x, &vy, what)) ||
        (s = check_weights(gamma, "gamma", x, vx.n, what)) || (s = check_weights(beta, "beta", x, vx.n, what)) ||
        (s = check_stat(mean, "mean", x, what)) || (s = check_stat(rstd, "rstd", x, what)) ||
        (s = check_in_place(y, x, "y", what)) ||
        (s = check_apart(y, "y", {{gamma, "gamma"}, {beta, "beta"}, {mean, "mean"}, {rstd, "rstd"}}, what)) ||
        (s = check_apart(mean, "mean", {{x, "x"}, {gamma, "gamma"}, {beta, "beta"}, {rstd, "rstd"}}, what)) ||
        (s = check_apart(rstd, "rstd", {{x, "x"}, {gamma, "gamma"}, {beta, "beta"}}, what)))
        return s;
    if (gamma->dtype != beta->dtype)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: gamma and beta must share a dtype", what);
    if (!vx.rows) return CHELIS_HIP_OK;
    if (is_float(x->dtype)) return layer_norm_rows(x, gamma, beta, epsilon, y, vx, vy, mean, rstd);
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    NormArgs a{};
    a.x = x->data, a.gamma = gamma->data, a.beta = beta->data, a.y = y->data;
    a.mean_out = mean->data, a.rstd_out = rstd->data;
    a.rows = vx.rows, a.ldx = vx.ld, a.ldy = vy.ld, a.n = (int)vx.n, a.eps = epsilon;
    return with_types(x->dtype, gamma->dtype, [&](auto t, auto w) -> int32_t {
        if constexpr (sizeof(t) == 2) return forward16<decltype(t), decltype(w)>(a, st);
        else return CHELIS_HIP_EUNSUPPORTED;
    });
}

extern "C" int32_t chelis_hip_layer_norm_adjoint(const chelis_gpu_tensor *x, const chelis_gpu_tensor *gamma,
                                                 const chelis_gpu_tensor *mean, const chelis_gpu_tensor *rstd,
                                                 const chelis_gpu_tensor *g, const chelis_gpu_tensor *dx,
                                                 const chelis_gpu_tensor *dgamma, const chelis_gpu_tensor *dbeta) {
    const char *what = "layer_norm_adjoint";
    RowView vx, vg, vd;
    int32_t s;
    if ((s = check_tensor(x, "x")) || (s = check_rows(x, "x", x, &vx, what)) || (s = check_rows(g, "g", x, &vg, what)) ||
        (s = check_weights(gamma, "gamma", x, vx.n, what)) || (s = check_stat(mean, "mean", x, what)) ||
        (s = check_stat(rstd, "rstd", x, what)))
        return s;
    if (!dx && !dgamma && !dbeta) return set_error(CHELIS_HIP_EDOMAIN, "%s: no gradient asked for", what);
    if (!dgamma != !dbeta) return set_error(CHELIS_HIP_EDOMAIN, "%s: dgamma and dbeta come together", what);
    if (dx && ((s = check_rows(dx, "dx", x, &vd, what)) || (s = check_in_place(dx, x, "dx", what)) ||
               (s = check_in_place(dx, g, "dx", what)) ||
               (s = check_apart(dx, "dx", {{gamma, "gamma"}, {mean, "mean"}, {rstd, "rstd"}}, what))))
        return s;
    if (dgamma) {
        if ((s = check_weights(dgamma, "dgamma", x, vx.n, what)) || (s = check_weights(dbeta, "dbeta", x, vx.n, what)))
            return s;
        if (dgamma->dtype != gamma->dtype || dbeta->dtype != gamma->dtype)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: dgamma and dbeta must have gamma's dtype", what);
        const std::initializer_list<NamedTensor> others = {{dx, "dx"}, {x, "x"}, {g, "g"}, {gamma, "gamma"},
                                                           {mean, "mean"}, {rstd, "rstd"}};
        if ((s = check_apart(dgamma, "dgamma", {{dbeta, "dbeta"}}, what)) ||
            (s = check_apart(dgamma, "dgamma", others, what)) || (s = check_apart(dbeta, "dbeta", others, what)))
            return s;
    }
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    NormArgs a{};
    a.x = x->data, a.gamma = gamma->data, a.g = g->data, a.mean = mean->data, a.rstd = rstd->data;
    a.dx = dx ? dx->data : nullptr;
    a.rows = vx.rows, a.ldx = vx.ld, a.ldg = vg.ld, a.ldy = dx ? vd.ld : 0, a.n = (int)vx.n;
    if (!a.rows && !dgamma) return CHELIS_HIP_OK;
    return with_types(x->dtype, gamma->dtype, [&](auto t, auto w) -> int32_t {
        return adjoint<decltype(t), decltype(w)>(a, dgamma ? dgamma->data : nullptr, dbeta ? dbeta->data : nullptr, st);
    });
}
