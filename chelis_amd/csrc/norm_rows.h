// Rows in registers, shared by the norm kernels: how a row's elements lie on the
// lanes of one or several waves, sums over it, the launch shape of a row length
// and the checks of row operands.
#pragma once

#include "elem.h"

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

// Rows past the register capacity: one workgroup a row.
constexpr int kLongThreads = 1024;

template <int N, typename A>
__device__ inline void block_sums(A (&v)[N]) {
    __shared__ A lds[2][2][kLongThreads / 64];
    __syncthreads();
    row_sums<kLongThreads / 64, 64>(v, lds, 0, threadIdx.x >> 6);
}

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
    if (!row_view(t, v) && (t->count || !t->shape[t->rank - 1]))
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
