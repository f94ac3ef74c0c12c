// The residual stream between two blocks in one pass: the norm after a block,
// its gate and scale, the sum, the norm before the next block; and the
// gradients of all of it.
//
//   v = N_post(b),  u = x + scale * gate * v,  h = N_pre(u)
//
//   t  = du + N_pre'(u; dh),          dx = t
//   dv = scale * gate * t,            db = N_post'(b; dv)
//   N'(x; g): k = (x - mean) * rstd, w = g gamma,
//             rstd * (w - avg(w) - k avg(w k))   (layer; rms without avg(w))
//
// The gradients of the weights come from four column sums, with k the unit rows
// of b (b itself without a norm) and m those of u:
//   S1 = sum t, S2 = sum t k (per gate row), S3 = sum dh m, S4 = sum dh
//   dgate = scale (gamma_post S2 + beta_post S1)
//   dgamma_post = scale sum gate S2, dbeta_post = scale sum gate S1
//   dgamma_pre = S3, dbeta_pre = S4
//
// A row stays in the registers of a wave, a part of one or several, so every
// operand is read once although two dependent averages (forward: statistics) a
// norm are taken over it. N_pre takes the sum before it is rounded to the stored
// type. Backward, a workgroup walks rows of one gate a fixed step apart and keeps
// its column sums in registers; they go to scratch once and a second launch adds
// them in workgroup order: no atomics, the same bits on every run. Statistics and
// sums are binary32 (binary64 for f64); a 16-bit result is rounded once.
//
// Bound by HBM: x + b of f32 [20000, 1000] with a layer norm after it 58 us (5.4
// TB/s), the gradients of bf16 [65536, 1024] with two rms norms and a gate 159 us (5.1
// TB/s). Short of the device they are bound by latency: [64, 1024] 5.3 us, the
// gradients of f32 [8, 512, 1024] 26 and 4.5 us in the two launches.
#include "norm_rows.h"

#include <algorithm>

namespace chelis {
namespace {

struct NormSide {
    int32_t kind;  // CHELIS_NORM_*
    const void *gamma, *beta;
    void *mean, *rstd;
};
struct ResidualArgs {
    const void *x, *b, *gate, *du, *dh;  // x: u in the gradients
    void *u, *h, *dx, *db, *part;
    NormSide post, pre;
    int64_t rows, group_rows, ldx, ldb, ldu, ldh, lddu, lddh, lddx, lddb;
    int64_t group_blocks;
    int32_t n, groups;
    int32_t has_b;  // b was given (its data may be null without rows)
    double scale, eps;
};

// ---------------------------------------------------------------- a row's parts
// Columns of a weight vector (ones or zeros where it is absent), widened.
template <typename WT, int V, int S>
struct Weights {
    Pack<WT, V> q[S];
    bool there;
    template <class C>
    __device__ void load(const void *p, int64_t at, const C &c) {
        there = p != nullptr;
        if (!there) return;
#pragma unroll
        for (int s = 0; s < S; ++s) q[s].load(static_cast<const WT *>(p) + at + c.at[s]);
    }
    template <typename A>
    __device__ A get(int s, int i, A absent) const {
        return there ? (A)q[s].get(i) : absent;
    }
};

template <typename A>
__device__ inline A inv_sqrt(A v) {
    if constexpr (sizeof(A) == 4) return 1.f / sqrtf(v);
    else return 1.0 / sqrt(v);
}

// Statistics of the row in v and the row at unit size; slot: row_sums'.
template <int W, int L, int S, int V, typename A, class C>
__device__ inline void unit_row(A (&v)[S][V], const C &c, const NormSide &side, int64_t row, bool first, int n, A eps,
                                A (*lds)[2][W], int &slot, int wave) {
    A mean = A(0);
    if (side.kind == CHELIS_NORM_LAYER) {
        A sum[1] = {};
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0] += i >= c.dup[s] ? v[s][i] : A(0);
        row_sums<W, L>(sum, lds, slot, wave);
        slot ^= 1;
        mean = sum[0] / (A)n;
    }
    A sq[1] = {};
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[s][i] -= mean;
            sq[0] += i >= c.dup[s] ? v[s][i] * v[s][i] : A(0);
        }
    row_sums<W, L>(sq, lds, slot, wave);
    slot ^= 1;
    const A rstd = inv_sqrt<A>(sq[0] / (A)n + eps);
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) v[s][i] *= rstd;
    if (first) {
        if (side.mean && side.kind == CHELIS_NORM_LAYER) static_cast<A *>(side.mean)[row] = canon_bits(mean);
        if (side.rstd) static_cast<A *>(side.rstd)[row] = canon_bits(rstd);
    }
}

// ---------------------------------------------------------------- forward
template <typename T, typename WT, int V, int S, int W, int R, int L>
__global__ __launch_bounds__(64 * W * R) void residual_kernel(ResidualArgs a) {
    using A = typename Wide<T>::type;
    __shared__ A lds[2][2][W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tid = L == 64 ? (wave % W) * 64 + lane : lane % L;
    int64_t row = (int64_t)blockIdx.x * R + wave / W;
    if (L < 64) row = row * (64 / L) + lane / L;
    const bool live = row < a.rows;
    if (!live) row = a.rows - 1;
    const bool first = live && tid == 0;
    const Columns<V, S, W, L> c(a.n, tid);
    int slot = 0;
    Pack<T, V> xq[S], bq[S];
#pragma unroll
    for (int s = 0; s < S; ++s) xq[s].load_streamed(static_cast<const T *>(a.x) + row * a.ldx + c.at[s]);
    if (a.has_b) {
#pragma unroll
        for (int s = 0; s < S; ++s) bq[s].load_streamed(static_cast<const T *>(a.b) + row * a.ldb + c.at[s]);
    }
    Weights<WT, V, S> gate, gamma, beta;
    gate.load(a.gate, a.groups > 1 ? row / a.group_rows * a.n : 0, c);
    gamma.load(a.post.gamma, 0, c);
    beta.load(a.post.beta, 0, c);
    A v[S][V];
    if (a.has_b) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) v[s][i] = bq[s].get(i);
        if (a.post.kind != CHELIS_NORM_NONE) {
            unit_row<W, L>(v, c, a.post, row, first, a.n, (A)a.eps, lds, slot, wave % W);
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) v[s][i] = v[s][i] * gamma.get(s, i, A(1)) + beta.get(s, i, A(0));
        }
        const A scale = (A)a.scale;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) v[s][i] = xq[s].get(i) + scale * gate.get(s, i, A(1)) * v[s][i];
        if (live) {
            T *u = static_cast<T *>(a.u) + row * a.ldu;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                Pack<T, V> out;
#pragma unroll
                for (int i = 0; i < V; ++i) out.set(i, v[s][i]);
                store_own<V>(out, u, c.at[s], c.dup[s]);
            }
        }
    } else {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) v[s][i] = xq[s].get(i);
    }
    if (a.pre.kind == CHELIS_NORM_NONE) return;
    gamma.load(a.pre.gamma, 0, c);
    beta.load(a.pre.beta, 0, c);
    unit_row<W, L>(v, c, a.pre, row, first, a.n, (A)a.eps, lds, slot, wave % W);
    if (!live) return;
    T *h = static_cast<T *>(a.h) + row * a.ldh;
#pragma unroll
    for (int s = 0; s < S; ++s) {
        Pack<T, V> out;
#pragma unroll
        for (int i = 0; i < V; ++i) out.set(i, v[s][i] * gamma.get(s, i, A(1)) + beta.get(s, i, A(0)));
        store_own<V>(out, h, c.at[s], c.dup[s]);
    }
}

// Rows past the register capacity: one workgroup a row, in vectors of V that move
// back inside the row at its end (f(at, dup), the first dup elements another
// thread's). Every pass forms the values it needs again from the inputs, which the
// caches hold by then.
template <typename WT, typename A>
__device__ inline A weight_at(const void *p, int64_t j, A absent) {
    return p ? (A)widen(static_cast<const WT *>(p)[j]) : absent;
}
template <int V, class F>
__device__ inline void for_columns(int n, F &&f) {
    for (int j = threadIdx.x * V; j < n; j += kLongThreads * V) {
        const int at = j < n - V ? j : n - V;
        f(at, j - at);
    }
}
template <typename WT, int V>
struct WeightVec {
    Pack<WT, V> q;
    bool there;
    __device__ WeightVec(const void *p, int64_t at) : there(p != nullptr) {
        if (there) q.load(static_cast<const WT *>(p) + at);
    }
    template <typename A>
    __device__ A get(int i, A absent) const {
        return there ? (A)q.get(i) : absent;
    }
};

// Statistics of the row whose vector at `at` value(at, out) forms.
template <int V, typename A, class F>
__device__ inline void long_stats(const NormSide &side, int64_t row, int n, A eps, A *mean, A *rstd, F &&value) {
    A m = A(0), v[V];
    if (side.kind == CHELIS_NORM_LAYER) {
        A sum[1] = {};
        for_columns<V>(n, [&](int at, int dup) {
            value(at, v);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0] += i >= dup ? v[i] : A(0);
        });
        block_sums(sum);
        m = sum[0] / (A)n;
    }
    A sq[1] = {};
    for_columns<V>(n, [&](int at, int dup) {
        value(at, v);
#pragma unroll
        for (int i = 0; i < V; ++i) sq[0] += i >= dup ? (v[i] - m) * (v[i] - m) : A(0);
    });
    block_sums(sq);
    *mean = m, *rstd = inv_sqrt<A>(sq[0] / (A)n + eps);
    if (threadIdx.x == 0) {
        if (side.mean && side.kind == CHELIS_NORM_LAYER) static_cast<A *>(side.mean)[row] = canon_bits(m);
        if (side.rstd) static_cast<A *>(side.rstd)[row] = canon_bits(*rstd);
    }
}

template <typename T, typename WT>
__global__ __launch_bounds__(kLongThreads) void residual_long_kernel(ResidualArgs a) {
    using A = typename Wide<T>::type;
    constexpr int V = 16 / sizeof(T);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + row * a.ldx, *b = static_cast<const T *>(a.b) + row * a.ldb;
        const int64_t gate_at = a.groups > 1 ? row / a.group_rows * a.n : 0;
        const bool post = a.post.kind != CHELIS_NORM_NONE, pre = a.pre.kind != CHELIS_NORM_NONE;
        A pm = A(0), pr = A(1), m, r;
        if (post)
            long_stats<V>(a.post, row, a.n, (A)a.eps, &pm, &pr, [&](int at, A(&v)[V]) {
                Pack<T, V> q;
                q.load(b + at);
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = q.get(i);
            });
        auto sum = [&](int at, A(&v)[V]) {
            Pack<T, V> xq, bq;
            xq.load(x + at);
            if (!a.has_b) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = xq.get(i);
                return;
            }
            bq.load(b + at);
            const WeightVec<WT, V> gamma(a.post.gamma, at), beta(a.post.beta, at), gate(a.gate, gate_at + at);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                A w = bq.get(i);
                if (post) w = (w - pm) * pr * gamma.get(i, A(1)) + beta.get(i, A(0));
                v[i] = xq.get(i) + (A)a.scale * gate.get(i, A(1)) * w;
            }
        };
        if (pre) long_stats<V>(a.pre, row, a.n, (A)a.eps, &m, &r, sum);
        T *u = static_cast<T *>(a.u) + row * a.ldu, *h = static_cast<T *>(a.h) + row * a.ldh;
        for_columns<V>(a.n, [&](int at, int dup) {
            A v[V];
            sum(at, v);
            Pack<T, V> out;
            if (a.has_b) {
#pragma unroll
                for (int i = 0; i < V; ++i) out.set(i, v[i]);
                store_own<V>(out, u, at, dup);
            }
            if (pre) {
                const WeightVec<WT, V> gamma(a.pre.gamma, at), beta(a.pre.beta, at);
#pragma unroll
                for (int i = 0; i < V; ++i) out.set(i, (v[i] - m) * r * gamma.get(i, A(1)) + beta.get(i, A(0)));
                store_own<V>(out, h, at, dup);
            }
        });
    }
}

// ---------------------------------------------------------------- backward
// One row's operands and statistics.
template <typename T, int V, int S>
struct RowIn {
    using A = typename Wide<T>::type;
    Pack<T, V> u[S], b[S], du[S], dh[S];
    A um, ur, bm, br;
    template <class C>
    __device__ void load(const ResidualArgs &a, int64_t row, const C &c) {
        if (a.pre.kind != CHELIS_NORM_NONE) {
#pragma unroll
            for (int s = 0; s < S; ++s) {
                u[s].load_streamed(static_cast<const T *>(a.x) + row * a.ldx + c.at[s]);
                dh[s].load_streamed(static_cast<const T *>(a.dh) + row * a.lddh + c.at[s]);
            }
        }
        if (a.du) {
#pragma unroll
            for (int s = 0; s < S; ++s) du[s].load_streamed(static_cast<const T *>(a.du) + row * a.lddu + c.at[s]);
        }
        if (a.has_b) {
#pragma unroll
            for (int s = 0; s < S; ++s) b[s].load_streamed(static_cast<const T *>(a.b) + row * a.ldb + c.at[s]);
        }
        um = a.pre.kind == CHELIS_NORM_LAYER ? static_cast<const A *>(a.pre.mean)[row] : A(0);
        ur = a.pre.kind != CHELIS_NORM_NONE ? static_cast<const A *>(a.pre.rstd)[row] : A(1);
        bm = a.post.kind == CHELIS_NORM_LAYER ? static_cast<const A *>(a.post.mean)[row] : A(0);
        br = a.post.kind != CHELIS_NORM_NONE ? static_cast<const A *>(a.post.rstd)[row] : A(1);
    }
};

// part holds S1 .. S4 of workgroup w at [(4 w + which) n ..]; workgroups
// g * group_blocks .. belong to gate row g. The weights (scale * gate, post's and
// pre's gamma) wait in LDS: in registers beside the four sums they spilled. 16-bit
// rows are requested one ahead of the arithmetic; f32 and f64 rows of four vectors a
// lane take 217-233 registers and have none left for that.
template <typename T, typename WT, int V, int S, int W, int R, int L>
__global__ __launch_bounds__(64 * W * R) void residual_adjoint_kernel(ResidualArgs a) {
    using A = typename Wide<T>::type;
    constexpr int G = R * (64 / L);  // rows the workgroup holds at a time
    constexpr int CAP = S * L * W * V, THREADS = 64 * W * R;
    constexpr bool AHEAD = sizeof(T) == 2;
    __shared__ A lds[2][2][W];
    __shared__ __attribute__((aligned(16))) A join[G > 1 ? G * CAP : 1], weight[3][CAP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tid = L == 64 ? (wave % W) * 64 + lane : lane % L;
    const int sub = L == 64 ? wave / W : wave * (64 / L) + lane / L;
    const Columns<V, S, W, L> col(a.n, tid);
    const int64_t group = blockIdx.x / a.group_blocks;
    const bool with_pre = a.pre.kind != CHELIS_NORM_NONE, with_post = a.post.kind != CHELIS_NORM_NONE;
    for (int j = threadIdx.x; j < a.n; j += THREADS) {
        weight[0][j] = (A)a.scale * weight_at<WT>(a.gate, (a.groups > 1 ? group * a.n : 0) + j, A(1));
        weight[1][j] = weight_at<WT>(a.post.gamma, j, A(1));
        weight[2][j] = weight_at<WT>(a.pre.gamma, j, A(1));
    }
    __syncthreads();
    A s1[S][V], s2[S][V], s3[S][V], s4[S][V];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
        for (int i = 0; i < V; ++i) s1[s][i] = s2[s][i] = s3[s][i] = s4[s][i] = A(0);
    const A inv_n = A(1) / (A)a.n;
    const int64_t step = a.group_blocks * G, row0 = group * a.group_rows, end = row0 + a.group_rows;
    int slot = 0;
    auto row_of = [&](int64_t base) { return base + sub < end ? base + sub : end - 1; };
    int64_t base = row0 + blockIdx.x % a.group_blocks * G;
    RowIn<T, V, S> in, next;
    if (AHEAD && base < end) next.load(a, row_of(base), col);
    for (; base < end; base += step) {
        const bool live = base + sub < end;
        const int64_t row = row_of(base);
        if constexpr (AHEAD) {
            in = next;
            next.load(a, row_of(base + step < end ? base + step : base), col);
        } else in.load(a, row, col);
        asm volatile("" ::: "memory");  // the weights are read again for every row, not held
        A t[S][V];
        if (with_pre) {
            A c[2] = {};
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const A m = (in.u[s].get(i) - in.um) * in.ur, g = in.dh[s].get(i), w = g * weight[2][col.at[s] + i];
                    const bool own = i >= col.dup[s];
                    c[0] += own ? w : A(0);
                    c[1] += own ? w * m : A(0);
                    t[s][i] = w;
                    if (live) {
                        s3[s][i] += g * m;
                        s4[s][i] += g;
                    }
                }
            row_sums<W, L>(c, lds, slot, wave % W);
            slot ^= 1;
            const A c1 = a.pre.kind == CHELIS_NORM_LAYER ? c[0] * inv_n : A(0), c2 = c[1] * inv_n;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) t[s][i] = in.ur * (t[s][i] - c1 - (in.u[s].get(i) - in.um) * in.ur * c2);
        } else {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) t[s][i] = A(0);
        }
        if (a.du) {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) t[s][i] += in.du[s].get(i);
        }
        if (live && a.dx) {
            T *dx = static_cast<T *>(a.dx) + row * a.lddx;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                Pack<T, V> out;
#pragma unroll
                for (int i = 0; i < V; ++i) out.set(i, t[s][i]);
                store_own<V>(out, dx, col.at[s], col.dup[s]);
            }
        }
        if (!a.has_b) continue;
        A c[2] = {};
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A k = (in.b[s].get(i) - in.bm) * in.br;
                if (live) {
                    s1[s][i] += t[s][i];
                    s2[s][i] += t[s][i] * k;
                }
                t[s][i] = weight[0][col.at[s] + i] * t[s][i] * weight[1][col.at[s] + i];
                const bool own = i >= col.dup[s];
                c[0] += own ? t[s][i] : A(0);
                c[1] += own ? t[s][i] * k : A(0);
            }
        if (with_post) {
            row_sums<W, L>(c, lds, slot, wave % W);
            slot ^= 1;
            const A c1 = a.post.kind == CHELIS_NORM_LAYER ? c[0] * inv_n : A(0), c2 = c[1] * inv_n;
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i) t[s][i] = in.br * (t[s][i] - c1 - (in.b[s].get(i) - in.bm) * in.br * c2);
        }
        if (live && a.db) {
            T *db = static_cast<T *>(a.db) + row * a.lddb;
#pragma unroll
            for (int s = 0; s < S; ++s) {
                Pack<T, V> out;
#pragma unroll
                for (int i = 0; i < V; ++i) out.set(i, t[s][i]);
                store_own<V>(out, db, col.at[s], col.dup[s]);
            }
        }
    }
    if (!a.part) return;
    A *part = static_cast<A *>(a.part) + (int64_t)blockIdx.x * 4 * a.n;
#pragma unroll
    for (int which = 0; which < 4; ++which) {
        if (which < 2 ? !a.has_b : !with_pre) continue;
        auto sum = [&](int s, int i) { return which == 0 ? s1[s][i] : which == 1 ? s2[s][i] : which == 2 ? s3[s][i] : s4[s][i]; };
        if constexpr (G == 1) {
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i >= col.dup[s]) part[(int64_t)which * a.n + col.at[s] + i] = sum(s, i);
        } else {
            __syncthreads();
#pragma unroll
            for (int s = 0; s < S; ++s)
#pragma unroll
                for (int i = 0; i < V; ++i)
                    if (i >= col.dup[s]) join[sub * CAP + col.at[s] + i] = sum(s, i);
            __syncthreads();
            for (int j = threadIdx.x; j < a.n; j += 64 * W * R) {
                A v = join[j];
#pragma unroll
                for (int k = 1; k < G; ++k) v += join[k * CAP + j];
                part[(int64_t)which * a.n + j] = v;
            }
        }
    }
}

// Long rows: the averages of both norms (avg(w), avg(w k); zero where absent),
// then the column sums, then the results, which may lie over the inputs.
template <typename T, typename WT, int V>
struct LongRow {
    using A = typename Wide<T>::type;
    const ResidualArgs &a;
    int64_t row, gate_at;
    A um, ur, bm, br;
    bool with_pre, with_post;
    // a vector of the row: unit rows m of u and k of b, dh, the cotangents that
    // arrive at u and the weights
    Pack<T, V> uq, bq, duq, dhq;
    __device__ LongRow(const ResidualArgs &args, int64_t r) : a(args), row(r) {
        gate_at = a.groups > 1 ? row / a.group_rows * a.n : 0;
        with_pre = a.pre.kind != CHELIS_NORM_NONE, with_post = a.post.kind != CHELIS_NORM_NONE;
        um = a.pre.kind == CHELIS_NORM_LAYER ? static_cast<const A *>(a.pre.mean)[row] : A(0);
        ur = with_pre ? static_cast<const A *>(a.pre.rstd)[row] : A(1);
        bm = a.post.kind == CHELIS_NORM_LAYER ? static_cast<const A *>(a.post.mean)[row] : A(0);
        br = with_post ? static_cast<const A *>(a.post.rstd)[row] : A(1);
    }
    __device__ void load(int64_t at) {
        if (with_pre) {
            uq.load(static_cast<const T *>(a.x) + row * a.ldx + at);
            dhq.load(static_cast<const T *>(a.dh) + row * a.lddh + at);
        }
        if (a.du) duq.load(static_cast<const T *>(a.du) + row * a.lddu + at);
        if (a.has_b) bq.load(static_cast<const T *>(a.b) + row * a.ldb + at);
    }
    __device__ A m(int i) const { return (uq.get(i) - um) * ur; }
    __device__ A k(int i) const { return (bq.get(i) - bm) * br; }
    __device__ A t(int i, A gamma, const A (&avg)[4]) const {
        const A v = with_pre ? ur * (dhq.get(i) * gamma - avg[0] - m(i) * avg[1]) : A(0);
        return a.du ? v + duq.get(i) : v;
    }
};

template <typename T, typename WT>
__global__ __launch_bounds__(kLongThreads) void residual_averages_kernel(ResidualArgs a, typename Wide<T>::type *avg) {
    using A = typename Wide<T>::type;
    constexpr int V = 16 / sizeof(T);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        LongRow<T, WT, V> r(a, row);
        A c[2] = {}, e[2] = {}, all[4] = {};
        if (r.with_pre) {
            for_columns<V>(a.n, [&](int at, int dup) {
                r.load(at);
                const WeightVec<WT, V> gamma(a.pre.gamma, at);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const A w = i >= dup ? r.dhq.get(i) * gamma.get(i, A(1)) : A(0);
                    c[0] += w;
                    c[1] += i >= dup ? w * r.m(i) : A(0);
                }
            });
            block_sums(c);
            all[0] = a.pre.kind == CHELIS_NORM_LAYER ? c[0] / (A)a.n : A(0);
            all[1] = c[1] / (A)a.n;
        }
        if (a.has_b && r.with_post) {
            for_columns<V>(a.n, [&](int at, int dup) {
                r.load(at);
                const WeightVec<WT, V> pre(a.pre.gamma, at), post(a.post.gamma, at), gate(a.gate, r.gate_at + at);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const A w = (A)a.scale * gate.get(i, A(1)) * r.t(i, pre.get(i, A(1)), all) * post.get(i, A(1));
                    e[0] += i >= dup ? w : A(0);
                    e[1] += i >= dup ? w * r.k(i) : A(0);
                }
            });
            block_sums(e);
            all[2] = a.post.kind == CHELIS_NORM_LAYER ? e[0] / (A)a.n : A(0);
            all[3] = e[1] / (A)a.n;
        }
        if (threadIdx.x < 4) avg[4 * row + threadIdx.x] = all[threadIdx.x];
    }
}

// Two neighbouring columns a thread, every group_blocks-th row of the gate's.
template <typename T, typename WT>
__global__ __launch_bounds__(256) void residual_columns_kernel(ResidualArgs a, const typename Wide<T>::type *avg) {
    using A = typename Wide<T>::type;
    constexpr int V = 2;
    const int64_t want = ((int64_t)blockIdx.x * 256 + threadIdx.x) * V, at = want < a.n - V ? want : a.n - V;
    if (want >= a.n) return;
    const int64_t group = blockIdx.y / a.group_blocks, end = (group + 1) * a.group_rows;
    const WeightVec<WT, V> gamma(a.pre.gamma, at);
    A s[4][V] = {};
#pragma unroll 2
    for (int64_t row = group * a.group_rows + blockIdx.y % a.group_blocks; row < end; row += a.group_blocks) {
        LongRow<T, WT, V> r(a, row);
        r.load(at);
        const A all[4] = {r.with_pre ? avg[4 * row] : A(0), r.with_pre ? avg[4 * row + 1] : A(0), A(0), A(0)};
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (a.has_b) {
                const A t = r.t(i, gamma.get(i, A(1)), all);
                s[0][i] += t;
                s[1][i] += t * r.k(i);
            }
            if (r.with_pre) {
                const A g = r.dhq.get(i);
                s[2][i] += g * r.m(i);
                s[3][i] += g;
            }
        }
    }
    A *part = static_cast<A *>(a.part) + (int64_t)blockIdx.y * 4 * a.n;
#pragma unroll
    for (int which = 0; which < 4; ++which)
#pragma unroll
        for (int i = 0; i < V; ++i) part[(int64_t)which * a.n + at + i] = s[which][i];
}

template <typename T, typename WT>
__global__ __launch_bounds__(kLongThreads) void residual_adjoint_long_kernel(ResidualArgs a,
                                                                             const typename Wide<T>::type *avg) {
    using A = typename Wide<T>::type;
    constexpr int V = 16 / sizeof(T);
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        LongRow<T, WT, V> r(a, row);
        A all[4] = {};
        if (avg) all[0] = avg[4 * row], all[1] = avg[4 * row + 1], all[2] = avg[4 * row + 2], all[3] = avg[4 * row + 3];
        for_columns<V>(a.n, [&](int at, int dup) {
            r.load(at);
            const WeightVec<WT, V> pre(a.pre.gamma, at), post(a.post.gamma, at), gate(a.gate, r.gate_at + at);
            Pack<T, V> dx, db;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const A t = r.t(i, pre.get(i, A(1)), all);
                dx.set(i, t);
                if (a.has_b) {
                    const A w = (A)a.scale * gate.get(i, A(1)) * t * post.get(i, A(1));
                    db.set(i, r.with_post ? r.br * (w - all[2] - r.k(i) * all[3]) : w);
                }
            }
            if (a.dx) store_own<V>(dx, static_cast<T *>(a.dx) + row * a.lddx, at, dup);
            if (a.db) store_own<V>(db, static_cast<T *>(a.db) + row * a.lddb, at, dup);
        });
    }
}

struct WeightGrads {
    void *dgate, *post_dgamma, *post_dbeta, *pre_dgamma, *pre_dbeta;
    bool any() const { return dgate || post_dgamma || post_dbeta || pre_dgamma || pre_dbeta; }
};

// The weights' gradients from the workgroups' sums: 32 columns a workgroup, 32
// threads a column, everything joined in order. blockIdx.y 0: S1 and S2 (the 32
// threads are dealt over as many gate rows as there are, up to 32, at a time);
// 1: S3 and S4.
template <typename A, typename WT>
__global__ __launch_bounds__(1024) void residual_weights_kernel(ResidualArgs a, WeightGrads d) {
    __shared__ A lds[2][32][33];
    const int col = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + col, n = a.n;
    const A *part = static_cast<const A *>(a.part);
    const bool ok = j < n;
    A p = A(0), q = A(0);
    if (blockIdx.y == 1) {
        if (a.pre.kind == CHELIS_NORM_NONE) return;
        const int64_t count = a.groups * a.group_blocks;
        if (ok) {
#pragma unroll 8
            for (int64_t w = k; w < count; w += 32) p += part[(4 * w + 2) * n + j], q += part[(4 * w + 3) * n + j];
        }
    } else {
        if (!a.has_b) return;
        int per = 32;  // threads to a gate row
        while (per > 1 && 32 / per < a.groups) per >>= 1;
        const A scale = (A)a.scale;
        const A gamma = ok ? weight_at<WT>(a.post.gamma, j, A(1)) : A(0), beta = ok ? weight_at<WT>(a.post.beta, j, A(0)) : A(0);
        for (int64_t g0 = 0; g0 < a.groups; g0 += 32 / per) {
            const int64_t g = g0 + k / per;
            const bool here = ok && g < a.groups;
            A s1 = A(0), s2 = A(0);
            if (here) {
#pragma unroll 8
                for (int64_t w = k % per; w < a.group_blocks; w += per) {
                    const A *at = part + 4 * (g * a.group_blocks + w) * n + j;
                    s1 += at[0], s2 += at[n];
                }
            }
            __syncthreads();
            lds[0][k][col] = s1, lds[1][k][col] = s2;
            __syncthreads();
            if (here && k % per == 0) {
                for (int i = 1; i < per; ++i) s1 += lds[0][k + i][col], s2 += lds[1][k + i][col];
                if (d.dgate)
                    static_cast<WT *>(d.dgate)[g * n + j] =
                        finalize<WT>((typename Wide<WT>::type)(scale * (gamma * s2 + beta * s1)));
                const A gate = weight_at<WT>(a.gate, (a.groups > 1 ? g * n : 0) + j, A(1));
                p += scale * gate * s2;
                q += scale * gate * s1;
            }
        }
        __syncthreads();
    }
    lds[0][k][col] = p, lds[1][k][col] = q;
    __syncthreads();
    if (k || !ok) return;
#pragma unroll
    for (int i = 1; i < 32; ++i) p += lds[0][i][col], q += lds[1][i][col];
    void *dgamma = blockIdx.y ? d.pre_dgamma : d.post_dgamma, *dbeta = blockIdx.y ? d.pre_dbeta : d.post_dbeta;
    if (dgamma) static_cast<WT *>(dgamma)[j] = finalize<WT>((typename Wide<WT>::type)p);
    if (dbeta) static_cast<WT *>(dbeta)[j] = finalize<WT>((typename Wide<WT>::type)q);
}

// ---------------------------------------------------------------- dispatch
template <typename T, typename WT>
int32_t forward(const ResidualArgs &a, hipStream_t st) {
    if (a.n > kCapacity<T>) {
        residual_long_kernel<T, WT><<<(unsigned)std::min<int64_t>(a.rows, 65536), kLongThreads, 0, st>>>(a);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    }
    return with_shape<T>(a.n, [&](auto V, auto S, auto W, auto R, auto L) -> int32_t {
        const unsigned grid = grid_for(a.rows, R * (64 / L));
        if (!grid_fits(grid, 64 * W * R))
            return set_error(CHELIS_HIP_EUNSUPPORTED, "residual_norm: %lld rows exceed one launch", (long long)a.rows);
        residual_kernel<T, WT, V, S, W, R, L><<<grid, 64 * W * R, 0, st>>>(a);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    });
}

// Four column sums and four rows to a lane: half of what the forward pass holds
// fits the registers, so the widest workgroup has eight waves.
template <typename T>
constexpr int64_t kAdjointCapacity = kCapacity<T> / 2;

template <typename T, typename WT>
int32_t adjoint(ResidualArgs a, const WeightGrads &d, hipStream_t st) {
    using A = typename Wide<T>::type;
    size_t bytes = 0, avg_bytes = 0;
    void *avg = nullptr;
    auto partials = [&]() -> int32_t {
        if (!d.any()) return CHELIS_HIP_OK;
        bytes = (size_t)a.groups * a.group_blocks * 4 * a.n * sizeof(A);
        a.part = scratch_alloc(bytes);
        return a.part ? CHELIS_HIP_OK : set_error(CHELIS_HIP_EHIP, "residual_norm_adjoint: scratch of %zu bytes", bytes);
    };
    int32_t status = CHELIS_HIP_OK;
    if (a.n > kAdjointCapacity<T>) {
        // at least 8 rows to a partial sum, about 64 partial sums
        a.group_blocks = std::max<int64_t>(1, std::min<int64_t>(64 / a.groups, (a.group_rows + 7) / 8));
        if (a.groups > 65535) return set_error(CHELIS_HIP_EUNSUPPORTED, "residual_norm_adjoint: over 65535 gates of rows this long");
        if ((status = partials())) return status;
        if (a.rows && (a.pre.kind != CHELIS_NORM_NONE || a.post.kind != CHELIS_NORM_NONE)) {
            avg_bytes = (size_t)a.rows * 4 * sizeof(A);
            avg = scratch_alloc(avg_bytes);
            if (!avg) {
                scratch_free(a.part, bytes);
                return set_error(CHELIS_HIP_EHIP, "residual_norm_adjoint: scratch of %zu bytes", avg_bytes);
            }
            const unsigned grid = (unsigned)std::min<int64_t>(a.rows, 65536);
            residual_averages_kernel<T, WT><<<grid, kLongThreads, 0, st>>>(a, static_cast<A *>(avg));
        }
        if (a.part)
            residual_columns_kernel<T, WT><<<dim3(grid_for(a.n, 512), (unsigned)(a.groups * a.group_blocks)), 256, 0, st>>>(
                a, static_cast<const A *>(avg));
        if (a.rows && (a.dx || a.db))
            residual_adjoint_long_kernel<T, WT><<<(unsigned)std::min<int64_t>(a.rows, 65536), kLongThreads, 0, st>>>(
                a, static_cast<const A *>(avg));
    } else {
        status = with_shape<T>(a.n, [&](auto V, auto S, auto W, auto R, auto L) -> int32_t {
            if constexpr (W <= 8) {
                constexpr int G = R * (64 / L);
                // two waves a SIMD over the whole device: more would only
                // write more partial sums
                const int64_t most = (int64_t)device_cus() * 8 / (W * R);
                a.group_blocks = std::max<int64_t>(1, std::min<int64_t>(most / a.groups, (a.group_rows + G - 1) / G));
                const int64_t grid = a.groups * a.group_blocks;
                if (!grid_fits(grid, 64 * W * R))
                    return set_error(CHELIS_HIP_EUNSUPPORTED, "residual_norm_adjoint: %d gates exceed one launch", a.groups);
                if (int32_t s = partials()) return s;
                residual_adjoint_kernel<T, WT, V, S, W, R, L><<<(unsigned)grid, 64 * W * R, 0, st>>>(a);
            }
            return CHELIS_HIP_OK;
        });
    }
    if (status == CHELIS_HIP_OK && a.part)
        residual_weights_kernel<A, WT><<<dim3(grid_for(a.n, 32), 2), 1024, 0, st>>>(a, d);
    const hipError_t e = hipGetLastError();
    scratch_free(avg, avg_bytes);
    scratch_free(a.part, bytes);
    if (status) return status;
    if (e != hipSuccess) return set_error(CHELIS_HIP_EHIP, "kernel launch: %s", hipGetErrorString(e));
    return CHELIS_HIP_OK;
}

// ---------------------------------------------------------------- checks
struct Checked {
    const chelis_gpu_tensor *x;
    const char *what;
    int64_t n = 0;
    chelis_dtype weights{};
    bool seen = false;  // a weight has set their dtype

    int32_t rows(const chelis_gpu_tensor *t, const char *name, int64_t *ld) {
        RowView v;
        if (int32_t s = check_rows(t, name, x, &v, what)) return s;
        *ld = v.ld;
        return CHELIS_HIP_OK;
    }
    int32_t weight_dtype(const chelis_gpu_tensor *w, const char *name) {
        if (seen && w->dtype != weights)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: gate and weights must share a dtype (%s)", what, name);
        weights = w->dtype, seen = true;
        return CHELIS_HIP_OK;
    }
    int32_t weight(const chelis_gpu_tensor *w, const char *name) {
        if (!w) return CHELIS_HIP_OK;
        if (int32_t s = check_weights(w, name, x, n, what)) return s;
        return weight_dtype(w, name);
    }
    // [hidden], or [leading axes of x .., hidden]: one gate for each run of rows
    int32_t gate(const chelis_gpu_tensor *t, const char *name, int32_t *groups) {
        if (int32_t s = check_tensor(t, name)) return s;
        if (!(t->dtype == x->dtype || (is_narrow16(x->dtype) && t->dtype == CHELIS_DTYPE_F32)))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must have x's dtype, or f32 beside 16-bit rows", what, name);
        bool fits = t->rank >= 1 && t->rank < x->rank + (t->rank == 1) && t->shape[t->rank - 1] == n && is_contiguous(t);
        int64_t g = 1;
        for (int32_t i = 0; fits && i + 1 < t->rank; ++i) fits = t->shape[i] == x->shape[i], g *= t->shape[i];
        if (!fits)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be contiguous [hidden] or [leading axes of x, hidden]", what, name);
        if (g > INT32_MAX) return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: over 2^31 gates", what);
        *groups = (int32_t)g;
        if (int32_t s = check_device(t, name)) return s;
        return weight_dtype(t, name);
    }
    int32_t norm(const chelis_hip_norm *side, const char *gamma, const char *beta, const char *mean, const char *rstd,
                 bool stats_needed, NormSide *out) {
        *out = NormSide{};
        if (!side || side->kind == CHELIS_NORM_NONE) {
            if (side && (side->gamma || side->beta || side->mean || side->rstd))
                return set_error(CHELIS_HIP_EDOMAIN, "%s: weights or statistics beside no norm", what);
            return CHELIS_HIP_OK;
        }
        if (side->kind != CHELIS_NORM_LAYER && side->kind != CHELIS_NORM_RMS)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: unknown norm %d", what, side->kind);
        if (side->reserved) return set_error(CHELIS_HIP_EDOMAIN, "%s: reserved field set", what);
        int32_t s;
        if ((s = weight(side->gamma, gamma)) || (s = weight(side->beta, beta))) return s;
        if (side->kind == CHELIS_NORM_RMS && side->mean)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s beside an rms norm", what, mean);
        if (stats_needed && (!side->rstd || (side->kind == CHELIS_NORM_LAYER && !side->mean)))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s (and %s for layer) must be given", what, rstd, mean);
        if (side->mean && (s = check_stat(side->mean, mean, x, what))) return s;
        if (side->rstd && (s = check_stat(side->rstd, rstd, x, what))) return s;
        out->kind = side->kind;
        out->gamma = side->gamma ? side->gamma->data : nullptr;
        out->beta = side->beta ? side->beta->data : nullptr;
        out->mean = side->mean ? side->mean->data : nullptr;
        out->rstd = side->rstd ? side->rstd->data : nullptr;
        return CHELIS_HIP_OK;
    }
};

// Rows t may lie over an input's very elements, nowhere else on one.
int32_t check_over(const chelis_gpu_tensor *t, const char *name, std::initializer_list<NamedTensor> inputs, const char *what) {
    for (const NamedTensor &in : inputs)
        if (in.t)
            if (int32_t s = check_in_place(t, in.t, name, what)) return s;
    return CHELIS_HIP_OK;
}

constexpr chelis_hip_norm kNoNorm{CHELIS_NORM_NONE, 0, nullptr, nullptr, nullptr, nullptr};

}  // namespace
}  // namespace chelis

using namespace chelis;

extern "C" int32_t chelis_hip_residual_norm(const chelis_gpu_tensor *x, const chelis_gpu_tensor *b,
                                            const chelis_hip_norm *post, const chelis_gpu_tensor *gate, double scale,
                                            const chelis_hip_norm *pre, double epsilon, const chelis_gpu_tensor *u,
                                            const chelis_gpu_tensor *h) {
    const char *what = "residual_norm";
    const chelis_hip_norm &po = post ? *post : kNoNorm, &pr = pre ? *pre : kNoNorm;
    int32_t s;
    if ((s = check_tensor(x, "x"))) return s;
    Checked c{x, what};
    ResidualArgs a{};
    RowView vx;
    if ((s = check_rows(x, "x", x, &vx, what))) return s;
    c.n = vx.n, a.groups = 1;
    if (!b && (po.kind != CHELIS_NORM_NONE || gate || u))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: post, gate and u come with b", what);
    if (b && !u) return set_error(CHELIS_HIP_EDOMAIN, "%s: b needs u", what);
    if ((pr.kind != CHELIS_NORM_NONE) != (h != nullptr))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: pre and h come together", what);
    if (!b && !h) return set_error(CHELIS_HIP_EDOMAIN, "%s: no result asked for", what);
    if (std::isnan(scale) || std::isinf(scale)) return set_error(CHELIS_HIP_EDOMAIN, "%s: scale must be finite", what);
    if (!(epsilon >= 0)) return set_error(CHELIS_HIP_EDOMAIN, "%s: epsilon must not be negative", what);
    if ((b && (s = c.rows(b, "b", &a.ldb))) || (u && (s = c.rows(u, "u", &a.ldu))) || (h && (s = c.rows(h, "h", &a.ldh))) ||
        (gate && (s = c.gate(gate, "gate", &a.groups))) ||
        (s = c.norm(&po, "post gamma", "post beta", "post mean", "post rstd", false, &a.post)) ||
        (s = c.norm(&pr, "pre gamma", "pre beta", "pre mean", "pre rstd", false, &a.pre)))
        return s;
    const std::initializer_list<NamedTensor> weights = {{gate, "gate"}, {po.gamma, "post gamma"}, {po.beta, "post beta"},
                                                        {pr.gamma, "pre gamma"}, {pr.beta, "pre beta"}};
    const NamedTensor stats[4] = {{po.mean, "post mean"}, {po.rstd, "post rstd"}, {pr.mean, "pre mean"}, {pr.rstd, "pre rstd"}};
    const NamedTensor rows[2] = {{u, "u"}, {h, "h"}};
    for (int i = 0; i < 2; ++i) {
        if (!rows[i].t) continue;
        if ((s = check_over(rows[i].t, rows[i].name, {{x, "x"}, {b, "b"}}, what)) ||
            (s = check_apart(rows[i].t, rows[i].name, weights, what)))
            return s;
        if (i && (s = check_apart(h, "h", {{u, "u"}}, what))) return s;
    }
    for (int i = 0; i < 4; ++i) {
        if (!stats[i].t) continue;
        if ((s = check_apart(stats[i].t, stats[i].name, weights, what)) ||
            (s = check_apart(stats[i].t, stats[i].name, {{x, "x"}, {b, "b"}, {u, "u"}, {h, "h"}}, what)))
            return s;
        for (int j = 0; j < i; ++j)
            if ((s = check_apart(stats[i].t, stats[i].name, {stats[j]}, what))) return s;
    }
    if (!vx.rows) return CHELIS_HIP_OK;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    a.x = x->data, a.b = b ? b->data : nullptr, a.has_b = b != nullptr, a.gate = gate ? gate->data : nullptr;
    a.u = u ? u->data : nullptr, a.h = h ? h->data : nullptr;
    a.rows = vx.rows, a.group_rows = vx.rows / a.groups, a.ldx = vx.ld, a.n = (int32_t)vx.n;
    a.scale = scale, a.eps = epsilon;
    return with_types(x->dtype, c.seen ? c.weights : x->dtype,
                      [&](auto t, auto w) -> int32_t { return forward<decltype(t), decltype(w)>(a, st); });
}

extern "C" int32_t chelis_hip_residual_norm_adjoint(
    const chelis_gpu_tensor *u, const chelis_gpu_tensor *b, const chelis_hip_norm *post, const chelis_gpu_tensor *gate,
    double scale, const chelis_hip_norm *pre, const chelis_gpu_tensor *du, const chelis_gpu_tensor *dh,
    const chelis_gpu_tensor *dx, const chelis_gpu_tensor *db, const chelis_gpu_tensor *dgate,
    const chelis_gpu_tensor *post_dgamma, const chelis_gpu_tensor *post_dbeta, const chelis_gpu_tensor *pre_dgamma,
    const chelis_gpu_tensor *pre_dbeta) {
    const char *what = "residual_norm_adjoint";
    const chelis_hip_norm &po = post ? *post : kNoNorm, &pr = pre ? *pre : kNoNorm;
    int32_t s;
    const bool with_pre = pr.kind != CHELIS_NORM_NONE;
    if (!du && !dh) return set_error(CHELIS_HIP_EDOMAIN, "%s: no cotangent given", what);
    if (!u && with_pre) return set_error(CHELIS_HIP_EDOMAIN, "%s: pre needs u", what);
    if (!u) u = du;  // without a norm before the next block its rows are not read
    if ((s = check_tensor(u, "u"))) return s;
    Checked c{u, what};
    ResidualArgs a{};
    RowView vu;
    if ((s = check_rows(u, "u", u, &vu, what))) return s;
    c.n = vu.n, a.groups = 1;
    if (with_pre != (dh != nullptr)) return set_error(CHELIS_HIP_EDOMAIN, "%s: pre and dh come together", what);
    if (!b && (po.kind != CHELIS_NORM_NONE || gate || db || dgate || post_dgamma || post_dbeta))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: post, gate and their gradients come with b", what);
    if (dgate && !gate) return set_error(CHELIS_HIP_EDOMAIN, "%s: dgate without gate", what);
    if ((post_dgamma || post_dbeta) && po.kind == CHELIS_NORM_NONE)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: post gradients without post", what);
    if ((pre_dgamma || pre_dbeta) && !with_pre) return set_error(CHELIS_HIP_EDOMAIN, "%s: pre gradients without pre", what);
    if (!dx && !db && !dgate && !post_dgamma && !post_dbeta && !pre_dgamma && !pre_dbeta)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: no gradient asked for", what);
    if (std::isnan(scale) || std::isinf(scale)) return set_error(CHELIS_HIP_EDOMAIN, "%s: scale must be finite", what);
    int32_t dgroups = 1;
    if ((b && (s = c.rows(b, "b", &a.ldb))) || (du && (s = c.rows(du, "du", &a.lddu))) ||
        (dh && (s = c.rows(dh, "dh", &a.lddh))) || (dx && (s = c.rows(dx, "dx", &a.lddx))) ||
        (db && (s = c.rows(db, "db", &a.lddb))) || (gate && (s = c.gate(gate, "gate", &a.groups))) ||
        (s = c.norm(&po, "post gamma", "post beta", "post mean", "post rstd", true, &a.post)) ||
        (s = c.norm(&pr, "pre gamma", "pre beta", "pre mean", "pre rstd", true, &a.pre)) ||
        (dgate && (s = c.gate(dgate, "dgate", &dgroups))) || (s = c.weight(post_dgamma, "post dgamma")) ||
        (s = c.weight(post_dbeta, "post dbeta")) || (s = c.weight(pre_dgamma, "pre dgamma")) ||
        (s = c.weight(pre_dbeta, "pre dbeta")))
        return s;
    if (dgate && !same_shape(dgate, gate)) return set_error(CHELIS_HIP_EDOMAIN, "%s: dgate must match gate", what);
    const std::initializer_list<NamedTensor> weights = {
        {gate, "gate"}, {po.gamma, "post gamma"}, {po.beta, "post beta"}, {po.mean, "post mean"}, {po.rstd, "post rstd"},
        {pr.gamma, "pre gamma"}, {pr.beta, "pre beta"}, {pr.mean, "pre mean"}, {pr.rstd, "pre rstd"}};
    const chelis_gpu_tensor *read_u = with_pre ? u : nullptr;
    const NamedTensor rows[2] = {{dx, "dx"}, {db, "db"}};
    for (const NamedTensor &r : rows)
        if (r.t && ((s = check_over(r.t, r.name, {{read_u, "u"}, {b, "b"}, {du, "du"}, {dh, "dh"}}, what)) ||
                    (s = check_apart(r.t, r.name, weights, what))))
            return s;
    if (dx && db && (s = check_apart(db, "db", {{dx, "dx"}}, what))) return s;
    const NamedTensor grads[5] = {{dgate, "dgate"}, {post_dgamma, "post dgamma"}, {post_dbeta, "post dbeta"},
                                  {pre_dgamma, "pre dgamma"}, {pre_dbeta, "pre dbeta"}};
    for (int i = 0; i < 5; ++i) {
        if (!grads[i].t) continue;
        if ((s = check_apart(grads[i].t, grads[i].name, weights, what)) ||
            (s = check_apart(grads[i].t, grads[i].name,
                             {{read_u, "u"}, {b, "b"}, {du, "du"}, {dh, "dh"}, {dx, "dx"}, {db, "db"}}, what)))
            return s;
        for (int j = 0; j < i; ++j)
            if ((s = check_apart(grads[i].t, grads[i].name, {grads[j]}, what))) return s;
    }
    const auto data = [](const chelis_gpu_tensor *t) { return t ? t->data : nullptr; };
    WeightGrads d{data(dgate), data(post_dgamma), data(post_dbeta), data(pre_dgamma), data(pre_dbeta)};
    if (!vu.rows && !d.any()) return CHELIS_HIP_OK;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    const bool no_gates = a.groups == 0;  // a leading axis without extent: the sums over no rows are zero
    if (no_gates) a.groups = 1, d.dgate = nullptr, gate = nullptr;
    a.x = u->data, a.b = data(b), a.has_b = b != nullptr, a.gate = data(gate), a.du = data(du), a.dh = data(dh), a.dx = data(dx), a.db = data(db);
    a.rows = vu.rows, a.group_rows = vu.rows / a.groups, a.ldx = vu.ld, a.n = (int32_t)vu.n;
    a.scale = scale;
    return with_types(u->dtype, c.seen ? c.weights : u->dtype,
                      [&](auto t, auto w) -> int32_t { return adjoint<decltype(t), decltype(w)>(a, d, st); });
}
