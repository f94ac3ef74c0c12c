// The global norm of many gradients and their clipping, for a training step.
//
//   norm = scale * sqrt(sum over every element of every tensor of g^2)
//   out  = g * factor,  factor = scale * (norm > max_norm ? max_norm / norm : 1)
//
// The tensors travel as a table in the kernel arguments, so a call is capturable
// as it stands and copies nothing to the device; a workgroup takes one run of
// one tensor and finds it by bisection over the runs' first workgroups. Squares
// and sums are binary64: every f32, bf16 and f16 square is exact there and no sum
// of them overflows. f64 elements whose squares would leave the range (from 2^480,
// under 2^-480) are summed apart, scaled by 2^-600 and 2^600, so that the norm is
// right wherever binary64 holds it (1 GiB of f64 in 188 us, 181 with one sum); a call
// without f64 gradients writes one sum a workgroup. One workgroup adds these in
// order: no atomics, the same bits on every run. The factor is formed on the device
// from the stored norm, so nothing waits for the host.
//
// Bound by HBM: the norm reads everything once, the clipping reads and writes it
// once. 184 M bf16 gradients in 193 tensors 202-209 us (5.4 TB/s): norm 76, clipping
// 133; four of a small classifier 15 us, three launches of 2-4 us each.
#include "elem.h"

#include <algorithm>
#include <cfloat>
#include <new>

namespace chelis {
namespace {

constexpr int kThreads = 256;

// What the launches of a call share. A launch's arguments stay under 4 KiB.
struct Common {
    int32_t count;
    uint32_t blocks;
    int64_t chunk;  // elements to a piece
    double *part;   // a sum a workgroup; beside f64 gradients those of large and of small elements follow
    int64_t apart;  // elements from one of these to the next, 0 where there is only the first
    const void *norm;
    double max_norm, scale;
    int32_t norm64, in_place;
};
// A dense tensor (or up to kRunMax elements of one): n elements from `in` on.
struct Run {
    const void *in;
    void *out;
    uint32_t n, first;  // its first workgroup in the launch, and the dtype's place in kRunTypes
};
constexpr uint32_t kFirstBits = 28, kFirstMask = (1u << kFirstBits) - 1;
constexpr int64_t kRunMax = int64_t(1) << 30, kMaxBlocks = (int64_t(1) << 23) - 1;
struct RunTable {
    static constexpr int kItems = 160;
    Common c;
    Run item[kItems];
};
// `rows` runs of n elements, ldi (ldo) apart, each dealt in `cuts` pieces.
struct Rows {
    const void *in;
    void *out;
    int64_t n, ldi, ldo;
    uint32_t rows, cuts, first, dtype;
};
struct RowTable {
    static constexpr int kItems = 64;
    Common c;
    Rows item[kItems];
};
static_assert(sizeof(RunTable) <= 4096 && sizeof(RowTable) <= 4096, "kernel arguments");

__device__ inline uint32_t first_of(const Run &r) { return r.first & kFirstMask; }
__device__ inline uint32_t first_of(const Rows &r) { return r.first; }

// A workgroup's elements lo .. hi of one run.
struct Piece {
    const char *in;
    char *out;
    int64_t lo, hi;
    uint32_t dtype;
};
constexpr uint32_t kRunTypes[4] = {CHELIS_DTYPE_F32, CHELIS_DTYPE_F64, CHELIS_DTYPE_BF16, CHELIS_DTYPE_F16};
template <class Table>
__device__ inline Piece piece_of(const Table &t, uint32_t block) {
    int lo = 0, hi = t.c.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first_of(t.item[mid]) <= block) lo = mid;
        else hi = mid;
    }
    const auto it = t.item[lo];
    const uint32_t k = block - first_of(it);
    Piece p{static_cast<const char *>(it.in), static_cast<char *>(it.out)};
    if constexpr (sizeof(Table::item[0]) == sizeof(Run)) {
        const uint32_t type = it.first >> kFirstBits;
        p.dtype = type == 0 ? CHELIS_DTYPE_F32 : type == 1 ? CHELIS_DTYPE_F64 : type == 2 ? CHELIS_DTYPE_BF16 : CHELIS_DTYPE_F16;
        p.lo = (int64_t)k * t.c.chunk;
    } else {
        const int64_t row = k / it.cuts, width = it.dtype == CHELIS_DTYPE_F32 ? 4 : it.dtype == CHELIS_DTYPE_F64 ? 8 : 2;
        p.dtype = it.dtype;
        p.in += row * it.ldi * width, p.out += row * it.ldo * width;
        p.lo = (int64_t)(k % it.cuts) * t.c.chunk;
    }
    p.hi = p.lo + t.c.chunk < (int64_t)it.n ? p.lo + t.c.chunk : (int64_t)it.n;
    return p;
}

template <class F>
__device__ inline void with_dtype(uint32_t d, F &&f) {
    switch (d) {
        case CHELIS_DTYPE_F32: f(float()); break;
        case CHELIS_DTYPE_F64: f(double()); break;
        case CHELIS_DTYPE_BF16: f(__bf16()); break;
        default: f(_Float16());
    }
}

// Sum of one value per thread over the workgroup, in thread 0.
__device__ inline double block_total(double s) {
    __shared__ double wave_sum[16];
    s = wave_tree_sum(s);
    __syncthreads();  // the last call's sums are read
    if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0)
        for (int w = 1; w < (int)((blockDim.x + 63) / 64); ++w) s += wave_sum[w];
    return s;
}

// Squares are exact enough as they are for magnitudes in [2^-480, 2^480): 2^63 of
// them stay under 2^1023 and each is a normal number. f64 elements past that (and
// those that are not finite) go times 2^-1200 to `large`, those below times 2^1200 to
// `small`.
constexpr double kLarge = 0x1p480, kSmall = 0x1p-480, kLift = 0x1p600, kDrop = 0x1p-600;
struct Sums {
    double mid = 0, large = 0, small = 0;
};
// What of v the middle sum takes.
template <typename T>
__device__ inline double kept(T q, Sums &far) {
    const double v = (double)widen(q);
    if constexpr (sizeof(T) == 8) {
        const double a = fabs(v);
        const bool up = !(a < kLarge), down = a < kSmall;
        if (up) far.large = fma(a * kDrop, a * kDrop, far.large);
        if (down) far.small = fma(a * kLift, a * kLift, far.small);
        return up || down ? 0.0 : v;
    }
    return v;
}

template <typename T, int V, int U>
__device__ inline Sums squares(const T *p, int64_t lo, int64_t hi) {
    double s[U] = {};
    Sums all;
    int64_t j = lo + (int64_t)threadIdx.x * V;
    for (; j + (int64_t)(U - 1) * kThreads * V + V <= hi; j += (int64_t)U * kThreads * V) {
        Pack<T, V> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u].load(p + j + (int64_t)u * kThreads * V);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double v = kept<T>(q[u].q[i], all);
                s[u] = fma(v, v, s[u]);
            }
    }
    for (; j + V <= hi; j += (int64_t)kThreads * V) {
        Pack<T, V> q;
        q.load(p + j);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const double v = kept<T>(q.q[i], all);
            s[0] = fma(v, v, s[0]);
        }
    }
    if (j < hi)
        for (int64_t e = j; e < hi; ++e) {
            const double v = kept<T>(p[e], all);
            s[0] = fma(v, v, s[0]);
        }
#pragma unroll
    for (int u = 1; u < U; ++u) s[0] += s[u];
    all.mid = s[0];
    return all;
}

template <class Table>
__global__ __launch_bounds__(kThreads) void norm_parts_kernel(Table t) {
    const Piece p = piece_of(t, blockIdx.x);
    Sums s;
    with_dtype(p.dtype, [&](auto z) {
        using T = decltype(z);
        s = squares<T, 16 / sizeof(T), 4>(reinterpret_cast<const T *>(p.in), p.lo, p.hi);
    });
    const double mid = block_total(s.mid);
    if (threadIdx.x == 0) t.c.part[blockIdx.x] = mid;
    if (!t.c.apart) return;
    double *rest = t.c.part + t.c.apart + blockIdx.x;
    const double large = block_total(s.large), small = block_total(s.small);
    if (threadIdx.x == 0) rest[0] = large, rest[t.c.apart] = small;
}

// scale * lift * root in the order that leaves the normal numbers only where the
// result does.
__device__ inline double scaled_root(double scale, double lift, double root) {
    return (scale < 1) == (lift > 1) ? scale * lift * root : scale * (root * lift);
}
__global__ __launch_bounds__(1024) void norm_join_kernel(const double *part, int64_t count, int64_t apart, double scale,
                                                         void *norm, int32_t norm64) {
    auto total = [&](const double *from) {
        double s = 0;
        for (int64_t i = threadIdx.x; i < count; i += 1024) s += from[i];
        return block_total(s);
    };
    const double mid = total(part);
    double large = 0, small = 0;
    if (apart) large = total(part + apart), small = total(part + 2 * apart);
    if (threadIdx.x == 0) {
        // small elements count for nothing beside large ones or a sum of 2^-200
        double v = scale * sqrt(mid);
        if (large != 0) v = scaled_root(scale, kLift, sqrt(large + mid * kDrop * kDrop));
        else if (small != 0 && mid < 0x1p-200) v = scaled_root(scale, kDrop, sqrt(small + mid * kLift * kLift));
        if (norm64) *static_cast<double *>(norm) = canon_bits(v);
        else *static_cast<float *>(norm) = canon_bits((float)v);
    }
}

// A product in binary64 for the wide types (rounded once), in binary32 for the
// 16-bit ones (the factor's own rounding is 2^-24 beside their 2^-9 and 2^-12)
// unless the factor leaves its normal range.
template <typename T>
__device__ inline T scaled(T v, double factor) {
    if constexpr (sizeof(T) == 2) {
        if (factor >= (double)FLT_MIN && factor <= (double)FLT_MAX) return finalize<T>(widen(v) * (float)factor);
        return finalize<T>((float)((double)widen(v) * factor));
    } else return finalize<T>((T)((double)v * factor));
}

template <typename T, int V, int U>
__device__ inline void scale_run(const T *p, T *o, int64_t lo, int64_t hi, double factor) {
    int64_t j = lo + (int64_t)threadIdx.x * V;
    for (; j + (int64_t)(U - 1) * kThreads * V + V <= hi; j += (int64_t)U * kThreads * V) {
        Pack<T, V> q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u].load(p + j + (int64_t)u * kThreads * V);
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int i = 0; i < V; ++i) q[u].q[i] = scaled<T>(q[u].q[i], factor);
            q[u].store_streamed(o + j + (int64_t)u * kThreads * V);
        }
    }
    for (; j + V <= hi; j += (int64_t)kThreads * V) {
        Pack<T, V> q;
        q.load(p + j);
#pragma unroll
        for (int i = 0; i < V; ++i) q.q[i] = scaled<T>(q.q[i], factor);
        q.store_streamed(o + j);
    }
    if (j < hi)
        for (int64_t e = j; e < hi; ++e) o[e] = scaled<T>(p[e], factor);
}

// Pieces from the last to the first: what the norm read last is still in the last
// level cache.
template <class Table>
__global__ __launch_bounds__(kThreads) void clip_kernel(Table t) {
    const double norm =
        t.c.norm64 ? *static_cast<const double *>(t.c.norm) : (double)*static_cast<const float *>(t.c.norm);
    const double factor = norm > t.c.max_norm ? t.c.scale * (t.c.max_norm / norm) : t.c.scale;
    if (t.c.in_place && factor == 1.0) return;
    const Piece p = piece_of(t, t.c.blocks - 1 - blockIdx.x);
    with_dtype(p.dtype, [&](auto z) {
        using T = decltype(z);
        scale_run<T, 16 / sizeof(T), 4>(reinterpret_cast<const T *>(p.in), reinterpret_cast<T *>(p.out), p.lo, p.hi, factor);
    });
}

// ---------------------------------------------------------------- host
// The elements of `in` (and the same ones of `out`, null: none) as rows of a
// contiguous run: axes in the order of in's strides, neighbours joined where
// both allow it.
bool collapse(const chelis_gpu_tensor *in, const chelis_gpu_tensor *out, Rows *it) {
    it->rows = 1, it->n = in->count, it->ldi = it->ldo = 0;
    if (is_contiguous(in) && (!out || is_contiguous(out))) return true;  // what a call of hundreds nearly always holds
    int32_t idx[8], k = 0;
    for (int32_t a = 0; a < in->rank; ++a)
        if (in->shape[a] > 1) idx[k++] = a;
    std::sort(idx, idx + k, [&](int32_t x, int32_t y) { return in->strides[x] > in->strides[y]; });
    int64_t ext[8], si[8], so[8];
    int32_t m = 0;
    for (int32_t i = 0; i < k; ++i) {
        const int64_t e = in->shape[idx[i]], s = in->strides[idx[i]], o = out ? out->strides[idx[i]] : s;
        if (m && si[m - 1] == s * e && so[m - 1] == o * e) ext[m - 1] *= e, si[m - 1] = s, so[m - 1] = o;
        else ext[m] = e, si[m] = s, so[m] = o, ++m;
    }
    it->n = 1;
    if (m == 0) return true;
    if (si[m - 1] == 1 && so[m - 1] == 1) it->n = ext[--m];
    if (m > 1 || (m == 1 && (ext[0] > UINT32_MAX))) return false;
    if (m == 1) it->rows = (uint32_t)ext[0], it->ldi = si[0], it->ldo = so[0];
    return true;
}

int32_t check_gradient(const chelis_gpu_tensor *g, const char *what) {
    if (int32_t s = check_tensor(g, "a gradient")) return s;
    if (!(is_float(g->dtype) || is_narrow16(g->dtype)))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: gradients must be f32, f64, bf16 or f16", what);
    if (!is_contiguous(g) && !non_overlapping(g)) return set_error(CHELIS_HIP_EDOMAIN, "%s: a gradient overlaps itself", what);
    return check_device(g, "a gradient");
}

int32_t check_norm(const chelis_gpu_tensor *norm, const char *what) {
    if (int32_t s = check_tensor(norm, "norm")) return s;
    if (!is_float(norm->dtype) || norm->count != 1)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: norm must be one f32 or f64 element", what);
    return check_device(norm, "norm");
}

int32_t check_factor(double v, const char *name, const char *what) {
    if (!(v > 0) || std::isinf(v)) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be positive and finite", what, name);
    return CHELIS_HIP_OK;
}

// Byte ranges of tensors for the overlap search.
struct Range {
    uintptr_t lo, hi;
    int32_t i;
    bool out;
};
Range range_of(const chelis_gpu_tensor *t, int32_t i, bool out) {
    int64_t reach = 1;
    for (int32_t a = 0; a < t->rank; ++a) reach += (t->shape[a] - 1) * t->strides[a];
    const uintptr_t lo = reinterpret_cast<uintptr_t>(t->data);
    return {lo, lo + (uintptr_t)(reach * dtype_width(t->dtype)), i, out};
}

// No result shares storage with another result, with another tensor's gradient
// or, other than element for element, with its own. Sorted by address, so a
// model's hundreds of gradients do not make a call of all pairs.
int32_t check_results(const chelis_gpu_tensor *const *gs, const chelis_gpu_tensor *const *outs, int32_t n) {
    Range *r = new (std::nothrow) Range[2 * (size_t)n + 1];
    if (!r) return set_error(CHELIS_HIP_EHIP, "clip_gradients: no memory to compare %d tensors", n);
    int32_t k = 0, status = CHELIS_HIP_OK;
    for (int32_t i = 0; i < n; ++i) {
        if (!gs[i]->count) continue;
        r[k++] = range_of(outs[i], i, true);
        if (!same_view(gs[i], outs[i])) r[k++] = range_of(gs[i], i, false);
    }
    const auto before = [](const Range &a, const Range &b) { return a.lo < b.lo; };
    if (!std::is_sorted(r, r + k, before)) std::sort(r, r + k, before);
    for (int32_t a = 0; a < k && !status; ++a)
        for (int32_t b = a + 1; b < k && r[b].lo < r[a].hi && !status; ++b) {
            if (!r[a].out && !r[b].out) continue;
            const chelis_gpu_tensor *x = r[a].out ? outs[r[a].i] : gs[r[a].i], *y = r[b].out ? outs[r[b].i] : gs[r[b].i];
            if (shares_storage(x, y))
                status = set_error(CHELIS_HIP_EDOMAIN, "clip_gradients: result %d overlaps %s %d", r[a].out ? r[a].i : r[b].i,
                                   r[a].out && r[b].out ? "result" : "gradient", r[a].out ? r[b].i : r[a].i);
        }
    delete[] r;
    return status;
}

// Elements to a workgroup's piece: 8192, more once that would be over 4096
// workgroups (their partial sums are joined by one).
int64_t chunk_for(const chelis_gpu_tensor *const *gs, int32_t n) {
    int64_t total = 0;
    for (int32_t i = 0; i < n; ++i) total += gs[i]->count;
    const int64_t step = 4 * 8 * kThreads;  // whole unrolled rounds of the widest vectors
    return std::max<int64_t>(1, (total / 4096 + step - 1) / step) * step;
}

// The call's launches, f(table): all dense tensors (in parts of kRunMax elements),
// then those in rows.
template <class F>
int32_t for_tables(const chelis_gpu_tensor *const *gs, const chelis_gpu_tensor *const *outs, int32_t n, const Common &common, F &&f) {
    RunTable runs;
    RowTable rows;
    runs.c = rows.c = common;
    auto add = [&](auto &t, const auto &item, int64_t blocks) -> int32_t {
        if (t.c.count == t.kItems || t.c.blocks + blocks > kMaxBlocks) {
            if (int32_t s = f(t)) return s;
            t.c.count = 0, t.c.blocks = 0;
        }
        t.item[t.c.count] = item;
        t.item[t.c.count++].first |= t.c.blocks;
        t.c.blocks += (uint32_t)blocks;
        return CHELIS_HIP_OK;
    };
    int32_t s;
    for (int pass = 0; pass < 2; ++pass)
        for (int32_t i = 0; i < n; ++i) {
            if (!gs[i]->count) continue;
            Rows it{};
            collapse(gs[i], outs ? outs[i] : nullptr, &it);
            it.in = gs[i]->data, it.out = outs ? outs[i]->data : nullptr, it.dtype = gs[i]->dtype;
            if ((it.rows == 1) != (pass == 0)) continue;
            const int64_t width = dtype_width(gs[i]->dtype);
            if (pass) {
                it.cuts = (uint32_t)((it.n + common.chunk - 1) / common.chunk);
                if ((s = add(rows, it, (int64_t)it.rows * it.cuts))) return s;
                continue;
            }
            const uint32_t type = (uint32_t)(std::find(kRunTypes, kRunTypes + 4, it.dtype) - kRunTypes);
            for (int64_t at = 0; at < it.n; at += kRunMax) {
                const int64_t part = std::min(kRunMax, it.n - at);
                const Run run{static_cast<const char *>(it.in) + at * width, it.out ? static_cast<char *>(it.out) + at * width : nullptr,
                              (uint32_t)part, type << kFirstBits};
                if ((s = add(runs, run, (part + common.chunk - 1) / common.chunk))) return s;
            }
        }
    if (runs.c.count && (s = f(runs))) return s;
    return rows.c.count ? f(rows) : CHELIS_HIP_OK;
}

// Workgroups of a tensor's pieces.
int64_t pieces_of(const Rows &it, int64_t chunk) {
    int64_t blocks = it.rows * ((it.n + chunk - 1) / chunk);
    if (it.rows == 1) {  // cut at whole parts too
        blocks = 0;
        for (int64_t at = 0; at < it.n; at += kRunMax) blocks += (std::min(kRunMax, it.n - at) + chunk - 1) / chunk;
    }
    return blocks;
}

int32_t check_layout(const chelis_gpu_tensor *g, const chelis_gpu_tensor *out, int32_t i, int64_t chunk, const char *what) {
    Rows it;
    if (!collapse(g, out, &it) || pieces_of(it, chunk) > kMaxBlocks)
        return set_error(CHELIS_HIP_EUNSUPPORTED,
                         "%s: gradient %d is neither dense nor at most 2^23 rows of contiguous elements a fixed step apart%s",
                         what, i, out ? ", or its result has another order of axes" : "");
    return CHELIS_HIP_OK;
}

}  // namespace
}  // namespace chelis

using namespace chelis;

extern "C" int32_t chelis_hip_gradient_norm(const chelis_gpu_tensor *const *gs, int32_t n, double scale,
                                            const chelis_gpu_tensor *norm) {
    const char *what = "gradient_norm";
    int32_t s;
    if (n < 0 || (n && !gs)) return set_error(CHELIS_HIP_EDOMAIN, "%s: %d gradients", what, n);
    if ((s = check_norm(norm, what)) || (s = check_factor(scale, "scale", what))) return s;
    for (int32_t i = 0; i < n; ++i) {
        if ((s = check_gradient(gs[i], what))) return s;
        if (shares_storage(norm, gs[i]))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: norm and gradient %d overlap", what, i);
    }
    const int64_t chunk = chunk_for(gs, n);
    int64_t parts = 0;
    bool wide = false;
    for (int32_t i = 0; i < n; ++i) {
        if ((s = check_layout(gs[i], nullptr, i, chunk, what))) return s;
        Rows it;
        wide = wide || (gs[i]->count && gs[i]->dtype == CHELIS_DTYPE_F64);
        if (gs[i]->count && collapse(gs[i], nullptr, &it)) parts += pieces_of(it, chunk);
    }
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    const size_t bytes = (size_t)std::max<int64_t>(1, parts) * (wide ? 3 : 1) * sizeof(double);
    double *part = static_cast<double *>(scratch_alloc(bytes));
    if (!part) return set_error(CHELIS_HIP_EHIP, "%s: scratch of %zu bytes", what, bytes);
    Common common{};
    common.chunk = chunk, common.apart = wide ? parts : 0;
    int64_t at = 0;
    s = for_tables(gs, nullptr, n, common, [&](auto &t) -> int32_t {
        t.c.part = part + at;
        at += t.c.blocks;
        norm_parts_kernel<<<t.c.blocks, kThreads, 0, st>>>(t);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    });
    if (!s) norm_join_kernel<<<1, 1024, 0, st>>>(part, parts, common.apart, scale, norm->data, norm->dtype == CHELIS_DTYPE_F64);
    const hipError_t e = hipGetLastError();
    scratch_free(part, bytes);
    if (s) return s;
    if (e != hipSuccess) return set_error(CHELIS_HIP_EHIP, "kernel launch: %s", hipGetErrorString(e));
    return CHELIS_HIP_OK;
}

extern "C" int32_t chelis_hip_clip_gradients(const chelis_gpu_tensor *const *gs, int32_t n,
                                             const chelis_gpu_tensor *norm, double max_norm, double scale,
                                             const chelis_gpu_tensor *const *outs) {
    const char *what = "clip_gradients";
    int32_t s;
    if (n < 0 || (n && (!gs || !outs))) return set_error(CHELIS_HIP_EDOMAIN, "%s: %d gradients", what, n);
    if ((s = check_norm(norm, what)) || (s = check_factor(scale, "scale", what)) ||
        (s = check_factor(max_norm, "max_norm", what)))
        return s;
    bool in_place = true;
    for (int32_t i = 0; i < n; ++i) {
        if ((s = check_gradient(gs[i], what)) || (s = check_gradient(outs[i], what))) return s;
        if (gs[i]->dtype != outs[i]->dtype || !same_shape(gs[i], outs[i]))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: result %d must match its gradient in shape and dtype", what, i);
        if (shares_storage(norm, outs[i])) return set_error(CHELIS_HIP_EDOMAIN, "%s: norm and result %d overlap", what, i);
        in_place = in_place && (!gs[i]->count || same_view(gs[i], outs[i]));
    }
    const int64_t chunk = n ? chunk_for(gs, n) : 1;
    for (int32_t i = 0; i < n; ++i)
        if ((s = check_layout(gs[i], outs[i], i, chunk, what))) return s;
    if ((s = check_results(gs, outs, n))) return s;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    Common common{};
    common.chunk = chunk, common.norm = norm->data, common.norm64 = norm->dtype == CHELIS_DTYPE_F64;
    common.max_norm = max_norm, common.scale = scale, common.in_place = in_place;
    return for_tables(gs, outs, n, common, [&](auto &t) -> int32_t {
        clip_kernel<<<t.c.blocks, kThreads, 0, st>>>(t);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    });
}
