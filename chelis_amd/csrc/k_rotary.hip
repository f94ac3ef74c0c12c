// Rotary positions over several axes (time, height, width, ...): the first
// 2 P elements of a head's width form P pairs; pair p turns by the angle
// t = position[axis of p] * freqs[p],
//   (u, v) -> (u cos t - v sin t, u sin t + v cos t),
// the gradient by -t, and the width past the pairs is copied.
//
// Bound by the reads and writes of x ([2, 8192, 16 + 16 heads of 64] f32, the
// heads inside the sequence axis: 47 us, 5.7 TB/s; 59 us while neighbouring
// threads took neighbouring tokens). Angles are binary64 (a position of 10^5
// leaves no correct digit of the fraction of a turn at binary32), brought to
// [-pi/4, pi/4] by quarter turns and then taken to the arithmetic width; one
// thread computes the sines of V pairs of a token once and turns them in
// several heads.
#include "elem.h"

#include <algorithm>

namespace chelis {
namespace {

constexpr int kAxes = 8;

struct RotaryTensor {
    const void *x;
    void *y;
    int64_t xb, xh, xs, yb, yh, ys;  // strides of batch, head, sequence
    int heads;
};

struct RotaryArgs {
    RotaryTensor t[2];
    const void *positions;
    const double *freqs;
    int64_t pa, pb, ps;  // strides of axis, batch, sequence
    int64_t seq, tokens;
    int wide;            // positions are i64
    int chunks;  // of the first tensor's heads; the second's follow
    int groups;  // neighbouring threads that take neighbouring heads
    int pairs, width, lanes, per_thread, end[kAxes - 1];  // pairs before axis 1, 2, ..
    double sign;
};

// sin and cos of the binary64 angle t at A's width: r = t - n pi/2 with the
// quarter turn in two parts, then the Taylor polynomials, whose first
// dropped terms at pi/4 are below 2e-9 (binary32).
__device__ inline void sin_cos(double t, float &s, float &c) {
    // n stops being the nearest quarter turn past 2^53 of them; the library's
    // reduction takes any angle (the registers it costs: the f32 prompt above
    // 47.3 -> 47.9 us, 64 bf16 tokens 6.5 us as before)
    if (!(fabs(t) < 0x1p50)) {
        double s64, c64;
        sincos(t, &s64, &c64);
        s = (float)s64, c = (float)c64;
        return;
    }
    const double n = rint(t * 0.63661977236758134308);
    const double r64 = fma(-n, 6.123233995736766036e-17, fma(-n, 1.5707963267948965580, t));
    const float r = (float)r64, z = r * r;
    const float ps = fmaf(z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), 0.f);
    const float sn = fmaf(r, ps, r);
    const float pc = fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f);
    const float cs = fmaf(z, pc, 1.f);
    const int q = (int)(int64_t)n & 3;
    s = q & 1 ? cs : sn;
    c = q & 1 ? sn : cs;
    s = q & 2 ? -s : s;
    c = (q + 1) & 2 ? -c : c;
}
__device__ inline void sin_cos(double t, double &s, double &c) { sincos(t, &s, &c); }

template <typename T, int V, bool HALVES>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    using A = typename Wide<T>::type;
    // a launch's threads are counted in 32 bits
    const uint32_t id = blockIdx.x * 256 + threadIdx.x, rest = id / (uint32_t)a.lanes;
    const int lane = (int)(id - rest * a.lanes), group = (int)(rest % (uint32_t)a.groups);
    const uint32_t token = rest / (uint32_t)a.groups;
    if (token >= a.tokens) return;
    const int64_t b = token / (uint32_t)a.seq, i = token % (uint32_t)a.seq;
    const bool second = (int)blockIdx.y >= a.chunks;
    const RotaryTensor &t = a.t[second];
    const int step = a.groups;
    const int first = ((int)blockIdx.y - (second ? a.chunks : 0)) * a.per_thread * step + group;
    const int last = min(first + a.per_thread * step, t.heads);
    if (first >= last) return;
    const T *x = static_cast<const T *>(t.x) + b * t.xb + i * t.xs;
    T *y = static_cast<T *>(t.y) + b * t.yb + i * t.ys;
    const int turned = HALVES ? a.pairs / V : 2 * a.pairs / V;
    if (lane >= turned) {  // past the pairs
        const int from = 2 * a.pairs + (lane - turned) * V;
        for (int h = first; h < last; h += step)
            for (int k = from; k < min(from + V, a.width); ++k) y[h * t.yh + k] = x[h * t.xh + k];
        return;
    }
    x += lane * V;
    y += lane * V;
    // the loads of four heads go out together, the first before the angles
    constexpr int G = 4;
    Pack<T, V> u[G], w[G];
    auto fetch = [&](int h) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
            const T *p = x + (h + g * step < last ? h + g * step : h) * t.xh;
            u[g].load_streamed(p);
            if constexpr (HALVES) w[g].load_streamed(p + a.pairs);
        }
    };
    fetch(first);
    constexpr int N = HALVES ? V : V / 2;  // pairs of this thread
    A sn[N], cs[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int p = lane * N + k;
        int axis = 0;
#pragma unroll
        for (int e = 0; e < kAxes - 1; ++e) axis += p >= a.end[e];
        const int64_t at = axis * a.pa + b * a.pb + i * a.ps;
        const double pos = a.wide ? (double)static_cast<const int64_t *>(a.positions)[at]
                                  : (double)static_cast<const int32_t *>(a.positions)[at];
        sin_cos(pos * a.freqs[p], sn[k], cs[k]);
        sn[k] = (A)a.sign * sn[k];
    }
    auto turn = [&](const Pack<T, V> &p, const Pack<T, V> &q, T *out) {
        Pack<T, V> rp, rq;
        if constexpr (HALVES) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                rp.set(k, p.get(k) * cs[k] - q.get(k) * sn[k]);
                rq.set(k, p.get(k) * sn[k] + q.get(k) * cs[k]);
            }
            rq.store_streamed(out + a.pairs);
        } else {
#pragma unroll
            for (int k = 0; k < N; ++k) {
                const A c = p.get(2 * k), d = p.get(2 * k + 1);
                rp.set(2 * k, c * cs[k] - d * sn[k]);
                rp.set(2 * k + 1, c * sn[k] + d * cs[k]);
            }
        }
        rp.store_streamed(out);
    };
    for (int h = first; h < last; h += G * step) {
#pragma unroll
        for (int g = 0; g < G; ++g)
            if (h + g * step < last) turn(u[g], w[g], y + (h + g * step) * t.yh);
        if (h + G * step < last) fetch(h + G * step);
    }
}

template <typename T, int V, bool HALVES>
int32_t launch(RotaryArgs a, hipStream_t st) {
    const int turned = HALVES ? a.pairs / V : 2 * a.pairs / V;
    a.lanes = turned + (a.width - 2 * a.pairs + V - 1) / V;
    // where a token's heads lie side by side, neighbouring threads take
    // neighbouring heads: a wave then reads whole kilobytes
    const int heads = a.t[0].heads + a.t[1].heads;
    a.groups = a.t[0].xh < a.t[0].xs && a.t[0].heads >= 4 ? 4 : 1;
    const int64_t threads = a.tokens * a.lanes * a.groups;
    // heads a thread turns with one set of sines: as many as leave two
    // workgroups a compute unit, at most eight
    const int64_t blocks = (threads + 255) / 256, want = 2 * (int64_t)device_cus();
    a.per_thread = (int)std::max<int64_t>(1, std::min<int64_t>(8, blocks * ((heads + a.groups - 1) / a.groups) / want));
    const int each = a.per_thread * a.groups;
    a.chunks = (a.t[0].heads + each - 1) / each;
    const dim3 grid((unsigned)std::min<int64_t>(blocks, 0xffffffffLL), (unsigned)(a.chunks + (a.t[1].heads + each - 1) / each));
    if (!grid_fits(blocks, 256) || grid.y > 65535)
        return set_error(CHELIS_HIP_EUNSUPPORTED, "rotary: grid too large");
    rotary_kernel<T, V, HALVES><<<grid, 256, 0, st>>>(a);
    CHELIS_LAUNCH_CHECK();
    return CHELIS_HIP_OK;
}

// The widest vector, up to 16 bytes and four pairs, that divides the pairs
// (halves) or the turned width (adjacent). With eight pairs a thread the sines,
// one after another, took longer than the narrower loads cost (bf16 heads of 128,
// 16 + 4 of them, eight against four pairs: 64 tokens 6.5 and 6.1 us, 1024 7.5 and
// 5.9, 8192 20.1 and 19.8, 32768 76.5 and 75.1; two pairs 22.9 at 8192).
template <typename T>
int32_t launch_widest(const RotaryArgs &a, bool halves, hipStream_t st) {
    if (halves) {
        constexpr int V = sizeof(T) == 8 ? 2 : 4;
        if (a.pairs % V == 0) return launch<T, V, true>(a, st);
        if constexpr (V > 2)
            if (a.pairs % (V / 2) == 0) return launch<T, V / 2, true>(a, st);
        return launch<T, 1, true>(a, st);
    }
    constexpr int V = 16 / sizeof(T);
    if (2 * a.pairs % V == 0) return launch<T, V, false>(a, st);
    return launch<T, 2, false>(a, st);
}

int32_t rotary(const chelis_gpu_tensor *const *xs, int32_t n, const chelis_gpu_tensor *positions,
               const chelis_gpu_tensor *freqs, const int64_t *sections, int32_t axes, int32_t pairing,
               const chelis_gpu_tensor *const *ys, double sign, const char *what) {
    if (n < 1 || n > 2 || !xs || !ys) return set_error(CHELIS_HIP_EDOMAIN, "%s: one or two tensors", what);
    if (axes < 1 || axes > kAxes || !sections)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: 1 to %d position axes", what, kAxes);
    if (pairing != CHELIS_ROTARY_HALVES && pairing != CHELIS_ROTARY_ADJACENT)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: unknown pairing %d", what, (int)pairing);
    int32_t s;
    if ((s = check_tensor(positions, "positions")) || (s = check_tensor(freqs, "freqs"))) return s;
    RotaryArgs a{};
    int64_t pairs = 0;
    for (int32_t k = 0; k < axes; ++k) {
        if (sections[k] < 1 || sections[k] > INT32_MAX / 4 - pairs)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: sections must be positive", what);
        pairs += sections[k];
        if (k < kAxes - 1) a.end[k] = (int)pairs;
    }
    for (int32_t k = axes - 1; k < kAxes - 1; ++k) a.end[k] = INT32_MAX;
    for (int32_t k = 0; k < n; ++k) {
        const chelis_gpu_tensor *x = xs[k], *y = ys[k];
        if ((s = check_tensor(x, "x")) || (s = check_tensor(y, "y")) || (s = check_device(x, "x")) ||
            (s = check_device(y, "y")))
            return s;
        if (x->rank != 4 || !(is_float(x->dtype) || is_narrow16(x->dtype)))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: x must be f32, f64, bf16 or f16 [batch, heads, seq, width]", what);
        if (y->dtype != x->dtype || !same_shape(x, y))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: x and y must share a shape and a dtype", what);
        if (x->dtype != xs[0]->dtype || x->shape[0] != xs[0]->shape[0] || x->shape[2] != xs[0]->shape[2] ||
            x->shape[3] != xs[0]->shape[3])
            return set_error(CHELIS_HIP_EDOMAIN, "%s: the tensors differ in more than their heads", what);
        if (2 * pairs > x->shape[3])
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %lld pairs do not fit a width of %lld", what, (long long)pairs,
                             (long long)x->shape[3]);
        if (x->shape[3] > INT32_MAX / 4 || x->shape[1] > 65535)
            return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: more than 65535 heads, or a head past 2^29", what);
        if ((x->shape[3] > 1 && (x->strides[3] != 1 || y->strides[3] != 1)))
            return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: the last axis must be contiguous", what);
        if (!non_overlapping(y)) return set_error(CHELIS_HIP_EDOMAIN, "%s: y overlaps itself", what);
        for (int32_t o = 0; o < n; ++o) {
            if (o != k && (s = check_tensor(xs[o], "x"))) return s;
            if (!(o == k && same_view(y, x)) && shares_storage(y, xs[o]))
                return set_error(CHELIS_HIP_EDOMAIN,
                                 "%s: y overlaps an input with other strides or from another element", what);
        }
        if (const char *other = shared_with(y, {{positions, "positions"}, {freqs, "freqs"}}))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: y and %s overlap", what, other);
        RotaryTensor &t = a.t[k];
        t.x = x->data, t.y = y->data, t.heads = (int)x->shape[1];
        t.xb = x->strides[0], t.xh = x->strides[1], t.xs = x->strides[2];
        t.yb = y->strides[0], t.yh = y->strides[1], t.ys = y->strides[2];
    }
    if (n == 2 && shares_storage(ys[0], ys[1]))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: the results overlap", what);
    const int64_t batch = xs[0]->shape[0], seq = xs[0]->shape[2];
    if ((positions->dtype != CHELIS_DTYPE_I32 && positions->dtype != CHELIS_DTYPE_I64) || positions->rank != 3 ||
        positions->shape[0] != axes || positions->shape[1] != batch || positions->shape[2] != seq)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: positions must be i32 or i64 [axes, batch, seq]", what);
    if (freqs->dtype != CHELIS_DTYPE_F64 || freqs->rank != 1 || freqs->shape[0] != pairs ||
        (pairs > 1 && freqs->strides[0] != 1))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: freqs must be contiguous f64 [pairs]", what);
    if ((s = check_device(positions, "positions")) || (s = check_device(freqs, "freqs"))) return s;
    a.positions = positions->data, a.wide = positions->dtype == CHELIS_DTYPE_I64;
    a.freqs = static_cast<const double *>(freqs->data);
    a.pa = positions->strides[0], a.pb = positions->strides[1], a.ps = positions->strides[2];
    a.seq = seq, a.tokens = batch * seq, a.pairs = (int)pairs, a.width = (int)xs[0]->shape[3];
    a.sign = sign;
    if (!a.tokens || !(a.t[0].heads + a.t[1].heads)) return CHELIS_HIP_OK;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    return with_elem(xs[0]->dtype,
                     [&](auto t) { return launch_widest<decltype(t)>(a, pairing == CHELIS_ROTARY_HALVES, st); });
}

}  // namespace
}  // namespace chelis

extern "C" int32_t chelis_hip_rotary(const chelis_gpu_tensor *const *xs, int32_t n, const chelis_gpu_tensor *positions,
                                     const chelis_gpu_tensor *freqs, const int64_t *sections, int32_t n_axes,
                                     int32_t pairing, const chelis_gpu_tensor *const *ys) {
    return chelis::rotary(xs, n, positions, freqs, sections, n_axes, pairing, ys, 1.0, "rotary");
}

extern "C" int32_t chelis_hip_rotary_adjoint(const chelis_gpu_tensor *const *gs, int32_t n,
                                             const chelis_gpu_tensor *positions, const chelis_gpu_tensor *freqs,
                                             const int64_t *sections, int32_t n_axes, int32_t pairing,
                                             const chelis_gpu_tensor *const *dxs) {
    return chelis::rotary(gs, n, positions, freqs, sections, n_axes, pairing, dxs, -1.0, "rotary_adjoint");
}
