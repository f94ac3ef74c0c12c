// The 16-bit product with bias, activation and residual in its epilogue, and its
// gradients.
//
//   z = x . w + bias,  y = act(z) + residual
//   dz = g * act'(z),  dx = dz . w^T,  dw = x^T . dz,  dbias = sum over rows of dz
//
// All products run on one kernel (dense_tile.h), which takes either operand
// along k or along its outer axis, so no gradient transposes anything; what it
// needs is whole 16-byte vectors. An operand without them (an odd extent or row
// stride) is first laid out with rows padded by zeros, which costs one pass over
// it. A transposed dw is the transposed product. dz is formed once, with the
// partial sums of dbias, and read by both products; without an activation g is
// dz. It is rounded to 16 bits for them, as the matrix cores take it (relative error
// of bf16 gradients 0.0023, where the result's own rounding makes 0.0017): carrying the
// bits below in a second operand would take twice the products. dbias sums it as it is.
//
// A long contraction with few tiles is cut into K slices whose sums go to
// scratch; a second launch adds them in order and finishes them: no atomics, the
// same bits on every run.
//
// Large products are bound by the card's power (bf16 16384 x 8192 x 4096 with bias
// and residual 1.0 ms, 1105 TFLOP/s; 8192^3 bare 937 us, 1174), middling ones by
// their epilogue, which the device's one round of tiles reaches all at once (4096 x
// 1024 x 4096 with GELU and z 55 us, 625 TFLOP/s), small ones by latency (one row of
// 1024 x 4096 5.5 us). Gradients of 8192 x 1024 x 4096 with GELU: dz and dbias 45 us
// (4.5 TB/s), the products 130 (1050 TFLOP/s).
#include "dense_rows.h"

#include <algorithm>
#include <initializer_list>

#include "hip_common.h"

namespace chelis {
namespace {

// i / d in 32 bits where both have no more (a fifth of the instructions).
__device__ inline int64_t quotient(int64_t i, int64_t d) {
    return (uint64_t)(i | d) >> 32 ? i / d : (int64_t)((uint32_t)i / (uint32_t)d);
}

// ---------------------------------------------------------------- slices' join
template <Narrow KIND>
__global__ __launch_bounds__(256) void dense_join_kernel(DenseProblem p) {
    const int64_t per = (p.N + 7) / 8, count = p.M * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t m = quotient(i, per), n = 8 * (i - m * per);
        float v[8] = {}, bias[8];
        load_bias<KIND>(p, n, p.N - n, bias);
        Vec16<KIND> resid;
        if (p.resid) resid = load8v<KIND>(p.resid + m * p.ldr + n, p.N - n);
        for (int s = 0; s < p.slices; ++s) {
            const float *q = p.part + ((int64_t)s * p.M + m) * p.N + n;
            if (n + 8 <= p.N) {
                const F4 a = *reinterpret_cast<const F4 *>(q), b = *reinterpret_cast<const F4 *>(q + 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += a[k], v[4 + k] += b[k];
            } else {
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (n + k < p.N) v[k] += q[k];
            }
        }
        finish8<KIND>(p, m * p.ldc + n, m * p.ldz + n, p.N - n, v, bias, resid);
    }
}

// ---------------------------------------------------------------- layout
// Rows of `inner` contiguous elements, ld apart, to rows of whole vectors, the
// rest zeros.
struct Layout {
    const uint16_t *from;
    uint16_t *to;
    int64_t rows, inner, ld;
};
struct Layouts {
    Layout of[2];
};
__global__ __launch_bounds__(256) void dense_layout_kernel(Layouts ls) {
    const Layout l = ls.of[blockIdx.y];
    const int64_t per = (l.inner + 7) / 8, count = l.rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t row = quotient(i, per), at = 8 * (i - row * per);
        const uint16_t *q = l.from + row * l.ld + at;
        uint4 v{};
        if (at + 8 <= l.inner) v = load8(q);
        else {
            uint16_t e[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = at + k < l.inner ? q[k] : (uint16_t)0;
            v = __builtin_bit_cast(uint4, e);
        }
        *reinterpret_cast<uint4 *>(l.to + 8 * i) = v;
    }
}

// ---------------------------------------------------------------- dz and dbias
// A workgroup's 256 columns and rows of its chunk: 32 threads of eight columns
// by eight rows at a time.
struct CotangentArgs {
    const uint16_t *g, *z;
    uint16_t *dz;  // rows of whole vectors, or null
    float *part;   // [chunks][N] sums, or null
    int64_t M, N, ldg, ldz, lddz, chunk;
    int32_t act;
};
template <Narrow KIND>
__global__ __launch_bounds__(256) void dense_cotangent_kernel(CotangentArgs a) {
    __shared__ float lds[8][256 + 8];
    const int vec = threadIdx.x & 31, r = threadIdx.x >> 5;
    const int64_t n = (int64_t)blockIdx.x * 256 + 8 * vec, count = a.N - n;
    const int64_t row0 = blockIdx.y * a.chunk, end = row0 + a.chunk < a.M ? row0 + a.chunk : a.M;
    float sum[8] = {};
    if (count > 0) {
        constexpr int U = 4;  // rows whose loads are under way together
        for (int64_t base = row0 + r; base < end; base += 8 * U) {
            Vec16<KIND> gq[U], zq[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t m = base + 8 * u < end ? base + 8 * u : end - 1;
                gq[u] = load8v<KIND>(a.g + m * a.ldg + n, count);
                if (a.act != CHELIS_ACT_NONE) zq[u] = load8v<KIND>(a.z + m * a.ldz + n, count);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int64_t m = base + 8 * u;
                if (m >= end) break;
                float g[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = i < count ? gq[u].get(i) : 0.f;
                if (a.act != CHELIS_ACT_NONE) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) g[i] = i < count ? act_adjoint(g[i], zq[u].get(i), a.act) : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += g[i];
                if (a.dz) store8<KIND>(a.dz + m * a.lddz + n, g, 8);
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) lds[r][8 * vec + i] = sum[i];
    __syncthreads();
    const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (col >= a.N) return;
    float s = lds[0][threadIdx.x];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += lds[k][threadIdx.x];
    a.part[blockIdx.y * a.N + col] = s;
}

// dbias from the chunks' sums: 32 columns a workgroup, THREADS / 32 threads a
// column, joined in order.
struct BiasArgs {
    const float *part;
    void *dbias;
    int64_t chunks, N;
    int32_t f32;
};
template <Narrow KIND, int THREADS>
__device__ inline void dense_bias(const BiasArgs &a, int64_t index, float *lds) {
    const int col = threadIdx.x & 31, k = threadIdx.x >> 5;
    const int64_t n = index * 32 + col;
    float s = 0.f;
    if (n < a.N) {
#pragma unroll 4
        for (int64_t c = k; c < a.chunks; c += THREADS / 32) s += a.part[c * a.N + n];
    }
    lds[k * 33 + col] = s;
    __syncthreads();
    if (k || n >= a.N) return;
#pragma unroll
    for (int i = 1; i < THREADS / 32; ++i) s += lds[i * 33 + col];
    if (a.f32) static_cast<float *>(a.dbias)[n] = canon_bits(s);
    else static_cast<typename Elem16<KIND>::type *>(a.dbias)[n] = finalize<typename Elem16<KIND>::type>(s);
}

// ---------------------------------------------------------------- gradients together
// dw, dx and dbias in one launch: workgroups 0 .. dw_groups belong to dw (its
// tiles walk all rows, the longest work, so they start first), the next to dx, the
// rest to dbias. Either product alone leaves a part of the device without work at
// its end, or all along where its tiles are fewer than the CUs; together they fill
// it. ([8192] 1024 x 4096 bf16: 130-157 us and 9 for joining dw's slices; one after
// the other 81 + 97 + 5.)
struct GradArgs {
    DenseProblem dw, dx;
    BiasArgs bias;
    uint32_t dw_groups, dx_groups;
};
template <Narrow KIND, int BLAY, class C>
__global__ __launch_bounds__(C::THREADS, C::OCC) void dense_gradients_kernel(GradArgs a) {
    __shared__ __attribute__((aligned(1024))) char lds[C::BYTES];
    const uint32_t i = blockIdx.x;
    if (i < a.dw_groups) dense_tile<KIND, 1, 1, C>(a.dw, i, lds);
    else if (i < a.dw_groups + a.dx_groups) dense_tile<KIND, 0, BLAY, C>(a.dx, i - a.dw_groups, lds);
    else dense_bias<KIND, C::THREADS>(a.bias, i - a.dw_groups - a.dx_groups, reinterpret_cast<float *>(lds));
}

// ---------------------------------------------------------------- dispatch
// A library call's scratch, given back when the call returns (in stream order).
struct Scratch {
    void *p[8] = {};
    size_t bytes[8] = {};
    int n = 0;
    void *take(size_t size) {
        void *q = scratch_alloc(size);
        if (q) p[n] = q, bytes[n++] = size;
        return q;
    }
    ~Scratch() {
        while (n--) scratch_free(p[n], bytes[n]);
    }
};

using TileL = TileShape<256, 256, 64, 2, 4, 1, 2, 2>;
using TileM = TileShape<128, 128, 64, 2, 2, 2, 2, 4>;   // two a CU
using TileN = TileShape<128, 128, 64, 2, 2, 4, 4, 4>;
using TileQ = TileShape<64, 128, 64, 2, 2, 2, 3, 4>;    // two a CU
using TileS = TileShape<64, 64, 128, 2, 2, 2, 3, 2>;
using TileT = TileShape<32, 32, 256, 1, 1, 8, 3, 2>;

// What a shape costs in us: a K step with the device full, a K step where every
// CU has at most one workgroup, the rest of a workgroup's work, the launch. Fitted
// to 36 products of 8 .. 16384 rows, 200 .. 8192 columns and 64 .. 8192 k, their
// operands from memory, each timed whole in every shape (root mean square 6-17 %). The
// plan that plan_for makes of them, beside every shape in every number of slices, all
// timed, over 40 products drawn from these ranges: within 3 % of the best in 26, within
// 10 % in 33, 27 % behind at worst (176 x 3912 x 720: slices whose join costs more than
// it counts); over 40 pairs of gradients 28, 37 and 15 %. Some of the shapes' best
// cases (us; the next best shape): L 4096^2 x 1024 45.5 (49.9), M 8192 x 1024 x 4096
// 74.8 (83.7), N 1024 x 4096 x 8192 87.6 (107), Q 2048^2 x 512 10.7 (11.9), S 1024^3
// 7.3 (10.5), T 8 x 4096 x 1024 5.6 (7.2).
struct ShapeCost {
    int bm, bn, bk, per_cu;
    double step, step_alone, fixed, launch;
};
constexpr ShapeCost kShapes[] = {
    {256, 256, 64, 1, 1.90, 1.41, 13.0, 0.9}, {128, 128, 64, 2, 1.14, 0.77, 4.9, 1.4}, {128, 128, 64, 1, 0.57, 0.49, 6.3, 0.6},
    {64, 128, 64, 2, 0.74, 0.39, 4.0, 0.8},   {64, 64, 128, 1, 0.51, 0.51, 2.4, 1.2},  {32, 32, 256, 1, 0.58, 0.58, 1.8, 2.4},
};
constexpr int kShapeCount = sizeof(kShapes) / sizeof(kShapes[0]);
// What the products reached of the memory's rate; tiles that take 64 bytes of each line
// of an operand along its outer axis reach less (a row of 8192 x 8192 along n: in T
// 35.1 us, in two slices of S 30.2 with their join).
constexpr double kBytesPerUs = 4.8e6, kNarrowBytesPerUs = 3.8e6;

// One product's part of a launch.
struct Extent3 {
    int64_t M, N, K;
    bool across;  // an operand lies along its outer axis
    double traffic() const { return 2.0 * (M * (double)K + K * (double)N + M * (double)N); }
};
struct Plan {
    int shape;
    int32_t slices[2];
};
// When n1 workgroups of time d1 and then n2 of time d2 are done on `room` places, each
// taking the next one as it falls free.
double makespan(double n1, double d1, double n2, double d2, double room) {
    const double full = std::floor(n1 / room), late = n1 - full * room, early = room - late;
    const double t0 = full * d1, t1 = late > 0 ? t0 + d1 : t0;  // when the early and the late places fall free
    if (!n2) return t1;
    // no place takes more than i, or i and what the early ones finish before t1
    for (double i = std::max(1.0, std::floor((n2 - early * (t1 - t0) / d2) / room));; ++i) {
        // the i-th workgroup on each early place, then on each late one
        if (early * i + late * std::max(0.0, std::floor((t0 + i * d2 - t1) / d2)) >= n2) return std::max(t1, t0 + i * d2);
        if (early * std::floor((t1 + i * d2 - t0) / d2) + late * i >= n2) return t1 + i * d2;
    }
}
// The shape and the numbers of K slices (powers of two) with the least estimated
// time for one product, or two in one launch. A slice's sums are written, read
// again and finished by one more launch.
Plan plan_for(const Extent3 *e, int count) {
    const double cus = std::max(1, device_cus());
    Plan best{0, {1, 1}};
    double least = 1e30;
    for (int i = 0; i < kShapeCount; ++i) {
        const ShapeCost &c = kShapes[i];
        const double room = cus * c.per_cu;
        double tiles[2] = {0, 2 * room}, steps[2] = {}, traffic = 0;
        for (int j = 0; j < count; ++j) {
            traffic += e[j].traffic() / (e[j].across && c.bn < 64 ? kNarrowBytesPerUs : kBytesPerUs);
            tiles[j] = (double)((e[j].M + c.bm - 1) / c.bm) * ((e[j].N + c.bn - 1) / c.bn);
            steps[j] = (double)std::max<int64_t>(1, (e[j].K + c.bk - 1) / c.bk);
        }
        // slices until one product's tiles fill the device by themselves
        const auto more = [&](int j, int32_t slices) {
            return slices == 1 || (slices <= 16 && slices <= steps[j] && tiles[j] * slices < 2 * room);
        };
        for (int32_t s0 = 1; more(0, s0); s0 *= 2)
            for (int32_t s1 = 1; more(1, s1); s1 *= 2) {
                const int32_t s[2] = {s0, s1};
                double one[2] = {}, n[2] = {}, groups = 0, alone = 0, joins = 0;
                for (int j = 0; j < count; ++j) {
                    const double per = std::ceil(steps[j] / s[j]);
                    one[j] = per * c.step + c.fixed;
                    n[j] = tiles[j] * s[j];
                    groups += n[j];
                    alone = std::max(alone, per * c.step_alone + c.fixed);
                    if (s[j] > 1) joins += 3.0 + 8.0 * e[j].M * e[j].N * s[j] / kBytesPerUs;
                }
                double t;
                if (groups <= cus) t = alone;
                else if (count == 1) {  // whole rounds, a last one with a workgroup a CU at most goes faster
                    const double full = std::floor(groups / room), rest = groups - full * room;
                    t = full * one[0] + (rest > cus ? one[0] : rest > 0 ? alone : 0.0);
                } else t = makespan(n[0], one[0], n[1], one[1], room);
                t = std::max(t + c.launch, traffic) + joins;
                if (t < least) least = t, best = Plan{i, {s0, s1}};
            }
    }
    return best;
}
void cut(DenseProblem *p, const ShapeCost &c, int32_t slices) {
    const int64_t steps = std::max<int64_t>(1, (p->K + c.bk - 1) / c.bk), per = (steps + slices - 1) / slices;
    p->kslice = per * c.bk, p->slices = (int32_t)((steps + per - 1) / per);
}
int64_t groups_of(const DenseProblem &p, const ShapeCost &c) {
    return ((p.M + c.bm - 1) / c.bm) * ((p.N + c.bn - 1) / c.bn) * p.slices;
}

// f(shape type) for a shape's number.
template <class F>
int32_t with_tiles(int shape, F &&f) {
    switch (shape) {
        case 0: return f(TileL());
        case 1: return f(TileM());
        case 2: return f(TileN());
        case 3: return f(TileQ());
        case 4: return f(TileS());
        default: return f(TileT());
    }
}

template <Narrow KIND>
int32_t join_slices(const DenseProblem &p, hipStream_t st) {
    if (p.slices == 1) return CHELIS_HIP_OK;
    dense_join_kernel<KIND><<<(unsigned)std::min<int64_t>((p.M * ((p.N + 7) / 8) + 255) / 256, 8192), 256, 0, st>>>(p);
    CHELIS_LAUNCH_CHECK();
    return CHELIS_HIP_OK;
}

// Offsets inside a tile are 31 bits: 256 lines of at most this many elements.
constexpr int64_t kMaxLine = int64_t(1) << 21, kMaxWidth = int64_t(1) << 20;

// An operand of the product: `inner` contiguous elements to a line, `lines` of
// them ld apart.
struct Side {
    const uint16_t *data;
    int64_t lines, inner, ld;
    bool whole() const {
        return (reinterpret_cast<uintptr_t>(data) & 15) == 0 && (lines < 2 || ld % 8 == 0) && inner % 8 == 0 && (lines < 2 || ld <= kMaxLine);
    }
};
int32_t lay_out(std::initializer_list<Side *> sides, Scratch &scratch, hipStream_t st) {
    Layouts ls{};
    int n = 0;
    int64_t most = 0;
    for (Side *s : sides) {
        if (!s || s->whole() || !s->lines || !s->inner) continue;
        const int64_t ld = (s->inner + 7) / 8 * 8;
        uint16_t *to = static_cast<uint16_t *>(scratch.take((size_t)s->lines * ld * 2));
        if (!to) return set_error(CHELIS_HIP_EHIP, "dense: scratch of %lld bytes", (long long)(s->lines * ld * 2));
        ls.of[n++] = Layout{s->data, to, s->lines, s->inner, s->ld};
        most = std::max(most, s->lines * ld / 8);
        s->data = to, s->ld = ld;
    }
    if (!n) return CHELIS_HIP_OK;
    dense_layout_kernel<<<dim3((unsigned)std::min<int64_t>((most + 255) / 256, 4096), (unsigned)n), 256, 0, st>>>(ls);
    CHELIS_LAUNCH_CHECK();
    return CHELIS_HIP_OK;
}

// The sides of a product whose operands are laid out, each along k (lay 0: lines
// are its outer axis) or along its outer axis (lay 1: lines are k), and its scratch
// for slices.
int32_t set_sides(DenseProblem *p, const Side &a, int alay, const Side &b, int blay, Scratch &scratch) {
    p->a = a.data, p->b = b.data;
    p->sam = alay ? 1 : a.ld, p->sak = alay ? a.ld : 1;
    p->sbn = blay ? 1 : b.ld, p->sbk = blay ? b.ld : 1;
    if (p->slices == 1) return CHELIS_HIP_OK;
    p->part = static_cast<float *>(scratch.take((size_t)p->slices * p->M * p->N * sizeof(float)));
    return p->part ? CHELIS_HIP_OK : set_error(CHELIS_HIP_EHIP, "dense: scratch for %d slices", p->slices);
}

// Whether a few rows by weights along k go to the vector units, from 300 products of
// 1 .. 14336 k and 8 .. 32001 columns timed there and in tiles (us there / in tiles,
// K x N). There the time grows with the rows, and short k leave threads without work;
// tiles take up to 32 rows for the time of one, but weights that are not whole vectors
// have to be laid out first.
//   one row, from 512 k or up to 512 columns: 512 x 4096 4.5 / 4.9, 4096^2 8.4 / 12.3,
//     257 x 333 5.3 / 7.8 (421 x 4096 9.6 / 8.9, 143 x 32001 39.3 / 15.3)
//   two, from 1500: 1536 x 4096 6.3 / 6.6, 8192 x 14336 42.2 / 48.8 (1024 x 8192 6.8 /
//     6.4); weights to lay out, from 1000: 1001 x 4096 9.4 / 12.8 (653 x 4096 11.8 / 10.5)
//   three and four, from 2000 while the workgroups go in one round of two a CU: 2048 x
//     4096 8.3 / 10.0, 4096^2 11.0 / 12.3 (1536 x 4096 7.8 / 6.6, 4096 x 8192 16.4 /
//     14.5); weights to lay out, from 1000 in one round and from 2000 in any: 1001 x
//     4096 11.0 / 12.8, 2053 x 32000 58.5 / 69.3 (1405 x 32000 68.5 / 48.6)
//   five to eight by weights to lay out, from 2000 in one round and from 8192 in any:
//     3001 x 4096 19.2 / 23.7, 8197 x 8192 60.2 / 67.5 (1405 x 2048 17.5 / 11.4, 4101 x
//     8192 44.7 / 37.6; whole 4096^2 15.0 / 12.5)
bool few_rows_pay(const DenseProblem &p, bool whole) {
    const bool one_round = p.N <= 16 * (int64_t)device_cus();
    if (p.M == 1) return p.K >= 512 || p.N <= 512;
    if (p.M == 2) return p.K >= (whole ? 1500 : 1000);
    if (p.M <= 4) return one_round ? p.K >= (whole ? 2000 : 1000) : !whole && p.K >= 2000;
    return p.M <= kFewRows && !whole && (p.K >= 8192 || (p.K >= 2000 && one_round));
}

template <Narrow KIND>
int32_t forward(DenseProblem p, Side a, Side b, int blay, Scratch &scratch, hipStream_t st) {
    if (blay == 0 && few_rows_pay(p, b.whole())) {
        p.a = a.data, p.b = b.data, p.sam = a.ld, p.sbk = p.sbn = b.ld;
        return few_rows<KIND>(p, st);
    }
    const Extent3 e{p.M, p.N, p.K, blay == 1};
    const Plan plan = plan_for(&e, 1);
    const ShapeCost &c = kShapes[plan.shape];
    cut(&p, c, plan.slices[0]);
    const int64_t groups = groups_of(p, c);
    int32_t s;
    if ((s = lay_out({&a, &b}, scratch, st)) || (s = set_sides(&p, a, 0, b, blay, scratch))) return s;
    s = with_tiles(plan.shape, [&](auto tile) -> int32_t {
        using T = decltype(tile);
        if (!grid_fits(groups, T::THREADS)) return set_error(CHELIS_HIP_EUNSUPPORTED, "dense: grid too large");
        if (blay) dense_tile_kernel<KIND, 0, 1, T><<<(unsigned)groups, T::THREADS, 0, st>>>(p);
        else dense_tile_kernel<KIND, 0, 0, T><<<(unsigned)groups, T::THREADS, 0, st>>>(p);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    });
    return s ? s : join_slices<KIND>(p, st);
}

// ---------------------------------------------------------------- checks
struct DenseChecks {
    const char *what;
    chelis_dtype dt;
    int64_t rows, K, N;

    int32_t row_operand(const chelis_gpu_tensor *t, const char *name, const chelis_gpu_tensor *x, int64_t width, int64_t *ld) {
        if (int32_t s = check_tensor(t, name)) return s;
        if (t->dtype != dt) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must have x's dtype", what, name);
        bool fits = t->rank == x->rank && t->shape[t->rank - 1] == width;
        for (int32_t i = 0; fits && i + 1 < t->rank; ++i) fits = t->shape[i] == x->shape[i];
        if (!fits) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be [x's leading axes, %lld]", what, name, (long long)width);
        RowView v;
        if (!row_view(t, &v) && t->count)
            return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: %s: last axis must be contiguous with uniform row stride", what, name);
        *ld = v.ld;
        return check_device(t, name);
    }
    int32_t operands(const chelis_gpu_tensor *x, const chelis_gpu_tensor *w, int64_t *ldx) {
        int32_t s;
        if ((s = check_tensor(x, "x")) || (s = check_tensor(w, "w"))) return s;
        if (!is_narrow16(x->dtype)) return set_error(CHELIS_HIP_EDOMAIN, "%s: x must be bf16 or f16 (f32 and f64: linear)", what);
        if (x->rank < 1) return set_error(CHELIS_HIP_EDOMAIN, "%s: x needs a last axis", what);
        if (w->dtype != x->dtype || w->rank != 2 || w->shape[0] != x->shape[x->rank - 1])
            return set_error(CHELIS_HIP_EDOMAIN, "%s: w must be [K, N] of x's dtype", what);
        dt = x->dtype, K = w->shape[0], N = w->shape[1];
        if (K > kMaxWidth || N > kMaxWidth) return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: widths past 2^20", what);
        if ((s = row_operand(x, "x", x, K, ldx)) || (s = check_device(w, "w"))) return s;
        rows = 1;
        for (int32_t i = 0; i + 1 < x->rank; ++i) rows *= x->shape[i];
        return CHELIS_HIP_OK;
    }
    // w or dw [K, N]: lines along n (k apart) or along k (n apart).
    int32_t matrix(const chelis_gpu_tensor *t, const char *name, bool *along_k) {
        const int64_t sk = t->strides[0], sn = t->strides[1];
        if (sk == 1 && (sn != 1 || N == 1)) *along_k = true;
        else if (sn == 1 || N == 1) *along_k = false;
        else if (K == 1) *along_k = true;
        else return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: %s: one axis must be contiguous", what, name);
        return CHELIS_HIP_OK;
    }
    int32_t activation(int32_t act) {
        if (act < CHELIS_ACT_NONE || act > CHELIS_ACT_SILU)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: unknown activation %d", what, act);
        return CHELIS_HIP_OK;
    }
    // dbias or bias [N], dw [K, N]: of x's dtype or f32
    int32_t dtype_or_f32(const chelis_gpu_tensor *t, const char *name) {
        if (t->dtype != dt && t->dtype != CHELIS_DTYPE_F32)
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must have x's dtype or f32", what, name);
        return check_device(t, name);
    }
    int32_t vector(const chelis_gpu_tensor *t, const char *name) {
        if (int32_t s = check_tensor(t, name)) return s;
        if (t->rank != 1 || t->shape[0] != N || (N > 1 && t->strides[0] != 1))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be contiguous [N]", what, name);
        return dtype_or_f32(t, name);
    }
    int32_t result(const chelis_gpu_tensor *t, const char *name, std::initializer_list<NamedTensor> others) {
        if (!non_overlapping(t)) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s overlaps itself", what, name);
        if (const char *other = shared_with(t, others))
            return set_error(CHELIS_HIP_EDOMAIN, "%s: %s and %s overlap", what, name, other);
        return CHELIS_HIP_OK;
    }
    Side weights(const chelis_gpu_tensor *w, bool along_k) {
        const uint16_t *d = static_cast<const uint16_t *>(w->data);
        return along_k ? Side{d, N, K, w->strides[1]} : Side{d, K, N, w->strides[0]};
    }
};

template <class F>
int32_t with_kind(chelis_dtype dt, F &&f) {
    return dt == CHELIS_DTYPE_BF16 ? f(std::integral_constant<Narrow, Narrow::Bf16>())
                                   : f(std::integral_constant<Narrow, Narrow::F16>());
}

}  // namespace
}  // namespace chelis

using namespace chelis;

extern "C" int32_t chelis_hip_dense(const chelis_gpu_tensor *x, const chelis_gpu_tensor *w, const chelis_gpu_tensor *bias,
                                    int32_t activation, const chelis_gpu_tensor *residual, const chelis_gpu_tensor *y,
                                    const chelis_gpu_tensor *z) {
    DenseChecks c{"dense"};
    DenseProblem p{};
    int64_t ldx;
    bool along_k;
    int32_t s;
    if ((s = c.operands(x, w, &ldx)) || (s = c.activation(activation)) || (s = c.matrix(w, "w", &along_k)) ||
        (bias && (s = c.vector(bias, "bias"))) || (s = c.row_operand(y, "y", x, c.N, &p.ldc)) ||
        (residual && (s = c.row_operand(residual, "residual", x, c.N, &p.ldr))) ||
        (z && (s = c.row_operand(z, "z", x, c.N, &p.ldz))) || (s = c.result(y, "y", {{x, "x"}, {w, "w"}, {bias, "bias"}})) ||
        (z && (s = c.result(z, "z", {{x, "x"}, {w, "w"}, {bias, "bias"}, {residual, "residual"}, {y, "y"}}))))
        return s;
    if (residual && !same_view(y, residual) && shares_storage(y, residual))
        return set_error(CHELIS_HIP_EDOMAIN, "dense: y overlaps residual with other strides or from another element");
    if (!c.rows || !c.N) return CHELIS_HIP_OK;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    p.M = c.rows, p.N = c.N, p.K = c.K;
    p.c = y->data, p.act = activation;
    if (bias) p.bias = bias->data, p.bias32 = bias->dtype == CHELIS_DTYPE_F32;
    if (residual) p.resid = static_cast<const uint16_t *>(residual->data);
    if (z) p.z = static_cast<uint16_t *>(z->data);
    const Side a{static_cast<const uint16_t *>(x->data), c.rows, c.K, ldx}, b = c.weights(w, along_k);
    return with_kind(c.dt, [&](auto kind) -> int32_t {
        Scratch scratch;
        return forward<decltype(kind)::value>(p, a, b, along_k ? 0 : 1, scratch, st);
    });
}

extern "C" int32_t chelis_hip_dense_adjoint(const chelis_gpu_tensor *x, const chelis_gpu_tensor *w, const chelis_gpu_tensor *z,
                                            int32_t activation, const chelis_gpu_tensor *g, const chelis_gpu_tensor *dx,
                                            const chelis_gpu_tensor *dw, const chelis_gpu_tensor *dbias) {
    DenseChecks c{"dense_adjoint"};
    CotangentArgs ca{};
    int64_t ldx, lddx = 0;
    bool along_k, dw_along_k = false;
    int32_t s;
    if ((s = c.operands(x, w, &ldx)) || (s = c.activation(activation)) || (s = c.matrix(w, "w", &along_k)) ||
        (s = c.row_operand(g, "g", x, c.N, &ca.ldg)))
        return s;
    if (!dx && !dw && !dbias) return set_error(CHELIS_HIP_EDOMAIN, "dense_adjoint: no gradient asked for");
    if (activation != CHELIS_ACT_NONE) {
        if (!z) return set_error(CHELIS_HIP_EDOMAIN, "dense_adjoint: an activation's gradient needs z");
        if ((s = c.row_operand(z, "z", x, c.N, &ca.ldz))) return s;
    } else z = nullptr;
    const std::initializer_list<NamedTensor> inputs = {{x, "x"}, {w, "w"}, {z, "z"}, {g, "g"}};
    if (dx && ((s = c.row_operand(dx, "dx", x, c.K, &lddx)) || (s = c.result(dx, "dx", inputs)))) return s;
    if (dw) {
        if ((s = check_tensor(dw, "dw"))) return s;
        if (!same_shape(dw, w)) return set_error(CHELIS_HIP_EDOMAIN, "dense_adjoint: dw must be [K, N]");
        if ((s = c.dtype_or_f32(dw, "dw")) || (s = c.matrix(dw, "dw", &dw_along_k)) || (s = c.result(dw, "dw", inputs)) ||
            (s = c.result(dw, "dw", {{dx, "dx"}})))
            return s;
    }
    if (dbias && ((s = c.vector(dbias, "dbias")) || (s = c.result(dbias, "dbias", inputs)) ||
                  (s = c.result(dbias, "dbias", {{dx, "dx"}, {dw, "dw"}}))))
        return s;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    return with_kind(c.dt, [&](auto kind) -> int32_t {
        constexpr Narrow KIND = decltype(kind)::value;
        Scratch scratch;
        GradArgs ga{};
        Side dz{static_cast<const uint16_t *>(g->data), c.rows, c.N, ca.ldg};
        const bool form = (dx || dw) && c.rows && c.N && (activation != CHELIS_ACT_NONE || !dz.whole());
        if (form || (dbias && c.N)) {
            ca.g = dz.data, ca.z = z ? static_cast<const uint16_t *>(z->data) : nullptr;
            ca.M = c.rows, ca.N = c.N, ca.act = activation;
            const int64_t cols = (c.N + 255) / 256;
            // sixteen workgroups a CU, five at a time, at least 32 rows to each ([8192, 4096] with
            // K = 64: 72 us; with eight 79, with 32 72)
            int64_t chunks = std::max<int64_t>(1, std::min<int64_t>((int64_t)device_cus() * 16 / cols, (c.rows + 31) / 32));
            ca.chunk = std::max<int64_t>(1, (c.rows + chunks - 1) / chunks);
            chunks = std::max<int64_t>(1, (c.rows + ca.chunk - 1) / ca.chunk);
            if (form) {
                ca.lddz = (c.N + 7) / 8 * 8;
                ca.dz = static_cast<uint16_t *>(scratch.take((size_t)c.rows * ca.lddz * 2));
                if (!ca.dz) return set_error(CHELIS_HIP_EHIP, "dense_adjoint: scratch for dz");
                dz.data = ca.dz, dz.ld = dz.inner = ca.lddz;  // whole vectors, zeros past N
            }
            if (dbias) {
                ca.part = static_cast<float *>(scratch.take((size_t)chunks * c.N * sizeof(float)));
                if (!ca.part) return set_error(CHELIS_HIP_EHIP, "dense_adjoint: scratch for dbias");
            }
            dense_cotangent_kernel<KIND><<<dim3((unsigned)cols, (unsigned)chunks), 256, 0, st>>>(ca);
            CHELIS_LAUNCH_CHECK();
            if (dbias) ga.bias = BiasArgs{ca.part, dbias->data, chunks, c.N, dbias->dtype == CHELIS_DTYPE_F32};
        }
        const bool with_dx = dx && c.rows && c.K, with_dw = dw && c.K && c.N;
        Side xs{static_cast<const uint16_t *>(x->data), c.rows, c.K, ldx}, ws = c.weights(w, along_k);
        ga.dx.M = c.rows, ga.dx.N = c.K, ga.dx.K = c.N, ga.dx.ldc = lddx, ga.dx.c = dx ? dx->data : nullptr;
        ga.dw.M = dw_along_k ? c.N : c.K, ga.dw.N = dw_along_k ? c.K : c.N, ga.dw.K = c.rows;
        if (dw) ga.dw.c = dw->data, ga.dw.c32 = dw->dtype == CHELIS_DTYPE_F32, ga.dw.ldc = dw->strides[dw_along_k ? 1 : 0];
        // planned for both products whichever are asked for: each has the same bits alone
        const Extent3 e[2] = {{ga.dw.M, ga.dw.N, ga.dw.K, true}, {ga.dx.M, ga.dx.N, ga.dx.K, along_k}};
        const Plan plan = plan_for(e, 2);
        const ShapeCost &shape = kShapes[plan.shape];
        int32_t s;
        if ((s = lay_out({with_dw ? &xs : nullptr, with_dx ? &ws : nullptr}, scratch, st))) return s;
        ga.dw.slices = ga.dx.slices = 1;
        if (with_dw) {
            cut(&ga.dw, shape, plan.slices[0]);
            ga.dw_groups = (uint32_t)groups_of(ga.dw, shape);
            if ((s = dw_along_k ? set_sides(&ga.dw, dz, 1, xs, 1, scratch) : set_sides(&ga.dw, xs, 1, dz, 1, scratch))) return s;
        }
        if (with_dx) {
            cut(&ga.dx, shape, plan.slices[1]);
            ga.dx_groups = (uint32_t)groups_of(ga.dx, shape);
            if ((s = set_sides(&ga.dx, dz, 0, ws, along_k ? 1 : 0, scratch))) return s;
        }
        const int64_t groups = groups_of(ga.dw, shape) * with_dw + groups_of(ga.dx, shape) * with_dx + (ga.bias.N + 31) / 32;
        if (!groups) return CHELIS_HIP_OK;
        s = with_tiles(plan.shape, [&](auto tile) -> int32_t {
            using T = decltype(tile);
            if (!grid_fits(groups, T::THREADS)) return set_error(CHELIS_HIP_EUNSUPPORTED, "dense_adjoint: grid too large");
            if (along_k) dense_gradients_kernel<KIND, 1, T><<<(unsigned)groups, T::THREADS, 0, st>>>(ga);
            else dense_gradients_kernel<KIND, 0, T><<<(unsigned)groups, T::THREADS, 0, st>>>(ga);
            CHELIS_LAUNCH_CHECK();
            return CHELIS_HIP_OK;
        });
        if (s || (s = join_slices<KIND>(ga.dw, st)) || (s = join_slices<KIND>(ga.dx, st))) return s;
        return CHELIS_HIP_OK;
    });
}
