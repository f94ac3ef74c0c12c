// The 16-bit product of the dense operators on whole 16-byte vectors: operand
// tiles go from memory straight to LDS (no registers, no waiting in between)
// several K steps ahead of the matrix instructions that read them.
#pragma once

#include "elem.h"
#include "gemm16_tile.h"
#include "gelu16_poly.h"

#include "chelis_hip.h"

namespace chelis {
namespace {

// c[m][n] = sum_k a[m][k] b[k][n] with its epilogue. Elements of a and b sit at
// m * sam + k * sak and k * sbk + n * sbn; one stride of each is 1.
struct DenseProblem {
    const uint16_t *a, *b;
    int64_t M, N, K, sam, sak, sbk, sbn;
    void *c;  // 16 bits, or f32 (c32)
    int64_t ldc;
    const void *bias;  // 16 bits, or f32 (bias32)
    const uint16_t *resid;
    int64_t ldr;
    uint16_t *z;
    int64_t ldz;
    int32_t c32, bias32, act;
    // K slices: sums of slice s go to part[s][m][n] instead, kslice k each
    float *part;
    int64_t kslice;
    int32_t slices;
};

// ---------------------------------------------------------------- activations
// Phi(-a) = q exp(-a^2 / 2) for a = |x|: q by the degree-8 polynomial of
// gelu16_poly.h (6.3e-8), the exponential in binary32 (its argument's rounding grows
// to 2^-16 relative at |x| = 13, 2^-18 at 6, where the tail is under 1e-9). Degree 6
// (2.5e-6) would be hundredths of a 16-bit rounding, but shows where a residual cancels
// most of the value and in a dbias stored in binary32; it is 0.4 us of 56 faster (4096 x
// 1024 x 4096). Past 30 both are 0 against 1, and infinities would meet 0.
__device__ inline void phi_tail(float x, float &q, float &e, float &a) {
    constexpr float kQ[CHELIS_GELU16_DEG + 1] = CHELIS_GELU16_Q;
    a = fminf(fabsf(x), 30.f);
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 1.f / CHELIS_GELU16_K, 1.f));
    q = kQ[CHELIS_GELU16_DEG];
#pragma unroll
    for (int d = CHELIS_GELU16_DEG - 1; d >= 0; --d) q = fmaf(q, t, kQ[d]);
    e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170368f);
}
// x - |x| Phi(-|x|) for x >= 0, -|x| Phi(-|x|) below (NaN takes the first way).
__device__ inline float act_gelu(float x) {
    float q, e, a;
    phi_tail(x, q, e, a);
    return fmaf(-(a * q), e, x < 0.f ? 0.f : x);
}
// Phi(x) + x phi(x)
__device__ inline float slope_gelu(float x) {
    float q, e, a;
    phi_tail(x, q, e, a);
    const float below = e * fmaf(a, -0.39894228040143267794f, q), r = x < 0.f ? below : 1.f - below;
    return x != x ? x : r;
}
// x clamped where the result has long reached its limit (NaN stays).
__device__ inline float sigmoid(float x) {
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * -1.44269504088896340736f));
}
__device__ inline float act_silu(float x) {
    x = x < -100.f ? -100.f : x;
    return x * sigmoid(x);
}
__device__ inline float slope_silu(float x) {
    x = x < -100.f ? -100.f : x > 100.f ? 100.f : x;
    const float s = sigmoid(x);
    return s * fmaf(x, 1.f - s, 1.f);
}
__device__ inline float activate(float x, int act) {
    switch (act) {
        case CHELIS_ACT_RELU: return x < 0.f ? 0.f : x;
        case CHELIS_ACT_GELU: return act_gelu(x);
        case CHELIS_ACT_SILU: return act_silu(x);
        default: return x;
    }
}
// g act'(x). relu's slope selects, as relu_adjoint does: where x <= 0 nothing of g
// arrives, infinities and NaN included.
__device__ inline float act_adjoint(float g, float x, int act) {
    switch (act) {
        case CHELIS_ACT_RELU: return x > 0.f ? g : x != x ? x : 0.f;
        case CHELIS_ACT_GELU: return g * slope_gelu(x);
        case CHELIS_ACT_SILU: return g * slope_silu(x);
        default: return g;
    }
}

// ---------------------------------------------------------------- epilogue
template <Narrow K>
struct Elem16;
template <>
struct Elem16<Narrow::Bf16> {
    using type = __bf16;
};
template <>
struct Elem16<Narrow::F16> {
    using type = _Float16;
};
template <Narrow KIND>
using Vec16 = Pack<typename Elem16<KIND>::type, 8>;

// Eight elements of a row, as far as `count` goes.
template <Narrow KIND>
__device__ inline void store8(uint16_t *p, const float (&v)[8], int64_t count) {
    using T = typename Elem16<KIND>::type;
    T *o = reinterpret_cast<T *>(p);
    Vec16<KIND> q;
#pragma unroll
    for (int i = 0; i < 8; ++i) q.set(i, v[i]);
    if (count >= 8) q.store(o);
    else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < count) o[i] = q.q[i];
    }
}
template <Narrow KIND>
__device__ inline Vec16<KIND> load8v(const uint16_t *p, int64_t count) {
    using T = typename Elem16<KIND>::type;
    const T *in = reinterpret_cast<const T *>(p);
    Vec16<KIND> q{};
    if (count >= 8) q.load(in);
    else {
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (i < count) q.q[i] = in[i];
    }
    return q;
}
template <Narrow KIND>
__device__ inline void load8f(const uint16_t *p, float (&v)[8], int64_t count) {
    const Vec16<KIND> q = load8v<KIND>(p, count);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = q.get(i);
}
typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));

// Eight neighbouring columns of a row, `count` of them there: the sums in v, the
// bias and (of the residual's type) the residual already loaded; at, at_z: their
// elements in the result and in z.
template <Narrow KIND>
__device__ inline void finish8(const DenseProblem &p, int64_t at, int64_t at_z, int64_t count, float (&v)[8],
                               const float (&bias)[8], const Vec16<KIND> &resid) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] += bias[i];
    if (p.z) store8<KIND>(p.z + at_z, v, count);
    if (p.act != CHELIS_ACT_NONE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = activate(v[i], p.act);
    }
    if (p.resid) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += resid.get(i);
    }
    if (p.c32) {
        float *o = static_cast<float *>(p.c) + at;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) o[i] = canon_bits(v[i]);
    } else store8<KIND>(static_cast<uint16_t *>(p.c) + at, v, count);
}
template <Narrow KIND>
__device__ inline void load_bias(const DenseProblem &p, int64_t n, int64_t count, float (&b)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) b[i] = 0.f;
    if (!p.bias) return;
    if (p.bias32) {
        const float *q = static_cast<const float *>(p.bias) + n;
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = i < count ? q[i] : 0.f;
    } else load8f<KIND>(static_cast<const uint16_t *>(p.bias) + n, b, count);
}
// The same for one K slice's sums.
__device__ inline void slice8(float *o, int64_t count, const float (&v)[8]) {
    if (count >= 8) {
        *reinterpret_cast<F4 *>(o) = F4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<F4 *>(o + 4) = F4{v[4], v[5], v[6], v[7]};
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < count) o[i] = v[i];
    }
}

// ---------------------------------------------------------------- tiles
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
#define CHELIS_LDS __attribute__((address_space(3)))

template <Narrow K>
__device__ inline f32x16 mfma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (K == Narrow::Bf16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
}

// 64 16-byte vectors, one a lane, from base + voff to 1 KiB of LDS at lds (the
// same in every lane). The hardware checks voff against the buffer's 2^31
// bytes: a lane with kNowhere reads nothing and stores zeros. Written in
// assembly because the compiler waits for such a load before the next
// transposed LDS read, whichever buffer that goes to; it writes no register (m0,
// where it takes the LDS address from, is an operand that the compiler sets), and
// load_wait below waits for it.
constexpr uint32_t kNowhere = 0x80000000u;
__device__ inline void load_to_lds(uint32_t lds, uint32_t voff, const uint16_t *base) {
    const uint64_t at = reinterpret_cast<uint64_t>(base);
    const i32x4 r = {(int)(uint32_t)at, (int)(uint32_t)(at >> 32 & 0xffff), (int)0x80000000u, 0x00027000};
    asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"{m0}"(lds), "v"(voff), "s"(r) : "memory");
}
// Until at most N of this wave's loads are under way (they land in order) and
// its LDS reads are done; then every wave of the workgroup.
template <int N>
__device__ inline void load_wait() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// One operand's tile of ROWS outer elements by BK.
//   LAY 0, contiguous along k: LDS holds [row][BK], the 16-byte vectors of a row
//     exchanged by the row, so that neighbouring lanes' rows lie on different
//     banks; a fragment is one 16-byte read.
//   LAY 1, contiguous along the outer axis: LDS holds [k][ROWS], the 32-byte
//     pairs of a k exchanged by k; a fragment is two transposing reads, each of
//     four k by 16 rows to 16 lanes.
template <int LAY, int ROWS, int BK, int THREADS_>
struct Operand {
    static constexpr int VEC = ROWS * BK / 8, NV = VEC / THREADS_, LINE = LAY == 0 ? BK / 8 : ROWS / 8;
    static_assert(VEC % THREADS_ == 0, "whole vectors a thread");
    static constexpr int BYTES = ROWS * BK * 2;
    uint32_t off[NV];
    const uint16_t *at;  // the tile at the next K step to load
    int64_t step;

    // row0: the tile's first outer element of `outer`; s: the stride of the
    // other axis.
    __device__ void init(const uint16_t *base, int64_t s, int64_t row0, int64_t outer, int64_t k0) {
        const int t = threadIdx.x;
        at = LAY == 0 ? base + row0 * s + k0 : base + row0 + k0 * s;
        step = LAY == 0 ? BK : BK * s;
        const int64_t left = outer - row0;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int slot = t + THREADS_ * j, line = slot / LINE, v = vector_at(line, slot % LINE);
            const bool there = LAY == 0 ? line < left : 8 * v < left;
            off[j] = there ? 2u * (uint32_t)(line * (uint32_t)s + 8 * v) : kNowhere;
        }
    }
    // the vector that LDS position p of a line holds (its own inverse)
    __device__ static int vector_at(int line, int p) {
        if constexpr (LAY == 0) return p ^ (BK >= 64 ? line & 7 : line >> 1 & 3);
        else return p ^ (ROWS >= 64 ? (line & 3) << 1 : (line >> 1 & 1) << 1);
    }
    // left: K elements from this step on
    __device__ void load(uint32_t lds, int64_t left) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds + wave * 1024);
        if (left >= BK) {
#pragma unroll
            for (int j = 0; j < NV; ++j) load_to_lds(to + j * THREADS_ * 16, off[j], at);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int slot = threadIdx.x + THREADS_ * j, line = slot / LINE;
                const int k = LAY == 0 ? 8 * vector_at(line, slot % LINE) : line;
                load_to_lds(to + j * THREADS_ * 16, k < left ? off[j] : kNowhere, at);
            }
        }
        at += step;
    }
    // rows row .. row + 31, k = 16 kk + 8 (lane / 32) ..: lane's fragment
    __device__ static uint4 fragment(const uint16_t *tile, int row, int kk) {
        const int lane = threadIdx.x & 63;
        if constexpr (LAY == 0) {
            const int r = row + (lane & 31), v = 2 * kk + (lane >> 5);
            return *reinterpret_cast<const uint4 *>(tile + r * BK + 8 * vector_at(r, v));
        } else {
            const int i = lane & 15, k = 16 * kk + 8 * (lane >> 5) + (i >> 2), r = row + 16 * (lane >> 4 & 1) + 4 * (i & 3);
            const uint16_t *at = tile + k * ROWS + 8 * vector_at(k, r >> 3) + (r & 7);
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CHELIS_LDS s16x4 *)at);
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((CHELIS_LDS s16x4 *)(at + 4 * ROWS));
            return __builtin_bit_cast(uint4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// A workgroup's tile: XCDs (workgroups are dealt to them in turn) get a run of
// tiles each, walked in groups of 8 tile rows so that a run shares operands. The
// divisions run on the vector units: their results go back to scalar registers, or
// every address formed from them takes two vector registers to the kernel's end.
__device__ inline uint32_t scalar(uint32_t v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, uint32_t *tm, uint32_t *tn) {
    constexpr uint32_t GM = 8;
    const uint32_t tiles = tiles_m * tiles_n, q = tiles / 8, r = tiles % 8, xcd = id % 8;
    id = xcd * q + (xcd < r ? xcd : r) + id / 8;
    const uint32_t group = scalar(id / (GM * tiles_n)), first = group * GM;
    const uint32_t size = tiles_m - first < GM ? tiles_m - first : GM, in = id - group * GM * tiles_n;
    *tn = scalar(in / size);
    *tm = first + in - *tn * size;
}

// BM x BN results a workgroup of WM x WN waves, WK times (each with its part of
// every step's k, joined at the end), K in steps of BK through ST buffers.
template <int BM_, int BN_, int BK_, int WM_, int WN_, int WK_, int ST_, int OCC_>
struct TileShape {
    static constexpr int BM = BM_, BN = BN_, BK = BK_, WM = WM_, WN = WN_, WK = WK_, ST = ST_, OCC = OCC_;
    static constexpr int THREADS = 64 * WM * WN * WK, MI = BM / WM / 32, NJ = BN / WN / 32;
    static constexpr int STAGE = (BM + BN) * BK * 2, PITCH = BN + 4, EPI = WM * 32 * PITCH * 4;
    static constexpr int EPI_UNROLL = MI > 2 ? 1 : MI;  // code size against registers moved
    static constexpr int BYTES = STAGE * ST > EPI * WK ? STAGE * ST : EPI * WK;
    static_assert(BK / 16 % WK == 0, "whole k blocks a wave");
};

// Workgroup `index` of a product: its slices' tiles, one slice after the other.
template <Narrow KIND, int ALAY, int BLAY, class C>
__device__ inline void dense_tile(const DenseProblem &p, uint32_t index, char *lds) {
    constexpr int BM = C::BM, BN = C::BN, BK = C::BK, ST = C::ST, MI = C::MI, NJ = C::NJ;
    const uint32_t tiles_m = (uint32_t)((p.M + BM - 1) / BM), tiles_n = (uint32_t)((p.N + BN - 1) / BN);
    const uint32_t slice = scalar(index / (tiles_m * tiles_n));
    uint32_t tm, tn;
    tile_of(index - slice * tiles_m * tiles_n, tiles_m, tiles_n, &tm, &tn);
    const int64_t m0 = (int64_t)tm * BM, n0 = (int64_t)tn * BN, k0 = slice * p.kslice;
    const int64_t K = p.K - k0 < p.kslice ? p.K - k0 : p.kslice;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wk = wave / (C::WM * C::WN);
    const int wm = wave / C::WN % C::WM, wn = wave % C::WN;

    Operand<ALAY, BM, BK, C::THREADS> a;
    Operand<BLAY, BN, BK, C::THREADS> b;
    a.init(p.a, ALAY == 0 ? p.sam : p.sak, m0, p.M, k0);
    b.init(p.b, BLAY == 0 ? p.sbn : p.sbk, n0, p.N, k0);
    const uint32_t lds0 = (uint32_t)reinterpret_cast<uintptr_t>((CHELIS_LDS char *)lds);
    const int steps = (int)((K + BK - 1) / BK);
    int64_t left = K;
    int into = 0;
    // past the last step nothing is read, the loads only keep the count
    auto load = [&]() {
        a.load(lds0 + into * C::STAGE, left);
        b.load(lds0 + into * C::STAGE + BM * BK * 2, left);
        left -= BK;
        into = into + 1 == ST ? 0 : into + 1;
    };
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) load();

    f32x16 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = f32x16{};
    constexpr int AHEAD = (ST - 2) * (a.NV + b.NV);
    int from = 0;
    for (int s = 0; s < steps; ++s) {
        load_wait<AHEAD>();
        load();
        const uint16_t *as = reinterpret_cast<const uint16_t *>(lds + from * C::STAGE), *bs = as + BM * BK;
        from = from + 1 == ST ? 0 : from + 1;
#pragma unroll
        for (int kk = 0; kk < BK / 16; kk += C::WK) {
            uint4 af[MI], bf[NJ];
#pragma unroll
            for (int i = 0; i < MI; ++i) af[i] = a.fragment(as, (wm * MI + i) * 32, kk + wk);
#pragma unroll
            for (int j = 0; j < NJ; ++j) bf[j] = b.fragment(bs, (wn * NJ + j) * 32, kk + wk);
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = mfma32<KIND>(af[i], bf[j], acc[i][j]);
        }
    }
    // 32 rows of every wave at a time through LDS: a thread then holds eight
    // neighbouring columns of some rows, and memory sees whole rows of the tile.
    // The residual's loads go ahead of the exchange that they do not wait for.
    constexpr int PER = BN / 8, ROWS = C::THREADS / PER, VPT = (C::WM * 32 + ROWS - 1) / ROWS;
    static_assert(C::THREADS % PER == 0 && (ROWS % 32 == 0 || 32 % ROWS == 0), "a thread keeps its columns");
    const int r0 = threadIdx.x / PER;
    const int64_t n = n0 + 8 * (threadIdx.x % PER), count = p.N - n;
    // row of the tile: a part of the thread's own and one that is the same for all
    const int64_t m_own = m0 + (r0 >> 5) * (MI * 32) + (r0 & 31);
    const auto further = [](int i, int k) { return i * 32 + (k * ROWS >> 5) * (MI * 32) + (k * ROWS & 31); };
    const int64_t at = m_own * p.ldc + n, at_z = m_own * p.ldz + n, at_part = (slice * p.M + m_own) * p.N + n;
    const uint16_t *resid_own = p.resid + (m_own * p.ldr + n);
    const bool mine_here = r0 < C::WM * 32 && count > 0;
    float bias[8];
    load_bias<KIND>(p, n, count, bias);
    float *stage = reinterpret_cast<float *>(lds), *mine = stage + wk * (C::EPI / 4);
    const float *from_stage = stage + r0 * C::PITCH + 8 * (threadIdx.x % PER);
    load_wait<0>();
#pragma unroll C::EPI_UNROLL
    for (int i = 0; i < MI; ++i) {
        Vec16<KIND> resid[VPT];
#pragma unroll
        for (int k = 0; k < VPT; ++k)
            if (p.resid && !p.part && mine_here && m_own + further(i, k) < p.M)
                resid[k] = load8v<KIND>(resid_own + further(i, k) * p.ldr, count);
        if (i) __syncthreads();
#pragma unroll
        for (int c = 0; c < MI; ++c)
            if (c == i) {
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        mine[(wm * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5)) * C::PITCH + (wn * NJ + j) * 32 + (lane & 31)] =
                            acc[c][j][r];
            }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int64_t more = further(i, k);
            __builtin_amdgcn_sched_barrier(0);  // one vector's arithmetic at a time: interleaved they spilled
            if (!mine_here || m_own + more >= p.M) continue;
            float x[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = from_stage[k * ROWS * C::PITCH + q];
#pragma unroll
            for (int w = 1; w < C::WK; ++w)
#pragma unroll
                for (int q = 0; q < 8; ++q) x[q] += from_stage[w * (C::EPI / 4) + k * ROWS * C::PITCH + q];
            if (p.part) slice8(p.part + at_part + more * p.N, count, x);
            else finish8<KIND>(p, at + more * p.ldc, at_z + more * p.ldz, count, x, bias, resid[k]);
        }
    }
}

template <Narrow KIND, int ALAY, int BLAY, class C>
__global__ __launch_bounds__(C::THREADS, C::OCC) void dense_tile_kernel(DenseProblem p) {
    __shared__ __attribute__((aligned(1024))) char lds[C::BYTES];
    dense_tile<KIND, ALAY, BLAY, C>(p, blockIdx.x, lds);
}

}  // namespace
}  // namespace chelis
