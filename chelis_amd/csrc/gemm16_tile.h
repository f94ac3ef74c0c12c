// What the 16-bit matrix kernels share: the 16x16x32 matrix instruction and the
// staging of an operand tile through registers into LDS, for operands of any
// alignment and extent. THREADS, BK and LD are the kernels' common tile.
#pragma once

#include "narrow.h"

#include <cstdint>

namespace chelis {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <Narrow K>
__device__ inline f32x4 mfma16(uint4 a, uint4 b, f32x4 c) {
    if constexpr (K == Narrow::Bf16)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b),
                                                       c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c,
                                                      0, 0, 0);
}

constexpr int THREADS = 256, BM = 128, BN = 128, BK = 64, LD = 72;

// One operand tile [ROWS][BK] staged in registers: LAY 0 = vectors along K,
// 8 values per 16-byte vector, stored as they are; 2 = element by element.
// LAY 1 = vectors along the outer axis (M of A, N of B), which LDS wants
// K-contiguous: thread t owns the 4 x 8 block of outer rows 4 nb + e (e < 4)
// and k = 8 kb + u (u < 8), nb = t % 4 + 4 (t / 32), kb = (t / 4) % 8. It
// reads one 8-byte vector of 4 rows per k, transposes the block in
// registers (one byte permute per output word) and writes one 16-byte
// vector of 8 k per row: with the 144-byte row pitch, 16 consecutive lanes
// write 16 distinct 4-bank groups (rows 4 nb + e, columns 8 kb), where the
// former element-by-element 2-byte stores took 32 LDS writes per thread.
// Vectors need only their element's alignment (a global access needs no more
// on gfx950): a [512, 213] operand is staged as a [512, 216] one.
typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t U2 __attribute__((ext_vector_type(2), aligned(2)));
__device__ inline uint4 load8(const uint16_t *p) {
    const U4 v = *reinterpret_cast<const U4 *>(p);
    return uint4{v.x, v.y, v.z, v.w};
}
__device__ inline uint2 load4(const uint16_t *p) {
    const U2 v = *reinterpret_cast<const U2 *>(p);
    return uint2{v.x, v.y};
}

template <int LAY, int ROWS>
struct Stage16 {
    static constexpr int NV = ROWS * BK / 8 / THREADS;
    static_assert(ROWS * BK == 32 * THREADS || ROWS * BK == 16 * THREADS, "a 4 x 8 block per thread, or per other thread");
    static constexpr int ACTIVE = ROWS * BK / 32;  // LAY 1: threads with a block
    uint4 r[LAY == 1 ? 1 : NV];
    uint2 q[LAY == 1 ? 8 : 1];

    // element (row, k) at base[row * s_row + k * s_k]; CHECK = false: the
    // whole tile is inside the operand. With CHECK a vector that would run
    // past the operand is moved back to end with it, and store() puts its
    // elements where they belong: no branch around a load, which made the
    // compiler wait for each before the next. Rows past the operand's hold
    // others of its values (nothing of theirs is stored); k past K is zero.
    // LAY 0 needs K >= 8, LAY 1 four rows. (Bounds branches: 1100 x 1100 x 33
    // bf16 13.9 us with both operands along the outer axis, 8191 x 65 x 4097
    // 315; element by element 10.5 and 171.)
    template <bool CHECK>
    __device__ void load(const uint16_t *__restrict__ base, int64_t s_row, int64_t s_k, int64_t row0, int64_t rows,
                         int64_t k0, int64_t K) {
        const int t = threadIdx.x;
        if constexpr (LAY == 1) {
            if (ACTIVE < THREADS && t >= ACTIVE) return;
            const int nb = t % 4 + 4 * (t / 32), kb = (t / 4) % 8;
            const int64_t gr = row0 + 4 * nb, at = CHECK && gr + 4 > rows ? rows - 4 : gr;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int64_t gk = k0 + 8 * kb + u;
                q[u] = load4(base + at + (CHECK && gk >= K ? K - 1 : gk) * s_k);
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int idx = t + THREADS * j;
            const int row = idx / (BK / 8), kv = (idx % (BK / 8)) * 8;
            const int64_t gr = row0 + row, gk = k0 + kv;
            if constexpr (LAY == 0) {
                r[j] = load8(base + (CHECK && gr >= rows ? rows - 1 : gr) * s_row + (CHECK && gk + 8 > K ? K - 8 : gk));
            } else {
                const uint16_t *p = base + gr * s_row + gk * s_k;
                uint16_t e[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) e[u] = (gr < rows && gk + u < K) ? p[u * s_k] : (uint16_t)0;
                r[j] = __builtin_bit_cast(uint4, e);
            }
        }
    }

    // row0 .. K: as the load's
    template <bool CHECK>
    __device__ void store(uint16_t *lds, int64_t row0, int64_t rows, int64_t k0, int64_t K) {
        const int t = threadIdx.x;
        if constexpr (LAY == 1) {
            if (ACTIVE < THREADS && t >= ACTIVE) return;
            const int nb = t % 4 + 4 * (t / 32), kb = (t / 4) % 8;
            if (CHECK && row0 + ROWS > rows) {
                const int64_t d = row0 + 4 * nb - (rows - 4);  // rows moved back; four and more: none of them is stored
                const int sh = d > 0 && d < 4 ? 16 * (int)d : 0;
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    q[u] = __builtin_bit_cast(uint2, __builtin_bit_cast(uint64_t, q[u]) >> sh);
            }
            if (CHECK && k0 + BK > K) {
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (k0 + 8 * kb + u >= K) q[u] = uint2{0, 0};
            }
            // output row e, word w: k = 2w in the low half, 2w + 1 in the high
            uint32_t w[4][4];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                const uint32_t a0 = q[2 * h].x, a1 = q[2 * h].y, b0 = q[2 * h + 1].x, b1 = q[2 * h + 1].y;
                w[0][h] = (a0 & 0xffffu) | (b0 << 16);
                w[1][h] = (a0 >> 16) | (b0 & 0xffff0000u);
                w[2][h] = (a1 & 0xffffu) | (b1 << 16);
                w[3][h] = (a1 >> 16) | (b1 & 0xffff0000u);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<uint4 *>(lds + (4 * nb + e) * LD + 8 * kb) = uint4{w[e][0], w[e][1], w[e][2], w[e][3]};
            return;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int idx = t + THREADS * j;
            const int row = idx / (BK / 8), kv = (idx % (BK / 8)) * 8;
            if (LAY == 0 && CHECK && k0 + BK > K) {
                const int64_t d = k0 + kv + 8 - K;  // elements moved back
                const uint64_t lo = (uint64_t)r[j].y << 32 | r[j].x, hi = (uint64_t)r[j].w << 32 | r[j].z;
                if (d > 0) {
                    const int sh = 16 * (int)(d & 3);
                    const uint64_t x = d < 4 ? lo : d < 8 ? hi : 0, y = d < 4 ? hi : 0;
                    const uint64_t l = sh ? x >> sh | y << (64 - sh) : x, h = y >> sh;
                    r[j] = uint4{(uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32)};
                }
            }
            *reinterpret_cast<uint4 *>(lds + row * LD + kv) = r[j];
        }
    }
};

}  // namespace
}  // namespace chelis
