// Attention with a sliding window and always-visible first tokens (sinks):
// query row i of a sequence of n keys stands at position p = start + i and
// sees key j when 0 <= j <= p < n and (p - j < window or j < sinks), so
//   o_i = sum_j P_ij v_j,  P_ij = exp(scale q_i.k_j - lse_i)
// over the visible j, o_i = 0 and lse_i = -inf where there is none, and with
// D_i = g_i . o_i and dS_ij = P_ij (g_i . v_j - D_i)
//   dq_i = scale sum_j dS_ij k_j, dk_j = scale sum_i dS_ij q_i,
//   dv_j = sum_i P_ij g_i
// summed over the query heads that share a key head.
//
// All products run on the matrix cores as 32 x 32 blocks (16 elements of the
// summed axis a step; binary32 operands as eight steps of 2). Layouts, for
// lane l with i = l % 32 and h = l / 32:
//   A and B hold eight elements of row (column) i: elements 8h .. 8h + 7 of
//   the step's 16, or any other order that both share;
//   C[8 (r / 4) + 4 h + r % 4][i] is item r of 16.
// Scores are formed so that the rows of C are what the next product sums
// over: eight consecutive items of C, rounded to the operand type, are then
// the B operand of the next product as they stand, in the order
// 4h .. 4h + 3, 8 + 4h .. 8 + 4h + 3 (and 16 more for items 8 .. 15), and
// nothing crosses lanes. The other operand reads the tile across its rows in
// the same order (16-bit types with the transposing LDS read).
//
// Scores, softmax statistics and sums are binary32. P and dS are rounded to
// the operand type for the products that sum over them, as the operands
// themselves are; the sum of P that divides the result is of the unrounded
// values.
#include "elem.h"

#include <algorithm>
#include <type_traits>

namespace chelis {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename T>
using V8 = T __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kKeys = 64;   // keys of a staged tile (forward, dq)
constexpr int kRows = 32;   // query rows of a staged tile (dk, dv)
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
// rows and keys: sums of three of them stay inside 32 bits
constexpr int64_t kMaxExtent = (int64_t(1) << 29) - 1024;

__device__ inline f32x16 mma(V8<__bf16> a, V8<__bf16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mma(V8<_Float16> a, V8<_Float16> b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mma(V8<float> a, V8<float> b, f32x16 c) {
#pragma unroll
    for (int t = 0; t < 8; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
    return c;
}

// LDS rows of D elements, 32 bytes apart from a multiple of the 256-byte
// bank span: 16-byte reads down a column of rows and the transposing reads
// of four rows both touch every bank once.
template <typename T, int D>
constexpr int kPitch = D + 32 / (int)sizeof(T);

// Eight elements of tile row `row` from element `at`.
template <typename T, int D>
__device__ inline V8<T> along(const T *tile, int row, int at) {
    return *reinterpret_cast<const V8<T> *>(tile + row * kPitch<T, D> + at);
}
// Column d0 + l % 32 of tile rows row0 + 4h .. + 3 and row0 + 8 + 4h .. + 3.
template <typename T, int D>
__device__ inline V8<T> across(const T *tile, int row0, int d0, int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        // each 16 lanes read four rows of 16 elements, lane i the four
        // elements 4 (i % 4) .. of row i / 4, and lane i gets column i
        const T *p = tile + (row0 + 4 * h + ((lane & 15) >> 2)) * kPitch<T, D> + d0 + (lane & 16) + 4 * (lane & 3);
        typedef __attribute__((address_space(3))) s16x4 *Lds;
        union {
            s16x4 q[2];
            V8<T> v;
        } u;
        u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p);
        u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 8 * kPitch<T, D>));
        return u.v;
    } else {
        const T *p = tile + (row0 + 4 * h) * kPitch<T, D> + d0 + (lane & 31);
        V8<T> v;
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = p[(t < 4 ? t : 4 + t) * kPitch<T, D>];
        return v;
    }
}

template <typename T>
__device__ inline bool not_finite(T v) {
    if constexpr (sizeof(T) == 2) {
        constexpr uint16_t e = std::is_same<T, _Float16>::value ? 0x7c00 : 0x7f80;
        return (__builtin_bit_cast(uint16_t, v) & e) == e;
    } else {
        return (f32_bits(v) & 0x7f800000u) == 0x7f800000u;
    }
}

// A hidden pair adds nothing, whatever it holds: its weight is 0, but 0 times
// an infinity or a NaN would be NaN. Tiles that some row or key does not see
// whole are looked over while they are staged; where one holds such an
// element, the pairs that see it get it added by themselves (add_special) and
// the tile is cleaned before its product. Rarely run.
template <typename T>
struct Largest {
    using U = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
    static constexpr U kInf = sizeof(T) == 4 ? (U)0x7f800000u : std::is_same<T, _Float16>::value ? (U)0x7c00 : (U)0x7f80;
    V8<U> m = {};
    __device__ void add(V8<T> v) {
        m = __builtin_elementwise_max(m, __builtin_bit_cast(V8<U>, v) & (U)~((U)1 << (8 * sizeof(U) - 1)));
    }
    __device__ bool special() const {
        using U4 = U __attribute__((ext_vector_type(4)));
        using U2 = U __attribute__((ext_vector_type(2)));
        const U4 a = __builtin_elementwise_max(U4(m.lo), U4(m.hi));
        const U2 b = __builtin_elementwise_max(U2(a.lo), U2(a.hi));
        return (b[0] >= kInf) | (b[1] >= kInf);
    }
};

// Adds the infinities and NaN of tile rows that `sees` holds for to the
// accumulated columns of weights >= 0.
template <typename T, int D, int N, class Sees>
__device__ inline void add_special(f32x16 (&acc)[D / 32], const T *tile, int h, Sees sees) {
#pragma unroll 1
    for (int row = 0; row < N; ++row) {
        const bool seen = sees(row);
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const T x = tile[row * kPitch<T, D> + 32 * d + 8 * (r >> 2) + 4 * h + (r & 3)];
                acc[d][r] += (seen & not_finite(x)) ? widen<T>(x) : 0.f;
            }
    }
}
// The same as marks, one bit an accumulated element, put in once the sums are
// whole: for kernels whose accumulators only the matrix cores touch while they
// run (any other use made the compiler move all of them between register files
// on every tile). With weights of either sign any special value makes the sum NaN.
template <int D>
struct Marks {
    static constexpr int W = (D / 2 + 31) / 32;
    uint32_t nan[W] = {}, up[W] = {}, down[W] = {};
    template <bool SIGNED, typename T, int N, class Sees>
    __device__ void note(const T *tile, int h, Sees sees) {
#pragma unroll 1
        for (int row = 0; row < N; ++row) {
            const bool seen = sees(row);
#pragma unroll
            for (int e = 0; e < D / 2; ++e) {
                const T x = tile[row * kPitch<T, D> + 32 * (e >> 4) + 8 * ((e & 15) >> 2) + 4 * h + (e & 3)];
                const bool hit = seen & not_finite(x), is_nan = SIGNED | (x != x);
                nan[e / 32] |= (uint32_t)(hit & is_nan) << (e % 32);
                up[e / 32] |= (uint32_t)(hit & !is_nan & (x > (T)0.f)) << (e % 32);
                down[e / 32] |= (uint32_t)(hit & !is_nan & (x < (T)0.f)) << (e % 32);
            }
        }
    }
    __device__ void apply(f32x16 (&acc)[D / 32]) const {
        uint32_t any = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) any |= nan[w] | up[w] | down[w];
        if (!__any(any != 0)) return;
#pragma unroll
        for (int e = 0; e < D / 2; ++e) {
            float x = (up[e / 32] >> (e % 32)) & 1 ? INFINITY : 0.f;
            x += (down[e / 32] >> (e % 32)) & 1 ? -INFINITY : 0.f;
            x = (nan[e / 32] >> (e % 32)) & 1 ? __builtin_nanf("") : x;
            acc[e >> 4][e & 15] += x;
        }
    }
};
// An infinity in v that a row sees makes its column infinite, whatever it
// weighs. But its weight may round to 0 (f16 holds e^-24 at least), or be scaled
// to 0 when a far larger score follows, and both make NaN of it. The columns it
// stands in are the only ones it reaches, so where a wave's sums came out
// infinite or NaN it looks over the keys it walked once more and sets those
// columns to what they hold. The look at the sums (64 multiply-adds at heads of
// 128) is all that other calls pay.
template <int D>
__device__ inline bool has_special(const f32x16 (&acc)[D / 32]) {
    float odd = 0.f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = fmaf(acc[d][r], 0.f, odd);
    return odd != 0.f;
}
// The infinities and NaN that a lane's row sees, a bit for each accumulated
// element; NaN sets both. `need`: the elements that no finite sum stands in.
template <typename T, int D>
struct SeenSpecials {
    uint64_t need = 0, up = 0, down = 0;
    __device__ SeenSpecials(const f32x16 (&acc)[D / 32], bool stored) {
#pragma unroll
        for (int e = 0; e < D / 2; ++e) need |= (uint64_t)(stored & not_finite(acc[e >> 4][e & 15])) << e;
    }
    // nothing that the wave's rows could still see would change them
    __device__ bool done() const { return !__any((need & ~(up & down)) != 0); }
    // keys k0 .. end - 1 of v, the whole wave together
    template <class Sees>
    __device__ void note(const T *V, int64_t step, int width, int k0, int end, int lane, Sees sees) {
        constexpr int C = D / 8, R = 64 / C;
        for (int j = k0; j < end; j += R) {
            const int key = j + lane / C, at = lane % C * 8;
            uint32_t mine = 0;  // which of the lane's eight, +inf in the low byte
            if (lane < R * C && key < end && at < width) {
                Pack<T, 8> x;
                x.load(V + key * step + at);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint32_t hit = not_finite(x.q[c]);
                    mine |= (x.q[c] < (T)0.f ? 0 : hit) << c | (x.q[c] > (T)0.f ? 0 : hit) << (8 + c);
                }
            }
            // four of eight columns belong to each half of the wave
            for (uint64_t hits = __ballot(mine != 0); hits; hits &= hits - 1) {
                const int lead = __ffsll((unsigned long long)hits) - 1, c0 = lead % C * 8;
                const uint32_t theirs = (uint32_t)__builtin_amdgcn_readlane((int)mine, lead) >> (lane >> 5) * 4;
                const uint64_t seen = sees(j + lead / C) ? 15 : 0;
                up |= (theirs & seen) << (c0 / 32 * 16 + c0 % 32 / 8 * 4);
                down |= (theirs >> 8 & seen) << (c0 / 32 * 16 + c0 % 32 / 8 * 4);
            }
        }
    }
    __device__ void put(f32x16 (&acc)[D / 32]) const {
#pragma unroll
        for (int e = 0; e < D / 2; ++e) {
            const bool u = up >> e & 1, d = down >> e & 1;
            const float x = (u ? INFINITY : 0.f) + (d ? -INFINITY : 0.f);
            acc[e >> 4][e & 15] = (u | d) ? x : acc[e >> 4][e & 15];
        }
    }
};
// The factor of a row's unscaled sums; a row whose every score is -inf is NaN.
__device__ inline float row_factor(bool empty, float l) {
    return empty ? 0.f : l > 0.f ? 1.f / l : __builtin_nanf("");
}
template <typename T, int D, int N, int THREADS>
__device__ inline void clean(T *tile, int tid) {
    for (int id = tid; id < N * (D / 8); id += THREADS) {
        V8<T> *p = reinterpret_cast<V8<T> *>(tile + id / (D / 8) * kPitch<T, D> + id % (D / 8) * 8);
        V8<T> v = *p;
#pragma unroll
        for (int t = 0; t < 8; ++t) v[t] = not_finite(v[t]) ? (T)0.f : v[t];
        *p = v;
    }
}

template <typename T>
__device__ inline V8<T> rounded(const f32x16 &s, int from) {
    V8<T> v;
#pragma unroll
    for (int t = 0; t < 8; ++t) v[t] = (T)s[from + t];
    return v;
}

// The order of a product loop's instructions: LDS reads for AHEAD products
// first, then one product and the reads for a later one in turn, so that no
// product waits for its own reads. (The compiler kept two reads in flight and
// waited for them before every second product.)
template <int PRODUCTS, int READS, int AHEAD>
__device__ inline void interleave() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS * AHEAD, 0);
#pragma unroll
    for (int k = 0; k < PRODUCTS - AHEAD; ++k) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
}

struct View {
    const void *p;
    int64_t b, h, s;  // strides of batch, head, sequence
};

struct WinArgs {
    View q, k, v, o, g, dq, dk, dv;
    const float *lse_in;
    float *lse, *delta, *range;
    const void *lengths, *starts;
    int64_t length_step, start_step;
    int lengths_wide, starts_wide;
    int sq, sk, window, sinks, heads, kv, group, width, flip;
    float c, signed_c, scale;  // |scale| log2(e), scale log2(e), scale
};

// Which tile of which head a workgroup takes. Workgroups go round robin over
// the eight XCDs, each with its own L2: `chunk` neighbouring tiles of a key
// head (of all its query heads) stay on one XCD, so the keys or rows that
// their windows share are read into one L2 instead of all eight. Later tiles
// go first: without a window they are the longest.
constexpr int kXcds = 8;
struct Deal {
    int tiles, heads, chunk;  // tiles of a pair (sequence, key head); query heads dealt with each tile
    int64_t pairs;
    __host__ __device__ int64_t chunks() const { return (int64_t)((tiles + chunk - 1) / chunk) * pairs; }
    __host__ __device__ int64_t blocks() const { return (chunks() + kXcds - 1) / kXcds * kXcds * chunk * heads; }
    // false: the workgroup has no tile. A launch's workgroups, and so its
    // pairs, are counted in 32 bits.
    __device__ bool take(uint32_t id, int &tile, int &head, uint32_t &pair) const {
        const uint32_t xcd = id % kXcds, j = id / kXcds, unit = chunk * heads, which = j / unit * kXcds + xcd;
        const uint32_t in = j % unit, each = (uint32_t)(tiles + chunk - 1) / chunk;
        pair = which / each;
        tile = tiles - 1 - (int)(which % each * chunk + in / heads);
        head = in % heads;
        return pair < pairs && tile >= 0;
    }
};
// At most 8 tiles to a chunk, and four chunks to an XCD while there are enough.
Deal deal(int64_t extent, int per_tile, int heads, int64_t pairs) {
    Deal d{(int)((extent + per_tile - 1) / per_tile), heads, 1, pairs};
    d.chunk = (int)std::max<int64_t>(1, std::min<int64_t>({8, d.tiles, d.tiles * pairs / (4 * kXcds)}));
    return d;
}

// The keys and the first row's position of sequence b. Stored lengths and
// starts are taken into the extents the launch was checked for.
struct Seq {
    int n, start;
    __device__ Seq(const WinArgs &a, int64_t b) {
        n = a.sk;
        if (a.lengths) n = (int)pick(a.lengths, a.lengths_wide, b * a.length_step, 0, a.sk);
        start = a.starts ? (int)pick(a.starts, a.starts_wide, b * a.start_step, -kMaxExtent, a.sk) : n - a.sq;
    }
    __device__ static int64_t pick(const void *p, int wide, int64_t at, int64_t lo, int64_t hi) {
        const int64_t v = wide ? static_cast<const int64_t *>(p)[at] : static_cast<const int32_t *>(p)[at];
        return v < lo ? lo : v > hi ? hi : v;
    }
};

template <typename T>
__device__ inline const T *head_of(const View &v, int64_t b, int64_t h) {
    return static_cast<const T *>(v.p) + b * v.b + h * v.h;
}

// Eight elements `at` .. of a row in memory, zero past the head's width or
// where the row is not `live` (row 0 is read in its place).
template <typename T>
__device__ inline V8<T> row_part(const T *row, int at, int width, bool live) {
    Pack<T, 8> p;
    p.load(row + (at < width ? at : 0));
    V8<T> z = {};
    return live && at < width ? p.q : z;
}

// Clears the columns of `rows` tile rows past the head's width, once for all
// tiles a buffer gets: the other factor is zero there, but 0 times an infinity
// in whatever else stood there would be NaN.
template <typename T, int D>
__device__ inline void clear_past(T *tile, int rows, int width, int tid, int threads) {
    if (width == D) return;
    for (int id = tid; id < rows * (D / 8); id += threads)
        if (id % (D / 8) * 8 >= width) *reinterpret_cast<V8<T> *>(tile + id / (D / 8) * kPitch<T, D> + id % (D / 8) * 8) = V8<T>{};
}

// A tile of N rows of D elements on its way from memory to LDS, staged by
// kThreads threads. Rows past `last` repeat others of the operand, hidden from
// every pair. A thread whose column lies past the width repeats the row's
// first one, in memory and in LDS (leaving its store out cost dk and dv of
// [1, 16 on 4, 8192, 128] bf16 20 us and spilled registers): the columns past
// the width keep the zeros of clear_past. Whole tiles take one address a
// thread and a uniform step between its parts (52 of the 380 vector
// instructions a tile went into addresses otherwise).
template <typename T, int D, int N>
struct Staged {
    static constexpr int C = D / 8, ALL = N * C, PARTS = (ALL + kThreads - 1) / kThreads;
    static constexpr bool EVEN = kThreads % C == 0;
    Pack<T, 8> part[PARTS];
    __device__ void load(const T *base, int64_t step, int row0, int last, int width, int tid) {
        const int own = tid % C * 8, at = own < width ? own : 0;
        if (EVEN && row0 + N - 1 <= last) {
            const T *p = base + row0 * step + (tid / C * step + at);
#pragma unroll
            for (int i = 0; i < PARTS; ++i) part[i].load(p + i * (kThreads / C) * step);
            return;
        }
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int id = tid + i * kThreads, r = min(row0 + id / C, last), e = id % C * 8;
            part[i].load(base + r * step + (e < width ? e : 0));
        }
    }
    __device__ bool special() const {
        Largest<T> m;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) m.add(part[i].q);
        return m.special();
    }
    __device__ void store(T *tile, int width, int tid) const {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int id = tid + i * kThreads, e = (EVEN ? tid : id) % C * 8;
            if (ALL % kThreads && id >= ALL) break;
            *reinterpret_cast<V8<T> *>(tile + id / C * kPitch<T, D> + (e < width ? e : 0)) = part[i].q;
        }
    }
};

// The key tiles that rows of positions first .. last see: those of the
// sinks, then those of the window.
template <int KEYS>
struct KeyWalk {
    int count, sink_tiles, window_from;
    __device__ KeyWalk(int first, int last, int n, int window, int sinks) {
        last = min(last, n - 1);
        count = sink_tiles = window_from = 0;
        if (last < 0 || first >= n) return;
        const int hi = last / KEYS, lo = max(0, first - window + 1) / KEYS;
        sink_tiles = min((sinks + KEYS - 1) / KEYS, hi + 1);
        window_from = max(sink_tiles, lo);
        count = sink_tiles + max(0, hi - window_from + 1);
    }
    __device__ int tile(int t) const { return t < sink_tiles ? t : window_from + t - sink_tiles; }
};

// What the rows from position `first` (at most 32; `live` of them, or more,
// are real) see of keys k0 .. k0 + count - 1.
enum Sight { kNone, kSome, kAll };
__device__ inline bool sees_all(int first, int last, int n, int window, int sinks, int k0, int k1) {
    return (k1 <= first) & (last < n) & ((k0 > last - window) | (k1 < sinks));
}
__device__ inline Sight sight(int first, int live, int n, int window, int sinks, int k0, int count) {
    const int end = first + min(live, 32) - 1, last = min(end, n - 1), k1 = k0 + count - 1;
    if ((live <= 0) | (first >= n) | (k0 > last) | ((k0 >= sinks) & (k1 <= first - window))) return kNone;
    return sees_all(first, end, n, window, sinks, k0, k1) ? kAll : kSome;
}
// The workgroup's answer to whether a wave staged an infinity or a NaN.
__device__ inline bool any_wave(const int *flags) {
    const int f = flags[0] | flags[1] | flags[2] | flags[3];
    return __builtin_amdgcn_readfirstlane(f) != 0;
}

// Which of the keys k0 + 8 (r / 4) + 4 h + r % 4, items r of a column of
// scores, a row sees whose last visible key is `top` (-1: none) and whose
// window starts behind key `low`. Selections only, no branches.
struct SeenKeys {
    int top, low, sinks;
    __device__ SeenKeys(int top_, int low_, int sinks_, int k0, int h)
        : top(top_ - k0 - 4 * h), low(low_ - k0 - 4 * h), sinks(sinks_ - k0 - 4 * h) {}
    __device__ bool operator()(int r) const { return at(8 * (r >> 2) + (r & 3)); }
    __device__ bool at(int k) const { return (k <= top) & ((k > low) | (k < sinks)); }
};
// Which of the rows r0 + 8 (r / 4) + 4 h + r % 4, of positions from start,
// see a key: those from the key's own position up to the window's end, or up
// to the last row inside the sequence for a sink.
struct SeenRows {
    int from, end;
    __device__ SeenRows(int key, int start, int r0, int h, int rows, int n, int window, int sinks) {
        const int base = r0 + 4 * h, last = min(rows, n - start);
        from = key - start - base;
        end = (key < sinks ? last : min(last, key - start + window)) - base;
    }
    __device__ bool operator()(int r) const { return at(8 * (r >> 2) + (r & 3)); }
    __device__ bool at(int k) const { return (k >= from) & (k < end); }
};

__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float other_half(float x) { return __shfl_xor(x, 32, 64); }

// Four consecutive elements of an accumulated column to memory.
template <typename T>
__device__ inline void store4(T *p, const f32x16 &c, int from, float f) {
    Pack<T, 4> out;
#pragma unroll
    for (int t = 0; t < 4; ++t) out.set(t, c[from + t] * f);
    out.store(p);
}
// Column block d0 .. of an accumulated result row.
template <typename T>
__device__ inline void store_column(T *row, const f32x16 &c, int d0, int width, int h, float f) {
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
        const int d = d0 + 2 * r + 4 * h;
        if (d < width) store4(row + d, c, r, f);
    }
}

// ---------------------------------------------------------------- forward
// f16 weights are held 2^10 times larger: the smallest keep their bits.
template <typename T>
constexpr float kShift = std::is_same<T, _Float16>::value ? 10.f : 0.f;
// The reference of a row's exponentials follows its running maximum only when
// that passes it by more than this (in powers of two; 2^15 is the largest f16
// weight then): nearly every tile leaves the results unscaled ([2, 16 on 4, 8192,
// 128] bf16, window 1024: 198 us with 8, 206 with 5).
template <typename T>
constexpr float kSlack = std::is_same<T, _Float16>::value ? 5.f : 8.f;

// LDS tiles of keys: two of each operand (one barrier a tile) where two
// workgroups then still fit a compute unit's 160 KB.
template <typename T>
constexpr int kBuffers = sizeof(T) == 2 ? 2 : 1;

// What the waves of a workgroup share of a walk over key tiles: staging ahead,
// and whether a tile holds infinities or NaN that some row does not see
// (LOOK: 0 looks over k, 1 over v).
template <typename T, int D, int LOOK>
struct KeyTiles {
    static constexpr int B = kBuffers<T>, SIZE = kKeys * kPitch<T, D>;
    struct Shared {
        T k[B][SIZE], v[B][SIZE];
        int flags[2][kWaves];
    };
    const WinArgs &a;
    Shared &sh;
    const T *K, *V;
    const KeyWalk<kKeys> &walk;
    int n, first, last, tid, wave;  // keys; positions of the workgroup's rows
    Staged<T, D, kKeys> ks, vs;
    __device__ bool whole(int k0) const { return sees_all(first, last, n, a.window, a.sinks, k0, k0 + kKeys - 1); }
    __device__ void load(int t) {
        if (t >= walk.count) return;
        ks.load(K, a.k.s, walk.tile(t) * kKeys, n - 1, a.width, tid);
        vs.load(V, a.v.s, walk.tile(t) * kKeys, n - 1, a.width, tid);
    }
    __device__ void store(int t) {
        if (t >= walk.count) return;
        ks.store(sh.k[t % B], a.width, tid);
        vs.store(sh.v[t % B], a.width, tid);
        if (!whole(walk.tile(t) * kKeys)) sh.flags[t & 1][wave] = __any(LOOK ? vs.special() : ks.special());
    }
    __device__ void begin() {
        load(0);
        clear_past<T, D>(sh.k[0], B * kKeys, a.width, tid, kThreads);
        clear_past<T, D>(sh.v[0], B * kKeys, a.width, tid, kThreads);
        if (B == 2) {
            store(0);
            load(1);
        }
    }
    // tile t is in LDS for every wave after this
    __device__ void next(int t) {
        __syncthreads();
        if (B == 2) {
            store(t + 1);
            load(t + 2);
        } else {
            store(t);
            __syncthreads();
            load(t + 1);
        }
    }
    __device__ bool special(int t) const { return !whole(walk.tile(t) * kKeys) && any_wave(sh.flags[t & 1]); }
};

// A workgroup takes 128 rows of one head, each wave 32 of them, which share
// the staged keys; the rows' q stays in registers. Bound by the softmax
// between the two products: each 32-cycle product comes with eight vector
// instructions that take as long, after it in the same wave. [2, 16 on 4,
// 8192, 128] bf16, window 1024, 197-201 us (matrix cores 29 %, LDS 38 % busy at
// 1.6 resident waves a SIMD; 650 TFLOP/s over the visible pairs, 540 without a
// window, where the last rows' workgroups end alone); [8, 16, 512, 64] f32,
// window 128, 51 us.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_forward_kernel(WinArgs a, Deal deal) {
    __shared__ __attribute__((aligned(16))) typename KeyTiles<T, D, 1>::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tile, member;
    uint32_t pair;
    if (!deal.take(blockIdx.x, tile, member, pair)) return;
    const int64_t b = pair / (uint32_t)a.kv, head = pair % (uint32_t)a.kv * a.group + member;
    const Seq seq(a, b);
    const int row0 = tile * (32 * kWaves), mine = row0 + 32 * wave, row = mine + i;
    const int live = a.sq - mine;  // rows past the last hold zeros and are not stored
    const T *Q = head_of<T>(a.q, b, head);
    V8<T> qf[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        qf[s] = row_part(Q + (row < a.sq ? row : 0) * a.q.s, 16 * s + 8 * h, a.width, row < a.sq);
        if (a.flip) qf[s] = -qf[s];
    }
    f32x16 acc[D / 32] = {};
    float m = -INFINITY, l = 0.f;
    const int first = seq.start + mine, p = first + i, top = row < a.sq && p < seq.n ? p : -1, low = p - a.window;
    const int group_first = seq.start + row0, group_last = seq.start + min(row0 + 32 * kWaves, a.sq) - 1;
    const KeyWalk<kKeys> walk(group_first, group_last, seq.n, a.window, a.sinks);
    KeyTiles<T, D, 1> tiles{a, sh, head_of<T>(a.k, b, head / a.group), head_of<T>(a.v, b, head / a.group), walk, seq.n,
                            group_first, group_last, tid, wave};
    tiles.begin();
    for (int t = 0; t < walk.count; ++t) {
        tiles.next(t);
        const int k0 = walk.tile(t) * kKeys;
        const T *Ks = sh.k[t % kBuffers<T>];
        T *Vs = sh.v[t % kBuffers<T>];
        const Sight see = sight(first, live, seq.n, a.window, a.sinks, k0, kKeys);
        // binary32 products cost sixteen times the 16-bit ones: there the
        // halves of a tile that a wave sees nothing of are left out ([8, 16,
        // 512, 64] with a window of 128: 54.7 -> 51.4 us); the branches cost
        // the 16-bit kernel more than they save (199 -> 216 us)
        constexpr bool HALVES = sizeof(T) == 4;
        bool half[2] = {true, true};
        if constexpr (HALVES) {
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
                half[kb] = sight(first, live, seq.n, a.window, a.sinks, k0 + 32 * kb, 32) != kNone;
        }
        f32x16 s[2] = {};
        if (see != kNone) {
            if constexpr (HALVES) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
                    if (half[kb]) {
#pragma unroll
                        for (int u = 0; u < D / 16; ++u) s[kb] = mma(along<T, D>(Ks, 32 * kb + i, 16 * u + 8 * h), qf[u], s[kb]);
                    }
            } else {
#pragma unroll
                for (int u = 0; u < D / 16; ++u)
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) s[kb] = mma(along<T, D>(Ks, 32 * kb + i, 16 * u + 8 * h), qf[u], s[kb]);
                interleave<D / 8, 1, 4>();
            }
            if (see == kSome) {
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const SeenKeys keys(top, low, a.sinks, k0 + 32 * kb, h);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[kb][r] = keys(r) ? s[kb][r] : -INFINITY;
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int r = 0; r < 32; ++r) mx = fmaxf(mx, s[r >> 4][r & 15]);
            mx = fmaxf(mx, other_half(mx)) * a.c;
            if (__any(mx > m + kSlack<T>)) {
                // by the row's own scores alone: no bit of it depends on its neighbours
                const float m_new = mx > m + kSlack<T> ? mx : m, alpha = exp2_(m - (m_new == -INFINITY ? 0.f : m_new));
                m = m_new;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < D / 32; ++d) acc[d] *= alpha;
            }
            // while every score is -inf, 0 in place of the maximum keeps the
            // weights 0 (-inf - -inf would be NaN, and stay)
            const float off = kShift<T> - (m == -INFINITY ? 0.f : m);
            float sum = 0.f;
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const float e = exp2_(fmaf(s[r >> 4][r & 15], a.c, off));
                s[r >> 4][r & 15] = e;
                sum += e;
            }
            l += sum;
        }
        if (tiles.special(t)) {
            if (see != kNone)
                add_special<T, D, kKeys>(acc, Vs, h, [&](int k) { return SeenKeys(top, low, a.sinks, k0, 0).at(k); });
            __syncthreads();
            clean<T, D, kKeys, kThreads>(Vs, tid);
            __syncthreads();
        }
        if (see == kNone) continue;
#pragma unroll
        for (int kc = 0; kc < 4; ++kc) {
            if (HALVES && !half[kc >> 1]) continue;
            const V8<T> pf = rounded<T>(s[kc >> 1], 8 * (kc & 1));
#pragma unroll
            for (int d = 0; d < D / 32; ++d) acc[d] = mma(across<T, D>(Vs, 16 * kc, 32 * d, lane), pf, acc[d]);
        }
        if (!HALVES) interleave<4 * D / 32, 2, 3>();
    }
    if (__any(has_special<D>(acc))) {
        SeenSpecials<T, D> specials(acc, row < a.sq && l == l);  // a row of NaN weights is NaN
        for (int t = 0; t < walk.count && !specials.done(); ++t) {
            const int k0 = walk.tile(t) * kKeys;
            specials.note(tiles.V, a.v.s, a.width, k0, min(k0 + kKeys, seq.n), lane,
                          [&](int k) { return SeenKeys(top, low, a.sinks, 0, 0).at(k); });
        }
        specials.put(acc);
    }
    l += other_half(l);
    if (row >= a.sq) return;
    const bool empty = top < 0;
    const float inv = row_factor(empty, l);
    T *O = const_cast<T *>(head_of<T>(a.o, b, head)) + row * a.o.s;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) store_column(O, acc[d], 32 * d, a.width, h, inv);
    if (a.lse && h == 0)
        a.lse[(b * a.heads + head) * a.sq + row] = empty ? -INFINITY : canon_bits((m - kShift<T> + log2f(l)) * kLn2);
}

// ---------------------------------------------------------------- few rows
// A few rows over many keys (single tokens over a cache): the rows of every
// query head that shares a key head are taken together, 32 to a task, and the
// key blocks of a task are dealt to `splits` waves, each on its own: it keeps
// its next 32 keys in flight in registers (a row of k per lane pair as the
// products want it, v on its way to the wave's own LDS tile) and no wave
// waits for another. With one split the wave stores its rows; else it leaves
// their sums, maxima and unscaled results in scratch and a second launch joins
// them in split order. Bound by the reads of k and v: one token of each of 64
// sequences of up to 16384 keys, window 4096, 32 heads of 128 on 8, bf16: 219
// us (4.9 TB/s); of one sequence 9.9 us, both launches' latency.
struct SplitArgs {
    float *part;  // per task, split and row: [width] results, then maxima and sums
    float *stat;
    int splits, rows, tiles, pack;  // rows of all heads of a group, row tiles, rows a part holds
    int64_t tasks;
};

// binary32 rows wider than 64 hold more than half a SIMD's registers: one wave a
// SIMD (two spilled them: one token of 64 sequences, window 4096, 32 heads of 128
// on 8, 954 and, with the look at the sums below, 1189 us; 515 now).
template <typename T, int D>
__global__ __launch_bounds__(kThreads, (sizeof(T) == 4 && D > 64 ? 1 : 2)) void window_split_kernel(WinArgs a, SplitArgs p) {
    constexpr int N = 32;
    __shared__ __attribute__((aligned(16))) T tiles[kWaves][N * kPitch<T, D>];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // a launch's waves, and so its tasks, are counted in 32 bits
    const uint32_t id = blockIdx.x * kWaves + wave, task = id / (uint32_t)p.splits;
    if (task >= p.tasks) return;
    const int split = (int)(id % (uint32_t)p.splits), rt = (int)(task % (uint32_t)p.tiles);
    const uint32_t pair = task / (uint32_t)p.tiles;
    const int64_t kvh = pair % (uint32_t)a.kv, b = pair / (uint32_t)a.kv;
    const Seq seq(a, b);
    const int r = rt * N + i, live = r < p.rows, rs = live ? r : 0;
    const int64_t head = kvh * a.group + rs / a.sq;
    const int row = rs % a.sq, pos = seq.start + row;
    const T *Q = head_of<T>(a.q, b, head) + row * a.q.s, *K = head_of<T>(a.k, b, kvh), *V = head_of<T>(a.v, b, kvh);
    V8<T> qf[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        qf[s] = row_part(Q, 16 * s + 8 * h, a.width, live);
        if (a.flip) qf[s] = -qf[s];
    }
    // the tile's rows: one head's run of them, or all where it spans heads
    const int last_row = min(rt * N + N, p.rows) - 1;
    const bool one = rt * N / a.sq == last_row / a.sq;
    const int first = seq.start + (one ? rt * N % a.sq : 0), last = seq.start + (one ? last_row % a.sq : a.sq - 1);
    const int top = live && pos < seq.n ? pos : -1, low = pos - a.window;
    const KeyWalk<N> walk(first, last, seq.n, a.window, a.sinks);
    f32x16 acc[D / 32] = {};
    float m = -INFINITY, l = 0.f;
    T *tile = tiles[wave];
    constexpr int PARTS = D / 16;  // 16-byte (f32: 32-byte) parts of a lane
    V8<T> kf[PARTS], vf[PARTS];
    auto load = [&](int t) {
        const int k0 = walk.tile(t) * N;
        const T *kr = K + min(k0 + i, seq.n - 1) * a.k.s;
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            const int at = 16 * s + 8 * h;
            Pack<T, 8> q;
            q.load_streamed(kr + (at < a.width ? at : 0));
            kf[s] = q.q;
        }
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            const int part = lane + 64 * s, at = part % (D / 8) * 8;
            Pack<T, 8> q;
            q.load_streamed(V + min(k0 + part / (D / 8), seq.n - 1) * a.v.s + (at < a.width ? at : 0));
            vf[s] = q.q;
        }
    };
    if (split < walk.count) load(split);
    for (int t = split; t < walk.count; t += p.splits) {
        const int k0 = walk.tile(t) * N;
        if (a.width < D) {  // zeros past the width, as in q
#pragma unroll
            for (int u = 0; u < PARTS; ++u) kf[u] = 16 * u + 8 * h < a.width ? kf[u] : V8<T>{};
        }
        f32x16 s = {};
#pragma unroll
        for (int u = 0; u < D / 16; ++u) s = mma(kf[u], qf[u], s);
#pragma unroll
        for (int u = 0; u < PARTS; ++u) {
            const int part = lane + 64 * u;
            *reinterpret_cast<V8<T> *>(tile + part / (D / 8) * kPitch<T, D> + part % (D / 8) * 8) = vf[u];
        }
        const bool all = sees_all(first, last, seq.n, a.window, a.sinks, k0, k0 + N - 1);
        bool special = false;
        if (!all) {
            Largest<T> most;
#pragma unroll
            for (int u = 0; u < PARTS; ++u) most.add(vf[u]);
            special = __any(most.special());
        }
        if (t + p.splits < walk.count) load(t + p.splits);
        if (!all) {
            const SeenKeys keys(top, low, a.sinks, k0, h);
#pragma unroll
            for (int c = 0; c < 16; ++c) s[c] = keys(c) ? s[c] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int c = 0; c < 16; ++c) mx = fmaxf(mx, s[c]);
        mx = fmaxf(mx, other_half(mx)) * a.c;
        const float m_new = fmaxf(m, mx), ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = exp2_(m - ref), off = kShift<T> - ref;
        m = m_new;
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 16; ++c) {
            s[c] = exp2_(fmaf(s[c], a.c, off));
            sum += s[c];
        }
        l = l * alpha + sum;
#pragma unroll
        for (int d = 0; d < D / 32; ++d) acc[d] *= alpha;
        if (special) {
            // the wave alone reads and writes its tile
            add_special<T, D, N>(acc, tile, h, [&](int k) { return SeenKeys(top, low, a.sinks, k0, 0).at(k); });
            clean<T, D, N, 64>(tile, lane);
        }
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            const V8<T> pf = rounded<T>(s, 8 * kc);
#pragma unroll
            for (int d = 0; d < D / 32; ++d) acc[d] = mma(across<T, D>(tile, 16 * kc, 32 * d, lane), pf, acc[d]);
        }
    }
    if (__any(has_special<D>(acc))) {
        SeenSpecials<T, D> specials(acc, live && l == l);  // a row of NaN weights is NaN
        for (int t = split; t < walk.count && !specials.done(); t += p.splits) {
            const int k0 = walk.tile(t) * N;
            specials.note(V, a.v.s, a.width, k0, min(k0 + N, seq.n), lane,
                          [&](int k) { return SeenKeys(top, low, a.sinks, 0, 0).at(k); });
        }
        specials.put(acc);
    }
    l += other_half(l);
    if (!live) return;
    if (p.splits > 1) {
        const int64_t at = (int64_t)id * p.pack + i;
        float *out = p.part + at * a.width;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
                const int e = 32 * d + 2 * c + 4 * h;
                if (e < a.width) *reinterpret_cast<f32x4 *>(out + e) = f32x4{acc[d][c], acc[d][c + 1], acc[d][c + 2], acc[d][c + 3]};
            }
        if (h == 0) {
            p.stat[2 * at] = m;
            p.stat[2 * at + 1] = l;
        }
        return;
    }
    const bool empty = top < 0;
    const float inv = row_factor(empty, l);
    T *O = const_cast<T *>(head_of<T>(a.o, b, head)) + row * a.o.s;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) store_column(O, acc[d], 32 * d, a.width, h, inv);
    if (a.lse && h == 0)
        a.lse[(b * a.heads + head) * a.sq + row] = empty ? -INFINITY : canon_bits((m - kShift<T> + log2f(l)) * kLn2);
}

// One row a workgroup: the splits' results under their common maximum, every
// eighth (or sixteenth) split to a group of threads, the groups joined in
// order. Latency bound: the statistics and a thread's first parts are read at
// once. (Statistics, sums and parts one after another took 4.0 us for a single
// token over 1024 keys, one wave walking its 35 splits 24 us.)
constexpr int kMaxSplits = 2048;

// A part's elements under its weight; infinities stay where the weight is 0.
__device__ inline f32x4 weighed(float w, f32x4 x) {
    f32x4 y;
#pragma unroll
    for (int t = 0; t < 4; ++t) y[t] = not_finite(x[t]) ? x[t] : w * x[t];
    return y;
}

template <typename T, int D>
__global__ __launch_bounds__(kThreads) void window_join_kernel(WinArgs a, SplitArgs p) {
    constexpr int LANES = D / 4, GROUPS = kThreads / LANES, AHEAD = 4;
    __shared__ float weight[kMaxSplits], waves[2][kWaves];
    __shared__ f32x4 join[GROUPS][LANES];
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const uint32_t id = blockIdx.x, sq = a.sq, bh = id / sq;
    const int64_t row = id % sq, b = bh / (uint32_t)a.heads;
    const uint32_t head = bh % (uint32_t)a.heads, kvh = head / (uint32_t)a.group;
    const int tid = threadIdx.x, r = (int)((head - kvh * a.group) * sq + row);
    const int64_t task = (b * a.kv + kvh) * p.tiles + r / 32, at = task * p.splits * p.pack + r % 32;
    const int lane = tid % LANES, group = tid / LANES;
    const bool own = group < GROUPS && 4 * lane < a.width;
    const f32x2 *stat = reinterpret_cast<const f32x2 *>(p.stat) + at;
    const float *part = p.part + at * a.width + 4 * lane;
    const int64_t step = (int64_t)p.pack * a.width;
    f32x2 mine = {-INFINITY, 0.f};  // maximum and sum of split tid
    if (tid < p.splits) mine = stat[(int64_t)tid * p.pack];
    f32x4 ahead[AHEAD] = {};
    if (own) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (group + k * GROUPS < p.splits) ahead[k] = *reinterpret_cast<const f32x4 *>(part + (group + k * GROUPS) * step);
    }
    const Seq seq(a, b);
    float m = mine[0];
    for (int s = tid + kThreads; s < p.splits; s += kThreads) m = fmaxf(m, stat[(int64_t)s * p.pack][0]);
    m = wave_vmax(m);
    if ((tid & 63) == 0) waves[0][tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(waves[0][0], waves[0][1]), fmaxf(waves[0][2], waves[0][3]));
    const float ref = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    for (int s = tid; s < p.splits; s += kThreads) {
        const f32x2 q = s == tid ? mine : stat[(int64_t)s * p.pack];
        const float f = exp2_(q[0] - ref);
        weight[s] = f;
        l = fmaf(f, q[1], l);
    }
    l = wave_tree_sum(l);
    if ((tid & 63) == 0) waves[1][tid >> 6] = l;
    __syncthreads();
    l = (waves[1][0] + waves[1][1]) + (waves[1][2] + waves[1][3]);
    f32x4 x = {};
    if (own) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
            if (group + k * GROUPS < p.splits) x += weighed(weight[group + k * GROUPS], ahead[k]);
#pragma unroll 4
        for (int s = group + AHEAD * GROUPS; s < p.splits; s += GROUPS)
            x += weighed(weight[s], *reinterpret_cast<const f32x4 *>(part + s * step));
        join[group][lane] = x;
    }
    __syncthreads();
    const int pos = seq.start + (int)row;
    const bool empty = pos < 0 || pos >= seq.n;
    if (own && group == 0) {
#pragma unroll
        for (int k = 1; k < GROUPS; ++k) x += join[k][lane];
        const float inv = row_factor(empty, l);
        Pack<T, 4> out;
#pragma unroll
        for (int t = 0; t < 4; ++t) out.set(t, x[t] * inv);
        out.store(const_cast<T *>(head_of<T>(a.o, b, head)) + row * a.o.s + 4 * lane);
    }
    if (a.lse && tid == 0)
        a.lse[id] = empty ? -INFINITY : canon_bits((m - kShift<T> + log2f(l)) * kLn2);
}

// ---------------------------------------------------------------- backward
// f16 holds dS times a power of two that brings its largest possible value,
// 2 max|g| max|v| width, just under f16's: gradients of any size keep their
// bits. A first launch takes both maxima (over kRanges workgroups each); the
// other types need no scale.
constexpr int kRanges = 256;

// Partial maxima of |g| over the rows inside their sequence (workgroups
// 0 .. kRanges - 1) and of |v| over its keys (the others); one row of one head
// to 16 lanes.
template <typename T>
__global__ __launch_bounds__(256) void window_range_kernel(WinArgs a, int batch) {
    __shared__ float waves[4];
    const bool keys = blockIdx.x >= kRanges;
    const View &x = keys ? a.v : a.g;
    const int heads = keys ? a.kv : a.heads, rows = keys ? a.sk : a.sq, at = threadIdx.x % 16 * 8;
    Largest<T> most;
    for (int b = 0; b < batch; ++b) {
        const Seq seq(a, b);
        const int from = keys ? 0 : max(0, -seq.start), to = keys ? seq.n : min(rows, seq.n - seq.start);
        if (to <= from) continue;
        const uint32_t count = to - from, all = min((int64_t)count * heads, (int64_t)UINT32_MAX);
        for (uint64_t id = blockIdx.x % kRanges * 16 + threadIdx.x / 16; id < (uint64_t)count * heads; id += kRanges * 16) {
            const int64_t h = all == UINT32_MAX ? id / count : (uint32_t)id / count;
            if (at < a.width) {
                Pack<T, 8> q;
                q.load(head_of<T>(x, b, h) + (int64_t)(from + (id - h * count)) * x.s + at);
#pragma unroll
                for (int t = 0; t < 8; ++t) q.q[t] = not_finite(q.q[t]) ? (T)0.f : q.q[t];
                most.add(q.q);
            }
        }
    }
    const V8<T> top = __builtin_bit_cast(V8<T>, most.m);
    float m = 0.f;
#pragma unroll
    for (int t = 0; t < 8; ++t) m = fmaxf(m, widen<T>(top[t]));
    m = wave_vmax(m);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.range[blockIdx.x] = fmaxf(fmaxf(waves[0], waves[1]), fmaxf(waves[2], waves[3]));
}

// The power of two; every thread of the workgroup calls it once.
template <typename T>
__device__ inline float gradient_scale(const WinArgs &a) {
    if constexpr (!std::is_same<T, _Float16>::value) return 1.f;
    __shared__ float waves[2][kWaves];
    static_assert(kRanges == kThreads, "one partial maximum a thread");
    const int t = threadIdx.x & (kThreads - 1);  // groups of threads do the same
    const float g = wave_vmax(a.range[t]), v = wave_vmax(a.range[kRanges + t]);
    if ((t & 63) == 0) {
        waves[0][t >> 6] = g;
        waves[1][t >> 6] = v;
    }
    __syncthreads();
    float mg = 0.f, mv = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        mg = fmaxf(mg, waves[0][w]);
        mv = fmaxf(mv, waves[1][w]);
    }
    const float most = 2.f * mg * mv * (float)a.width;
    // most < 2^(ilogb + 1), taken to less than 2^15
    return most > 0.f ? ldexpf(1.f, min(14 - ilogbf(most), 100)) : 1.f;
}

// dq, and D for the second kernel: rows as in the forward kernel, q and g in
// registers, three products a block. [1, 16 on 4, 8192, 128] bf16, window
// 1024: 140 us (matrix cores 28 %, LDS 34 % busy).
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 2) void window_dq_kernel(WinArgs a, Deal deal) {
    __shared__ __attribute__((aligned(16))) typename KeyTiles<T, D, 0>::Shared sh;
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tile, member;
    uint32_t pair;
    if (!deal.take(blockIdx.x, tile, member, pair)) return;
    const int64_t b = pair / (uint32_t)a.kv, head = pair % (uint32_t)a.kv * a.group + member;
    const Seq seq(a, b);
    const int row0 = tile * (32 * kWaves), mine = row0 + 32 * wave, row = mine + i;
    const int live = min(32, a.sq - mine), safe = row < a.sq ? row : 0;
    const T *Q = head_of<T>(a.q, b, head);
    const T *G = head_of<T>(a.g, b, head), *O = head_of<T>(a.o, b, head);
    V8<T> qf[D / 16], gf[D / 16];
    float delta = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
        const int at = 16 * s + 8 * h;
        qf[s] = row_part(Q + safe * a.q.s, at, a.width, row < a.sq);
        gf[s] = row_part(G + safe * a.g.s, at, a.width, row < a.sq);
        const V8<T> of = row_part(O + safe * a.o.s, at, a.width, row < a.sq);
#pragma unroll
        for (int t = 0; t < 8; ++t) delta = fmaf(widen<T>(gf[s][t]), widen<T>(of[t]), delta);
    }
    delta += other_half(delta);
    const int64_t stat = (b * a.heads + head) * a.sq + safe;
    if (row < a.sq && h == 0) a.delta[stat] = delta;
    const float lse = a.lse_in[stat] * kLog2e, up = gradient_scale<T>(a);
    f32x16 acc[D / 32] = {};
    Marks<D> marks;
    const int first = seq.start + mine, p = first + i, top = row < a.sq && p < seq.n ? p : -1, low = p - a.window;
    const int group_first = seq.start + row0, group_last = seq.start + min(row0 + 32 * kWaves, a.sq) - 1;
    const KeyWalk<kKeys> walk(group_first, group_last, seq.n, a.window, a.sinks);
    KeyTiles<T, D, 0> tiles{a, sh, head_of<T>(a.k, b, head / a.group), head_of<T>(a.v, b, head / a.group), walk, seq.n,
                            group_first, group_last, tid, wave};
    tiles.begin();
    for (int t = 0; t < walk.count; ++t) {
        tiles.next(t);
        const int k0 = walk.tile(t) * kKeys;
        T *Ks = sh.k[t % kBuffers<T>];
        const T *Vs = sh.v[t % kBuffers<T>];
        const bool special = tiles.special(t);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int kk = k0 + 32 * kb;
            const Sight see = sight(first, live, seq.n, a.window, a.sinks, kk, 32);
            f32x16 s = {}, dp = {};
            if (see != kNone) {
#pragma unroll
                for (int u = 0; u < D / 16; ++u) {
                    s = mma(along<T, D>(Ks, 32 * kb + i, 16 * u + 8 * h), qf[u], s);
                    dp = mma(along<T, D>(Vs, 32 * kb + i, 16 * u + 8 * h), gf[u], dp);
                }
                if (sizeof(T) == 2) interleave<D / 8, 1, 4>();
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = exp2_(fmaf(s[r], a.signed_c, -lse)) * ((dp[r] - delta) * up);
                if (see == kSome) {
                    const SeenKeys keys(top, low, a.sinks, kk, h);
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] = keys(r) ? s[r] : 0.f;
                }
            }
            if (special) {
                T *half = Ks + 32 * kb * kPitch<T, D>;
                marks.template note<true, T, 32>(half, h, [&](int k) { return SeenKeys(top, low, a.sinks, kk, 0).at(k); });
                __syncthreads();
                clean<T, D, 32, kThreads>(half, tid);
                __syncthreads();
            }
            if (see == kNone) continue;
#pragma unroll
            for (int kc = 0; kc < 2; ++kc) {
                const V8<T> df = rounded<T>(s, 8 * kc);
#pragma unroll
                for (int d = 0; d < D / 32; ++d) acc[d] = mma(across<T, D>(Ks, 32 * kb + 16 * kc, 32 * d, lane), df, acc[d]);
            }
            if (sizeof(T) == 2) interleave<2 * D / 32, 2, 3>();
        }
    }
    marks.apply(acc);
    if (row >= a.sq) return;
    T *DQ = const_cast<T *>(head_of<T>(a.dq, b, head)) + row * a.dq.s;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) store_column(DQ, acc[d], 32 * d, a.width, h, a.scale / up);
}

// dk and dv. A wave holds 32 keys of one key head and takes tiles of 32 query
// rows, staged in LDS with their lse and D.
template <typename T, int D>
struct KeyGradients {
    f32x16 dk[D / 32] = {}, dv[D / 32] = {};
    Marks<D> mk, mv;
    // columns of keys past the sequence are zero
    static __device__ V8<T> part(const T *base, int64_t step, int key, int n, int at, int width) {
        if (n <= 0) return V8<T>{};
        return row_part(base + (key < n ? key : 0) * step, at, width, key < n);
    }
    // Weights and dS of a tile, one key a column. Ls holds
    // shift - lse log2(e), Ds the rows' D; half scales dS.
    template <int READS, class Keys, class Values>  // LDS reads a product
    __device__ void scores(f32x16 &s, f32x16 &dp, Keys keys, Values values, const T *Qs, const T *Gs, const float *Ls, const float *Ds, float c,
                           float half, bool all, const SeenRows &rows, int lane) const {
        const int i = lane & 31, h = lane >> 5;
        s = dp = f32x16{};
#pragma unroll
        for (int u = 0; u < D / 16; ++u) {
            s = mma(along<T, D>(Qs, i, 16 * u + 8 * h), keys(u), s);
            dp = mma(along<T, D>(Gs, i, 16 * u + 8 * h), values(u), dp);
        }
        if (sizeof(T) == 2) interleave<D / 8, READS, 2>();
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            const f32x4 lr = *reinterpret_cast<const f32x4 *>(Ls + 8 * r4 + 4 * h);
            const f32x4 dr = *reinterpret_cast<const f32x4 *>(Ds + 8 * r4 + 4 * h);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 4 * r4 + j;
                const float p = exp2_(fmaf(s[r], c, lr[j]));
                s[r] = p;
                dp[r] = p * ((dp[r] - dr[j]) * half);
            }
        }
        if (!all) {
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[r] = rows(r) ? s[r] : 0.f;
                dp[r] = rows(r) ? dp[r] : 0.f;
            }
        }
    }
    __device__ void add(const f32x16 &s, const f32x16 &dp, const T *Qs, const T *Gs, int lane) {
#pragma unroll
        for (int kc = 0; kc < 2; ++kc) {
            const V8<T> pf = rounded<T>(s, 8 * kc), df = rounded<T>(dp, 8 * kc);
#pragma unroll
            for (int d = 0; d < D / 32; ++d) {
                dv[d] = mma(across<T, D>(Gs, 16 * kc, 32 * d, lane), pf, dv[d]);
                dk[d] = mma(across<T, D>(Qs, 16 * kc, 32 * d, lane), df, dk[d]);
            }
        }
        if (sizeof(T) == 2) interleave<4 * D / 32, 2, 3>();
    }
    __device__ void special(const T *Qs, const T *Gs, const SeenRows &rows, int h) {
        mv.template note<false, T, kRows>(Gs, h, [&](int r) { return rows.at(r); });
        mk.template note<true, T, kRows>(Qs, h, [&](int r) { return rows.at(r); });
    }
    __device__ void finish() {
        mv.apply(dv);
        mk.apply(dk);
    }
};

// Rows far behind the window see the sinks alone. A workgroup of keys would
// walk all of them (one workgroup of 128 keys walking 8192 rows of four heads
// took 3.8 ms beside 0.2 ms for the others), so they are dealt to `splits`
// workgroups of their own for each block of 32 sink keys. Such a block's sums
// are then unscaled parts in scratch: part 0 from the near rows, the others
// from the far workgroups, joined in order by a last launch.
struct FarArgs {
    float *part;  // [block][1 + splits][dk, dv][32 keys][width]; null: none are dealt out
    int splits, blocks;
    __device__ float *at(int64_t pair, int block, int part_index, int width) const {
        return part + ((pair * blocks + block) * (1 + splits) + part_index) * 64 * width;
    }
};

// First position whose rows are far for the workgroup of keys from tile0.
__device__ inline int far_from(int tile0, int window) { return tile0 + 32 * kWaves - 1 + window; }

template <typename T, int D>
__device__ inline void store_part(float *part, const KeyGradients<T, D> &w, int i, int h, int width, bool keep) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const int e = 32 * d + 2 * r + 4 * h;
            if (e >= width) continue;
            const f32x16 &k = w.dk[d], &v = w.dv[d];
            f32x4 x = {k[r], k[r + 1], k[r + 2], k[r + 3]}, y = {v[r], v[r + 1], v[r + 2], v[r + 3]};
            *reinterpret_cast<f32x4 *>(part + i * width + e) = keep ? x : f32x4{};
            *reinterpret_cast<f32x4 *>(part + (32 + i) * width + e) = keep ? y : f32x4{};
        }
}

// The near rows: a workgroup takes 128 keys, 32 to a wave, in `GROUPS` groups
// of four waves that take the row tiles in turn and add their sums up at the
// end. k and v stay in LDS. Row tiles are double buffered, one barrier a tile.
// [1, 16 on 4, 8192, 128] bf16, window 1024: 212 us, bound by LDS (48 % busy)
// with one workgroup a CU. k and v in registers at one wave a SIMD took 240-245;
// two groups with k alone there spill (325); four waves for dv and four for
// dk, which form the scores twice, 262-278.
template <typename T, int D>
constexpr int kGroups = sizeof(T) == 4 && D > 64 ? 1 : 2;

template <typename T, int D>
__global__ __launch_bounds__((kThreads * kGroups<T, D>), 1) void window_dkv_kernel(WinArgs a, FarArgs f, Deal deal) {
    constexpr int GROUPS = kGroups<T, D>, TILE = kRows * kPitch<T, D>, KEYS = 32 * kWaves;
    struct Buffers {
        T q[2][GROUPS][TILE], g[2][GROUPS][TILE], v[KEYS * kPitch<T, D>], k[GROUPS > 1 ? KEYS * kPitch<T, D> : 1];
    };
    union Shared {
        Buffers in;
        float sums[GROUPS > 1 ? kWaves * D / 2 * 64 : 1];
    };
    __shared__ __attribute__((aligned(16))) Shared sh;
    __shared__ __attribute__((aligned(16))) float Ls[2][GROUPS][kRows], Ds[2][GROUPS][kRows];
    __shared__ int flags[2][kWaves * GROUPS];
    const int tid = threadIdx.x & (kThreads - 1), lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), group = __builtin_amdgcn_readfirstlane(threadIdx.x / kThreads);
    int tile, member;
    uint32_t pair;
    if (!deal.take(blockIdx.x, tile, member, pair)) return;
    const int64_t b = pair / (uint32_t)a.kv, kvh = pair % (uint32_t)a.kv;
    const Seq seq(a, b);
    const int tile0 = tile * KEYS, mine = tile0 + 32 * wave, key = mine + i;
    KeyGradients<T, D> w;
    for (int id = threadIdx.x; id < KEYS * (D / 8); id += kThreads * GROUPS) {
        const int r = id / (D / 8), at = id % (D / 8) * 8, to = r * kPitch<T, D> + at;
        *reinterpret_cast<V8<T> *>(sh.in.v + to) = KeyGradients<T, D>::part(head_of<T>(a.v, b, kvh), a.v.s, tile0 + r, seq.n, at, a.width);
        if constexpr (GROUPS > 1)
            *reinterpret_cast<V8<T> *>(sh.in.k + to) = KeyGradients<T, D>::part(head_of<T>(a.k, b, kvh), a.k.s, tile0 + r, seq.n, at, a.width);
    }
    const T *Vs = sh.in.v + (32 * wave + i) * kPitch<T, D> + 8 * h, *Ks = sh.in.k + (32 * wave + i) * kPitch<T, D> + 8 * h;
    V8<T> kf[GROUPS > 1 ? 1 : D / 16];
    if constexpr (GROUPS == 1) {
#pragma unroll
        for (int u = 0; u < D / 16; ++u)
            kf[u] = KeyGradients<T, D>::part(head_of<T>(a.k, b, kvh), a.k.s, key, seq.n, 16 * u + 8 * h, a.width);
    }
    auto keys = [&](int u) -> V8<T> {
        if constexpr (GROUPS > 1) return *reinterpret_cast<const V8<T> *>(Ks + 16 * u);
        else return kf[u];
    };
    auto values = [&](int u) { return *reinterpret_cast<const V8<T> *>(Vs + 16 * u); };
    const float up = gradient_scale<T>(a), half = up * exp2_(-kShift<T>);
    // rows lo .. rows - 1 see some key of the tile
    const int64_t end = tile0 < a.sinks && !f.part ? 2 * kMaxExtent : far_from(tile0, a.window);
    const int lo = max(0, tile0 - seq.start);
    const int rows = (int)min(min((int64_t)a.sq, (int64_t)seq.n - seq.start), end - seq.start);
    const int from = lo / kRows, tiles = rows <= lo || tile0 >= seq.n ? 0 : (rows - 1) / kRows - from + 1;
    const int items = tiles * a.group, turns = (items + GROUPS - 1) / GROUPS;
    Staged<T, D, kRows> qs, gs;
    float ls = 0.f, ds = 0.f;
    // the group's tile of a turn: its head and first row
    struct Item {
        int head, r0;
        bool live;
    };
    auto item = [&](int turn) {
        const int t = turn * GROUPS + group;
        return Item{t / max(tiles, 1), (from + t % max(tiles, 1)) * kRows, t < items};
    };
    auto load = [&](int turn) {
        const Item x = item(turn);
        if (!x.live) return;
        const int64_t head = kvh * a.group + x.head;
        qs.load(head_of<T>(a.q, b, head), a.q.s, x.r0, a.sq - 1, a.width, tid);
        gs.load(head_of<T>(a.g, b, head), a.g.s, x.r0, a.sq - 1, a.width, tid);
        if (tid < kRows) {
            const int64_t stat = (b * a.heads + head) * a.sq + min(x.r0 + tid, a.sq - 1);
            ls = a.lse_in[stat];
            ds = a.delta[stat];
        }
    };
    auto whole = [&](const Item &x) {
        const int p0 = seq.start + x.r0;
        return (int)(x.r0 + kRows <= rows) & (int)sees_all(p0, p0 + kRows - 1, seq.n, a.window, a.sinks, tile0, tile0 + KEYS - 1);
    };
    auto store = [&](int turn) {
        const Item x = item(turn);
        const int to = turn & 1;
        bool special = false;
        if (x.live) {
            qs.store(sh.in.q[to][group], a.width, tid);
            gs.store(sh.in.g[to][group], a.width, tid);
            if (tid < kRows) {
                Ls[to][group][tid] = kShift<T> - ls * kLog2e;
                Ds[to][group][tid] = ds;
            }
            if (!whole(x)) special = __any((int)qs.special() | (int)gs.special());
        }
        flags[to][group * kWaves + wave] = special;
    };
    if (turns) {
        load(0);
        clear_past<T, D>(sh.in.q[0][0], 2 * GROUPS * kRows, a.width, threadIdx.x, kThreads * GROUPS);
        clear_past<T, D>(sh.in.g[0][0], 2 * GROUPS * kRows, a.width, threadIdx.x, kThreads * GROUPS);
        store(0);
        if (turns > 1) load(1);
    }
    for (int turn = 0; turn < turns; ++turn) {
        __syncthreads();
        if (turn + 1 < turns) store(turn + 1);
        if (turn + 2 < turns) load(turn + 2);
        const Item x = item(turn);
        const int at = turn & 1;
        T *Qs = sh.in.q[at][group], *Gs = sh.in.g[at][group];
        const Sight see = x.live ? sight(seq.start + x.r0, rows - x.r0, seq.n, a.window, a.sinks, mine, 32) : kNone;
        const bool all = see == kAll && x.r0 + kRows <= rows;  // a row past the last is hidden from every key
        f32x16 s, dp;
        if (see != kNone)
            w.template scores<GROUPS>(s, dp, keys, values, Qs, Gs, Ls[at][group], Ds[at][group], a.signed_c, half, all,
                     SeenRows(key, seq.start, x.r0, h, rows, seq.n, a.window, a.sinks), lane);
        if (any_wave(flags[at]) || (GROUPS > 1 && any_wave(flags[at] + kWaves * (GROUPS - 1)))) {
            if (see != kNone) w.special(Qs, Gs, SeenRows(key, seq.start, x.r0, 0, rows, seq.n, a.window, a.sinks), h);
            __syncthreads();
            clean<T, D, kRows, kThreads>(Qs, tid);
            clean<T, D, kRows, kThreads>(Gs, tid);
            __syncthreads();
        }
        if (see != kNone) w.add(s, dp, Qs, Gs, lane);
    }
    w.finish();
    if constexpr (GROUPS > 1) {
        // the second group's sums through LDS, dk and then dv
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            f32x16(&acc)[D / 32] = which ? w.dv : w.dk;
            float *mineat = sh.sums + wave * (D / 2) * 64 + lane;
            __syncthreads();
            if (group == 1) {
#pragma unroll
                for (int e = 0; e < D / 2; ++e) mineat[e * 64] = acc[e >> 4][e & 15];
            }
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int e = 0; e < D / 2; ++e) acc[e >> 4][e & 15] += mineat[e * 64];
            }
        }
        if (group) return;
    }
    if (f.part && mine < a.sinks) {
        store_part(f.at(b * a.kv + kvh, mine / 32, 0, a.width), w, i, h, a.width, true);
        return;
    }
    if (key >= a.sk) return;
    T *DK = const_cast<T *>(head_of<T>(a.dk, b, kvh)) + key * a.dk.s, *DV = const_cast<T *>(head_of<T>(a.dv, b, kvh)) + key * a.dv.s;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) {
        store_column(DK, w.dk[d], 32 * d, a.width, h, a.scale / up);
        store_column(DV, w.dv[d], 32 * d, a.width, h, exp2_(-kShift<T>));
    }
}

// The far rows of one block of sink keys: the tiles dealt to the waves, each of
// which stages its own.
template <typename T, int D>
__global__ __launch_bounds__(kThreads, 1) void window_far_kernel(WinArgs a, FarArgs f) {
    __shared__ __attribute__((aligned(16))) T tiles[kWaves][2][kRows * kPitch<T, D>];
    __shared__ __attribute__((aligned(16))) float stats[kWaves][2][kRows];
    const int tid = threadIdx.x, lane = tid & 63, i = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const float up = gradient_scale<T>(a), half = up * exp2_(-kShift<T>);
    const int64_t b = blockIdx.z / f.blocks, kvh = blockIdx.y;
    const int block = blockIdx.z % f.blocks, split = blockIdx.x * kWaves + wave, splits = f.splits * kWaves;
    const Seq seq(a, b);
    const int key = block * 32 + i;
    KeyGradients<T, D> w;
    V8<T> kf[D / 16], vf[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        kf[s] = KeyGradients<T, D>::part(head_of<T>(a.k, b, kvh), a.k.s, key, seq.n, 16 * s + 8 * h, a.width),
        vf[s] = KeyGradients<T, D>::part(head_of<T>(a.v, b, kvh), a.v.s, key, seq.n, 16 * s + 8 * h, a.width);
    const int from = max(0, far_from(block / kWaves * 32 * kWaves, a.window) - seq.start);
    const int rows = min(a.sq, seq.n - seq.start), count = rows > from ? (rows - from + kRows - 1) / kRows : 0;
    T *Qs = tiles[wave][0], *Gs = tiles[wave][1];
    float *Ls = stats[wave][0], *Ds = stats[wave][1];
    constexpr int PARTS = D / 16;
    V8<T> qr[PARTS], gr[PARTS];
    float ls = 0.f;
    auto load = [&](int t) {
        const int64_t head = kvh * a.group + t / count;
        const int r0 = from + t % count * kRows;
        const T *Q = head_of<T>(a.q, b, head), *G = head_of<T>(a.g, b, head);
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            const int part = lane + 64 * s, at = part % (D / 8) * 8, r = min(r0 + part / (D / 8), a.sq - 1);
            Pack<T, 8> x, y;
            x.load(Q + r * a.q.s + (at < a.width ? at : 0));
            y.load(G + r * a.g.s + (at < a.width ? at : 0));
            qr[s] = x.q;
            gr[s] = y.q;
        }
        const int64_t stat = (b * a.heads + head) * a.sq + min(r0 + i, a.sq - 1);
        ls = h ? a.delta[stat] : kShift<T> - a.lse_in[stat] * kLog2e;
    };
    const int items = count * a.group;
    clear_past<T, D>(Qs, 2 * kRows, a.width, lane, 64);  // of both tiles
    if (split < items) load(split);
    for (int t = split; t < items; t += splits) {
        const int r0 = from + t % count * kRows;
#pragma unroll
        for (int s = 0; s < PARTS; ++s) {
            const int part = lane + 64 * s, e = part % (D / 8) * 8, at = part / (D / 8) * kPitch<T, D> + (e < a.width ? e : 0);
            *reinterpret_cast<V8<T> *>(Qs + at) = qr[s];
            *reinterpret_cast<V8<T> *>(Gs + at) = gr[s];
        }
        (h ? Ds : Ls)[i] = ls;
        const bool whole = r0 + kRows <= rows;
        bool special = false;
        if (!whole) {
            Largest<T> most;
#pragma unroll
            for (int s = 0; s < PARTS; ++s) {
                most.add(qr[s]);
                most.add(gr[s]);
            }
            special = __any(most.special());
        }
        if (t + splits < items) load(t + splits);
        // the wave alone writes and reads its tile
        __builtin_amdgcn_wave_barrier();
        f32x16 s, dp;
        w.template scores<1>(s, dp, [&](int u) { return kf[u]; }, [&](int u) { return vf[u]; }, Qs, Gs, Ls, Ds, a.signed_c, half, whole, SeenRows(key, seq.start, r0, h, rows, seq.n, a.window, key + 1), lane);
        if (special) {
            w.special(Qs, Gs, SeenRows(key, seq.start, r0, 0, rows, seq.n, a.window, key + 1), h);
            clean<T, D, kRows, 64>(Qs, lane);
            clean<T, D, kRows, 64>(Gs, lane);
        }
        w.add(s, dp, Qs, Gs, lane);
        __builtin_amdgcn_wave_barrier();
    }
    w.finish();
    // the waves' sums through LDS, dk and then dv
    float *sums = reinterpret_cast<float *>(&tiles[0][0][0]) + lane;
    static_assert(sizeof tiles >= sizeof(float) * (kWaves - 1) * D / 2 * 64, "sums of three waves");
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        f32x16(&acc)[D / 32] = which ? w.dv : w.dk;
        __syncthreads();
        if (wave) {
#pragma unroll
            for (int e = 0; e < D / 2; ++e) sums[((wave - 1) * (D / 2) + e) * 64] = acc[e >> 4][e & 15];
        }
        __syncthreads();
        if (!wave) {
#pragma unroll
            for (int e = 0; e < D / 2; ++e)
                acc[e >> 4][e & 15] += (sums[e * 64] + sums[(D / 2 + e) * 64]) + sums[(D + e) * 64];
        }
    }
    if (wave) return;
    store_part(f.at(b * a.kv + kvh, block, 1 + blockIdx.x, a.width), w, i, h, a.width, key < a.sinks);
}

// One key of a sink block, dk and dv: every fourth part to a wave.
template <typename T>
__global__ __launch_bounds__(kThreads) void window_sinks_kernel(WinArgs a, FarArgs f) {
    __shared__ f32x4 join[kWaves][64];
    const float up = gradient_scale<T>(a);
    const int64_t b = blockIdx.z / f.blocks, kvh = blockIdx.y;
    const int block = blockIdx.z % f.blocks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int which = lane >> 5, at = 4 * (lane & 31), i = blockIdx.x, key = block * 32 + i;
    if (key >= a.sk) return;
    f32x4 x = {};
    if (at < a.width) {
        const float *part = f.at(b * a.kv + kvh, block, 0, a.width) + (32 * which + i) * a.width + at;
#pragma unroll 8
        for (int s = wave; s <= f.splits; s += kWaves) x += *reinterpret_cast<const f32x4 *>(part + (int64_t)s * 64 * a.width);
    }
    join[wave][lane] = x;
    __syncthreads();
    if (wave || at >= a.width) return;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) x += join[w][lane];
    const View &out = which ? a.dv : a.dk;
    const float scale = which ? exp2_(-kShift<T>) : a.scale / up;
    Pack<T, 4> y;
#pragma unroll
    for (int t = 0; t < 4; ++t) y.set(t, x[t] * scale);
    y.store(const_cast<T *>(head_of<T>(out, b, kvh)) + key * out.s + at);
}

// ---------------------------------------------------------------- dispatch
// f(T(), D): the operand type and the head width the registers hold.
template <class F>
int32_t with_head(chelis_dtype dt, int width, F &&f) {
    auto by_width = [&](auto t) -> int32_t {
        if (width <= 64) return f(t, std::integral_constant<int, 64>());
        if (width <= 96) return f(t, std::integral_constant<int, 96>());
        return f(t, std::integral_constant<int, 128>());
    };
    if (dt == CHELIS_DTYPE_F32) return by_width(float());
    if (dt == CHELIS_DTYPE_BF16) return by_width(__bf16());
    return by_width(_Float16());
}

View view_of(const chelis_gpu_tensor *t) { return {t->data, t->strides[0], t->strides[1], t->strides[2]}; }

int32_t check_part(const chelis_gpu_tensor *t, const char *name, const chelis_gpu_tensor *like, const char *what) {
    if (int32_t s = check_tensor(t, name)) return s;
    if (t->rank != 4 || !(t->dtype == CHELIS_DTYPE_F32 || is_narrow16(t->dtype)))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be f32, bf16 or f16 [batch, heads, seq, width]", what, name);
    if (t->dtype != like->dtype) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must have q's dtype", what, name);
    if (t->shape[3] > 1 && t->strides[3] != 1)
        return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: %s: the last axis must be contiguous", what, name);
    return check_device(t, name);
}

int32_t check_same(const chelis_gpu_tensor *t, const char *name, const chelis_gpu_tensor *like, const char *other,
                   const char *what) {
    if (!same_shape(t, like)) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must have %s's shape", what, name, other);
    return CHELIS_HIP_OK;
}

int32_t check_stat(const chelis_gpu_tensor *t, const char *name, const chelis_gpu_tensor *q, const char *what) {
    if (int32_t s = check_tensor(t, name)) return s;
    bool fits = t->dtype == CHELIS_DTYPE_F32 && t->rank == 3 && is_contiguous(t);
    for (int32_t i = 0; fits && i < 3; ++i) fits = t->shape[i] == q->shape[i];
    if (!fits) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be contiguous f32 [batch, heads, seq]", what, name);
    return check_device(t, name);
}

int32_t check_index(const chelis_gpu_tensor *t, const char *name, int64_t batch, const char *what) {
    if (int32_t s = check_tensor(t, name)) return s;
    if ((t->dtype != CHELIS_DTYPE_I32 && t->dtype != CHELIS_DTYPE_I64) || t->rank != 1 || t->shape[0] != batch)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s must be i32 or i64 [batch]", what, name);
    return check_device(t, name);
}

// Checks what both directions share and fills the arguments.
int32_t window_args(const chelis_gpu_tensor *q, const chelis_gpu_tensor *k, const chelis_gpu_tensor *v,
                    const chelis_gpu_tensor *lengths, const chelis_gpu_tensor *starts, int64_t window, int64_t sinks,
                    double scale, WinArgs *a, const char *what) {
    int32_t s;
    if ((s = check_tensor(q, "q")) || (s = check_part(q, "q", q, what)) || (s = check_part(k, "k", q, what)) ||
        (s = check_part(v, "v", q, what)) || (s = check_same(v, "v", k, "k", what)))
        return s;
    const int64_t B = q->shape[0], H = q->shape[1], KV = k->shape[1], W = q->shape[3];
    if (k->shape[0] != B || k->shape[3] != W)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: q and k must share batch and width", what);
    if (KV ? H % KV != 0 : H != 0)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %lld query heads over %lld key heads", what, (long long)H, (long long)KV);
    if (W < 8 || W > 128 || W % 8)
        return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: heads of %lld: a multiple of 8 up to 128", what, (long long)W);
    if (window < 1 || sinks < 0)
        return set_error(CHELIS_HIP_EDOMAIN, "%s: window must be at least 1 and sinks not negative", what);
    if (!std::isfinite(scale) || !std::isfinite((float)(std::fabs(scale) * kLog2e)))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: scale must be finite", what);
    if (q->shape[2] > kMaxExtent || k->shape[2] > kMaxExtent || B > 65535 || H > 65535)
        return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: more than 2^29 - 1024 rows or keys, or 65535 sequences or heads", what);
    if ((lengths && (s = check_index(lengths, "lengths", B, what))) ||
        (starts && (s = check_index(starts, "starts", B, what))))
        return s;
    a->q = view_of(q), a->k = view_of(k), a->v = view_of(v);
    if (lengths) {
        a->lengths = lengths->data, a->length_step = lengths->strides[0];
        a->lengths_wide = lengths->dtype == CHELIS_DTYPE_I64;
    }
    if (starts) {
        a->starts = starts->data, a->start_step = starts->strides[0];
        a->starts_wide = starts->dtype == CHELIS_DTYPE_I64;
    }
    a->sq = (int)q->shape[2], a->sk = (int)k->shape[2];
    // sinks that hold every key leave nothing to the window: plain causal rows
    if (sinks >= a->sk) window = a->sk, sinks = 0;
    a->window = (int)std::min<int64_t>(window, std::max(a->sk, 1)), a->sinks = (int)sinks;
    a->heads = (int)H, a->kv = (int)KV, a->group = KV ? (int)(H / KV) : 1, a->width = (int)W;
    a->flip = scale < 0, a->scale = (float)scale, a->c = (float)(std::fabs(scale) * 1.4426950408889634074);
    // hidden scores are -inf, and 0 times that is NaN
    if (a->c == 0.f) a->c = 0x1p-126f;
    a->signed_c = a->flip ? -a->c : a->c;
    return CHELIS_HIP_OK;
}

int32_t check_result(const chelis_gpu_tensor *t, const char *name, std::initializer_list<NamedTensor> others,
                     const char *what) {
    if (!non_overlapping(t)) return set_error(CHELIS_HIP_EDOMAIN, "%s: %s overlaps itself", what, name);
    if (const char *other = shared_with(t, others))
        return set_error(CHELIS_HIP_EDOMAIN, "%s: %s overlaps another operand (%s)", what, name, other);
    return CHELIS_HIP_OK;
}

// Key blocks of 32 that a run of `rows` query rows can see.
int64_t seen_blocks(const WinArgs &a, int64_t rows) {
    const int64_t span = std::min<int64_t>(a.sk, a.window + rows - 1) / 32 + 2 + (a.sinks + 31) / 32;
    return std::max<int64_t>(1, std::min<int64_t>((a.sk + 31) / 32, span));
}

// The rows are taken together over the heads of a group and the keys split
// over waves when that is estimated to be faster. Measured with bf16 heads of
// 128 (us, split against whole rows): 16 heads on 4, 16384 keys: one row 19
// against 490, 256 rows 137 against 366; window 1024 of 8 sequences: 16 rows
// 23 against 40, 32 rows 34-41 against 32; 2048 keys of 32 sequences, 32 heads on
// 8: 8 rows 77 against 143, 16 rows 136 against 110, 32 rows 233 against 110.
// Narrow heads cost the split what the 64 columns in registers cost: heads of 8,
// 16 on 16, 2048 keys: 512 rows 25 against 39, 2048 rows 73 against 40; binary32
// 512 rows 60 against 167, 2048 rows 197 against 168, and of 64, 75 against 168 and
// 243 against 169. Both kernels' times follow these lines.
bool few_rows(const WinArgs &a, chelis_dtype dt, int64_t batch) {
    const double f32 = dt == CHELIS_DTYPE_F32 ? 1 : 0;
    // a join takes a workgroup a row, and the split counts its rows in 32 bits
    if (!grid_fits(batch * a.heads * a.sq, kThreads)) return false;
    const int64_t tasks = batch * a.kv * (((int64_t)a.group * a.sq + 31) / 32);
    const int64_t groups = batch * a.heads * ((a.sq + 127) / 128), rounds = (groups + 511) / 512;
    const double idle = 24 + 16 * f32, width = std::max<double>(a.width, idle + a.width * (1 - idle / 64));
    const double split = 8 + (double)tasks * seen_blocks(a, a.sq) * width / 32000 * (1 + f32);
    const double whole = 5 + rounds * (seen_blocks(a, std::min(a.sq, 128)) / 2.0) * (0.75 + 0.005 * a.width) * (1 + 3 * f32);
    return split < whole;
}

int32_t window_split(const WinArgs &a, chelis_dtype dt, int64_t batch, hipStream_t st, const char *what) {
    SplitArgs p{};
    p.rows = a.group * a.sq;
    p.tiles = (p.rows + 31) / 32;
    p.pack = std::min(p.rows, 32);
    p.tasks = batch * a.kv * p.tiles;
    // eight waves a compute unit, a key block each at least; past 8 MB of
    // parts, no more of them than a quarter of the keys and values read
    const int64_t blocks = seen_blocks(a, a.sq), fill = 8 * (int64_t)device_cus() / p.tasks;
    const int64_t cheap = std::max<int64_t>(blocks * 8 / p.pack, (int64_t(8) << 20) / (p.tasks * p.pack * a.width * 4));
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({blocks, fill, cheap, kMaxSplits}));
    const int64_t grid = (p.tasks * p.splits + kWaves - 1) / kWaves, parts = p.tasks * p.splits * p.pack;
    const int64_t rows = batch * a.heads * a.sq;
    if (!grid_fits(grid, kThreads) || !grid_fits(rows, kThreads))
        return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: grid too large", what);
    const size_t bytes = p.splits > 1 ? (size_t)parts * (a.width + 2) * sizeof(float) : 0;
    if (bytes) {
        p.part = static_cast<float *>(scratch_alloc(bytes));
        if (!p.part) return set_error(CHELIS_HIP_EHIP, "%s: scratch of %zu bytes", what, bytes);
        p.stat = p.part + parts * a.width;
    }
    const int32_t s = with_head(dt, a.width, [&](auto t, auto d) -> int32_t {
        using T = decltype(t);
        window_split_kernel<T, d><<<(unsigned)grid, kThreads, 0, st>>>(a, p);
        if (bytes) window_join_kernel<T, d><<<(unsigned)rows, kThreads, 0, st>>>(a, p);
        return CHELIS_HIP_OK;
    });
    const hipError_t e = hipGetLastError();
    scratch_free(p.part, bytes);
    if (e != hipSuccess) return set_error(CHELIS_HIP_EHIP, "kernel launch: %s", hipGetErrorString(e));
    return s;
}

}  // namespace
}  // namespace chelis

using namespace chelis;

extern "C" int32_t chelis_hip_window_attention(const chelis_gpu_tensor *q, const chelis_gpu_tensor *k,
                                               const chelis_gpu_tensor *v, const chelis_gpu_tensor *lengths,
                                               const chelis_gpu_tensor *starts, int64_t window, int64_t sinks,
                                               double scale, const chelis_gpu_tensor *o,
                                               const chelis_gpu_tensor *lse) {
    const char *what = "window_attention";
    WinArgs a{};
    int32_t s;
    if ((s = window_args(q, k, v, lengths, starts, window, sinks, scale, &a, what)) ||
        (s = check_part(o, "o", q, what)) || (s = check_same(o, "o", q, "q", what)) ||
        (lse && (s = check_stat(lse, "lse", q, what))) ||
        (s = check_result(o, "o", {{q, "q"}, {k, "k"}, {v, "v"}, {lse, "lse"}, {lengths, "lengths"}, {starts, "starts"}}, what)) ||
        (lse && (s = check_result(lse, "lse", {{q, "q"}, {k, "k"}, {v, "v"}, {lengths, "lengths"}, {starts, "starts"}}, what))))
        return s;
    a.o = view_of(o);
    a.lse = lse ? static_cast<float *>(lse->data) : nullptr;
    if (!q->count) return CHELIS_HIP_OK;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    if (few_rows(a, q->dtype, q->shape[0])) return window_split(a, q->dtype, q->shape[0], st, what);
    const Deal rows = deal(a.sq, 32 * kWaves, a.group, q->shape[0] * a.kv);
    if (!grid_fits(rows.blocks(), kThreads)) return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: grid too large", what);
    return with_head(q->dtype, a.width, [&](auto t, auto d) -> int32_t {
        window_forward_kernel<decltype(t), d><<<(unsigned)rows.blocks(), kThreads, 0, st>>>(a, rows);
        CHELIS_LAUNCH_CHECK();
        return CHELIS_HIP_OK;
    });
}

extern "C" int32_t chelis_hip_window_attention_adjoint(
    const chelis_gpu_tensor *q, const chelis_gpu_tensor *k, const chelis_gpu_tensor *v, const chelis_gpu_tensor *o,
    const chelis_gpu_tensor *lse, const chelis_gpu_tensor *g, const chelis_gpu_tensor *lengths,
    const chelis_gpu_tensor *starts, int64_t window, int64_t sinks, double scale, const chelis_gpu_tensor *dq,
    const chelis_gpu_tensor *dk, const chelis_gpu_tensor *dv) {
    const char *what = "window_attention_adjoint";
    WinArgs a{};
    int32_t s;
    if ((s = window_args(q, k, v, lengths, starts, window, sinks, scale, &a, what))) return s;
    for (auto [t, name] : {std::pair(o, "o"), std::pair(g, "g"), std::pair(dq, "dq")})
        if ((s = check_part(t, name, q, what)) || (s = check_same(t, name, q, "q", what))) return s;
    for (auto [t, name] : {std::pair(dk, "dk"), std::pair(dv, "dv")})
        if ((s = check_part(t, name, q, what)) || (s = check_same(t, name, k, "k", what))) return s;
    if ((s = check_stat(lse, "lse", q, what))) return s;
    const std::initializer_list<NamedTensor> ins = {{q, "q"}, {k, "k"}, {v, "v"}, {o, "o"}, {g, "g"}, {lse, "lse"},
                                                    {lengths, "lengths"}, {starts, "starts"}};
    if ((s = check_result(dq, "dq", ins, what)) || (s = check_result(dk, "dk", ins, what)) ||
        (s = check_result(dv, "dv", ins, what)) || (s = check_result(dq, "dq", {{dk, "dk"}, {dv, "dv"}}, what)) ||
        (s = check_result(dk, "dk", {{dv, "dv"}}, what)))
        return s;
    a.o = view_of(o), a.g = view_of(g), a.dq = view_of(dq), a.dk = view_of(dk), a.dv = view_of(dv);
    a.lse_in = static_cast<const float *>(lse->data);
    if (!q->count && !k->count) return CHELIS_HIP_OK;
    hipStream_t st = stream();
    if (!st) return set_error(CHELIS_HIP_EHIP, "no HIP device");
    const Deal rows = deal(a.sq, 32 * kWaves, a.group, q->shape[0] * a.kv);
    const Deal keys = deal(a.sk, 32 * kWaves, 1, q->shape[0] * a.kv);
    if (!grid_fits(rows.blocks(), kThreads) || !grid_fits(keys.blocks(), 2 * kThreads))
        return set_error(CHELIS_HIP_EUNSUPPORTED, "%s: grid too large", what);
    // rows far behind the window of the first keys: dealt out a tile to a wave,
    // over no more workgroups than fill the device. Many sinks fill it as they
    // are, with less work and no parts: past eight sink blocks a compute unit
    // whose parts outgrow k, the keys' own workgroups walk those rows too
    // (bf16, dealt against walked, us: [8, 16 on 16, 2048, 128] of 256 sinks
    // 569 and 663, of 1024 1087 and 950; [64, 16 on 8, 1024, 64] of 64 sinks
    // 755 and 939, of 256 1138 and 987; [1, 16 on 4, 8192, 128] of 4096, 512
    // blocks in all, 1354 and 1781).
    FarArgs f{};
    const int64_t pairs = q->shape[0] * a.kv, far = (int64_t)a.sk - (32 * kWaves - 1) - a.window;
    const int64_t blocks = (a.sinks + 31) / 32;
    const bool many = pairs * blocks > 8 * (int64_t)device_cus() &&
                      2 * pairs * blocks * 64 * a.width * (int64_t)sizeof(float) > k->count * dtype_width(k->dtype);
    if (a.sinks > 0 && q->count && far > 0 && !many && q->shape[0] * blocks <= 65535) {
        f.blocks = (int)blocks;
        const int64_t tiles = (std::min<int64_t>(far, a.sq) + kRows - 1) / kRows * a.group;
        f.splits = (int)std::max<int64_t>(1, std::min<int64_t>((tiles + kWaves - 1) / kWaves, (int64_t)device_cus() / (pairs * f.blocks)));
    }
    const size_t parts = f.blocks ? (size_t)pairs * f.blocks * (1 + f.splits) * 64 * a.width : 0;
    const size_t bytes = (2 * kRanges + parts + (size_t)lse->count) * sizeof(float);
    a.range = static_cast<float *>(scratch_alloc(bytes));
    if (!a.range) return set_error(CHELIS_HIP_EHIP, "%s: scratch of %zu bytes", what, bytes);
    f.part = parts ? a.range + 2 * kRanges : nullptr;
    a.delta = a.range + 2 * kRanges + parts;
    s = with_head(q->dtype, a.width, [&](auto t, auto d) -> int32_t {
        using T = decltype(t);
        if constexpr (std::is_same<T, _Float16>::value) {
            window_range_kernel<T><<<2 * kRanges, 256, 0, st>>>(a, (int)q->shape[0]);
        }
        if (q->count) window_dq_kernel<T, d><<<(unsigned)rows.blocks(), kThreads, 0, st>>>(a, rows);
        if (k->count) window_dkv_kernel<T, d><<<(unsigned)keys.blocks(), kThreads * kGroups<T, d>, 0, st>>>(a, f, keys);
        if (parts) {
            const unsigned z = (unsigned)(q->shape[0] * f.blocks);
            window_far_kernel<T, d><<<dim3(f.splits, a.kv, z), kThreads, 0, st>>>(a, f);
            window_sinks_kernel<T><<<dim3(32, a.kv, z), kThreads, 0, st>>>(a, f);
        }
        return CHELIS_HIP_OK;
    });
    const hipError_t e = hipGetLastError();
    scratch_free(a.range, bytes);
    if (e != hipSuccess) return set_error(CHELIS_HIP_EHIP, "kernel launch: %s", hipGetErrorString(e));
    return s;
}
