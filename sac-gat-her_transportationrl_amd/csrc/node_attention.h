// node_attention.h -- what the attention kernels share (node_attention_fwd.h,
// node_attention_bwd.h): matrix fragments, staged tiles, scores.
//
// Fragments.  The 16 x 16 matrix instructions take, in lane l (g = l / 16, c = l
// % 16), eight operand elements of row or column c at depth 8g .. 8g+7 of a
// 32-deep step (float32: eight 4-deep instructions, instruction j takes element
// j of each lane, so the depth it covers is {8g + j}), and give rows 4g .. 4g+3
// of column c.  Scores are computed as a transposed tile whose column is the row
// that the next product keeps (the query in the forward and in grad_q, the key
// in grad_k / grad_v).  Its results then already lie as the next product's
// second operand, with depth slot (g, j) meaning row 4g + j of one 16-row tile
// (j < 4) and row 4g + j - 4 of the next: probabilities never pass through LDS.
// The first operand follows that order when it is read from its staged
// row-major tile: LDS transposing reads give a lane four rows of its column at
// once for two-byte types, plain reads for float32.
#pragma once
#include <hip/hip_runtime.h>

#include <cmath>
#include <type_traits>

#include "float_types.h"
#include "trx_internal.h"

namespace trx {

// How a pass over kept rows (tiles of them) and an axis that is run over (splits of it) is cut
struct AttentionCut {
    bool narrow;   // one wave
    int mq;        // its 16-row tiles
    int64_t tiles;
    int splits;
};

namespace {

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

using Args = trx_node_attention_args;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Frag;
template <>
struct Frag<__bf16> {
    typedef __bf16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Frag<_Float16> {
    typedef _Float16 type __attribute__((ext_vector_type(8)));
};
template <>
struct Frag<float> {
    typedef float type __attribute__((ext_vector_type(8)));
};
template <typename T>
using frag = typename Frag<T>::type;

__device__ __forceinline__ f32x4 mma(frag<__bf16> a, frag<__bf16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(frag<_Float16> a, frag<_Float16> b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(frag<float> a, frag<float> b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

template <typename T>
__device__ __forceinline__ frag<T> zero_frag() {
    frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)0.0f;
    return f;
}
template <typename T>
__device__ __forceinline__ frag<T> load_frag(const T* p) {
    return __builtin_bit_cast(frag<T>, load8(p));
}

// LDS row of a staged tile: 16 bytes longer than CP elements, so that the 16
// rows of a fragment start in different banks
template <typename T, int CP>
constexpr int kRow = CP + 16 / (int)sizeof(T);

// elements of column col + c at rows 4g .. 4g+3 behind row0 and behind row1
template <typename T, int CP>
__device__ __forceinline__ frag<T> turned(const T* tile, int row0, int row1, int col, int lane) {
    const int g = lane / 16, c = lane % 16;
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4 lds4;
        const T* p = tile + (row0 + 4 * g + c / 4) * kRow<T, CP> + col + 4 * (c % 4);
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + (row1 - row0) * kRow<T, CP>));
        return __builtin_bit_cast(frag<T>, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    } else {
        frag<T> f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            f[j] = tile[(row0 + 4 * g + j) * kRow<T, CP> + col + c];
            f[4 + j] = tile[(row1 + 4 * g + j) * kRow<T, CP> + col + c];
        }
        return f;
    }
}

// ROWS x CP elements of consecutive rows on their way from memory to LDS through
// registers.  Rows and channels behind the last come from the last: nothing is
// masked, because what a tile holds there meets weights of zero (rows) or zero
// operands and results that are not stored (channels).
template <typename T, int CP, int ROWS, int THREADS>
struct Staged {
    static constexpr int kChunks = ROWS * (CP / 8), kEach = (kChunks + THREADS - 1) / THREADS;
    Eight<T> r[kEach];

    static __device__ __forceinline__ int row_of(int e) { return (threadIdx.x + e * THREADS) / (CP / 8); }
    static __device__ __forceinline__ int channel_of(int e) { return 8 * ((threadIdx.x + e * THREADS) % (CP / 8)); }

    // rows first .. of `rows` (at least one)
    __device__ __forceinline__ void load(const T* base, int64_t row, int first, int rows, int C) {
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            r[e] = load8(base + min(first + row_of(e), rows - 1) * row + min(channel_of(e), C - 8));
    }
    // the same with a pointer of its own for each row
    template <typename F>
    __device__ __forceinline__ void load_rows(int first, int rows, int C, F&& row) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) r[e] = load8(row(min(first + row_of(e), rows - 1)) + min(channel_of(e), C - 8));
    }
    __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (kChunks % THREADS == 0 || row_of(e) < ROWS) store8(tile + row_of(e) * kRow<T, CP> + channel_of(e), r[e]);
    }
};

// n / d for 0 <= n < 2^31 by a multiplication
struct Divide {
    uint32_t mul, shift, by;
    __device__ __forceinline__ int operator()(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};
inline Divide divide_by(int d) {
    uint32_t s = 0;
    while ((int64_t(1) << s) < d) ++s;
    return {(uint32_t)((uint64_t(1) << (31 + s)) / d + 1), 31 + s, (uint32_t)d};
}

// The arguments of a launch.  The grid: every (tile, split, graph, key/value head) in this order, last tiles first:
// only large graphs have them, and their workgroups, the longest, had better not start last.  Behind them kRestBlocks
// workgroups for the rows of no graph; they must not lie between the others, or every second compute unit gets nothing
// else.  Eight dies take workgroups in turn, so the tiles of one (graph, head), which read the same keys, lie behind one
// L2 where there are 8 k heads.  Where there are distances, the heads of a tile go to one die instead: they read the
// same 4 bytes a pair and head, which would otherwise come through the fabric once a die.
constexpr int kRestBlocks = 16;
// What scores are counted in: a power of two, so that products with it are exact.  Natural units where a bias or a cap
// comes in; else the power of two below the scale, so that a scale like 1 / 8 leaves the products as they come.
struct Unit {
    float pre;     // what the products <q, k> are multiplied by (where scores are capped: to the tanh's argument)
    float log2;    // from scores to log 2
    float nat;     // from scores to natural units, and back
    float per;
};
inline Unit unit_of(const Args& a) {
    if (a.cap > 0.0f) return {a.scale / a.cap, kLog2e, 1.0f, 1.0f};
    if (a.dist) return {a.scale, kLog2e, 1.0f, 1.0f};
    int e = a.scale == 0.0f ? 0 : std::ilogb(a.scale);
    e = e < -100 ? -100 : e > 100 ? 100 : e;
    return {std::ldexp(a.scale, -e), std::ldexp(kLog2e, e), std::ldexp(1.0f, e), std::ldexp(1.0f, -e)};
}

struct Call {
    Args a;
    Divide group, kv, units;   // by heads of a group, key/value heads, (graph, key/value head)s
    Divide splits;
    int tiles, blocks;
    Unit unit;
};
inline Call call_of(const Args& a, const AttentionCut& c) {
    const int units = a.num_graphs * a.kv_heads;
    return {a, divide_by(a.heads / a.kv_heads), divide_by(a.kv_heads), divide_by(units > 0 ? units : 1),
            divide_by(c.splits), (int)c.tiles, (int)c.tiles * c.splits * units, unit_of(a)};
}

// one column's four distances behind key j: +inf from `limit` on
__device__ __forceinline__ f32x4 distances(const float* row, int j, int limit, bool whole) {
    if (whole || j + 4 <= limit) return *reinterpret_cast<const f32x4u*>(row + j);
    f32x4 d{INFINITY, INFINITY, INFINITY, INFINITY};
    if (j < limit) {
        d[0] = row[j];
        if (j + 1 < limit) d[1] = row[j + 1];
        if (j + 2 < limit) d[2] = row[j + 2];
    }
    return d;
}

// ROWS query rows' distances to KT keys, through registers to LDS like the tiles.  A fragment's lanes hold sixteen
// rows side by side, so reading them where they are used would touch sixteen cache lines for every sixteen lanes;
// here the lanes run along the rows.
//
// Where rows go in equal steps, one 32-bit offset a lane and scalars address them all.  The last tile's window then
// ends at the matrix's last row and key instead of passing them: `shift` is how far its rows lie behind where the
// tile's first row would be (rows behind the last that is read meet nothing), and lanes that were moved back along
// the keys move their values.  Every other shape takes each row by itself.
template <int ROWS, int KT, int THREADS>
struct StagedDistances {
    static constexpr int kLanes = KT / 4, kStep = THREADS / kLanes, kEach = ROWS / kStep, kPitch = KT + 4;
    f32x4 r[kEach];
    int shift;

    // rows row0 .. row0 + ROWS of the graph's (query, head of the group)s, `rows` of them there; keys from j on
    __device__ __forceinline__ void load(const Call& call, const float* graph, int row0, int rows, int keys, int j) {
        const Args& a = call.a;
        const int G = call.group.by, mine = threadIdx.x / kLanes, col = 4 * (threadIdx.x % kLanes);
        const int limit = min(keys, a.dist_cols), i0 = call.group(row0), end = min(row0 + ROWS, rows);
        const int first = min(i0, a.dist_rows - ROWS / G);
        shift = 0;
        if (kStep % G == 0 && row0 % G == 0 && a.dist_row < (1 << 24) && limit >= 4 && first >= 0 &&
            call.group(end - 1) < a.dist_rows) {
            shift = (i0 - first) * G;
            const int j1 = min(j, limit - 4), at = min(j + col, limit - 4), back = j + col - at;
            const float* base = graph + first * a.dist_row + j1;
            const uint32_t off = call.group(mine) * (uint32_t)a.dist_row + (at - j1);
#pragma unroll
            for (int e = 0; e < kEach; ++e)
                r[e] = *reinterpret_cast<const f32x4u*>(base + e * (kStep / G) * a.dist_row + off);
            if (j + KT > limit) {
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const f32x4 v = r[e];
                    r[e][0] = back == 0 ? v[0] : back == 1 ? v[1] : back == 2 ? v[2] : back == 3 ? v[3] : INFINITY;
                    r[e][1] = back == 0 ? v[1] : back == 1 ? v[2] : back == 2 ? v[3] : INFINITY;
                    r[e][2] = back == 0 ? v[2] : back == 1 ? v[3] : INFINITY;
                    r[e][3] = back == 0 ? v[3] : INFINITY;
                }
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int row = row0 + mine + kStep * e, i = call.group(min(row, rows - 1));
            r[e] = distances(graph + i * a.dist_row, j + col, i < a.dist_rows ? limit : 0, false);
        }
    }
    __device__ __forceinline__ void store(float* tile) const {
        const int mine = threadIdx.x / kLanes, col = 4 * (threadIdx.x % kLanes);
#pragma unroll
        for (int e = 0; e < kEach; ++e) *reinterpret_cast<f32x4*>(tile + (mine + kStep * e) * kPitch + col) = r[e];
    }
};

// four elements of a result; where `low` is given, what rounding took from them goes there
template <typename T>
__device__ __forceinline__ void put4(T* out, T* low, int64_t at, f32x4 v) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    T4 y;
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = (T)v[r];
    *reinterpret_cast<T4*>(out + at) = y;
    if (low) {
        T4 z;
#pragma unroll
        for (int r = 0; r < 4; ++r) z[r] = (T)(v[r] - (float)y[r]);
        *reinterpret_cast<T4*>(low + at) = z;
    }
}

// 16-row tiles of a wave in a workgroup of four: two, one where float32's accumulators and operands of 128 channels
// would not leave registers for two waves
template <typename T, int CP>
constexpr int kTilesOfWave = sizeof(T) == 4 && CP == 128 ? 1 : 2;

// Waves of a SIMD that registers are left for.  For a workgroup of one wave the compiler's own choice takes accumulator
// registers beside the others and so fits fewer: 4096 networks of 24 nodes, 4 heads of 64, forward, 42 us with 2 asked
// for, 50 us without, 66 us with 4 (spills).
template <typename T, int CP, int WAVES>
constexpr int kWavesPerSimd = WAVES > 1 || CP <= 64 ? 2 : 1;

// calls f with the padded channels, whether there are distances, whether scores are capped
template <typename T, typename F>
inline hipError_t by_shape(const Args& a, F&& f) {
    auto second = [&](auto cp) {
        if (a.dist)
            return a.cap > 0.0f ? f(cp, std::true_type{}, std::true_type{}) : f(cp, std::true_type{}, std::false_type{});
        return a.cap > 0.0f ? f(cp, std::false_type{}, std::true_type{}) : f(cp, std::false_type{}, std::false_type{});
    };
    if (a.channels <= 32) return second(std::integral_constant<int, 32>{});
    if (a.channels <= 64) return second(std::integral_constant<int, 64>{});
    return second(std::integral_constant<int, 128>{});
}

// what a workgroup does
struct Work {
    int tile, split, graph, head;   // key/value head
};
template <bool DIST>
__device__ __forceinline__ Work work_of(const Call& call) {
    int id = blockIdx.x;
    const int heads = call.a.kv_heads, groups = call.kv(call.blocks) & ~7;
    if (DIST && id < groups * heads) {
        // eight graphs' worth at a time, turned from lot to lot, or a graph would always meet the same die
        const int slot = id >> 3, lot = call.kv(slot), turn = lot + (lot >> 3) + (lot >> 6);
        id = (lot * 8 + ((id + turn) & 7)) * heads + (slot - lot * heads);
    }
    const int of = call.units(id), unit = id - of * call.units.by, tile = call.splits(of), graph = call.kv(unit);
    return {call.tiles - 1 - tile, of - tile * (int)call.splits.by, graph, unit - graph * heads};
}

struct Span {
    int64_t at;
    int n;
};
// graph b's rows, clamped to the tensor
__device__ __forceinline__ Span span(const int64_t* ptr, int b, int64_t rows) {
    int64_t lo = ptr[b], hi = ptr[b + 1];
    lo = lo < 0 ? 0 : lo > rows ? rows : lo;
    hi = hi < lo ? lo : hi > rows ? rows : hi;
    return {lo, (int)(hi - lo)};
}
// the rows of all graphs
__device__ __forceinline__ Span all_rows(const int64_t* ptr, int graphs, int64_t rows) {
    int64_t lo = graphs > 0 ? ptr[0] : 0, hi = graphs > 0 ? ptr[graphs] : 0;
    lo = lo < 0 ? 0 : lo > rows ? rows : lo;
    hi = hi < lo ? lo : hi > rows ? rows : hi;
    return {lo, (int)(hi - lo)};
}
// zeros in the rows of no graph (before the first and behind the last)
template <typename T>
__device__ __forceinline__ void zero_rest(T* out, const int64_t* ptr, int graphs, int64_t rows, int64_t width,
                                          int block) {
    const Span s = all_rows(ptr, graphs, rows);
    const int64_t at = (int64_t)block * blockDim.x + threadIdx.x, step = (int64_t)kRestBlocks * blockDim.x;
    for (int64_t e = at; e < s.at * width; e += step) out[e] = (T)0.0f;
    for (int64_t e = (s.at + s.n) * width + at; e < rows * width; e += step) out[e] = (T)0.0f;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// sums and maxima over the four lanes that share a column (same c)
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// A row's weights are 2^(w unit - R) for some reference R near its largest score's.  Everything is divided by their sum in
// the end, so R need not be anything in particular, but it must be the same number for each of them, and near: log2 of
// the sum, rounded into R, would be lost where scores are large and alike (24 nodes at one distance of 1e9).
//   Near zero (|R| below some 2^20) R = c, c = at unit rounded, and one multiply-add a score is exact up to the result's
// own step.  Farther, at unit would be rounded by more than the exponents that matter: there R = at unit as it is, and
// scores have `at` subtracted first, which is exact where they are close.  A wave takes that form for all its rows as
// soon as one needs it; add = at unit - R says the same of the others.
//   `lift` puts R that far below at unit.
struct Around {
    float at, c;
    __device__ __forceinline__ bool far(float limit) const { return fabsf(c) >= limit && fabsf(at) < INFINITY; }
    __device__ __forceinline__ float add(float unit, float limit, float lift = 0.0f) const {
        return fabsf(c) < limit ? __builtin_fmaf(at, unit, -c) : lift;
    }
};
__device__ __forceinline__ Around around(float at, float unit, float lift = 0.0f) {
    return {at, __builtin_fmaf(at, unit, -lift)};
}
constexpr float kFar = 1048576.0f;
// float16 ends at 2^16 and loses bits below 2^-14, so what is rounded to it is brought into that range first.
// Forward: weights are 2^7 at the reference and at most 2^15; without, those below 2^-14 of the largest lose bits and
// those below 2^-25 of it vanish from the product though the sum has them.  A probability in grad_v: by 2^15.
template <typename T>
constexpr bool kHalf = std::is_same_v<T, _Float16>;
template <typename T>
constexpr float kLift = kHalf<T> ? 7.0f : 0.0f;
template <typename T>
constexpr float kWeight = kHalf<T> ? 32768.0f : 1.0f;
// A score's gradient has no scale that is known beforehand (it is as large as the incoming gradient over the nodes):
// each column keeps a power of two that brings its largest so far to 2^8 .. 2^14, and its accumulators follow when one
// passes that.  Nothing of it is left in the result.  (bfloat16 has float32's range and needs none of this.)
struct Raise {
    float by;
    template <int N>
    __device__ __forceinline__ void over(float most, f32x4 (&acc)[N]) {
        if (__any(!(most * by <= 16384.0f))) {
            const float top = column_max(most);
            const float next =
                top * by > 16384.0f ? __uint_as_float((262u - (__float_as_uint(top) >> 23)) << 23) : by;   // 2^8 / top
#pragma unroll
            for (int x = 0; x < N; ++x) acc[x] = acc[x] * (next / by);
            by = next;
        }
    }
};
constexpr float kRaiseAll = 0x1p100f;   // until something has been seen
// In the backward passes R comes from lse, and near zero two-byte types take the weights around it for probabilities:
// up to 2^10 their sum is 1 within 2^-14 (half a step of lse and one of c), an eighth of half a step of float16.
template <typename T>
constexpr float kFarBack = sizeof(T) == 2 ? 1024.0f : kFar;
// what is done to every score of a lane's column: n over its tiles, r over a tile's four rows
#define TRX_EACH_SCORE _Pragma("unroll") for (int n = 0; n < kTiles; ++n) _Pragma("unroll") for (int r = 0; r < 4; ++r)
// Scores capped: cap tanh(s * pre), and with SLACK the tanh's slope 1 - tanh^2.  float32 takes the library's tanh.  For
// two-byte types, a tile whose arguments all lie within a quarter of zero takes the series to x^7 (off by 4e-7 of x at
// the end), seven operations; others 1 - 2 / (1 + e^2x) by the hardware's exp2 and reciprocal, twelve, off by 2^-23:
// 8e-6 in a score at a cap of 64, far below what rounding its probability takes.  With larger caps that error would
// grow past the scores' own, so there arguments within a quarter of zero take the series wherever they are.  So they do
// where `alone`: a score is then the same number in whatever tile it is computed.  The backward passes need that beside
// biases so large that the least difference moves the sum to its neighbour, which may weigh 2^90 times as much.
template <typename T, int kTiles, bool SLACK>
__device__ __forceinline__ void cap_scores(f32x4 (&s)[kTiles], f32x4 (&slack)[kTiles], float pre, float cap, bool alone) {
    if constexpr (sizeof(T) == 4) {
        TRX_EACH_SCORE {
            const float th = tanhf(s[n][r] * pre);
            s[n][r] = cap * th;
            if (SLACK) slack[n][r] = __builtin_fmaf(-th, th, 1.0f);
        }
    } else {
        float most = 0.0f;
        TRX_EACH_SCORE {
            s[n][r] *= pre;
            most = fmaxf(most, fabsf(s[n][r]));
        }
        auto series = [](float x) {
            const float y = x * x;
            return x * __builtin_fmaf(y, __builtin_fmaf(y, __builtin_fmaf(y, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f), 1.0f);
        };
        if (__all(most < 0.25f)) {
            TRX_EACH_SCORE {
                const float th = series(s[n][r]);
                s[n][r] = cap * th;
                if (SLACK) slack[n][r] = __builtin_fmaf(-th, th, 1.0f);
            }
        } else if (cap <= 64.0f && !alone) {
            TRX_EACH_SCORE {
                const float e = exp2_fast(s[n][r] * (2.0f * kLog2e));
                const float th = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
                s[n][r] = cap * th;
                if (SLACK) slack[n][r] = __builtin_fmaf(-th, th, 1.0f);
            }
        } else {
            TRX_EACH_SCORE {
                const float x = s[n][r], e = exp2_fast(x * (2.0f * kLog2e));
                const float th = fabsf(x) < 0.25f ? series(x) : __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + e), 1.0f);
                s[n][r] = cap * th;
                if (SLACK) slack[n][r] = __builtin_fmaf(-th, th, 1.0f);
            }
        }
    }
}
// the products of a tile to scores: with the scale, or capped
template <typename T, bool CAP, bool SLACK, int kTiles>
__device__ __forceinline__ void scores(const Call& call, f32x4 (&s)[kTiles], f32x4 (&slack)[kTiles], bool alone) {
    if (CAP) {
        cap_scores<T, kTiles, SLACK>(s, slack, call.unit.pre, call.a.cap, alone);
    } else if (call.unit.pre != 1.0f) {
        TRX_EACH_SCORE s[n][r] *= call.unit.pre;
    }
}
template <int N>
__device__ __forceinline__ bool ordinary(const f32x4 (&d)[N]) {
    uint32_t most = 0;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) most = max(most, __float_as_uint(d[n][r]));
    return __all(most <= 0x7f800000u);   // neither negative nor NaN
}

}  // namespace

// node_attention_fwd.h, node_attention_bwd.h; instantiated in node_attention_{f32,bf16,f16}.hip
template <typename T>
hipError_t launch_attention_fwd(const trx_node_attention_args& a, hipStream_t stream);
template <typename T>
hipError_t launch_attention_bwd(const trx_node_attention_args& a, hipStream_t stream);
AttentionCut cut_fwd(const trx_node_attention_args& a);
AttentionCut cut_bwd_q(const trx_node_attention_args& a);
AttentionCut cut_bwd_kv(const trx_node_attention_args& a);
size_t attention_row_floats(const trx_node_attention_args& a);
constexpr int kSlopeChunks = 64;   // of the rows, each with its own sum of the slopes' gradients

}  // namespace trx
