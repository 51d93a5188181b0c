// node_attention.h -- what the attention kernels share (node_attention.hip,
// node_attention_bwd.hip): matrix fragments, staged tiles, scores.
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

#include "float_types.h"
#include "trx_internal.h"

namespace trx {
namespace {

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f;

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

// ROWS x CP elements on their way from memory to LDS through registers: loaded
// while the tile before is worked on
template <typename T, int CP, int ROWS, int THREADS>
struct Staged {
    static constexpr int kChunks = ROWS * (CP / 8), kEach = (kChunks + THREADS - 1) / THREADS;
    Eight<T> r[kEach];

    // row(i) -> pointer to row i's first element, or null where there is none
    template <typename F>
    __device__ __forceinline__ void load(int C, F&& row) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int x = threadIdx.x + e * THREADS, i = x / (CP / 8), c = 8 * (x % (CP / 8));
            const T* p = x < kChunks ? row(i) : nullptr;
            r[e] = p && c < C ? load8(p + c) : Eight<T>{};
        }
    }
    __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int x = threadIdx.x + e * THREADS, i = x / (CP / 8), c = 8 * (x % (CP / 8));
            if (x < kChunks) store8(tile + i * kRow<T, CP> + c, r[e]);
        }
    }
};

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
__device__ __forceinline__ void zero_rest(T* out, const int64_t* ptr, int graphs, int64_t rows, int64_t width, int at,
                                          int step) {
    const Span s = all_rows(ptr, graphs, rows);
    for (int64_t e = at; e < s.at * width; e += step) out[e] = (T)0.0f;
    for (int64_t e = (s.at + s.n) * width + at; e < rows * width; e += step) out[e] = (T)0.0f;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh(x * mul): for two-byte types 1 - 2 / (1 + e^2x) with the hardware's exp2
// and reciprocal, off by about 2^-23 absolute, far below their products' own
// rounding; float32 takes the library's
template <typename T>
__device__ __forceinline__ float tanh_of(float x, float mul) {
    if constexpr (sizeof(T) == 2)
        return __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + exp2_fast(x * (mul * 2.0f * kLog2e))), 1.0f);
    else
        return tanhf(x * mul);
}

// sums and maxima over the four lanes that share a column (same c)
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// one column's four distances behind key j: +inf from `limit` on
__device__ __forceinline__ f32x4 distances(const float* row, int j, int limit, bool whole) {
    if (whole) return *reinterpret_cast<const f32x4u*>(row + j);
    f32x4 d;
#pragma unroll
    for (int r = 0; r < 4; ++r) d[r] = j + r < limit ? row[j + r] : INFINITY;
    return d;
}

}  // namespace

// node_attention_bwd.hip
hipError_t launch_attention_bwd(const trx_node_attention_args& a, hipStream_t stream);
size_t attention_bwd_workspace(const trx_node_attention_args& a);

}  // namespace trx
