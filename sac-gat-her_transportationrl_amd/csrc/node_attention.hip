// node_attention.hip -- softmax attention of query rows over the nodes of their
// own network (include/trafficrl.h, trx_node_attention_*): scores scaled,
// optionally capped by a tanh, lowered by slope[h] times the pair's distance,
// pairs at no finite distance unseen.
//
// Forward: one wave per (query row, head), its lanes over the channels, one
// pass over the keys with the running maximum and sum.  Backward: one wave per
// (query row, head) for grad_q and the slope, one per (node, kv head) for
// grad_k and grad_v; the probabilities come back from the saved lse.
#include <hip/hip_runtime.h>

#include "float_types.h"
#include "trx_internal.h"

namespace trx {
namespace {

constexpr int kWave = 64;
constexpr float kLog2e = 1.44269504088896340736f;

using Args = trx_node_attention_args;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

struct Span {
    int64_t at;
    int n;
};

// graph b's rows, clamped to the tensor; graph num_graphs: none
__device__ __forceinline__ Span span(const int64_t* ptr, int b, int64_t rows) {
    int64_t lo = ptr[b], hi = ptr[b + 1];
    lo = lo < 0 ? 0 : lo > rows ? rows : lo;
    hi = hi < lo ? lo : hi > rows ? rows : hi;
    return {lo, (int)(hi - lo)};
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// the distance of pair (i, j) of graph b, +inf where the pair is not seen
__device__ __forceinline__ float distance(const Args& a, int b, int i, int j) {
    if (!a.dist) return 0.0f;
    if (i >= a.dist_rows || j >= a.dist_cols) return INFINITY;
    const float d = a.dist[b * a.dist_graph + i * a.dist_row + j];
    return finite(d) ? d : INFINITY;
}

// rows of no graph: before the first and behind the last
template <typename T>
__device__ __forceinline__ void zero_rest(T* out, const int64_t* ptr, int graphs, int64_t rows, int64_t width, int at,
                                          int step) {
    if (!out) return;
    int64_t begin = graphs > 0 ? ptr[0] : 0, end = graphs > 0 ? ptr[graphs] : 0;
    begin = begin < 0 ? 0 : begin > rows ? rows : begin;
    end = end < begin ? begin : end > rows ? rows : end;
    for (int64_t e = at; e < begin * width; e += step) out[e] = (T)0.0f;
    for (int64_t e = end * width + at; e < rows * width; e += step) out[e] = (T)0.0f;
}

struct Score {
    float w, slack, d;   // the biased score in units of log 2, dz/d(scaled product), the distance
    bool seen;
};
__device__ __forceinline__ Score score(const Args& a, float dot, float d, float slope) {
    float z = dot * a.scale, slack = 1.0f;
    if (a.cap > 0.0f) {
        const float t = tanhf(z / a.cap);
        z = a.cap * t;
        slack = 1.0f - t * t;
    }
    if (!finite(d)) return {-INFINITY, 0.0f, 0.0f, false};
    return {(z - slope * d) * kLog2e, slack, d, true};
}

template <typename T>
__device__ __forceinline__ float2 two(const T* row, int C, int lane) {
    return {lane < C ? (float)row[lane] : 0.0f, lane + kWave < C ? (float)row[lane + kWave] : 0.0f};
}
template <typename T>
__device__ __forceinline__ void put(T* row, int C, int lane, float x, float y) {
    if (lane < C) row[lane] = (T)x;
    if (lane + kWave < C) row[lane + kWave] = (T)y;
}

template <typename T>
__global__ void __launch_bounds__(kWave) attention_fwd_kernel(Args a) {
    const int lane = threadIdx.x, b = blockIdx.x, h = blockIdx.z, C = a.channels;
    T* out = static_cast<T*>(a.out);
    if (b == a.num_graphs) {
        const int at = (blockIdx.z * gridDim.y + blockIdx.y) * kWave + lane, step = gridDim.y * gridDim.z * kWave;
        zero_rest(out, a.q_ptr, b, a.num_queries, (int64_t)a.heads * C, at, step);
        return;
    }
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int hk = h / (a.heads / a.kv_heads);
    const float slope = a.slope ? a.slope[h] : 0.0f;
    for (int i = blockIdx.y; i < qs.n; i += gridDim.y) {
        const int64_t row = qs.at + i;
        const float2 q = two(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head, C, lane);
        float m = -INFINITY, l = 0.0f, ox = 0.0f, oy = 0.0f;
        for (int j = 0; j < ks.n; ++j) {
            const float2 k = two(static_cast<const T*>(a.k) + (ks.at + j) * a.k_row + hk * a.k_head, C, lane);
            const Score s = score(a, wave_sum(q.x * k.x + q.y * k.y), distance(a, b, i, j), slope);
            if (s.w == -INFINITY) continue;
            const float2 v = two(static_cast<const T*>(a.v) + (ks.at + j) * a.v_row + hk * a.v_head, C, lane);
            const float mn = s.w > m ? s.w : m, f = exp2f(m - mn), p = exp2f(s.w - mn);
            l = l * f + p;
            ox = ox * f + p * v.x;
            oy = oy * f + p * v.y;
            m = mn;
        }
        const float r = l == 0.0f ? 0.0f : 1.0f / l;
        put(out + (row * a.heads + h) * C, C, lane, ox * r, oy * r);
        if (a.lse && lane == 0) a.lse[row * a.heads + h] = l == 0.0f ? -INFINITY : m + log2f(l);
    }
}

template <typename T>
__global__ void __launch_bounds__(kWave) attention_bwd_q_kernel(Args a, float* dots, float* slopes) {
    const int lane = threadIdx.x, b = blockIdx.x, h = blockIdx.z, C = a.channels;
    const int at = (blockIdx.z * gridDim.y + blockIdx.y) * kWave + lane, step = gridDim.y * gridDim.z * kWave;
    T* gq = static_cast<T*>(a.grad_q);
    if (b == a.num_graphs) {
        zero_rest(gq, a.q_ptr, b, a.num_queries, (int64_t)a.heads * C, at, step);
        zero_rest(slopes, a.q_ptr, b, a.num_queries, (int64_t)a.heads, at, step);
        return;
    }
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int hk = h / (a.heads / a.kv_heads);
    const float slope = a.slope ? a.slope[h] : 0.0f;
    for (int i = blockIdx.y; i < qs.n; i += gridDim.y) {
        const int64_t row = qs.at + i, o = row * a.heads + h;
        const float2 q = two(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head, C, lane);
        const float2 go = two(static_cast<const T*>(a.grad_out) + o * C, C, lane);
        const float2 ov = two(static_cast<const T*>(a.out) + o * C, C, lane);
        const float D = wave_sum(go.x * ov.x + go.y * ov.y), lse = a.lse[o];
        float gx = 0.0f, gy = 0.0f, pd = 0.0f, u = 0.0f, ud = 0.0f;
        for (int j = 0; j < ks.n && lse > -INFINITY; ++j) {
            const float2 k = two(static_cast<const T*>(a.k) + (ks.at + j) * a.k_row + hk * a.k_head, C, lane);
            const float2 v = two(static_cast<const T*>(a.v) + (ks.at + j) * a.v_row + hk * a.v_head, C, lane);
            const Score s = score(a, wave_sum(q.x * k.x + q.y * k.y), distance(a, b, i, j), slope);
            if (s.w == -INFINITY) continue;
            const float p = exp2f(s.w - lse), gp = wave_sum(go.x * v.x + go.y * v.y);
            const float w = p * (gp - D), t = w * s.slack * a.scale;
            gx += t * k.x;
            gy += t * k.y;
            pd += p * s.d;
            u += w;
            ud += w * s.d;
        }
        put(gq + o * C, C, lane, gx, gy);
        if (lane == 0) {
            dots[o] = D;
            slopes[o] = u * pd - ud;   // D stands on the rounded out: what is left of sum w corrects it
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kWave) attention_bwd_kv_kernel(Args a, const float* dots) {
    const int lane = threadIdx.x, b = blockIdx.x, hk = blockIdx.z, C = a.channels;
    const int at = (blockIdx.z * gridDim.y + blockIdx.y) * kWave + lane, step = gridDim.y * gridDim.z * kWave;
    T *gk = static_cast<T*>(a.grad_k), *gv = static_cast<T*>(a.grad_v);
    if (b == a.num_graphs) {
        zero_rest(gk, a.k_ptr, b, a.num_nodes, (int64_t)a.kv_heads * C, at, step);
        zero_rest(gv, a.k_ptr, b, a.num_nodes, (int64_t)a.kv_heads * C, at, step);
        return;
    }
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int G = a.heads / a.kv_heads;
    for (int j = blockIdx.y; j < ks.n; j += gridDim.y) {
        const float2 k = two(static_cast<const T*>(a.k) + (ks.at + j) * a.k_row + hk * a.k_head, C, lane);
        const float2 v = two(static_cast<const T*>(a.v) + (ks.at + j) * a.v_row + hk * a.v_head, C, lane);
        float kx = 0.0f, ky = 0.0f, vx = 0.0f, vy = 0.0f;
        for (int i = 0; i < qs.n; ++i) {
            const float d = distance(a, b, i, j);
            if (!finite(d)) continue;
            for (int h = hk * G; h < hk * G + G; ++h) {
                const int64_t row = qs.at + i, o = row * a.heads + h;
                const float lse = a.lse[o];
                const float2 q = two(static_cast<const T*>(a.q) + row * a.q_row + h * a.q_head, C, lane);
                const float2 go = two(static_cast<const T*>(a.grad_out) + o * C, C, lane);
                const Score s = score(a, wave_sum(q.x * k.x + q.y * k.y), d, a.slope ? a.slope[h] : 0.0f);
                if (s.w == -INFINITY || lse == -INFINITY) continue;
                const float p = exp2f(s.w - lse), gp = wave_sum(go.x * v.x + go.y * v.y);
                const float t = p * (gp - dots[o]) * s.slack * a.scale;
                kx += t * q.x;
                ky += t * q.y;
                vx += p * go.x;
                vy += p * go.y;
            }
        }
        const int64_t o = (ks.at + j) * a.kv_heads + hk;
        put(gk + o * C, C, lane, kx, ky);
        put(gv + o * C, C, lane, vx, vy);
    }
}

// grad_slope[h] = the sum of its column, in a fixed order: 16 waves over the rows, lanes over their rows
__global__ void __launch_bounds__(kWave * 16) slope_sum_kernel(const float* slopes, int64_t rows, int heads, float* out) {
    __shared__ float part[16];
    const int h = blockIdx.x, lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
    float v = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += kWave * 16) v += slopes[r * heads + h];
    v = wave_sum(v);
    if (lane == 0) part[w] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) v += part[k];
        out[h] = v;
    }
}

unsigned rows_of(int64_t most, int64_t rows) {
    const int64_t n = most < rows ? most : rows;
    return (unsigned)(n < 1 ? 1 : n > 4096 ? 4096 : n);
}

}  // namespace

size_t node_attention_workspace(const trx_node_attention_args& a, bool backward) {
    return backward ? (size_t)a.num_queries * a.heads * 2 * sizeof(float) : 0;
}

hipError_t launch_node_attention_fwd(const trx_node_attention_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const dim3 grid(a.num_graphs + 1, rows_of(a.max_queries, a.num_queries), a.heads);
        hipLaunchKernelGGL(attention_fwd_kernel<T>, grid, dim3(kWave), 0, stream, a);
        return hipGetLastError();
    });
}

hipError_t launch_node_attention_bwd(const trx_node_attention_args& a, hipStream_t stream) {
    float *dots = static_cast<float*>(a.workspace), *slopes = dots + a.num_queries * a.heads;
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a.num_queries > 0) {
            const dim3 grid(a.num_graphs + 1, rows_of(a.max_queries, a.num_queries), a.heads);
            hipLaunchKernelGGL(attention_bwd_q_kernel<T>, grid, dim3(kWave), 0, stream, a, dots, slopes);
        }
        if (a.num_nodes > 0) {
            const dim3 grid(a.num_graphs + 1, rows_of(a.max_nodes, a.num_nodes), a.kv_heads);
            hipLaunchKernelGGL(attention_bwd_kv_kernel<T>, grid, dim3(kWave), 0, stream, a, dots);
        }
        if (a.grad_slope)
            hipLaunchKernelGGL(slope_sum_kernel, dim3(a.heads), dim3(kWave * 16), 0, stream, slopes, a.num_queries,
                               a.heads, a.grad_slope);
        return hipGetLastError();
    });
}

}  // namespace trx
