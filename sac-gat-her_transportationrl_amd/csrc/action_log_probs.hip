// action_log_probs.hip -- the masked categorical policy over each row's links:
// log probability of a given action, entropy and the best alternatives, with
// the gradient for the logits (include/trafficrl.h, trx_action_log_probs_*).
//
// With m = max x, s = sum e^(x - m) and t = sum e^(x - m) (x - m) over the links
// that may be chosen: log p_j = x_j - m - log s and entropy = log s - t / s.
#include <hip/hip_runtime.h>

#include "float_types.h"
#include "trx_internal.h"

namespace trx {
namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint64_t u = __shfl_xor((unsigned long long)v, o);
        v = u > v ? u : v;
    }
    return v;
}

// Ranking key: larger logits first, then lower links; 0 ranks nothing.  The
// float's bits in an order that whole numbers keep, over the link's complement.
// NaN ranks above +inf.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t link) {
    x = x == 0.0f ? 0.0f : x;   // -0 and +0 are a tie
    uint32_t u = __float_as_uint(x);
    if (x != x) u = 0x7fffffffu;
    u = u & 0x80000000u ? ~u : u | 0x80000000u;
    return ((uint64_t)u << 32) | (uint32_t)~link;
}
__device__ __forceinline__ uint32_t key_link(uint64_t key) { return ~(uint32_t)key; }
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

struct Row {
    int64_t at, len, mask_at;
};

__device__ __forceinline__ Row find_row(const trx_action_log_probs_args& a, int64_t r) {
    if (!a.row_ptr) return {r * a.row_stride, a.row_len, r * a.mask_stride};
    int64_t lo = a.row_ptr[r], hi = a.row_ptr[r + 1];
    lo = lo < 0 ? 0 : lo > a.total ? a.total : lo;
    hi = hi < lo ? lo : hi > a.total ? a.total : hi;
    return {lo, hi - lo, lo};
}

__device__ __forceinline__ bool may_choose(const trx_action_log_probs_args& a, int64_t at) {
    if (!a.mask) return true;
    return a.mask_dtype == 0 ? static_cast<const float*>(a.mask)[at] > 0.0f
                             : static_cast<const uint8_t*>(a.mask)[at] != 0;
}

template <typename T>
__device__ __forceinline__ float logit(const trx_action_log_probs_args& a, const Row& row, int64_t j) {
    return may_choose(a, row.mask_at + j) ? (float)static_cast<const T*>(a.logits)[row.at + j] : -INFINITY;
}

template <typename T>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_fwd_kernel(trx_action_log_probs_args a) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t r = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (r >= a.rows) return;
    const Row row = find_row(a, r);
    uint64_t best = 0;
    for (int64_t j = lane; j < row.len; j += kWave) {
        const float x = logit<T>(a, row, j);
        if (x != -INFINITY) {
            const uint64_t key = rank_key(x, (uint32_t)j);
            best = key > best ? key : best;
        }
    }
    best = wave_max(best);
    const float m = best ? key_logit(best) : 0.0f;
    float s = 0.0f, t = 0.0f;
    for (int64_t j = lane; j < row.len; j += kWave) {
        const float x = logit<T>(a, row, j);
        if (x != -INFINITY) {
            const float e = expf(x - m);
            s += e;
            t += e > 0.0f ? e * (x - m) : 0.0f;
        }
    }
    s = wave_sum(s);
    t = wave_sum(t);
    const float ls = best ? logf(s) : 0.0f, entropy = best ? ls - t / s : 0.0f;
    uint64_t key = best;
    for (int k = 0; k < a.top_k; ++k) {
        if (lane == 0) {
            a.top_log_prob[r * a.top_k + k] = key ? key_logit(key) - m - ls : -INFINITY;
            a.top_action[r * a.top_k + k] = key ? (int64_t)key_link(key) : -1;
        }
        uint64_t next = 0;
        for (int64_t j = lane; j < row.len && key; j += kWave) {
            const float x = logit<T>(a, row, j);
            const uint64_t u = x != -INFINITY ? rank_key(x, (uint32_t)j) : 0;
            if (u < key && u > next) next = u;
        }
        key = wave_max(next);
    }
    if (lane == 0) {
        const int64_t act = a.action[r];
        const float x = act >= 0 && act < row.len ? logit<T>(a, row, act) : -INFINITY;
        a.log_prob[r] = x != -INFINITY ? x - m - ls : -INFINITY;
        a.entropy[r] = entropy;
        float* st = a.stats + 4 * r;
        st[0] = m;
        st[1] = ls;
        st[2] = entropy;
        st[3] = x != -INFINITY ? 1.0f : 0.0f;
    }
}

template <typename T>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_bwd_kernel(trx_action_log_probs_args a) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t r = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
    T* grad = static_cast<T*>(a.grad_logits);
    if (r >= a.rows) {   // packed elements before the first and behind the last row
        if (r == a.rows && a.row_ptr) {
            int64_t begin = 0, end = 0;
            if (a.rows > 0) {
                const Row first = find_row(a, 0), last = find_row(a, a.rows - 1);
                begin = first.at;
                end = last.at + last.len;
            }
            for (int64_t j = lane; j < begin; j += kWave) grad[j] = (T)0.0f;
            for (int64_t j = end + lane; j < a.total; j += kWave) grad[j] = (T)0.0f;
        }
        return;
    }
    const Row row = find_row(a, r);
    const float* st = a.stats + 4 * r;
    const float m = st[0], ls = st[1], entropy = st[2];
    const float g1 = a.g_log_prob && st[3] != 0.0f ? a.g_log_prob[r] : 0.0f, g2 = a.g_entropy ? a.g_entropy[r] : 0.0f;
    float all = g1;
    if (a.g_top)
        for (int k = 0; k < a.top_k; ++k) all += a.top_action[r * a.top_k + k] >= 0 ? a.g_top[r * a.top_k + k] : 0.0f;
    const int64_t act = a.action[r], to = a.row_ptr ? row.at : r * a.row_len;
    for (int64_t j = lane; j < row.len; j += kWave) {
        const float x = logit<T>(a, row, j);
        float g = 0.0f;
        if (x != -INFINITY) {
            const float lp = x - m - ls, p = expf(lp);
            g = -all * p - (p > 0.0f ? g2 * p * (lp + entropy) : 0.0f);
            if (j == act) g += g1;
            if (a.g_top)
                for (int k = 0; k < a.top_k; ++k)
                    if (a.top_action[r * a.top_k + k] == j) g += a.g_top[r * a.top_k + k];
        }
        grad[to + j] = (T)g;
    }
}

}  // namespace

size_t action_log_probs_workspace(const trx_action_log_probs_args&) { return 0; }

hipError_t launch_action_log_probs_fwd(const trx_action_log_probs_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL(log_probs_fwd_kernel<T>, dim3((unsigned)((a.rows + kWaves - 1) / kWaves)),
                           dim3(kWave * kWaves), 0, stream, a);
        return hipGetLastError();
    });
}

hipError_t launch_action_log_probs_bwd(const trx_action_log_probs_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL(log_probs_bwd_kernel<T>, dim3((unsigned)((a.rows + kWaves) / kWaves)),
                           dim3(kWave * kWaves), 0, stream, a);
        return hipGetLastError();
    });
}

}  // namespace trx
