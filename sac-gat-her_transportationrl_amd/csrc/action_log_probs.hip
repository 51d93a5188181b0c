// action_log_probs.hip -- the masked categorical policy over each row's links:
// log probability of a given action, entropy and the best alternatives, with
// the gradient for the logits (include/trafficrl.h, trx_action_log_probs_*).
//
// With m = max x, s = sum e^(x - m) and t = sum e^(x - m) (x - m) over the links
// that may be chosen: log p_j = x_j - m - log s and entropy = log s - t / s.
// One read of the logits forward, one read and one write backward: rows of up
// to 1024 links stay in one wave's registers, longer ones pass through a
// workgroup's in chunks, split over several workgroups where there are few rows.
// Ranking compares whole numbers made of the logit's bits and the link, so ties
// go to the lower link whatever the order of anything.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "float_types.h"
#include "trx_internal.h"

namespace trx {
namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4;
constexpr float kLog2e = 1.44269504088896340736f;
using Args = trx_action_log_probs_args;

#define TRX_DPP(v, ctrl) __builtin_amdgcn_update_dpp(0, (int)(v), ctrl, 0xf, 0xf, false)
__device__ __forceinline__ float wave_sum(float v) {
    v += __int_as_float(TRX_DPP(__float_as_int(v), 0xB1));
    v += __int_as_float(TRX_DPP(__float_as_int(v), 0x4E));
    v += __int_as_float(TRX_DPP(__float_as_int(v), 0x141));
    v += __int_as_float(TRX_DPP(__float_as_int(v), 0x140));
    auto at = [&](int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); };
    return (at(0) + at(16)) + (at(32) + at(48));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = max(v, (uint32_t)TRX_DPP(v, 0xB1));
    v = max(v, (uint32_t)TRX_DPP(v, 0x4E));
    v = max(v, (uint32_t)TRX_DPP(v, 0x141));
    v = max(v, (uint32_t)TRX_DPP(v, 0x140));
    auto at = [&](int l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, l); };
    return max(max(at(0), at(16)), max(at(32), at(48)));
}
#undef TRX_DPP
// the largest of the lanes' keys
__device__ __forceinline__ uint64_t wave_max(uint64_t key) {
    const uint32_t high = (uint32_t)(key >> 32), top = wave_max(high);
    return ((uint64_t)top << 32) | wave_max(high == top ? (uint32_t)key : 0u);
}

// Whole numbers in the floats' order; 0 for -inf, NaN above +inf, the two zeros alike.
__device__ __forceinline__ uint32_t order_of(float x) {
    if (x == -INFINITY) return 0;
    uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
    if (x != x) u = 0x7fffffffu;
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Ranking keys: larger logits first, then lower links; 0 ranks nothing.
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t link) {
    const uint32_t o = order_of(x);
    return o ? ((uint64_t)o << 32) | (uint32_t)~link : 0;
}
__device__ __forceinline__ uint32_t key_link(uint64_t key) { return ~(uint32_t)key; }
__device__ __forceinline__ float key_logit(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

struct Row {
    int64_t at, len, mask_at;
};
__device__ __forceinline__ Row find_row(const Args& a, int64_t r) {
    if (!a.row_ptr) return {r * a.row_stride, a.row_len, r * a.mask_stride};
    int64_t lo = a.row_ptr[r], hi = a.row_ptr[r + 1];
    lo = lo < 0 ? 0 : lo > a.total ? a.total : lo;
    hi = hi < lo ? lo : hi > a.total ? a.total : hi;
    return {lo, hi - lo, lo};
}
__device__ __forceinline__ bool may_choose(const Args& a, int64_t at) {
    if (!a.mask) return true;
    return a.mask_dtype == 0 ? static_cast<const float*>(a.mask)[at] > 0.0f
                             : static_cast<const uint8_t*>(a.mask)[at] != 0;
}
// link j's logit, -inf where it may not be chosen
template <typename T>
__device__ __forceinline__ float logit(const Args& a, const Row& row, int64_t j) {
    return may_choose(a, row.mask_at + j) ? (float)static_cast<const T*>(a.logits)[row.at + j] : -INFINITY;
}
// eight consecutive ones from j on, at whatever alignment the row has; -inf behind the row's end
template <typename T>
__device__ __forceinline__ void logits8(const Args& a, const Row& row, int64_t j, float (&x)[8]) {
    if (j + 8 > row.len) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = j + e < row.len ? logit<T>(a, row, j + e) : -INFINITY;
        return;
    }
    typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
    const vec v = *reinterpret_cast<const vec*>(static_cast<const T*>(a.logits) + row.at + j);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
    if (!a.mask) return;
    if (a.mask_dtype == 0) {
        typedef float fvec __attribute__((ext_vector_type(8), aligned(4)));
        const fvec k = *reinterpret_cast<const fvec*>(static_cast<const float*>(a.mask) + row.mask_at + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = k[e] > 0.0f ? x[e] : -INFINITY;
    } else {
        typedef uint8_t bvec __attribute__((ext_vector_type(8), aligned(1)));
        const bvec k = *reinterpret_cast<const bvec*>(static_cast<const uint8_t*>(a.mask) + row.mask_at + j);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = k[e] != 0 ? x[e] : -INFINITY;
    }
}

// max, sum and first moment of some of a row's links; m = -inf: none
struct Stats {
    float m, s, t;
};
__device__ __forceinline__ void add(Stats& x, float v, float m) {
    const float d = v - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
    x.s += e;
    x.t = __builtin_fmaf(e, fmaxf(d, -1e30f), x.t);   // where e is 0, d may be -inf
}
__device__ __forceinline__ Stats joined(const Stats& x, const Stats& y) {
    if (x.m == -INFINITY && x.s == 0.0f) return y;
    if (y.m == -INFINITY && y.s == 0.0f) return x;
    const float m = fmaxf(x.m, y.m), dx = x.m - m, dy = y.m - m, fx = expf(dx), fy = expf(dy);
    return {m, x.s * fx + y.s * fy,
            fx * __builtin_fmaf(x.s, fmaxf(dx, -1e30f), x.t) + fy * __builtin_fmaf(y.s, fmaxf(dy, -1e30f), y.t)};
}

// a row's results from its statistics; one lane
template <typename T>
__device__ __forceinline__ void put_stats(const Args& a, const Row& row, int64_t r, const Stats& x) {
    const bool none = x.m == -INFINITY && x.s == 0.0f;
    const float m = none ? 0.0f : x.m, ls = none ? 0.0f : logf(x.s), entropy = none ? 0.0f : ls - x.t / x.s;
    const int64_t act = a.action[r];
    const float v = act >= 0 && act < row.len ? logit<T>(a, row, act) : -INFINITY;
    a.log_prob[r] = v != -INFINITY ? v - m - ls : -INFINITY;
    a.entropy[r] = entropy;
    float* st = a.stats + 4 * r;
    st[0] = m;
    st[1] = ls;
    st[2] = entropy;
    st[3] = v != -INFINITY ? 1.0f : 0.0f;
}
__device__ __forceinline__ void put_top(const Args& a, int64_t r, int k, uint64_t key, const Stats& x) {
    a.top_log_prob[r * a.top_k + k] = key ? key_logit(key) - x.m - logf(x.s) : -INFINITY;
    a.top_action[r * a.top_k + k] = key ? (int64_t)key_link(key) : -1;
}

// A row too long for the wave's registers (its length was not announced): passes over memory.
template <typename T>
__device__ __forceinline__ void long_row(const Args& a, const Row& row, int64_t r, int lane) {
    float m = -INFINITY;
    for (int64_t j = lane; j < row.len; j += kWave) m = fmaxf(m, logit<T>(a, row, j));
    uint64_t key = ~0ull;
    const uint32_t top = wave_max(order_of(m));
    Stats x{top ? key_logit((uint64_t)top << 32) : -INFINITY, 0.0f, 0.0f};
    for (int64_t j = lane; j < row.len; j += kWave) {
        const float v = logit<T>(a, row, j);
        if (v != -INFINITY) add(x, v, x.m == -INFINITY ? 0.0f : x.m);
    }
    x.s = wave_sum(x.s);
    x.t = wave_sum(x.t);
    for (int k = 0; k < a.top_k; ++k) {
        uint64_t next = 0;
        for (int64_t j = lane; j < row.len && key; j += kWave) {
            const uint64_t u = rank_key(logit<T>(a, row, j), (uint32_t)j);
            if (u < key && u > next) next = u;
        }
        key = wave_max(next);
        if (lane == 0) put_top(a, r, k, key, x);
    }
    if (lane == 0) put_stats<T>(a, row, r, x);
}

// one wave to a row of up to 64 V links
template <typename T, int V>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_short_kernel(Args a) {
    const int lane = threadIdx.x % kWave;
    const int64_t r = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (r >= a.rows) return;
    const Row row = find_row(a, r);
    if (row.len > kWave * V) return long_row<T>(a, row, r, lane);
    const int n = (int)row.len;
    float x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = lane + kWave * i < n ? logit<T>(a, row, lane + kWave * i) : -INFINITY;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) m = fmaxf(m, x[i]);
    const uint32_t top = wave_max(order_of(m));
    Stats st{top ? key_logit((uint64_t)top << 32) : -INFINITY, 0.0f, 0.0f};
    const float base = top ? st.m : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) add(st, x[i], base);
    st.s = wave_sum(st.s);
    st.t = wave_sum(st.t);
    if (lane == 0) put_stats<T>(a, row, r, st);
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top_k; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint64_t key = rank_key(x[i], lane + kWave * i);
            if (key < last && key > best) best = key;
        }
        last = wave_max(best);
        if (lane == 0) put_top(a, r, k, last, st);
    }
}

// Longer rows: a workgroup holds kChunk links at a time, 32 a thread.
constexpr int kEach = 4, kThreads = kWave * kWaves, kChunk = kThreads * 8 * kEach, kRoom = 64;

struct Parts {
    float4* stats;     // [rows, slots]: m, s, t
    uint64_t* keys;    // [rows, slots, top_k]
};
__device__ __forceinline__ Parts parts_of(const Args& a, int slots) {
    float4* s = static_cast<float4*>(a.workspace);
    return {s, reinterpret_cast<uint64_t*>(s + a.rows * slots)};
}

// The alternatives are found by value first: the top_k-th largest of the lanes' own maxima is a bound that at least
// top_k of the wave's logits reach, and few others do, so one comparison a logit leaves a short list in LDS.  Where
// many tie at the bound, or a NaN ranks, the wave takes its top_k one after the other from its registers instead.
template <typename T>
__global__ void __launch_bounds__(kThreads) log_probs_long_kernel(Args a, int slots) {
    __shared__ uint64_t listed[kWaves][kRoom], kept[TRX_TOP_MAX];
    __shared__ float red[3][kWaves];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const int64_t r = blockIdx.x;
    const Row row = find_row(a, r);
    Stats all{-INFINITY, 0.0f, 0.0f};
    if (threadIdx.x < TRX_TOP_MAX) kept[threadIdx.x] = 0;
    for (int64_t j0 = (int64_t)blockIdx.y * kChunk; j0 < row.len; j0 += (int64_t)slots * kChunk) {
        float x[kEach][8];
#pragma unroll
        for (int i = 0; i < kEach; ++i) logits8<T>(a, row, j0 + 8 * (threadIdx.x + kThreads * i), x[i]);
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) m = fmaxf(m, x[i][e]);
        const uint32_t mine = order_of(m), wave_top = wave_max(mine);
        const float base = wave_top ? key_logit((uint64_t)wave_top << 32) : 0.0f;
        Stats st{wave_top ? base : -INFINITY, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < kEach; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) add(st, x[i][e], base);
        st.s = wave_sum(st.s);
        st.t = wave_sum(st.t);
        if (a.top_k > 0) {
            uint32_t left = mine, bound = 0;
            for (int k = 0; k < a.top_k; ++k) {
                bound = wave_max(left);
                if (!bound) break;
                // one lane of the maximum is done with
                const uint64_t who = __ballot(left == bound);
                if (lane == __ffsll((unsigned long long)who) - 1) left = 0;
            }
            int count = 0;
            bool fits = st.s == st.s;   // a NaN: by keys
            if (fits && wave_top) {
                const float limit = bound ? key_logit((uint64_t)bound << 32) : -INFINITY;
#pragma unroll
                for (int i = 0; i < kEach; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const bool in = x[i][e] >= limit && x[i][e] > -INFINITY;
                        const uint64_t who = __ballot(in);
                        if (who) {
                            const int at = count + __popcll(who & ((1ull << lane) - 1));
                            if (in && at < kRoom)
                                listed[w][at] = rank_key(x[i][e], (uint32_t)(j0 + 8 * (threadIdx.x + kThreads * i) + e));
                            count += __popcll(who);
                        }
                    }
                fits = count <= kRoom;
            }
            if (!fits) {
                uint64_t last = ~0ull;
                count = 0;
                for (int k = 0; k < a.top_k && last; ++k) {
                    uint64_t best = 0;
#pragma unroll
                    for (int i = 0; i < kEach; ++i)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const uint64_t key = rank_key(x[i][e], (uint32_t)(j0 + 8 * (threadIdx.x + kThreads * i) + e));
                            if (key < last && key > best) best = key;
                        }
                    last = wave_max(best);
                    if (last) {
                        if (lane == 0) listed[w][k] = last;
                        count = k + 1;
                    }
                }
            }
            if (lane >= count) listed[w][lane] = 0;
        }
        if (lane == 0) {
            red[0][w] = st.m;
            red[1][w] = st.s;
            red[2][w] = st.t;
        }
        __syncthreads();
        // every thread of wave 0 joins the waves' statistics; their lists and what was kept so far become top_k again
        if (w == 0) {
#pragma unroll
            for (int v = 0; v < kWaves; ++v) all = joined(all, Stats{red[0][v], red[1][v], red[2][v]});
            if (a.top_k > 0) {
                uint64_t key[kWaves + 1];
#pragma unroll
                for (int v = 0; v < kWaves; ++v) key[v] = listed[v][lane];
                key[kWaves] = lane < TRX_TOP_MAX ? kept[lane] : 0;
                uint64_t last = ~0ull, mine_kept = 0;
                for (int k = 0; k < a.top_k; ++k) {
                    uint64_t best = 0;
#pragma unroll
                    for (int v = 0; v <= kWaves; ++v)
                        if (key[v] < last && key[v] > best) best = key[v];
                    last = wave_max(best);
                    if (lane == k) mine_kept = last;
                }
                if (lane < TRX_TOP_MAX) kept[lane] = lane < a.top_k ? mine_kept : 0;
            }
        }
        __syncthreads();
    }
    if (w != 0) return;
    if (slots == 1) {
        if (lane < a.top_k) put_top(a, r, lane, kept[lane], all);
        if (lane == 0) put_stats<T>(a, row, r, all);
    } else {
        const Parts p = parts_of(a, slots);
        const int64_t at = r * slots + blockIdx.y;
        if (lane == 0) p.stats[at] = make_float4(all.m, all.s, all.t, 0.0f);
        if (lane < a.top_k) p.keys[at * a.top_k + lane] = kept[lane];
    }
}

// one wave to a row: its slots' statistics in their order, their sorted alternatives merged
template <typename T>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_join_kernel(Args a, int slots) {
    const int lane = threadIdx.x % kWave;
    const int64_t r = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (r >= a.rows) return;
    const Parts p = parts_of(a, slots);
    Stats x{-INFINITY, 0.0f, 0.0f};
    for (int s = 0; s < slots; ++s) {
        const float4 v = p.stats[r * slots + s];
        x = joined(x, Stats{v.x, v.y, v.z});
    }
    uint64_t last = ~0ull;
    for (int k = 0; k < a.top_k; ++k) {
        uint64_t best = 0;
        for (int i = lane; i < slots * a.top_k; i += kWave) {
            const uint64_t key = p.keys[r * slots * a.top_k + i];
            if (key < last && key > best) best = key;
        }
        last = wave_max(best);
        if (lane == 0) put_top(a, r, k, last, x);
    }
    if (lane == 0) put_stats<T>(a, find_row(a, r), r, x);
}

// ---------------------------------------------------------------- backward
// What a row's gradient needs.  Lane 0 holds the action and its incoming gradient, lanes 1 .. top_k the alternatives
// and theirs (link -1: none): the links that get more than their share of the sums.
struct Grad {
    float norm, entropy, all, g2;   // m + log s, the entropy, the sum of the incoming log probability gradients
    int64_t link;
    float extra;
};
__device__ __forceinline__ Grad grad_of(const Args& a, int64_t r, int lane) {
    const float* st = a.stats + 4 * r;
    Grad g;
    g.entropy = st[2];
    g.norm = st[0] + st[1];
    g.g2 = a.g_entropy ? a.g_entropy[r] : 0.0f;
    g.link = -1;
    g.extra = 0.0f;
    if (lane == 0 && a.g_log_prob && st[3] != 0.0f) {
        g.link = a.action[r];
        g.extra = a.g_log_prob[r];
    } else if (lane > 0 && lane <= a.top_k && a.g_top) {
        g.link = a.top_action[r * a.top_k + lane - 1];
        g.extra = g.link >= 0 ? a.g_top[r * a.top_k + lane - 1] : 0.0f;
    }
    g.all = wave_sum(g.extra);
    return g;
}
__device__ __forceinline__ float base_grad(const Grad& g, float x) {
    const float lp = x - g.norm, p = __builtin_amdgcn_exp2f(lp * kLog2e);
    // where p is 0, lp may be -inf; a link that may not be chosen gets 0 in a row of NaN too
    const float d = -p * __builtin_fmaf(g.g2, fmaxf(lp, -1e30f) + g.entropy, g.all);
    return x == -INFINITY ? 0.0f : d;
}

// packed elements before the first and behind the last row
template <typename T>
__device__ __forceinline__ void zero_rest(const Args& a, int64_t at, int64_t step) {
    if (!a.row_ptr) return;
    int64_t begin = 0, end = 0;
    if (a.rows > 0) {
        const Row first = find_row(a, 0), last = find_row(a, a.rows - 1);
        begin = first.at;
        end = last.at + last.len;
    }
    T* grad = static_cast<T*>(a.grad_logits);
    for (int64_t j = at; j < begin; j += step) grad[j] = (T)0.0f;
    for (int64_t j = end + at; j < a.total; j += step) grad[j] = (T)0.0f;
}

// one wave to a row, a link a lane
template <typename T>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_short_bwd_kernel(Args a, int blocks) {
    const int lane = threadIdx.x % kWave;
    if ((int)blockIdx.x >= blocks)
        return zero_rest<T>(a, (int64_t)(blockIdx.x - blocks) * kThreads + threadIdx.x,
                            (int64_t)(gridDim.x - blocks) * kThreads);
    const int64_t r = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (r >= a.rows) return;
    const Row row = find_row(a, r);
    const Grad g = grad_of(a, r, lane);
    T* grad = static_cast<T*>(a.grad_logits) + (a.row_ptr ? row.at : r * a.row_len);
    for (int64_t j0 = 0; j0 < row.len; j0 += kWave) {
        const int64_t j = j0 + lane;
        float d = j < row.len ? base_grad(g, logit<T>(a, row, j)) : 0.0f;
        uint64_t who = __ballot(g.link >= j0 && g.link < j0 + kWave);
        while (who) {
            const int l = __ffsll((unsigned long long)who) - 1;
            who &= who - 1;
            const int at = __builtin_amdgcn_readlane((int)(g.link - j0), l);
            const float extra = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g.extra), l));
            d += lane == at ? extra : 0.0f;
        }
        if (j < row.len) grad[j] = (T)d;
    }
}

// a workgroup to a chunk of a row, eight links a lane at a time
template <typename T>
__global__ void __launch_bounds__(kThreads) log_probs_long_bwd_kernel(Args a) {
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    if ((int64_t)blockIdx.x >= a.rows)
        return zero_rest<T>(a, (int64_t)blockIdx.y * kThreads + threadIdx.x, (int64_t)gridDim.y * kThreads);
    const int64_t r = blockIdx.x;
    const Row row = find_row(a, r);
    if ((int64_t)blockIdx.y * kChunk >= row.len) return;
    const Grad g = grad_of(a, r, lane);
    T* grad = static_cast<T*>(a.grad_logits) + (a.row_ptr ? row.at : r * a.row_len);
    for (int64_t c0 = (int64_t)blockIdx.y * kChunk; c0 < row.len; c0 += (int64_t)gridDim.y * kChunk) {
        float x[kEach][8];
#pragma unroll
        for (int i = 0; i < kEach; ++i) logits8<T>(a, row, c0 + 8 * (threadIdx.x + kThreads * i), x[i]);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int64_t j0 = c0 + 8 * (kWave * w + kThreads * i), j = j0 + 8 * lane;   // this wave's 512 links
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = base_grad(g, x[i][e]);
            uint64_t who = __ballot(g.link >= j0 && g.link < j0 + 8 * kWave);
            while (who) {
                const int l = __ffsll((unsigned long long)who) - 1;
                who &= who - 1;
                const int at = __builtin_amdgcn_readlane((int)(g.link - j0), l);
                const float extra = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(g.extra), l));
#pragma unroll
                for (int e = 0; e < 8; ++e) x[i][e] += 8 * lane + e == at ? extra : 0.0f;
            }
            if (j + 8 <= row.len) {
                typedef T vec __attribute__((ext_vector_type(8), aligned(sizeof(T))));
                vec v;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = (T)x[i][e];
                *reinterpret_cast<vec*>(grad + j) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (j + e < row.len) grad[j + e] = (T)x[i][e];
            }
        }
    }
}

// up to here one wave holds a row: 16 links a lane
constexpr int kShort = 16 * kWave;

int64_t longest(const Args& a) { return a.row_ptr ? a.max_row : a.row_len; }
// workgroups to a long row: as many as fill the chip four times, but no more than it has chunks
int slots_of(const Args& a) {
    const int64_t chunks = (longest(a) + kChunk - 1) / kChunk, want = (1024 + a.rows - 1) / std::max<int64_t>(1, a.rows);
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min(chunks, want), 1024));
}

}  // namespace

size_t action_log_probs_workspace(const trx_action_log_probs_args& a) {
    if (longest(a) <= kShort) return 0;
    const int slots = slots_of(a);
    return slots > 1 ? (size_t)a.rows * slots * (sizeof(float4) + a.top_k * sizeof(uint64_t)) : 0;
}

hipError_t launch_action_log_probs_fwd(const trx_action_log_probs_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const int64_t n = longest(a);
        const dim3 by_four((unsigned)((a.rows + kWaves - 1) / kWaves)), block(kThreads);
        if (n <= 2 * kWave) {
            hipLaunchKernelGGL((log_probs_short_kernel<T, 2>), by_four, block, 0, stream, a);
        } else if (n <= kShort) {
            hipLaunchKernelGGL((log_probs_short_kernel<T, kShort / kWave>), by_four, block, 0, stream, a);
        } else {
            const int slots = slots_of(a);
            hipLaunchKernelGGL(log_probs_long_kernel<T>, dim3((unsigned)a.rows, slots), block, 0, stream, a, slots);
            if (slots > 1) hipLaunchKernelGGL(log_probs_join_kernel<T>, by_four, block, 0, stream, a, slots);
        }
        return hipGetLastError();
    });
}

hipError_t launch_action_log_probs_bwd(const trx_action_log_probs_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const int64_t n = longest(a);
        if (n <= kShort) {
            const int blocks = (int)((a.rows + kWaves - 1) / kWaves), rest = a.row_ptr ? 16 : 0;
            hipLaunchKernelGGL(log_probs_short_bwd_kernel<T>, dim3(blocks + rest), dim3(kThreads), 0, stream, a, blocks);
        } else {
            const unsigned chunks = (unsigned)std::min<int64_t>((n + kChunk - 1) / kChunk, 65535);
            hipLaunchKernelGGL(log_probs_long_bwd_kernel<T>, dim3((unsigned)a.rows + (a.row_ptr ? 1 : 0), chunks),
                               dim3(kThreads), 0, stream, a);
        }
        return hipGetLastError();
    });
}

}  // namespace trx
