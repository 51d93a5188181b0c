// action_log_probs.hip -- the masked categorical policy over each row's links:
// log probability of a given action, entropy and the best alternatives, with
// the gradient for the logits (include/trafficrl.h, trx_action_log_probs_*).
//
// With m = max x, s = sum e^(x - m) and t = sum e^(x - m) (x - m) over the links
// that may be chosen: log p_j = x_j - m - log s and entropy = log s - t / s.
// One read of the logits forward, one read and one write backward: rows pass
// through registers, of one wave where they are short, of sixteen where they are
// long, of several workgroups where there are few.
// Ranking compares whole numbers made of the logit's bits and the link, so ties
// go to the lower link whatever the order of anything.
//
// Bound by memory and vector instructions alike where rows are many and long: 2048 x
// 50000 bfloat16, called again on the same 205 MB (part of them in the last cache),
// 45 us, 12 vector instructions a link issuing in 78% of the cycles; with 8
// alternatives 81 us, 22 of them in 82%.  By latency otherwise: one row of 914 links
// with 8 alternatives 6 us, 4096 x 76 with 4 of them 8 us and 4 us back, 256 x 50001
// bfloat16 with 8 25 us and 14 us back (77 MB in all, 2.0 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>

#include "float_types.h"
#include "trx_internal.h"

namespace trx {
namespace {

constexpr int kWave = 64;
constexpr int kWaves = 4, kThreads = kWave * kWaves;
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
// the largest of the lanes' keys
__device__ __forceinline__ uint64_t wave_max(uint64_t key) {
    const uint32_t high = (uint32_t)(key >> 32), top = wave_max(high);
    return ((uint64_t)top << 32) | wave_max(high == top ? (uint32_t)key : 0u);
}

// A number that at least `count` <= 16 of the lanes reach: the least of the maxima of 16, 8 or 4 groups of lanes
__device__ __forceinline__ uint32_t reached_by(uint32_t v, int count) {
    v = max(v, (uint32_t)TRX_DPP(v, 0xB1));
    v = max(v, (uint32_t)TRX_DPP(v, 0x4E));            // 16 groups of four
    if (count <= 8) v = max(v, (uint32_t)TRX_DPP(v, 0x141));
    if (count <= 4) v = max(v, (uint32_t)TRX_DPP(v, 0x140));
    return ~wave_max(~v);
}
#undef TRX_DPP
// the lane's word for the whole wave
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
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
__device__ __forceinline__ void add(float& s, float& t, float v, float m) {
    const float d = v - m, e = __builtin_amdgcn_exp2f(d * kLog2e);
    s += e;
    t = __builtin_fmaf(e, fmaxf(d, -1e30f), t);   // where e is 0, d may be -inf
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

// Longer rows: a wave takes kPiece links at a time, two lots of eight consecutive ones a lane, and keeps running
// statistics and its best top_k.  Nothing is shared between waves until the end.
constexpr int kLots = 2, kPiece = kWave * 8 * kLots, kRoom = 64;

struct Wave {
    float m = -INFINITY;   // of the wave
    float s = 0.0f, t = 0.0f;   // of the lane, around m
    uint64_t kept = 0;     // lane k: the k-th best key
};

// The best top_k of up to 64 different keys in LDS, in order, one a lane: each lane counts the keys above its own.
__device__ __forceinline__ uint64_t ranked(uint64_t* listed, int count, int top_k, int lane) {
    __builtin_amdgcn_wave_barrier();
    const uint64_t key = lane < count ? listed[lane] : 0;
    int above = 0;
    for (int i = 0; i < count; ++i) above += from_lane(key, i) > key;
    __builtin_amdgcn_wave_barrier();
    if (lane < count && above < top_k) listed[above] = key;
    __builtin_amdgcn_wave_barrier();
    return lane < top_k && lane < count ? listed[lane] : 0;
}
// The same of N keys a lane (0: none): what reaches a bound that top_k lanes reach goes through the list; where too
// many do, top_k rounds of the wave's maximum.
template <int N>
__device__ __forceinline__ uint64_t best_of(const uint64_t (&key)[N], uint64_t* listed, int top_k, int lane) {
    uint32_t high = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) high = max(high, (uint32_t)(key[i] >> 32));
    const uint32_t bound = max(reached_by(high, top_k), 1u);
    int count = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const bool in = (uint32_t)(key[i] >> 32) >= bound;
        const uint64_t who = __ballot(in);
        const int at = count + __popcll(who & ((1ull << lane) - 1));
        if (in && at < kRoom) listed[at] = key[i];
        count += __popcll(who);
    }
    if (count <= kRoom) return ranked(listed, count, top_k, lane);
    uint64_t last = ~0ull, kept = 0;
    for (int k = 0; k < top_k; ++k) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (key[i] < last && key[i] > best) best = key[i];
        last = wave_max(best);
        if (lane == k) kept = last;
    }
    return kept;
}

// The alternatives are found by value first: of the lanes' own maxima, some bound is reached by at least top_k, and
// few other logits of the piece reach it, so one comparison a logit leaves a short list in LDS.  Where many tie at
// the bound, the wave takes its top_k one after the other from its registers instead.
template <typename T>
__device__ __forceinline__ void wave_pass(const Args& a, const Row& row, int64_t first, int64_t end, int64_t step,
                                          int lane, uint64_t* listed, Wave& w) {
    float x[kLots][8], next[kLots][8];
    auto fetch = [&](int64_t j0) {
#pragma unroll
        for (int i = 0; i < kLots; ++i) logits8<T>(a, row, j0 + 8 * (lane + kWave * i), next[i]);
    };
    if (first < end) fetch(first);
    for (int64_t j0 = first; j0 < end; j0 += step) {
#pragma unroll
        for (int i = 0; i < kLots; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = next[i][e];
        if (j0 + step < end) fetch(j0 + step);
        float mine = -INFINITY;
#pragma unroll
        for (int i = 0; i < kLots; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) mine = fmaxf(mine, x[i][e]);
        const uint32_t left = order_of(mine), top = wave_max(left);
        const float m = top ? key_logit((uint64_t)top << 32) : -INFINITY;
        if (m > w.m) {
            const float d = w.m - m, f = __builtin_amdgcn_exp2f(d * kLog2e);
            w.t = f * __builtin_fmaf(w.s, fmaxf(d, -1e30f), w.t);
            w.s *= f;
            w.m = m;
        }
        const float base = w.m == -INFINITY ? 0.0f : w.m;
#pragma unroll
        for (int i = 0; i < kLots; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) add(w.s, w.t, x[i][e], base);
        if (a.top_k == 0 || !top) continue;
        // once top_k are kept, a logit has to pass the last of them: links only grow, so a tie loses
        const uint64_t lowest = __shfl(w.kept, a.top_k - 1);
        const float limit = lowest ? key_logit(lowest) : -INFINITY;
        if (lowest && !(m > limit)) continue;
        float reach = limit;
        if (!lowest) {
            const uint32_t bound = reached_by(left, a.top_k);
            if (bound) reach = key_logit((uint64_t)bound << 32);
        }
        int count = 0;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < kLots; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const bool in = x[i][e] >= reach && x[i][e] > limit;
                const uint64_t who = __ballot(in);
                if (who) {
                    const int at = count + __popcll(who & ((1ull << lane) - 1));
                    if (in && at < kRoom) listed[at] = rank_key(x[i][e], (uint32_t)(j0 + 8 * (lane + kWave * i) + e));
                    count += __popcll(who);
                }
            }
        if (lowest && count <= a.top_k) {   // few: each goes in at its place
            __builtin_amdgcn_wave_barrier();
            const uint64_t fresh = lane < count ? listed[lane] : 0;
            for (int i = 0; i < count; ++i) {
                const uint64_t key = from_lane(fresh, i), before = __shfl_up(w.kept, 1);
                const int at = __popcll(__ballot(w.kept > key));
                if (lane >= at && lane < a.top_k) w.kept = lane == at ? key : before;
            }
        } else if (count + a.top_k <= kRoom) {
            const uint64_t old = __ballot(w.kept != 0);   // the lanes from 0 on
            if (w.kept) listed[count + lane] = w.kept;
            w.kept = ranked(listed, count + __popcll(old), a.top_k, lane);
        } else {
            const uint64_t old = w.kept;
            uint64_t last = ~0ull;
            for (int k = 0; k < a.top_k; ++k) {
                uint64_t best = old < last ? old : 0;
#pragma unroll
                for (int i = 0; i < kLots; ++i)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint64_t key = rank_key(x[i][e], (uint32_t)(j0 + 8 * (lane + kWave * i) + e));
                        if (key < last && key > best) best = key;
                    }
                last = wave_max(best);
                if (lane == k) w.kept = last;
            }
        }
    }
}

// the best top_k of some of a row's links by their keys alone, passes over memory: for rows in which a NaN ranks
template <typename T>
__device__ __forceinline__ uint64_t ranked_by_keys(const Args& a, const Row& row, int64_t first, int64_t end, int lane) {
    uint64_t kept = 0, last = ~0ull;
    for (int k = 0; k < a.top_k && last; ++k) {
        uint64_t best = 0;
        for (int64_t j = first + lane; j < end; j += kWave) {
            const uint64_t key = rank_key(logit<T>(a, row, j), (uint32_t)j);
            if (key < last && key > best) best = key;
        }
        last = wave_max(best);
        if (lane == k) kept = last;
    }
    return kept;
}

// One wave to a row.  Up to 64 V links: a link a lane at a time, all ranked by keys; more: in pieces.  At 76 links the
// pieces' eight a lane would leave five lanes of six idle.
template <typename T, int V>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_short_kernel(Args a) {
    __shared__ uint64_t listed[kWaves][kRoom];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const int64_t r = (int64_t)blockIdx.x * kWaves + w;
    if (r >= a.rows) return;
    const Row row = find_row(a, r);
    if (row.len > kWave * V) {
        Wave x;
        wave_pass<T>(a, row, 0, row.len, kPiece, lane, listed[w], x);
        const Stats st{x.m, wave_sum(x.s), wave_sum(x.t)};
        if (st.s != st.s) x.kept = ranked_by_keys<T>(a, row, 0, row.len, lane);
        if (lane < a.top_k) put_top(a, r, lane, x.kept, st);
        if (lane == 0) put_stats<T>(a, row, r, st);
        return;
    }
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
    for (int i = 0; i < V; ++i) add(st.s, st.t, x[i], base);
    st.s = wave_sum(st.s);
    st.t = wave_sum(st.t);
    if (lane == 0) put_stats<T>(a, row, r, st);
    if (a.top_k == 0) return;
    uint64_t key[V];
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = rank_key(x[i], lane + kWave * i);
    const uint64_t kept = best_of(key, listed[w], a.top_k, lane);
    if (lane < a.top_k) put_top(a, r, lane, kept, st);
}

struct Parts {
    float4* stats;     // [rows, slots]: m, s, t
    uint64_t* keys;    // [rows, slots, top_k]
};
__device__ __forceinline__ Parts parts_of(const Args& a, int slots) {
    float4* s = static_cast<float4*>(a.workspace);
    return {s, reinterpret_cast<uint64_t*>(s + a.rows * slots)};
}
// one wave: the lanes' statistics as one
__device__ __forceinline__ Stats joined(float m, float s, float t) {
    const uint32_t top = wave_max(order_of(m));
    const float all = top ? key_logit((uint64_t)top << 32) : -INFINITY, d = m == -INFINITY ? 0.0f : m - all;
    const float f = expf(d);
    return {all, wave_sum(s * f), wave_sum(f * __builtin_fmaf(s, d, t))};
}

// W waves to a row, or to one of its slots: consecutive `each` links (a multiple of kPiece)
template <typename T, int W>
__global__ void __launch_bounds__(kWave * W) log_probs_long_kernel(Args a, int slots) {
    __shared__ uint64_t listed[W][kRoom], lists[W * TRX_TOP_MAX];
    __shared__ float red[3][W];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    const int64_t r = blockIdx.x;
    const Row row = find_row(a, r);
    const int64_t each = ((row.len + kPiece - 1) / kPiece + slots - 1) / slots * kPiece;
    const int64_t first = min(row.len, blockIdx.y * each), end = min(row.len, first + each);
    Wave x;
    wave_pass<T>(a, row, first + w * kPiece, end, W * kPiece, lane, listed[w], x);
    x.s = wave_sum(x.s);
    x.t = wave_sum(x.t);
    if (lane < TRX_TOP_MAX) lists[w * TRX_TOP_MAX + lane] = lane < a.top_k ? x.kept : 0;
    if (lane == 0) {
        red[0][w] = x.m;
        red[1][w] = x.s;
        red[2][w] = x.t;
    }
    __syncthreads();
    if (w != 0) return;
    const bool has = lane < W;
    const Stats st = joined(has ? red[0][lane] : -INFINITY, has ? red[1][lane] : 0.0f, has ? red[2][lane] : 0.0f);
    if (a.top_k > 0) {
        if (st.s != st.s) {
            x.kept = ranked_by_keys<T>(a, row, first, end, lane);
        } else {
            constexpr int kLists = (W * TRX_TOP_MAX + kWave - 1) / kWave;
            uint64_t key[kLists];
#pragma unroll
            for (int i = 0; i < kLists; ++i) key[i] = lists[lane + kWave * i];
            x.kept = best_of(key, listed[0], a.top_k, lane);
        }
    }
    if (slots == 1) {
        if (lane < a.top_k) put_top(a, r, lane, x.kept, st);
        if (lane == 0) put_stats<T>(a, row, r, st);
    } else {
        const Parts p = parts_of(a, slots);
        const int64_t at = r * slots + blockIdx.y;
        if (lane == 0) p.stats[at] = make_float4(st.m, st.s, st.t, 0.0f);
        if (lane < a.top_k) p.keys[at * a.top_k + lane] = x.kept;
    }
}

// one wave to a row: the statistics of its slots (at most 64), their alternatives merged
template <typename T>
__global__ void __launch_bounds__(kWave * kWaves) log_probs_join_kernel(Args a, int slots) {
    __shared__ uint64_t listed[kWaves][kRoom];
    const int lane = threadIdx.x % kWave;
    const int64_t r = (int64_t)blockIdx.x * kWaves + threadIdx.x / kWave;
    if (r >= a.rows) return;
    const Parts p = parts_of(a, slots);
    const float4 v = lane < slots ? p.stats[r * slots + lane] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
    const Stats st = joined(v.x, v.y, v.z);
    constexpr int kLists = TRX_TOP_MAX;   // 64 slots' lists over 64 lanes
    uint64_t key[kLists], kept = 0;
#pragma unroll
    for (int i = 0; i < kLists; ++i)
        key[i] = lane + kWave * i < slots * a.top_k ? p.keys[r * slots * a.top_k + lane + kWave * i] : 0;
    if (a.top_k > 0) kept = best_of(key, listed[threadIdx.x / kWave], a.top_k, lane);
    if (lane < a.top_k) put_top(a, r, lane, kept, st);
    if (lane == 0) put_stats<T>(a, find_row(a, r), r, st);
}

// ---------------------------------------------------------------- backward
// What a row's gradient needs.  Lane 0 holds the action and its incoming gradient, lanes 1 .. top_k the alternatives
// and theirs (link -1: none): the links that get more than their share of the sums.
struct Grad {
    float m, ls, entropy, all, g2;   // m, log s, the entropy, the sum of the incoming log probability gradients
    int64_t link;
    float extra;
};
__device__ __forceinline__ Grad grad_of(const Args& a, int64_t r, int lane) {
    const float* st = a.stats + 4 * r;
    Grad g;
    g.entropy = st[2];
    g.m = st[0];
    g.ls = st[1];
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
    // in two steps as forward: m + log s in one float would lose log s where |m| is large (a row whose links all hold
    // the same -1e9 would get p = 1 for each of them)
    const float lp = x - g.m - g.ls, p = __builtin_amdgcn_exp2f(lp * kLog2e);
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

// a workgroup to kChunk links of a row at a time, four lots of eight a lane
constexpr int kEach = 4, kChunk = kThreads * 8 * kEach;
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

int64_t longest(const Args& a) { return a.row_ptr ? a.max_row : a.row_len; }

// Waves to a row: one up to 1024 links (four such rows a workgroup), four up to 8192 or where a thousand rows fill the
// chip by themselves (each wave finds its first alternatives anew, so fewer waves do less), sixteen beyond.  Rows are
// split into slots where they alone would leave compute units idle, each of at least sixteen pieces (a slot costs its
// part of the joining launch).
constexpr int kOneWave = kPiece, kFourWaves = 8 * kPiece, kManyRows = 1024;
int slots_of(const Args& a) {
    const int64_t n = longest(a), pieces = (n + kPiece - 1) / kPiece, rows = std::max<int64_t>(1, a.rows);
    if (n <= kFourWaves || rows >= kManyRows) return 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(pieces / 16, 64), 256 / rows));
}

}  // namespace

size_t action_log_probs_workspace(const trx_action_log_probs_args& a) {
    const int slots = slots_of(a);
    return slots > 1 ? (size_t)a.rows * slots * (sizeof(float4) + a.top_k * sizeof(uint64_t)) : 0;
}

hipError_t launch_action_log_probs_fwd(const trx_action_log_probs_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const int64_t n = longest(a);
        const dim3 by_four((unsigned)((a.rows + kWaves - 1) / kWaves)), by_one((unsigned)a.rows);
        const int slots = slots_of(a);
        if (n <= kOneWave) {
            hipLaunchKernelGGL((log_probs_short_kernel<T, 2>), by_four, dim3(kThreads), 0, stream, a);
        } else if (n <= kFourWaves || a.rows >= kManyRows) {
            hipLaunchKernelGGL((log_probs_long_kernel<T, 4>), by_one, dim3(kThreads), 0, stream, a, 1);
        } else {
            hipLaunchKernelGGL((log_probs_long_kernel<T, 16>), dim3((unsigned)a.rows, slots), dim3(16 * kWave), 0, stream,
                               a, slots);
            if (slots > 1) hipLaunchKernelGGL(log_probs_join_kernel<T>, by_four, dim3(kThreads), 0, stream, a, slots);
        }
        return hipGetLastError();
    });
}

hipError_t launch_action_log_probs_bwd(const trx_action_log_probs_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const int64_t n = longest(a);
        if (n <= kOneWave) {
            const int blocks = (int)((a.rows + kWaves - 1) / kWaves), rest = a.row_ptr ? 16 : 0;
            hipLaunchKernelGGL(log_probs_short_bwd_kernel<T>, dim3(blocks + rest), dim3(kThreads), 0, stream, a, blocks);
        } else {
            // packed rows may be much shorter than the longest (or than `max_row` says): about 2^15 workgroups then, which
            // loop over a row's further chunks; a chunk each would be rows x total of them (32768 rows of
            // 76, longest not given: 2747 us, 137 now, 61 where it is given).
            const int64_t most = a.row_ptr ? std::max<int64_t>(1, (1 << 15) / std::max<int64_t>(1, a.rows)) : 65535;
            const unsigned chunks = (unsigned)std::min<int64_t>((n + kChunk - 1) / kChunk, std::min<int64_t>(most, 65535));
            hipLaunchKernelGGL(log_probs_long_bwd_kernel<T>, dim3((unsigned)a.rows + (a.row_ptr ? 1 : 0), chunks),
                               dim3(kThreads), 0, stream, a);
        }
        return hipGetLastError();
    });
}

}  // namespace trx
