// node_attention_bwd.h -- node_attention's gradients, one element type to a
// translation unit (node_attention_{f32,bf16,f16}.hip): with p the probabilities,
// brought back from the saved lse, go the incoming gradient, gp = go v^T and D =
// <go, out> of each row,
//   t = p (gp - D);  grad_slope = -sum t d;  u = t (1 - tanh^2)
//   grad_q = scale u k;  grad_k = scale u^T q;  grad_v = p^T go.
// Two passes and no atomics: one workgroup keeps query rows and runs over the
// keys (grad_q, D, the slopes' sums), one keeps keys and runs over the query
// rows of every head that shares them (grad_k, grad_v).  Seven products where
// five would do, for results that do not depend on the order of anything.
//
// D = <grad_out, out> is subtracted from <grad_out, v>, and its error does not
// shrink with the difference.  out alone, rounded to bfloat16, leaves grad_q off by
// 0.0041 (relative to float64) where all values are shifted by 1, 0.0139 by 4,
// 0.0042 where the softmax is peaked; with out_low 0.0024 to 0.0025.  Inputs of
// mean zero gain nothing.  out_low costs 0.5 us forward and 2 us here at 4001 nodes.
//
// p and u are rounded to the type for their products, as the forward's weights are
// (float16's range is kept, see Raise).  Gradients in bfloat16 are off by 0.0024
// (relative to float64) where rounding the results alone costs 0.0017.
//
// What bounds them: as forward, vector instructions (15.0 and 15.4 a score, issuing
// in 50% and 40% of the cycles, the matrix pipe busy in 19%) and waiting (36% and 52%
// of the waves' cycles), with two waves a SIMD.  4001 nodes, 8 heads of 64, bfloat16,
// distances: 132 us (grad_q) and 154 us (grad_k, grad_v), 280 TFLOP/s of the five
// products that are needed with the sums; 4096 nodes without distances 192 us
// together with the sums (448 TFLOP/s).
#pragma once
#include <algorithm>

#include "node_attention.h"

namespace trx {
namespace {

// Per (query row, head), summed with weights around lse: their sum, which is 1 but for what rounding took from lse
// and divides everything else, and what the slope's gradient needs.  D is off by its own roundings, so sum t is not
// quite zero; what is left of it corrects sum t d: grad_slope of the row = (sum t)(sum p d) - sum t d.
struct Sums {
    float e, t, pd, td;
    __device__ __forceinline__ float inverse() const { return e == 0.0f ? 0.0f : 1.0f / e; }
    __device__ __forceinline__ float slope(float inv) const {
        return __builtin_fmaf(t * inv, pd * inv, -(td * inv));
    }
};
// where they go, for the pass over the keys and for the slopes' sums (slopes: NULL where not wanted)
struct RowSums {
    float *dots, *inverse, *slopes;
};

template <typename T, int CP, int MQ, int WAVES, int KT, bool DIST, bool CAP>
__global__ void __launch_bounds__(kWave* WAVES) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, CP, WAVES>)))
attention_bwd_q_kernel(Call call, RowSums out, float* part) {
    constexpr int kThreads = kWave * WAVES, kRows = 16 * MQ * WAVES, kSteps = CP / 32, kTiles = KT / 16;
    constexpr bool kAhead = WAVES > 1;   // one wave's registers are better spent on more waves
    constexpr bool kStageD = DIST && WAVES > 1;
    using Distances = StagedDistances<kStageD ? kRows : kTiles * 16, KT, kThreads>;
    __shared__ __attribute__((aligned(16))) float d_tile[kStageD ? kRows * Distances::kPitch : 4];
    __shared__ __attribute__((aligned(16))) T k_tile[KT * kRow<T, CP>], v_tile[KT * kRow<T, CP>];
    const Args& a = call.a;
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, c = lane % 16;
    const int G = call.group.by, C = a.channels;
    const float unit = call.unit.log2;
    T* grad_q = static_cast<T*>(a.grad_q);
    if ((int)blockIdx.x >= call.blocks) {
        if (!part) zero_rest(grad_q, a.q_ptr, a.num_graphs, a.num_queries, (int64_t)a.heads * C, blockIdx.x - call.blocks);
        return;
    }
    const Work work = work_of<DIST>(call);
    const int b = work.graph, hk = work.head, split = work.split, splits = call.splits.by;
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int rows = qs.n * G;
    int first = 0, last = ks.n;
    if (splits > 1) {
        const int each = ((ks.n + KT - 1) / KT + splits - 1) / splits * KT;
        first = min((int64_t)ks.n, (int64_t)split * each);
        last = min((int64_t)ks.n, (int64_t)first + each);
    }
    const T* k_base = static_cast<const T*>(a.k) + ks.at * a.k_row + hk * a.k_head;
    const T* v_base = static_cast<const T*>(a.v) + ks.at * a.v_row + hk * a.v_head;

    for (int tile = work.tile; (int64_t)tile * kRows < rows; tile += call.tiles) {
        const int row0 = tile * kRows + w * 16 * MQ;
        Staged<T, CP, KT, kThreads> k_next, v_next;
        auto fetch = [&](int j0) {
            k_next.load(k_base, a.k_row, j0, ks.n, C);
            v_next.load(v_base, a.v_row, j0, ks.n, C);
        };
        if (kAhead && first < last) fetch(first);
        frag<T> q[MQ][kSteps], go[MQ][kSteps];
        const float* dist[MQ];
        Around ref[MQ];
        bool far[MQ];
        float slope[MQ], D[MQ];
        int limit[MQ];
        Sums sums[MQ];
        f32x4 acc[MQ][CP / 16];
        Raise raise[MQ];
#pragma unroll
        for (int t = 0; t < MQ; ++t) {
            const int row = min(row0 + 16 * t + c, rows - 1);
            const int i = call.group(row), h = hk * G + (row - i * G);
            const int64_t at = (qs.at + i) * a.heads + h;
            const T* p = static_cast<const T*>(a.q) + (qs.at + i) * a.q_row + h * a.q_head;
            const T *po = static_cast<const T*>(a.out) + at * C, *pg = static_cast<const T*>(a.grad_out) + at * C;
            const T* pl = a.out_low ? static_cast<const T*>(a.out_low) + at * C : nullptr;
            float dot = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const bool in = 32 * s + 8 * g < C;
                q[t][s] = in ? load_frag(p + 32 * s + 8 * g) : zero_frag<T>();
                go[t][s] = in ? load_frag(pg + 32 * s + 8 * g) : zero_frag<T>();
                const frag<T> o = in ? load_frag(po + 32 * s + 8 * g) : zero_frag<T>();
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = __builtin_fmaf((float)go[t][s][e], (float)o[e], dot);
                if (pl && in) {   // what rounding took from out: else D's error would be as large as all others' together
                    const frag<T> low = load_frag(pl + 32 * s + 8 * g);
#pragma unroll
                    for (int e = 0; e < 8; ++e) dot = __builtin_fmaf((float)go[t][s][e], (float)low[e], dot);
                }
            }
            D[t] = column_sum(dot);
            slope[t] = DIST && a.slope ? -a.slope[h] : 0.0f;
            if (DIST && !kStageD) {
                dist[t] = a.dist + b * a.dist_graph + i * a.dist_row;
                limit[t] = i < a.dist_rows ? min(ks.n, a.dist_cols) : 0;
            }
            const float lse = a.lse[at];   // an empty row: every weight comes out as zero
            ref[t] = around(lse == -INFINITY ? INFINITY : lse * call.unit.per, unit);
            far[t] = __any(ref[t].far(kFarBack<T>));
            if (split == 0 && g == 0 && row0 + 16 * t + c < rows) out.dots[at] = D[t];
            sums[t] = {0.0f, 0.0f, 0.0f, 0.0f};
            raise[t] = {kRaiseAll};
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) acc[t][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        const float* graph = DIST ? a.dist + b * a.dist_graph : nullptr;
        Distances d_next;
        int d_row[MQ];
        if (kStageD && first < last) d_next.load(call, graph, tile * kRows, rows, ks.n, first);
#pragma unroll
        for (int t = 0; t < MQ; ++t) d_row[t] = min(w * 16 * MQ + 16 * t + c + d_next.shift, kRows - 1) * Distances::kPitch;
        for (int j0 = first; j0 < last; j0 += KT) {
            f32x4 d[MQ][kTiles];
            if (!kAhead) fetch(j0);
            if (DIST && !kStageD) {
#pragma unroll
                for (int t = 0; t < MQ; ++t) {
                    const bool whole = __all(j0 + KT <= limit[t]);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) d[t][n] = distances(dist[t], j0 + 16 * n + 4 * g, limit[t], whole);
                }
            }
            __syncthreads();
            k_next.store(k_tile);
            v_next.store(v_tile);
            if (kStageD) d_next.store(d_tile);
            __syncthreads();
            if (kAhead && j0 + KT < last) {
                fetch(j0 + KT);
                if (kStageD) d_next.load(call, graph, tile * kRows, rows, ks.n, j0 + KT);
            }
            if (row0 >= rows) continue;
            f32x4 s[MQ][kTiles], gp[MQ][kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                for (int t = 0; t < MQ; ++t) s[t][n] = gp[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const frag<T> f = load_frag(k_tile + (16 * n + c) * kRow<T, CP> + 32 * x + 8 * g);
#pragma unroll
                    for (int t = 0; t < MQ; ++t) s[t][n] = mma(f, q[t][x], s[t][n]);
                }
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const frag<T> f = load_frag(v_tile + (16 * n + c) * kRow<T, CP> + 32 * x + 8 * g);
#pragma unroll
                    for (int t = 0; t < MQ; ++t) gp[t][n] = mma(f, go[t][x], gp[t][n]);
                }
            }
            frag<T> u[MQ][KT / 32];
#pragma unroll
            for (int t = 0; t < MQ; ++t) {
                if (kStageD) {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
                        d[t][n] = *reinterpret_cast<const f32x4*>(d_tile + d_row[t] + 16 * n + 4 * g);
                }
                f32x4 slack[kTiles];
                scores<T, CAP, true>(call, s[t], slack, far[t]);
                if (DIST) {
                    // beside weights of zero a distance must not be infinite in the slopes' sums
                    if (__all(slope[t] < 0.0f) && ordinary(d[t])) {
                        TRX_EACH_SCORE s[t][n][r] = __builtin_fmaf(slope[t], d[t][n][r], s[t][n][r]);
                        if (out.slopes) TRX_EACH_SCORE d[t][n][r] = fminf(d[t][n][r], 3.402823466e38f);
                    } else {
                        TRX_EACH_SCORE {
                            const bool seen = finite(d[t][n][r]);
                            s[t][n][r] = seen ? __builtin_fmaf(slope[t], d[t][n][r], s[t][n][r]) : -INFINITY;
                            d[t][n][r] = seen ? d[t][n][r] : 0.0f;
                        }
                    }
                } else if (j0 + KT > last) {
                    TRX_EACH_SCORE if (j0 + 16 * n + 4 * g + r >= last) s[t][n][r] = -INFINITY;
                }
                float minus = -ref[t].c;
                if (far[t]) {   // a weight is at most 1: a score rounded otherwise than in the forward must not pass it
                    TRX_EACH_SCORE s[t][n][r] = fminf(s[t][n][r] - ref[t].at, 0.0f);
                    minus = ref[t].add(unit, kFarBack<T>);
                }
                TRX_EACH_SCORE {
                    const float e = exp2_fast(__builtin_fmaf(s[t][n][r], unit, minus));
                    s[t][n][r] = e;
                    sums[t].e += e;
                    gp[t][n][r] = e * (gp[t][n][r] - D[t]);
                }
                if (DIST && out.slopes) {
                    TRX_EACH_SCORE {
                        sums[t].t += gp[t][n][r];
                        sums[t].pd = __builtin_fmaf(s[t][n][r], d[t][n][r], sums[t].pd);
                        sums[t].td = __builtin_fmaf(gp[t][n][r], d[t][n][r], sums[t].td);
                    }
                }
                // rounded to the type for the product with k
                if (CAP) TRX_EACH_SCORE gp[t][n][r] *= slack[n][r];
                if constexpr (kHalf<T>) {
                    float most = 0.0f;
                    TRX_EACH_SCORE most = fmaxf(most, fabsf(gp[t][n][r]));
                    raise[t].over(most, acc[t]);
                    TRX_EACH_SCORE gp[t][n][r] *= raise[t].by;
                }
                TRX_EACH_SCORE u[t][n / 2][4 * (n % 2) + r] = (T)gp[t][n][r];
            }
#pragma unroll
            for (int x = 0; x < CP / 16; ++x)
#pragma unroll
                for (int y = 0; y < KT / 32; ++y) {
                    const frag<T> f = turned<T, CP>(k_tile, 32 * y, 32 * y + 16, 16 * x, lane);
#pragma unroll
                    for (int t = 0; t < MQ; ++t) acc[t][x] = mma(f, u[t][y], acc[t][x]);
                }
        }
#pragma unroll
        for (int t = 0; t < MQ; ++t) {
            const int row = row0 + 16 * t + c;
            Sums sum{column_sum(sums[t].e), 0.0f, 0.0f, 0.0f};
            if (DIST && out.slopes) {
                sum.t = column_sum(sums[t].t);
                sum.pd = column_sum(sums[t].pd);
                sum.td = column_sum(sums[t].td);
            }
            if (row >= rows) continue;
            const int i = call.group(row), h = hk * G + (row - i * G);
            const int64_t all = a.num_queries * a.heads, at = (qs.at + i) * a.heads + h;
            if constexpr (kHalf<T>) {
#pragma unroll
                for (int x = 0; x < CP / 16; ++x) acc[t][x] = acc[t][x] * (1.0f / raise[t].by);
            }
            if (part) {
                const int64_t mine = split * all + at;
                if (g == 0) reinterpret_cast<Sums*>(part + (int64_t)splits * all * C)[mine] = sum;
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) *reinterpret_cast<f32x4*>(part + mine * C + 16 * x + 4 * g) = acc[t][x];
            } else {
                const float inv = sum.inverse();
                if (g == 0) {
                    out.inverse[at] = inv;
                    if (out.slopes) out.slopes[at] = sum.slope(inv);
                }
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C)
                        put4(grad_q, static_cast<T*>(nullptr), at * C + 16 * x + 4 * g, acc[t][x] * inv * a.scale);
            }
        }
    }
}

// grad_q, its rows' sums and slope gradients from the splits'; rows of no graph zero: four channels a thread
template <typename T>
__global__ void __launch_bounds__(256) join_grad_q_kernel(Args a, RowSums out, const float* part, int splits) {
    const Span qs = all_rows(a.q_ptr, a.num_graphs, a.num_queries);
    const int C = a.channels, C4 = C / 4;
    const int64_t all = a.num_queries * a.heads, step = (int64_t)gridDim.x * 256;
    const Sums* sums = reinterpret_cast<const Sums*>(part + splits * all * C);
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < all * C4; x += step) {
        const int64_t at = x / C4, row = at / a.heads, e = x * 4;
        f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
        if (row >= qs.at && row < qs.at + qs.n) {
            Sums sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (int k = 0; k < splits; ++k) {
                v = v + *reinterpret_cast<const f32x4*>(part + k * all * C + e);
                const Sums s = sums[k * all + at];
                sum = {sum.e + s.e, sum.t + s.t, sum.pd + s.pd, sum.td + s.td};
            }
            const float inv = sum.inverse();
            v = v * inv;
            if (x == at * C4) {
                out.inverse[at] = inv;
                if (out.slopes) out.slopes[at] = sum.slope(inv);
            }
        }
        put4(static_cast<T*>(a.grad_q), static_cast<T*>(nullptr), e, v * a.scale);
    }
}

// Distances are read where they are used: a fragment's sixteen lanes lie along a row already.  Staged through LDS as
// in the other passes this one took 184 us at 4001 nodes; it took 157 us once that and some of its score code went.
template <typename T, int CP, int MK, int WAVES, int RT, bool DIST, bool CAP>
__global__ void __launch_bounds__(kWave* WAVES) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, CP, WAVES>)))
attention_bwd_kv_kernel(Call call, const float* dots, const float* inverse, float* part) {
    constexpr int kThreads = kWave * WAVES, kKeys = 16 * MK * WAVES, kSteps = CP / 32, kTiles = RT / 16;
    constexpr bool kAhead = WAVES > 1, kDivide = sizeof(T) == 4;   // kDivide: by the weights' sum, near zero too
    __shared__ __attribute__((aligned(16))) T q_tile[RT * kRow<T, CP>], go_tile[RT * kRow<T, CP>];
    __shared__ __attribute__((aligned(16))) float row_at[RT], row_minus[RT], row_inv[RT], row_D[RT], row_slope[RT];
    __shared__ int tile_far;
    const Args& a = call.a;
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, c = lane % 16;
    const int G = call.group.by, C = a.channels;
    const float unit = call.unit.log2;
    T *grad_k = static_cast<T*>(a.grad_k), *grad_v = static_cast<T*>(a.grad_v);
    if ((int)blockIdx.x >= call.blocks) {
        if (part) return;
        zero_rest(grad_k, a.k_ptr, a.num_graphs, a.num_nodes, (int64_t)a.kv_heads * C, blockIdx.x - call.blocks);
        zero_rest(grad_v, a.k_ptr, a.num_graphs, a.num_nodes, (int64_t)a.kv_heads * C, blockIdx.x - call.blocks);
        return;
    }
    const Work work = work_of<DIST>(call);
    const int b = work.graph, hk = work.head, split = work.split, splits = call.splits.by;
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int rows = qs.n * G;
    int first = 0, last = rows;
    if (splits > 1) {
        const int each = ((rows + RT - 1) / RT + splits - 1) / splits * RT;
        first = min((int64_t)rows, (int64_t)split * each);
        last = min((int64_t)rows, (int64_t)first + each);
    }
    bool falls = DIST && a.slope;   // all the group's slopes are positive
    if (falls)
        for (int h = lane; h < G; h += kWave) falls = falls && a.slope[hk * G + h] > 0.0f;
    falls = __all(falls);

    for (int tile = work.tile; (int64_t)tile * kKeys < ks.n; tile += call.tiles) {
        const int key0 = tile * kKeys + w * 16 * MK;
        frag<T> k[MK][kSteps], v[MK][kSteps];
        const float* dist[MK];
        uint32_t d_off[MK];
        // (16 n + 4 g + r) / G = 16 n / G + 4 g / G + r / G for every power of two up to 16; r0 is a multiple of 32
        const bool steps = DIST && WAVES > 1 && 16 % G == 0 && a.dist_row < (1 << 22) && a.dist_cols >= ks.n;
        f32x4 gk[MK][CP / 16], gv[MK][CP / 16];
        Raise raise[MK];
#pragma unroll
        for (int t = 0; t < MK; ++t) {
            const int j = min(key0 + 16 * t + c, ks.n - 1);
            const T* pk = static_cast<const T*>(a.k) + (ks.at + j) * a.k_row + hk * a.k_head;
            const T* pv = static_cast<const T*>(a.v) + (ks.at + j) * a.v_row + hk * a.v_head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const bool in = 32 * s + 8 * g < C;
                k[t][s] = in ? load_frag(pk + 32 * s + 8 * g) : zero_frag<T>();
                v[t][s] = in ? load_frag(pv + 32 * s + 8 * g) : zero_frag<T>();
            }
            if (DIST) {
                dist[t] = j < a.dist_cols ? a.dist + b * a.dist_graph + j : nullptr;
                d_off[t] = call.group(4 * g) * (uint32_t)a.dist_row + j;
            }
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) gk[t][x] = gv[t][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            raise[t] = {kRaiseAll};
        }
        Staged<T, CP, RT, kThreads> q_next, go_next;
        Around next{0.0f, 0.0f};
        float next_inv = 0.0f, next_D = 0.0f, next_slope = 0.0f;
        auto fetch = [&](int r0) {
            q_next.load_rows(r0, rows, C, [&](int row) {
                const int i = call.group(row), h = hk * G + (row - i * G);
                return static_cast<const T*>(a.q) + (qs.at + i) * a.q_row + h * a.q_head;
            });
            go_next.load_rows(r0, rows, C, [&](int row) {
                const int i = call.group(row), h = hk * G + (row - i * G);
                return static_cast<const T*>(a.grad_out) + ((qs.at + i) * a.heads + h) * C;
            });
            next = {INFINITY, INFINITY};   // rows that are not there, and empty ones: every weight comes out as zero
            next_D = next_inv = 0.0f;
            next_slope = -1.0f;    // as any row's where all fall: with 0, a distance of +inf would make NaN
            if (threadIdx.x < RT && r0 + (int)threadIdx.x < last) {
                const int row = r0 + threadIdx.x, i = call.group(row), h = hk * G + (row - i * G);
                const int64_t at = (qs.at + i) * a.heads + h;
                if (a.lse[at] != -INFINITY) {
                    next = around(a.lse[at] * call.unit.per, unit);
                    next_inv = inverse[at];
                    next_D = dots[at];
                }
                if (DIST) next_slope = a.slope ? -a.slope[h] : 0.0f;
            }
        };
        f32x4 d[MK][kTiles];
        if (kAhead && first < last) fetch(first);
        for (int r0 = first; r0 < last; r0 += RT) {
            if (!kAhead) fetch(r0);
            if (DIST && key0 < ks.n) {
                if (steps && r0 + RT <= rows && call.group(r0 + RT - 1) < a.dist_rows) {
                    // rows in equal steps and all there: one 32-bit offset a lane, the rest is scalar
                    const float* base = a.dist + b * a.dist_graph + (int64_t)call.group(r0) * a.dist_row;
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float* row = base + (int64_t)call.group(16 * n + r) * a.dist_row;
#pragma unroll
                            for (int t = 0; t < MK; ++t) d[t][n][r] = row[d_off[t]];
                        }
                } else {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int row = min(r0 + 16 * n + 4 * g + r, rows - 1), i = call.group(row);
                            const int64_t at = i * a.dist_row;
                            const bool in = i < a.dist_rows;
#pragma unroll
                            for (int t = 0; t < MK; ++t) d[t][n][r] = in && dist[t] ? dist[t][at] : INFINITY;
                        }
                }
            }
            __syncthreads();
            q_next.store(q_tile);
            go_next.store(go_tile);
            if (threadIdx.x < RT) {
                const bool far = __any(next.far(kFarBack<T>));   // RT threads of the first wave
                float minus = -next.c;
                if (far) minus = next.add(unit, kFarBack<T>) + (kDivide ? 0.0f : log2f(next_inv));
                row_at[threadIdx.x] = next.at;
                row_minus[threadIdx.x] = minus;
                if (kDivide) row_inv[threadIdx.x] = next_inv;
                row_D[threadIdx.x] = next_D;
                tile_far = far;
                if (DIST) row_slope[threadIdx.x] = next_slope;
            }
            __syncthreads();
            if (kAhead && r0 + RT < last) fetch(r0 + RT);
            if (key0 >= ks.n) continue;
            f32x4 s[MK][kTiles], gp[MK][kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                for (int t = 0; t < MK; ++t) s[t][n] = gp[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const frag<T> f = load_frag(q_tile + (16 * n + c) * kRow<T, CP> + 32 * x + 8 * g);
#pragma unroll
                    for (int t = 0; t < MK; ++t) s[t][n] = mma(f, k[t][x], s[t][n]);
                }
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const frag<T> f = load_frag(go_tile + (16 * n + c) * kRow<T, CP> + 32 * x + 8 * g);
#pragma unroll
                    for (int t = 0; t < MK; ++t) gp[t][n] = mma(f, v[t][x], gp[t][n]);
                }
            }
            frag<T> p[MK][RT / 32], u[MK][RT / 32];
            const bool far = tile_far;
            f32x4 minus[kTiles], inv[kTiles], D[kTiles], slope[kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                minus[n] = *reinterpret_cast<const f32x4*>(row_minus + 16 * n + 4 * g);
                if (kDivide) inv[n] = *reinterpret_cast<const f32x4*>(row_inv + 16 * n + 4 * g);
                D[n] = *reinterpret_cast<const f32x4*>(row_D + 16 * n + 4 * g);
                if (DIST) slope[n] = *reinterpret_cast<const f32x4*>(row_slope + 16 * n + 4 * g);
            }
#pragma unroll
            for (int t = 0; t < MK; ++t) {
                f32x4 slack[kTiles];
                scores<T, CAP, true>(call, s[t], slack, far);
                if (DIST) {
                    if (falls && ordinary(d[t])) {
                        TRX_EACH_SCORE s[t][n][r] = __builtin_fmaf(slope[n][r], d[t][n][r], s[t][n][r]);
                    } else {
                        TRX_EACH_SCORE s[t][n][r] =
                            finite(d[t][n][r]) ? __builtin_fmaf(slope[n][r], d[t][n][r], s[t][n][r]) : -INFINITY;
                    }
                }
                if (far) {
                    TRX_EACH_SCORE s[t][n][r] = fminf(s[t][n][r] - row_at[16 * n + 4 * g + r], 0.0f);
                }
                TRX_EACH_SCORE {   // both rounded to the type for their products
                    float e = exp2_fast(__builtin_fmaf(s[t][n][r], unit, minus[n][r]));
                    if (kDivide) e *= inv[n][r];
                    const float v = e * (gp[t][n][r] - D[n][r]);
                    p[t][n / 2][4 * (n % 2) + r] = (T)(e * kWeight<T>);
                    s[t][n][r] = CAP ? v * slack[n][r] : v;
                }
                if constexpr (kHalf<T>) {
                    float most = 0.0f;
                    TRX_EACH_SCORE most = fmaxf(most, fabsf(s[t][n][r]));
                    raise[t].over(most, gk[t]);
                    TRX_EACH_SCORE s[t][n][r] *= raise[t].by;
                }
                TRX_EACH_SCORE u[t][n / 2][4 * (n % 2) + r] = (T)s[t][n][r];
            }
#pragma unroll
            for (int x = 0; x < CP / 16; ++x)
#pragma unroll
                for (int y = 0; y < RT / 32; ++y) {
                    const frag<T> f = turned<T, CP>(go_tile, 32 * y, 32 * y + 16, 16 * x, lane);
#pragma unroll
                    for (int t = 0; t < MK; ++t) gv[t][x] = mma(f, p[t][y], gv[t][x]);
                    const frag<T> e = turned<T, CP>(q_tile, 32 * y, 32 * y + 16, 16 * x, lane);
#pragma unroll
                    for (int t = 0; t < MK; ++t) gk[t][x] = mma(e, u[t][y], gk[t][x]);
                }
        }
#pragma unroll
        for (int t = 0; t < MK; ++t) {
            const int j = key0 + 16 * t + c;
            if (j >= ks.n) continue;
            const int64_t all = a.num_nodes * a.kv_heads, at = (ks.at + j) * a.kv_heads + hk;
            if constexpr (kHalf<T>) {
#pragma unroll
                for (int x = 0; x < CP / 16; ++x) {
                    gk[t][x] = gk[t][x] * (1.0f / raise[t].by);
                    gv[t][x] = gv[t][x] * (1.0f / kWeight<T>);
                }
            }
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) {
                const int ch = 16 * x + 4 * g;
                if (ch >= C) continue;
                if (part) {   // [split][k, v][node, head, channel]
                    float* mine = part + ((int64_t)split * 2 * all + at) * C + ch;
                    *reinterpret_cast<f32x4*>(mine) = gk[t][x];
                    *reinterpret_cast<f32x4*>(mine + all * C) = gv[t][x];
                } else {
                    put4(grad_k, static_cast<T*>(nullptr), at * C + ch, gk[t][x] * a.scale);
                    put4(grad_v, static_cast<T*>(nullptr), at * C + ch, gv[t][x]);
                }
            }
        }
    }
}

// One output's splits: out[e] = scale x the sum of part[k * stride + e] over the splits k in their order; rows of no
// graph: zeros
struct SplitSum {
    const float* part;
    void* out;
    float scale;
};
template <typename T>
__global__ void __launch_bounds__(256) sum_splits_kernel(SplitSum first, SplitSum second, int splits, int64_t stride,
                                                         int64_t n, int64_t width, const int64_t* ptr, int graphs,
                                                         int64_t rows) {
    const SplitSum& x = blockIdx.y == 0 ? first : second;
    const Span s = all_rows(ptr, graphs, rows);
    const int64_t step = (int64_t)gridDim.x * 256 * 4;
    for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < n; e += step) {
        f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
        if (e >= s.at * width && e < (s.at + s.n) * width) {
#pragma unroll 4
            for (int k = 0; k < splits; ++k) v = v + *reinterpret_cast<const f32x4*>(x.part + k * stride + e);
        }
        put4(static_cast<T*>(x.out), static_cast<T*>(nullptr), e, v * x.scale);
    }
}

// A (head, chunk of the query rows) each: the sum of the rows' slope gradients; chunk by chunk to out[head + heads *
// chunk].  A fixed order throughout.
template <int kBlock>
__device__ __forceinline__ float block_sum(float v) {
    __shared__ float part[kBlock / kWave];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int k = 1; k < kBlock / kWave; ++k) v += part[k];
    return v;
}
template <typename T>
__global__ void __launch_bounds__(1024)
    slope_rows_kernel(Args a, const float* slopes, float* out) {
    const int h = blockIdx.x;
    const int64_t each = (a.num_queries + gridDim.y - 1) / gridDim.y;
    const Span s = all_rows(a.q_ptr, a.num_graphs, a.num_queries);
    const int64_t begin = max(s.at, (int64_t)blockIdx.y * each), end = min(s.at + s.n, (int64_t)(blockIdx.y + 1) * each);
    float v = 0.0f;
#pragma unroll 4
    for (int64_t r = begin + threadIdx.x; r < end; r += 1024) v += slopes[r * a.heads + h];
    v = block_sum<1024>(v);
    if (threadIdx.x == 0) out[blockIdx.y * a.heads + h] = v;
}
template <typename T>
__global__ void __launch_bounds__(kWave) slope_chunks_kernel(const float* chunks, int count, int heads, float* out) {
    const float v = block_sum<kWave>((int)threadIdx.x < count ? chunks[threadIdx.x * heads + blockIdx.x] : 0.0f);
    if (threadIdx.x == 0) out[blockIdx.x] = v;
}

template <typename T, int CP, bool DIST, bool CAP>
void launch_bwd(const Args& a, hipStream_t stream) {
    const int64_t rows = a.num_queries * a.heads;
    float *dots = static_cast<float*>(a.workspace), *inverse = dots + rows, *slopes = inverse + rows;
    float *chunks = slopes + rows, *split = dots + attention_row_floats(a);
    const bool want_slopes = DIST && a.grad_slope && a.slope;
    const RowSums sums{dots, inverse, want_slopes ? slopes : nullptr};
    auto blocks = [](int64_t n) { return (unsigned)std::min<int64_t>(2048, (n / 4 + 255) / 256); };
    // 128 channels: of 32 rows a wave, operands, accumulators and both score tiles leave no registers to load ahead
    constexpr int M = kTilesOfWave<T, CP>, MQ = CP == 128 ? 1 : 2, MK = CP == 128 ? 1 : 2;
    if (a.num_queries > 0) {
        const AttentionCut c = cut_bwd_q(a);
        float* part = c.splits > 1 ? split : nullptr;
        const Call call = call_of(a, c);
        const dim3 grid(call.blocks + kRestBlocks);
        if (c.narrow)
            hipLaunchKernelGGL((attention_bwd_q_kernel<T, CP, M, 1, 32, DIST, CAP>), grid, dim3(64), 0, stream, call, sums,
                               part);
        else
            hipLaunchKernelGGL((attention_bwd_q_kernel<T, CP, MQ, 4, 32, DIST, CAP>), grid, dim3(256), 0, stream, call, sums,
                               part);
        const int64_t n = a.num_queries * a.heads * a.channels;
        if (part)
            hipLaunchKernelGGL(join_grad_q_kernel<T>, dim3(blocks(n)), dim3(256), 0, stream, a, sums, part, c.splits);
        if (want_slopes) {
            const int count = (int)std::max<int64_t>(1, std::min<int64_t>(kSlopeChunks, a.num_queries / 16384));
            hipLaunchKernelGGL(slope_rows_kernel<T>, dim3(a.heads, count), dim3(1024), 0, stream, a, slopes,
                               count > 1 ? chunks : a.grad_slope);
            if (count > 1)
                hipLaunchKernelGGL(slope_chunks_kernel<T>, dim3(a.heads), dim3(kWave), 0, stream, chunks, count, a.heads,
                                   a.grad_slope);
        }
    } else if (want_slopes) {
        hipLaunchKernelGGL(slope_rows_kernel<T>, dim3(a.heads), dim3(1024), 0, stream, a, slopes, a.grad_slope);
    }
    if (a.num_nodes > 0) {
        const AttentionCut c = cut_bwd_kv(a);
        float* part = c.splits > 1 ? split : nullptr;
        const Call call = call_of(a, c);
        const dim3 grid(call.blocks + kRestBlocks);
        if (c.narrow)
            hipLaunchKernelGGL((attention_bwd_kv_kernel<T, CP, MK, 1, 32, DIST, CAP>), grid, dim3(64), 0, stream, call, dots,
                               inverse, part);
        else
            hipLaunchKernelGGL((attention_bwd_kv_kernel<T, CP, MK, 4, 32, DIST, CAP>), grid, dim3(256), 0, stream, call,
                               dots, inverse, part);
        if (part) {
            const int64_t n = a.num_nodes * a.kv_heads * a.channels;
            hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks(n), 2), dim3(256), 0, stream,
                               SplitSum{part, a.grad_k, a.scale}, SplitSum{part + n, a.grad_v, 1.0f}, c.splits, 2 * n, n,
                               (int64_t)a.kv_heads * a.channels, a.k_ptr, a.num_graphs, a.num_nodes);
        }
    }
}

}  // namespace

template <typename T>
hipError_t launch_attention_bwd(const trx_node_attention_args& a, hipStream_t stream) {
    return by_shape<T>(a, [&](auto cp, auto dist, auto cap) {
        launch_bwd<T, decltype(cp)::value, decltype(dist)::value, decltype(cap)::value>(a, stream);
        return hipGetLastError();
    });
}

}  // namespace trx
