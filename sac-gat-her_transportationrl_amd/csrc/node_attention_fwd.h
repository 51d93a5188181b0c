// node_attention_fwd.h -- node_attention's forward kernels, one element type to
// a translation unit (node_attention_{f32,bf16,f16}.hip).
//
// One pass over a graph's keys with the running maximum and sum of the softmax.
// A workgroup holds WAVES x 16 MQ rows of one (graph, key/value head): the
// query rows of all heads that share the key/value head, row-major (query, head
// of the group), so a shared head's keys are read once.  Keys, values and
// distances pass through LDS in tiles of KT, the next tile on its way in registers.
//
// Weights are rounded to the type for the product with v, because the matrix
// instructions take operands of it; their sum is not.  Results in bfloat16 are off
// by 0.0019 to 0.0020 (relative to float64), where rounding the result alone costs
// 0.0016 to 0.0017.
//
// What bounds it.  Large graphs: the vector instructions of the scores and waiting.
// 4096 nodes, 8 heads of 64, bfloat16, with distances: 11.8 vector instructions a
// score issue in 50% of the cycles, the matrix pipe is busy in 16%, waves wait in
// 31% of theirs; registers allow two waves a SIMD (three: 183 us against 132 when
// tried).  With the splits' join, 4096 nodes, 8 heads, bfloat16: 110 us at 128
// channels (623 TFLOP/s), 72 to 78 at 64 (442 to 477); with distances 145 and 100.
// 64 keys a tile at 64 channels with distances (32: 120 us against 107 when tried),
// 32 at 128.  Small graphs and single queries: memory.  4096
// networks of 24 nodes, 4 heads of 64: 43 us (201 MB at 4.7 TB/s, a large copy's
// rate); 8 queries over 32768 nodes each, 16 heads on 2 of 128: 50 us and 7 us for
// joining the splits (270 MB at 4.7 TB/s together).
#pragma once
#include <algorithm>

#include "node_attention.h"

namespace trx {
namespace {

template <typename T, int CP, int MQ, int WAVES, int KT, bool DIST, bool CAP>
__global__ void __launch_bounds__(kWave* WAVES) __attribute__((amdgpu_waves_per_eu(kWavesPerSimd<T, CP, WAVES>)))
attention_fwd_kernel(Call call, float* part) {
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
    T* out = static_cast<T*>(a.out);
    if ((int)blockIdx.x >= call.blocks) {
        if (!part) zero_rest(out, a.q_ptr, a.num_graphs, a.num_queries, (int64_t)a.heads * C, blockIdx.x - call.blocks);
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
        frag<T> q[MQ][kSteps];
        const float* dist[MQ];
        Around ref[MQ];
        float m[MQ], l[MQ], slope[MQ];   // the reference's score (-inf: none yet), the sum, -slope
        bool far[MQ];                    // of the wave
        int limit[MQ];
        f32x4 o[MQ][CP / 16];
#pragma unroll
        for (int t = 0; t < MQ; ++t) {
            const int row = min(row0 + 16 * t + c, rows - 1);
            const int i = call.group(row), h = hk * G + (row - i * G);
            const T* p = static_cast<const T*>(a.q) + (qs.at + i) * a.q_row + h * a.q_head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[t][s] = 32 * s + 8 * g < C ? load_frag(p + 32 * s + 8 * g) : zero_frag<T>();
            slope[t] = DIST && a.slope ? -a.slope[h] : 0.0f;
            if (DIST && !kStageD) {
                dist[t] = a.dist + b * a.dist_graph + i * a.dist_row;
                limit[t] = i < a.dist_rows ? min(ks.n, a.dist_cols) : 0;
            }
            m[t] = -INFINITY;
            ref[t] = {0.0f, 0.0f};
            far[t] = false;
            l[t] = 0.0f;
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) o[t][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
            f32x4 s[MQ][kTiles];
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
#pragma unroll
                for (int t = 0; t < MQ; ++t) s[t][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int x = 0; x < kSteps; ++x) {
                    const frag<T> f = load_frag(k_tile + (16 * n + c) * kRow<T, CP> + 32 * x + 8 * g);
#pragma unroll
                    for (int t = 0; t < MQ; ++t) s[t][n] = mma(f, q[t][x], s[t][n]);
                }
            }
            frag<T> p[MQ][KT / 32];
#pragma unroll
            for (int t = 0; t < MQ; ++t) {
                if (kStageD) {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
                        d[t][n] = *reinterpret_cast<const f32x4*>(d_tile + d_row[t] + 16 * n + 4 * g);
                }
                scores<T, CAP, false>(call, s[t], s[t], false);
                if (DIST) {
                    if (__all(slope[t] < 0.0f) && ordinary(d[t])) {   // a distance of +inf makes its -inf by itself
                        TRX_EACH_SCORE s[t][n][r] = __builtin_fmaf(slope[t], d[t][n][r], s[t][n][r]);
                    } else {
                        TRX_EACH_SCORE s[t][n][r] =
                            finite(d[t][n][r]) ? __builtin_fmaf(slope[t], d[t][n][r], s[t][n][r]) : -INFINITY;
                    }
                } else if (j0 + KT > last) {
                    TRX_EACH_SCORE if (j0 + 16 * n + 4 * g + r >= last) s[t][n][r] = -INFINITY;
                }
                float top = -INFINITY;
                TRX_EACH_SCORE top = fmaxf(top, s[t][n][r]);
                top = column_max(top);
                // The reference point moves only when a score passes it by 2^8: nothing is lost in float32, and the
                // accumulators are rescaled once or twice a row instead of at every new maximum.
                const bool move = (top - m[t]) * unit > 8.0f;
                if (__any(move)) {
                    const Around next = around(top, unit, kLift<T>);
                    const float by = next.add(unit, kFar, kLift<T>) - ref[t].add(unit, kFar, kLift<T>);
                    const float f = move ? exp2_fast(__builtin_fmaf(m[t] - top, unit, by)) : 1.0f;
                    if (move) {
                        m[t] = top;
                        ref[t] = next;
                    }
                    far[t] = __any(ref[t].far(kFar));
                    l[t] *= f;
#pragma unroll
                    for (int x = 0; x < CP / 16; ++x) o[t][x] = o[t][x] * f;
                }
                float minus = -ref[t].c;
                if (far[t]) {
                    TRX_EACH_SCORE s[t][n][r] -= ref[t].at;
                    minus = ref[t].add(unit, kFar, kLift<T>);
                }
                TRX_EACH_SCORE {
                    const float e = exp2_fast(__builtin_fmaf(s[t][n][r], unit, minus));
                    l[t] += e;
                    p[t][n / 2][4 * (n % 2) + r] = (T)e;   // rounded to the type for the product with v
                }
            }
#pragma unroll
            for (int x = 0; x < CP / 16; ++x)
#pragma unroll
                for (int u = 0; u < KT / 32; ++u) {
                    const frag<T> f = turned<T, CP>(v_tile, 32 * u, 32 * u + 16, 16 * x, lane);
#pragma unroll
                    for (int t = 0; t < MQ; ++t) o[t][x] = mma(f, p[t][u], o[t][x]);
                }
        }
#pragma unroll
        for (int t = 0; t < MQ; ++t) {
            const float sum = column_sum(l[t]);
            const int row = row0 + 16 * t + c;
            if (row >= rows) continue;
            const int i = call.group(row), h = hk * G + (row - i * G);
            const int64_t at = (qs.at + i) * a.heads + h;
            const float add = ref[t].add(unit, kFar, kLift<T>);   // 0 where m is still -inf
            if (part) {   // this split's sum and accumulator around m unit, for the joining kernels
                const int64_t all = a.num_queries * a.heads, mine = split * all + at;
                float* stat = part + (int64_t)splits * all * C;
                const float f = exp2_fast(-add);
                if (g == 0) {
                    stat[2 * mine] = m[t];
                    stat[2 * mine + 1] = sum * f;
                }
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) *reinterpret_cast<f32x4*>(part + mine * C + 16 * x + 4 * g) = o[t][x] * f;
            } else {
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (a.lse && g == 0)
                    a.lse[at] = sum == 0.0f ? -INFINITY : __builtin_fmaf(log2f(sum) - add, kLn2, m[t] * call.unit.nat);
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) put4(out, static_cast<T*>(a.out_low), at * C + 16 * x + 4 * g, o[t][x] * f);
            }
        }
    }
}

// out, out_low and lse from few splits' sums, rows of no graph zero: four channels a thread
template <typename T>
__global__ void __launch_bounds__(256) attention_join_few_kernel(Args a, Unit unit, const float* part, int splits) {
    const Span qs = all_rows(a.q_ptr, a.num_graphs, a.num_queries);
    const int C = a.channels, C4 = C / 4;
    const int64_t all = a.num_queries * a.heads, step = (int64_t)gridDim.x * 256;
    const float* stat = part + splits * all * C;
    for (int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x; x < all * C4; x += step) {
        const int64_t at = x / C4, row = at / a.heads, e = x * 4;
        if (row < qs.at || row >= qs.at + qs.n) {
            put4(static_cast<T*>(a.out), static_cast<T*>(nullptr), e, f32x4{0.0f, 0.0f, 0.0f, 0.0f});
            continue;
        }
        float top = -INFINITY, sum = 0.0f;
        for (int s = 0; s < splits; ++s) top = fmaxf(top, stat[2 * (s * all + at)]);
        f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
        for (int s = 0; s < splits; ++s) {
            const float m = stat[2 * (s * all + at)], l = stat[2 * (s * all + at) + 1];
            // a split without a finite score adds its sum as it is: zero, or the NaN that it saw
            const float f = m == -INFINITY ? 0.0f : exp2_fast((m - top) * unit.log2);
            sum += m == -INFINITY ? l : l * f;
            v = v + *reinterpret_cast<const f32x4*>(part + s * all * C + e) * f;
        }
        put4(static_cast<T*>(a.out), static_cast<T*>(a.out_low), e, v * (sum == 0.0f ? 0.0f : 1.0f / sum));
        if (a.lse && x == at * C4) a.lse[at] = sum == 0.0f ? -INFINITY : __builtin_fmaf(log2f(sum), kLn2, top * unit.nat);
    }
}

// The same from many: a workgroup to a (row, head), its four waves
// each over every fourth split, two channels a lane
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(Args a, Unit unit, const float* part, int splits) {
    __shared__ float sums[4][2 * kWave];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, C = a.channels;
    const int64_t all = a.num_queries * a.heads, at = blockIdx.x;
    const Span qs = all_rows(a.q_ptr, a.num_graphs, a.num_queries);
    const int64_t row = at / a.heads;
    if (row < qs.at || row >= qs.at + qs.n) {
        if (threadIdx.x < C) static_cast<T*>(a.out)[at * C + threadIdx.x] = (T)0.0f;
        return;
    }
    const float* stat = part + splits * all * C;
    const bool has = lane < splits;   // at most 64
    const float m = has ? stat[2 * (lane * all + at)] : -INFINITY, l = has ? stat[2 * (lane * all + at) + 1] : 0.0f;
    float top = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    // a split without a finite score adds its sum as it is: zero, or the NaN that it saw
    const float f = m == -INFINITY ? 0.0f : exp2_fast((m - top) * unit.log2);
    float sum = m == -INFINITY ? l : l * f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    float x = 0.0f, y = 0.0f;
    const int mine = min(2 * lane, C - 2);   // every lane takes part: the factors come from lanes of all splits
    for (int s = w; s < splits; s += 4) {
        const float2 v = *reinterpret_cast<const float2*>(part + (s * all + at) * C + mine);
        const float fs = __shfl(f, s);
        x = __builtin_fmaf(v.x, fs, x);
        y = __builtin_fmaf(v.y, fs, y);
    }
    sums[w][2 * lane] = x;
    sums[w][2 * lane + 1] = y;
    __syncthreads();
    if (threadIdx.x < C) {
        const int ch = threadIdx.x;
        const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
        const float v = ((sums[0][ch] + sums[1][ch]) + (sums[2][ch] + sums[3][ch])) * r;
        const T t = (T)v;
        static_cast<T*>(a.out)[at * C + ch] = t;
        if (a.out_low) static_cast<T*>(a.out_low)[at * C + ch] = (T)(v - (float)t);
    }
    if (a.lse && threadIdx.x == 0) a.lse[at] = sum == 0.0f ? -INFINITY : __builtin_fmaf(log2f(sum), kLn2, top * unit.nat);
}

template <typename T, int CP, bool DIST, bool CAP>
void launch_fwd(const Args& a, hipStream_t stream) {
    const AttentionCut c = cut_fwd(a);
    float* part = c.splits > 1 ? static_cast<float*>(a.workspace) : nullptr;
    const Call call = call_of(a, c);
    const dim3 grid(call.blocks + kRestBlocks);
    constexpr int kWide = sizeof(T) == 2 && CP <= 64 ? 64 : 32;
    if (!c.narrow)
        hipLaunchKernelGGL((attention_fwd_kernel<T, CP, kTilesOfWave<T, CP>, 4, kWide, DIST, CAP>), grid, dim3(256), 0,
                           stream, call, part);
    else if (c.mq == 2)
        hipLaunchKernelGGL((attention_fwd_kernel<T, CP, 2, 1, 32, DIST, CAP>), grid, dim3(64), 0, stream, call, part);
    else
        hipLaunchKernelGGL((attention_fwd_kernel<T, CP, 1, 1, 32, DIST, CAP>), grid, dim3(64), 0, stream, call, part);
    if (part && c.splits <= 8)
        hipLaunchKernelGGL(attention_join_few_kernel<T>,
                           dim3((unsigned)std::min<int64_t>(4096, (a.num_queries * a.heads * a.channels / 4 + 255) / 256)),
                           dim3(256), 0, stream, a, call.unit, part, c.splits);
    else if (part)
        hipLaunchKernelGGL(attention_join_kernel<T>, dim3((unsigned)(a.num_queries * a.heads)), dim3(256), 0, stream, a,
                           call.unit, part, c.splits);
}

}  // namespace

template <typename T>
hipError_t launch_attention_fwd(const trx_node_attention_args& a, hipStream_t stream) {
    return by_shape<T>(a, [&](auto cp, auto dist, auto cap) {
        launch_fwd<T, decltype(cp)::value, decltype(dist)::value, decltype(cap)::value>(a, stream);
        return hipGetLastError();
    });
}

}  // namespace trx
