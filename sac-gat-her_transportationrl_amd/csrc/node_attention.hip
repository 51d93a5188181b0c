// node_attention.hip -- softmax attention of query rows over the nodes of their
// own network, forward (include/trafficrl.h, trx_node_attention_*; backward:
// node_attention_bwd.hip): scores scaled, optionally capped by a tanh, lowered
// by slope[h] times the pair's distance, pairs at no finite distance unseen.
//
// One pass over a graph's keys with the running maximum and sum of the softmax.
// A workgroup holds WAVES x 16 MQ rows of one (graph, key/value head): the
// query rows of all heads that share the key/value head, row-major (query, head
// of the group), so a shared head's keys are read once.  Keys and values pass
// through LDS in tiles of KT, the next tile on its way in registers.
#include <algorithm>

#include "node_attention.h"

namespace trx {
namespace {

template <typename T, int CP, int MQ, int WAVES, int KT>
__global__ void __launch_bounds__(kWave* WAVES) attention_fwd_kernel(Args a, float* part) {
    constexpr int kThreads = kWave * WAVES, kRows = 16 * MQ * WAVES, kSteps = CP / 32, kTiles = KT / 16;
    __shared__ __attribute__((aligned(16))) T k_tile[KT * kRow<T, CP>], v_tile[KT * kRow<T, CP>];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, c = lane % 16;
    const int b = blockIdx.x / a.kv_heads, hk = blockIdx.x % a.kv_heads, G = a.heads / a.kv_heads, C = a.channels;
    T* out = static_cast<T*>(a.out);
    if (b == a.num_graphs) {
        if (!part && hk == 0)
            zero_rest(out, a.q_ptr, b, a.num_queries, (int64_t)a.heads * C, blockIdx.y * kThreads + threadIdx.x,
                      gridDim.y * kThreads);
        return;
    }
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int64_t rows = (int64_t)qs.n * G;
    const int keys_each = ((ks.n + KT - 1) / KT + gridDim.z - 1) / gridDim.z * KT;
    const int first = min((int64_t)ks.n, (int64_t)blockIdx.z * keys_each), last = min(ks.n, first + keys_each);
    const T* k_base = static_cast<const T*>(a.k) + ks.at * a.k_row + hk * a.k_head;
    const T* v_base = static_cast<const T*>(a.v) + ks.at * a.v_row + hk * a.v_head;
    const float mul = a.cap > 0.0f ? a.scale / a.cap : a.scale;

    for (int64_t tile = blockIdx.y; tile * kRows < rows; tile += gridDim.y) {
        const int64_t row0 = tile * kRows + w * 16 * MQ;
        frag<T> q[MQ][kSteps];
        const float* dist[MQ];
        float slope[MQ], m[MQ], l[MQ];
        int limit[MQ];
        f32x4 o[MQ][CP / 16];
#pragma unroll
        for (int t = 0; t < MQ; ++t) {
            const int64_t row = min(row0 + 16 * t + c, rows - 1);
            const int i = (int)(row / G), h = hk * G + (int)(row % G);
            const T* p = static_cast<const T*>(a.q) + (qs.at + i) * a.q_row + h * a.q_head;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) q[t][s] = 32 * s + 8 * g < C ? load_frag(p + 32 * s + 8 * g) : zero_frag<T>();
            slope[t] = a.slope ? -a.slope[h] : 0.0f;
            dist[t] = a.dist ? a.dist + b * a.dist_graph + i * a.dist_row : nullptr;
            limit[t] = !a.dist ? ks.n : i < a.dist_rows ? min(ks.n, a.dist_cols) : 0;
            m[t] = -INFINITY;
            l[t] = 0.0f;
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) o[t][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        Staged<T, CP, KT, kThreads> k_next, v_next;
        auto fetch = [&](int j0) {
            k_next.load(C, [&](int j) { return j0 + j < ks.n ? k_base + (j0 + j) * a.k_row : nullptr; });
            v_next.load(C, [&](int j) { return j0 + j < ks.n ? v_base + (j0 + j) * a.v_row : nullptr; });
        };
        if (first < last) fetch(first);
        for (int j0 = first; j0 < last; j0 += KT) {
            __syncthreads();
            k_next.store(k_tile);
            v_next.store(v_tile);
            __syncthreads();
            if (j0 + KT < last) fetch(j0 + KT);
            if (row0 >= rows) continue;
            f32x4 d[MQ][kTiles];
            if (a.dist) {
#pragma unroll
                for (int t = 0; t < MQ; ++t) {
                    const bool whole = __all(j0 + KT <= limit[t]);
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) d[t][n] = distances(dist[t], j0 + 16 * n + 4 * g, limit[t], whole);
                }
            }
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
                // scores, and their maximum
                if (a.cap > 0.0f) {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[t][n][r] = a.cap * tanh_of<T>(s[t][n][r], mul);
                } else {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n) s[t][n] = s[t][n] * mul;
                }
                if (a.dist) {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            s[t][n][r] = finite(d[t][n][r]) ? __builtin_fmaf(slope[t], d[t][n][r], s[t][n][r]) : -INFINITY;
                } else if (j0 + KT > ks.n) {
#pragma unroll
                    for (int n = 0; n < kTiles; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (j0 + 16 * n + 4 * g + r >= ks.n) s[t][n][r] = -INFINITY;
                }
                float top = -INFINITY;
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][n][r]);
                top = column_max(top);
                // The reference point moves only when a score passes it by 5.5, a factor of 2^8 in the sums: nothing
                // is lost in float32, and the accumulators are rescaled once or twice a row instead of at every new
                // maximum.
                const bool move = top > m[t] + 5.5f;
                if (__any(move)) {
                    const float f = move ? exp2_fast((m[t] - top) * kLog2e) : 1.0f;
                    m[t] = move ? top : m[t];
                    l[t] *= f;
#pragma unroll
                    for (int x = 0; x < CP / 16; ++x) o[t][x] = o[t][x] * f;
                }
                const float base = m[t] == -INFINITY ? 0.0f : -m[t] * kLog2e;
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float e = exp2_fast(__builtin_fmaf(s[t][n][r], kLog2e, base));
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
            const int64_t row = row0 + 16 * t + c;
            if (row >= rows) continue;
            const int i = (int)(row / G), h = hk * G + (int)(row % G);
            const int64_t at = (qs.at + i) * a.heads + h;
            if (part) {   // this split's sum and accumulator, for join_kernel
                const int64_t all = a.num_queries * a.heads, mine = blockIdx.z * all + at;
                float* stat = part + (int64_t)gridDim.z * all * C;
                if (g == 0) {
                    stat[2 * mine] = m[t] * kLog2e;
                    stat[2 * mine + 1] = sum;
                }
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) *reinterpret_cast<f32x4*>(part + mine * C + 16 * x + 4 * g) = o[t][x];
            } else {
                const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                if (a.lse && g == 0) a.lse[at] = sum == 0.0f ? -INFINITY : m[t] * kLog2e + log2f(sum);
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) {
                        typedef T T4 __attribute__((ext_vector_type(4)));
                        T4 y;
#pragma unroll
                        for (int r = 0; r < 4; ++r) y[r] = (T)(o[t][x][r] * f);
                        *reinterpret_cast<T4*>(out + at * C + 16 * x + 4 * g) = y;
                    }
            }
        }
    }
}

// out and lse from the splits' sums: one wave per (row, head), rows of no graph zero
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(Args a, const float* part, int splits) {
    const int lane = threadIdx.x % kWave;
    const int64_t all = a.num_queries * a.heads, at = (int64_t)blockIdx.x * 4 + threadIdx.x / kWave;
    if (at >= all) return;
    const Span qs = all_rows(a.q_ptr, a.num_graphs, a.num_queries);
    const int64_t row = at / a.heads;
    T* out = static_cast<T*>(a.out) + at * a.channels;
    const float* stat = part + splits * all * a.channels;
    float m = -INFINITY, l = 0.0f, x = 0.0f, y = 0.0f;
    if (row >= qs.at && row < qs.at + qs.n) {
        for (int s = 0; s < splits; ++s) m = fmaxf(m, stat[2 * (s * all + at)]);
        for (int s = 0; s < splits; ++s) {
            const int64_t mine = s * all + at;
            const float f = stat[2 * mine] == -INFINITY ? 0.0f : exp2_fast(stat[2 * mine] - m);
            // a split without a finite score adds its sum as it is: zero, or the NaN that it saw
            l += stat[2 * mine] == -INFINITY ? stat[2 * mine + 1] : stat[2 * mine + 1] * f;
            if (lane < a.channels) x += part[mine * a.channels + lane] * f;
            if (lane + kWave < a.channels) y += part[mine * a.channels + lane + kWave] * f;
        }
        if (a.lse && lane == 0) a.lse[at] = l == 0.0f ? -INFINITY : m + log2f(l);
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    if (lane < a.channels) out[lane] = (T)(x * f);
    if (lane + kWave < a.channels) out[lane + kWave] = (T)(y * f);
}

// How a forward pass is cut.  Up to 32 rows to a (graph, head), one wave has them all and a workgroup of more would
// idle; else four waves share each tile of keys.  Keys are split where the rows alone leave most of the 256 compute
// units without a workgroup, into pieces of at least 256 keys (a piece costs its accumulator's round trip).
struct Cut {
    bool narrow;   // one wave
    int mq;        // 16-row tiles of a wave
    int64_t tiles;
    int splits;
};
Cut cut_fwd(const Args& a) {
    const int64_t G = a.heads / a.kv_heads, units = (int64_t)a.num_graphs * a.kv_heads;
    const int64_t rows = std::min(a.max_queries, a.num_queries) * G, keys = std::min(a.max_nodes, a.num_nodes);
    Cut c;
    c.narrow = rows <= 32;
    c.mq = c.narrow && rows <= 16 ? 1 : 2;
    const int64_t each = c.narrow ? 16 * c.mq : 128;
    c.tiles = std::max<int64_t>(1, std::min<int64_t>((rows + each - 1) / each, 65535));
    const int64_t blocks = std::max<int64_t>(1, units * c.tiles), want = c.narrow ? 2048 : 512;
    const int64_t most = std::min<int64_t>(64, std::min(keys / 256, (int64_t(1) << 28) / std::max<int64_t>(1, a.num_queries * a.heads * (a.channels + 2) * 4)));
    c.splits = (int)std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, most));
    return c;
}

}  // namespace

size_t node_attention_workspace(const trx_node_attention_args& a, bool backward) {
    if (backward) return attention_bwd_workspace(a);
    const int splits = cut_fwd(a).splits;
    return splits > 1 ? (size_t)splits * a.num_queries * a.heads * (a.channels + 2) * sizeof(float) : 0;
}

template <typename T, int CP>
static void launch_fwd(const Args& a, const Cut& c, hipStream_t stream) {
    float* part = c.splits > 1 ? static_cast<float*>(a.workspace) : nullptr;
    const dim3 grid((unsigned)((a.num_graphs + 1) * (int64_t)a.kv_heads), (unsigned)c.tiles, c.splits);
    constexpr int kWide = sizeof(T) == 2 ? 64 : 32;
    if (!c.narrow)
        hipLaunchKernelGGL((attention_fwd_kernel<T, CP, 2, 4, kWide>), grid, dim3(256), 0, stream, a, part);
    else if (c.mq == 2)
        hipLaunchKernelGGL((attention_fwd_kernel<T, CP, 2, 1, 32>), grid, dim3(64), 0, stream, a, part);
    else
        hipLaunchKernelGGL((attention_fwd_kernel<T, CP, 1, 1, 32>), grid, dim3(64), 0, stream, a, part);
    if (part)
        hipLaunchKernelGGL(attention_join_kernel<T>, dim3((unsigned)((a.num_queries * a.heads + 3) / 4)), dim3(256), 0,
                           stream, a, part, c.splits);
}

hipError_t launch_node_attention_fwd(const trx_node_attention_args& a, hipStream_t stream) {
    const Cut c = cut_fwd(a);
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a.channels <= 32)
            launch_fwd<T, 32>(a, c, stream);
        else if (a.channels <= 64)
            launch_fwd<T, 64>(a, c, stream);
        else
            launch_fwd<T, 128>(a, c, stream);
        return hipGetLastError();
    });
}

hipError_t launch_node_attention_bwd(const trx_node_attention_args& a, hipStream_t stream) {
    return launch_attention_bwd(a, stream);
}

}  // namespace trx
