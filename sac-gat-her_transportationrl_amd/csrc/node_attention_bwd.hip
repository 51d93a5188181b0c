// node_attention_bwd.hip -- gradients of node_attention (include/trafficrl.h):
// with p the probabilities, brought back from the saved lse, go the incoming
// gradient, gp = go v^T and D = <go, out> of each row,
//   t = p (gp - D);  grad_slope = -sum t d;  u = t (1 - tanh^2)
//   grad_q = scale u k;  grad_k = scale u^T q;  grad_v = p^T go.
// Two passes and no atomics: one workgroup keeps query rows and runs over the
// keys (grad_q, D, the slopes' sums), one keeps keys and runs over the query
// rows of every head that shares them (grad_k, grad_v).  Seven products where
// five would do, for results that do not depend on the order of anything.
#include <algorithm>

#include "node_attention.h"

namespace trx {
namespace {

// Per (query row, head): what the slope's gradient needs.  D stands on the rounded out, so sum t is not quite zero;
// what is left of it corrects sum t d: grad_slope of the row = (sum t)(sum p d) - sum t d.
struct SlopeSums {
    float t, pd, td;
};

template <typename T, int CP, int MQ, int WAVES, int KT>
__global__ void __launch_bounds__(kWave* WAVES)
    attention_bwd_q_kernel(Args a, float* dots, float* slopes, float* part) {
    constexpr int kThreads = kWave * WAVES, kRows = 16 * MQ * WAVES, kSteps = CP / 32, kTiles = KT / 16;
    __shared__ __attribute__((aligned(16))) T k_tile[KT * kRow<T, CP>], v_tile[KT * kRow<T, CP>];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, c = lane % 16;
    const int b = blockIdx.x / a.kv_heads, hk = blockIdx.x % a.kv_heads, G = a.heads / a.kv_heads, C = a.channels;
    T* grad_q = static_cast<T*>(a.grad_q);
    if (b == a.num_graphs) {
        if (hk != 0) return;
        const int at = blockIdx.y * kThreads + threadIdx.x, step = gridDim.y * kThreads;
        if (!part) zero_rest(grad_q, a.q_ptr, b, a.num_queries, (int64_t)a.heads * C, at, step);
        if (!part && slopes) zero_rest(slopes, a.q_ptr, b, a.num_queries, (int64_t)a.heads, at, step);
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
        frag<T> q[MQ][kSteps], go[MQ][kSteps];
        const float* dist[MQ];
        float slope[MQ], lse[MQ], D[MQ];
        int limit[MQ];
        SlopeSums sums[MQ];
        f32x4 acc[MQ][CP / 16];
#pragma unroll
        for (int t = 0; t < MQ; ++t) {
            const int64_t row = min(row0 + 16 * t + c, rows - 1);
            const int i = (int)(row / G), h = hk * G + (int)(row % G);
            const int64_t at = (qs.at + i) * a.heads + h;
            const T* p = static_cast<const T*>(a.q) + (qs.at + i) * a.q_row + h * a.q_head;
            const T *po = static_cast<const T*>(a.out) + at * C, *pg = static_cast<const T*>(a.grad_out) + at * C;
            float dot = 0.0f;
#pragma unroll
            for (int s = 0; s < kSteps; ++s) {
                const bool in = 32 * s + 8 * g < C;
                q[t][s] = in ? load_frag(p + 32 * s + 8 * g) : zero_frag<T>();
                go[t][s] = in ? load_frag(pg + 32 * s + 8 * g) : zero_frag<T>();
                const frag<T> o = in ? load_frag(po + 32 * s + 8 * g) : zero_frag<T>();
#pragma unroll
                for (int e = 0; e < 8; ++e) dot = __builtin_fmaf((float)go[t][s][e], (float)o[e], dot);
            }
            D[t] = column_sum(dot);
            slope[t] = a.slope ? -a.slope[h] : 0.0f;
            dist[t] = a.dist ? a.dist + b * a.dist_graph + i * a.dist_row : nullptr;
            limit[t] = !a.dist ? ks.n : i < a.dist_rows ? min(ks.n, a.dist_cols) : 0;
            lse[t] = a.lse[at];
            if (lse[t] == -INFINITY) lse[t] = INFINITY;   // an empty row: every probability comes out as zero
            if (blockIdx.z == 0 && g == 0 && row0 + 16 * t + c < rows) dots[at] = D[t];
            sums[t] = {0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) acc[t][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
                const bool cut = !a.dist && j0 + KT > ks.n;
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float z = s[t][n][r], slack = 1.0f;
                        if (a.cap > 0.0f) {
                            const float th = tanh_of<T>(z, mul);
                            z = a.cap * th;
                            slack = __builtin_fmaf(-th, th, 1.0f);
                        } else {
                            z = z * mul;
                        }
                        bool seen = !cut || j0 + 16 * n + 4 * g + r < ks.n;
                        float dd = 0.0f;
                        if (a.dist) {
                            dd = d[t][n][r];
                            seen = finite(dd);
                            z = __builtin_fmaf(slope[t], dd, z);
                        }
                        const float p = seen ? exp2_fast(__builtin_fmaf(z, kLog2e, -lse[t])) : 0.0f;
                        const float v = seen ? p * (gp[t][n][r] - D[t]) : 0.0f;
                        if (a.slope) {
                            dd = seen ? dd : 0.0f;
                            sums[t].t += v;
                            sums[t].pd = __builtin_fmaf(p, dd, sums[t].pd);
                            sums[t].td = __builtin_fmaf(v, dd, sums[t].td);
                        }
                        u[t][n / 2][4 * (n % 2) + r] = (T)(v * slack);   // rounded to the type for the product with k
                    }
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
            const int64_t row = row0 + 16 * t + c;
            const float st = column_sum(sums[t].t), spd = column_sum(sums[t].pd), std_ = column_sum(sums[t].td);
            if (row >= rows) continue;
            const int i = (int)(row / G), h = hk * G + (int)(row % G);
            const int64_t all = a.num_queries * a.heads, at = (qs.at + i) * a.heads + h;
            if (part) {
                const int64_t mine = blockIdx.z * all + at;
                float* stat = part + (int64_t)gridDim.z * all * C;
                if (slopes && g == 0) {
                    stat[3 * mine] = st;
                    stat[3 * mine + 1] = spd;
                    stat[3 * mine + 2] = std_;
                }
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) *reinterpret_cast<f32x4*>(part + mine * C + 16 * x + 4 * g) = acc[t][x];
            } else {
                if (slopes && g == 0) slopes[at] = __builtin_fmaf(st, spd, -std_);
#pragma unroll
                for (int x = 0; x < CP / 16; ++x)
                    if (16 * x + 4 * g < C) {
                        typedef T T4 __attribute__((ext_vector_type(4)));
                        T4 y;
#pragma unroll
                        for (int r = 0; r < 4; ++r) y[r] = (T)(acc[t][x][r] * a.scale);
                        *reinterpret_cast<T4*>(grad_q + at * C + 16 * x + 4 * g) = y;
                    }
            }
        }
    }
}

template <typename T, int CP, int MK, int WAVES, int RT>
__global__ void __launch_bounds__(kWave* WAVES) attention_bwd_kv_kernel(Args a, const float* dots, float* part) {
    constexpr int kThreads = kWave * WAVES, kKeys = 16 * MK * WAVES, kSteps = CP / 32, kTiles = RT / 16;
    __shared__ __attribute__((aligned(16))) T q_tile[RT * kRow<T, CP>], go_tile[RT * kRow<T, CP>];
    __shared__ __attribute__((aligned(16))) float row_lse[RT], row_D[RT], row_slope[RT];
    __shared__ __attribute__((aligned(16))) int64_t row_dist[RT];
    const int lane = threadIdx.x % kWave, w = threadIdx.x / kWave, g = lane / 16, c = lane % 16;
    const int b = blockIdx.x / a.kv_heads, hk = blockIdx.x % a.kv_heads, G = a.heads / a.kv_heads, C = a.channels;
    T *grad_k = static_cast<T*>(a.grad_k), *grad_v = static_cast<T*>(a.grad_v);
    if (b == a.num_graphs) {
        if (hk != 0 || part) return;
        const int at = blockIdx.y * kThreads + threadIdx.x, step = gridDim.y * kThreads;
        zero_rest(grad_k, a.k_ptr, b, a.num_nodes, (int64_t)a.kv_heads * C, at, step);
        zero_rest(grad_v, a.k_ptr, b, a.num_nodes, (int64_t)a.kv_heads * C, at, step);
        return;
    }
    const Span qs = span(a.q_ptr, b, a.num_queries), ks = span(a.k_ptr, b, a.num_nodes);
    const int64_t rows = (int64_t)qs.n * G;
    const int64_t rows_each = ((rows + RT - 1) / RT + gridDim.z - 1) / gridDim.z * RT;
    const int64_t first = min(rows, blockIdx.z * rows_each), last = min(rows, first + rows_each);
    const float mul = a.cap > 0.0f ? a.scale / a.cap : a.scale;

    for (int64_t tile = blockIdx.y; tile * kKeys < ks.n; tile += gridDim.y) {
        const int key0 = (int)tile * kKeys + w * 16 * MK;
        frag<T> k[MK][kSteps], v[MK][kSteps];
        const float* dist[MK];
        f32x4 gk[MK][CP / 16], gv[MK][CP / 16];
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
            dist[t] = a.dist && j < a.dist_cols ? a.dist + b * a.dist_graph + j : nullptr;
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) gk[t][x] = gv[t][x] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        Staged<T, CP, RT, kThreads> q_next, go_next;
        float next_lse = 0.0f, next_D = 0.0f, next_slope = 0.0f;
        int64_t next_dist = -1;
        auto fetch = [&](int64_t r0) {
            q_next.load(C, [&](int x) -> const T* {
                const int64_t row = r0 + x;
                if (row >= rows) return nullptr;
                const int64_t i = G == 1 ? row : row / G, h = hk * G + (row - i * G);
                return static_cast<const T*>(a.q) + (qs.at + i) * a.q_row + h * a.q_head;
            });
            go_next.load(C, [&](int x) -> const T* {
                const int64_t row = r0 + x;
                if (row >= rows) return nullptr;
                const int64_t i = G == 1 ? row : row / G, h = hk * G + (row - i * G);
                return static_cast<const T*>(a.grad_out) + ((qs.at + i) * a.heads + h) * C;
            });
            const int64_t row = r0 + threadIdx.x;
            next_lse = INFINITY;   // rows that are not there, and empty ones: every probability comes out as zero
            next_D = next_slope = 0.0f;
            next_dist = -1;
            if (threadIdx.x < RT && row < rows) {
                const int64_t i = G == 1 ? row : row / G, h = hk * G + (row - i * G), at = (qs.at + i) * a.heads + h;
                if (a.lse[at] != -INFINITY) {
                    next_lse = a.lse[at];
                    next_D = dots[at];
                }
                next_slope = a.slope ? -a.slope[h] : 0.0f;
                if (i < a.dist_rows) next_dist = i * a.dist_row;
            }
        };
        if (first < last) fetch(first);
        for (int64_t r0 = first; r0 < last; r0 += RT) {
            __syncthreads();
            q_next.store(q_tile);
            go_next.store(go_tile);
            if (threadIdx.x < RT) {
                row_lse[threadIdx.x] = next_lse;
                row_D[threadIdx.x] = next_D;
                row_slope[threadIdx.x] = next_slope;
                row_dist[threadIdx.x] = next_dist;
            }
            __syncthreads();
            if (r0 + RT < last) fetch(r0 + RT);
            if (key0 >= ks.n) continue;
            f32x4 d[MK][kTiles];
            if (a.dist) {
#pragma unroll
                for (int n = 0; n < kTiles; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int64_t at = row_dist[16 * n + 4 * g + r];
#pragma unroll
                        for (int t = 0; t < MK; ++t) d[t][n][r] = dist[t] && at >= 0 ? dist[t][at] : INFINITY;
                    }
            }
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
#pragma unroll
            for (int n = 0; n < kTiles; ++n) {
                const f32x4 lse = *reinterpret_cast<const f32x4*>(row_lse + 16 * n + 4 * g);
                const f32x4 D = *reinterpret_cast<const f32x4*>(row_D + 16 * n + 4 * g);
                const f32x4 slope = *reinterpret_cast<const f32x4*>(row_slope + 16 * n + 4 * g);
#pragma unroll
                for (int t = 0; t < MK; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float z = s[t][n][r], slack = 1.0f;
                        if (a.cap > 0.0f) {
                            const float th = tanh_of<T>(z, mul);
                            z = a.cap * th;
                            slack = __builtin_fmaf(-th, th, 1.0f);
                        } else {
                            z = z * mul;
                        }
                        bool seen = true;
                        if (a.dist) {
                            seen = finite(d[t][n][r]);
                            z = __builtin_fmaf(slope[r], d[t][n][r], z);
                        }
                        const float e = seen ? exp2_fast(__builtin_fmaf(z, kLog2e, -lse[r])) : 0.0f;
                        const float x = seen ? e * (gp[t][n][r] - D[r]) * slack : 0.0f;
                        p[t][n / 2][4 * (n % 2) + r] = (T)e;   // both rounded to the type for their products
                        u[t][n / 2][4 * (n % 2) + r] = (T)x;
                    }
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
#pragma unroll
            for (int x = 0; x < CP / 16; ++x) {
                const int ch = 16 * x + 4 * g;
                if (ch >= C) continue;
                if (part) {   // [split][k, v][node, head, channel]
                    float* mine = part + ((int64_t)blockIdx.z * 2 * all + at) * C + ch;
                    *reinterpret_cast<f32x4*>(mine) = gk[t][x];
                    *reinterpret_cast<f32x4*>(mine + all * C) = gv[t][x];
                } else {
                    typedef T T4 __attribute__((ext_vector_type(4)));
                    T4 y, z;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        y[r] = (T)(gk[t][x][r] * a.scale);
                        z[r] = (T)gv[t][x][r];
                    }
                    *reinterpret_cast<T4*>(grad_k + at * C + ch) = y;
                    *reinterpret_cast<T4*>(grad_v + at * C + ch) = z;
                }
            }
        }
    }
}

// out[e] = scale x the splits' sum of part[e] in their order, four elements a thread; rows of no graph: zeros
template <typename T>
__global__ void __launch_bounds__(256)
    sum_splits_kernel(const float* part, int splits, int64_t stride, int64_t n, int64_t width, const int64_t* ptr,
                      int graphs, int64_t rows, float scale, T* out) {
    const Span s = all_rows(ptr, graphs, rows);
    const int64_t step = (int64_t)gridDim.x * 256 * 4;
    for (int64_t e = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < n; e += step) {
        f32x4 v{0.0f, 0.0f, 0.0f, 0.0f};
        if (e >= s.at * width && e < (s.at + s.n) * width)
            for (int k = 0; k < splits; ++k) v = v + *reinterpret_cast<const f32x4*>(part + k * stride + e);
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 y;
#pragma unroll
        for (int r = 0; r < 4; ++r) y[r] = (T)(v[r] * scale);
        *reinterpret_cast<T4*>(out + e) = y;
    }
}

// each row's slope gradient from its splits' sums
__global__ void __launch_bounds__(256)
    join_slopes_kernel(Args a, const float* stat, int splits, float* slopes) {
    const Span s = all_rows(a.q_ptr, a.num_graphs, a.num_queries);
    const int64_t all = a.num_queries * a.heads;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < all; at += (int64_t)gridDim.x * 256) {
        float t = 0.0f, pd = 0.0f, td = 0.0f;
        const int64_t row = at / a.heads;
        if (row >= s.at && row < s.at + s.n)
            for (int k = 0; k < splits; ++k) {
                t += stat[3 * (k * all + at)];
                pd += stat[3 * (k * all + at) + 1];
                td += stat[3 * (k * all + at) + 2];
            }
        slopes[at] = __builtin_fmaf(t, pd, -td);
    }
}

// out[h] = the sum of column h in a fixed order: threads over the rows, then a tree
__global__ void __launch_bounds__(1024) slope_sum_kernel(const float* slopes, int64_t rows, int heads, float* out) {
    __shared__ float part[16];
    const int h = blockIdx.x, lane = threadIdx.x % kWave, w = threadIdx.x / kWave;
    float v = 0.0f;
    for (int64_t r = threadIdx.x; r < rows; r += 1024) v += slopes[r * heads + h];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (lane == 0) part[w] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < 16; ++k) v += part[k];
        out[h] = v;
    }
}

// How both passes are cut, as in the forward: one wave where a (graph, head) has up to 32 rows to keep, four
// otherwise; the axis that is run over is split where the workgroups would not fill the 256 compute units.
struct Cut {
    bool narrow;
    int64_t tiles;
    int splits;
};
Cut cut(int64_t kept, int64_t run, int64_t units, int64_t row_bytes) {
    Cut c;
    c.narrow = kept <= 32;
    const int64_t each = c.narrow ? 32 : 128;
    c.tiles = std::max<int64_t>(1, std::min<int64_t>((kept + each - 1) / each, 65535));
    const int64_t blocks = std::max<int64_t>(1, units * c.tiles), want = c.narrow ? 2048 : 512;
    const int64_t most = std::min<int64_t>(64, std::min(run / 256, (int64_t(1) << 28) / std::max<int64_t>(1, row_bytes)));
    c.splits = (int)std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, most));
    return c;
}
Cut cut_q(const Args& a) {
    const int64_t G = a.heads / a.kv_heads;
    return cut(std::min(a.max_queries, a.num_queries) * G, std::min(a.max_nodes, a.num_nodes),
               (int64_t)a.num_graphs * a.kv_heads, a.num_queries * a.heads * (a.channels + 3) * 4);
}
Cut cut_kv(const Args& a) {
    const int64_t G = a.heads / a.kv_heads;
    return cut(std::min(a.max_nodes, a.num_nodes), std::min(a.max_queries, a.num_queries) * G,
               (int64_t)a.num_graphs * a.kv_heads, a.num_nodes * a.kv_heads * a.channels * 8);
}
size_t split_floats_q(const Args& a, const Cut& c) {
    return c.splits > 1 ? (size_t)c.splits * a.num_queries * a.heads * (a.channels + 3) : 0;
}
size_t split_floats_kv(const Args& a, const Cut& c) {
    return c.splits > 1 ? (size_t)c.splits * a.num_nodes * a.kv_heads * a.channels * 2 : 0;
}
// each row's <go, out> and slope gradient, then the splits of one pass after the other
size_t row_floats(const Args& a) { return ((size_t)a.num_queries * a.heads * 2 + 3) / 4 * 4; }

template <typename T, int CP>
void launch(const Args& a, hipStream_t stream) {
    float *dots = static_cast<float*>(a.workspace), *slopes = dots + a.num_queries * a.heads;
    float *row_slopes = a.grad_slope && a.slope ? slopes : nullptr, *split = dots + row_floats(a);
    const unsigned gx = (unsigned)((a.num_graphs + 1) * (int64_t)a.kv_heads);
    if (a.num_queries > 0) {
        const Cut c = cut_q(a);
        float* part = c.splits > 1 ? split : nullptr;
        const dim3 grid(gx, (unsigned)c.tiles, c.splits);
        if (c.narrow)
            hipLaunchKernelGGL((attention_bwd_q_kernel<T, CP, 2, 1, 32>), grid, dim3(64), 0, stream, a, dots, row_slopes,
                               part);
        else
            hipLaunchKernelGGL((attention_bwd_q_kernel<T, CP, 2, 4, 32>), grid, dim3(256), 0, stream, a, dots, row_slopes,
                               part);
        if (part) {
            const int64_t n = a.num_queries * a.heads * a.channels;
            const unsigned blocks = (unsigned)std::min<int64_t>(2048, (n / 4 + 255) / 256);
            hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks), dim3(256), 0, stream, part, c.splits, n, n,
                               (int64_t)a.heads * a.channels, a.q_ptr, a.num_graphs, a.num_queries, a.scale,
                               static_cast<T*>(a.grad_q));
            if (row_slopes)
                hipLaunchKernelGGL(join_slopes_kernel, dim3((unsigned)std::min<int64_t>(2048, (a.num_queries * a.heads + 255) / 256)),
                                   dim3(256), 0, stream, a, part + c.splits * n, c.splits, row_slopes);
        }
    }
    if (a.num_nodes > 0) {
        const Cut c = cut_kv(a);
        float* part = c.splits > 1 ? split : nullptr;
        const dim3 grid(gx, (unsigned)c.tiles, c.splits);
        if (c.narrow)
            hipLaunchKernelGGL((attention_bwd_kv_kernel<T, CP, 2, 1, 32>), grid, dim3(64), 0, stream, a, dots, part);
        else
            hipLaunchKernelGGL((attention_bwd_kv_kernel<T, CP, 2, 4, 32>), grid, dim3(256), 0, stream, a, dots, part);
        if (part) {
            const int64_t n = a.num_nodes * a.kv_heads * a.channels, width = (int64_t)a.kv_heads * a.channels;
            const unsigned blocks = (unsigned)std::min<int64_t>(2048, (n / 4 + 255) / 256);
            hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks), dim3(256), 0, stream, part, c.splits, 2 * n, n, width,
                               a.k_ptr, a.num_graphs, a.num_nodes, a.scale, static_cast<T*>(a.grad_k));
            hipLaunchKernelGGL(sum_splits_kernel<T>, dim3(blocks), dim3(256), 0, stream, part + n, c.splits, 2 * n, n,
                               width, a.k_ptr, a.num_graphs, a.num_nodes, 1.0f, static_cast<T*>(a.grad_v));
        }
    }
    if (row_slopes)
        hipLaunchKernelGGL(slope_sum_kernel, dim3(a.heads), dim3(1024), 0, stream, slopes, a.num_queries, a.heads,
                           a.grad_slope);
}

}  // namespace

size_t attention_bwd_workspace(const trx_node_attention_args& a) {
    return (row_floats(a) + std::max(split_floats_q(a, cut_q(a)), split_floats_kv(a, cut_kv(a)))) * sizeof(float);
}

hipError_t launch_attention_bwd(const trx_node_attention_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (a.channels <= 32)
            launch<T, 32>(a, stream);
        else if (a.channels <= 64)
            launch<T, 64>(a, stream);
        else
            launch<T, 128>(a, stream);
        return hipGetLastError();
    });
}

}  // namespace trx
