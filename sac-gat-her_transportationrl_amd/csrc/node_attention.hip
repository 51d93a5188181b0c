// node_attention.hip -- softmax attention of query rows over the nodes of their
// own network (include/trafficrl.h, trx_node_attention_*): how its passes are
// cut into workgroups.  Kernels: node_attention_fwd.h, node_attention_bwd.h.
#include <algorithm>

#include "node_attention.h"

namespace trx {

namespace {

// kept, run: the rows that are kept and run over of the largest (graph, key/value head); all: the kept rows of all
// graphs; heads: key/value heads; row_bytes: a split's part of the workspace.  Up to 32 kept rows, one wave has them
// all and a workgroup of four would idle.  The axis that is run over is split where the tiles that there are about
// leave compute units without work, into pieces of at least `least` rows (a piece costs its accumulator's round trip),
// up to 64 and 256 MB.  512 workgroups of four waves, two to a compute unit: 4001 nodes, 8 heads of 64, forward and
// backward together 396 us, against 587 us with 256 and 434 us with 1024 (compared side by side; the passes have
// changed by a few percent since).
AttentionCut cut(int64_t kept, int64_t run, int64_t all, int64_t graphs, int64_t heads, int64_t row_bytes, int wide,
                 int least) {
    AttentionCut c;
    const int64_t units = std::max<int64_t>(1, graphs * heads);
    c.narrow = kept <= 32;
    c.mq = c.narrow && kept <= 16 ? 1 : 2;
    const int64_t each = c.narrow ? 16 * c.mq : wide;
    // Workgroups of no rows cost 0.9 us a thousand: no more of them than four times those that can have rows, or 2^17
    // in all; a graph's further tiles are looped over.  4096 graphs of 24 nodes and 4 heads whose
    // largest is not given: forward 360 us, 7525 with up to 2^23 workgroups, 43 where it is given.
    const int64_t filled = heads * (all / each + graphs);
    const int64_t limit = std::min<int64_t>(1 << 23, std::max<int64_t>(1 << 17, 4 * filled));
    c.tiles = std::max<int64_t>(1, std::min<int64_t>((kept + each - 1) / each, limit / units));
    const int64_t blocks = std::max<int64_t>(1, std::min(units * c.tiles, filled));
    const int64_t want = c.narrow ? 2048 : 512;
    const int64_t most = std::min<int64_t>(64, std::min(run / least, (int64_t(1) << 28) / std::max<int64_t>(1, row_bytes)));
    c.splits = (int)std::max<int64_t>(1, std::min((want + blocks - 1) / blocks, most));
    c.splits = (int)std::max<int64_t>(1, std::min<int64_t>(c.splits, (1 << 23) / (units * c.tiles)));   // the grid x 256 < 2^32
    return c;
}
int wide_rows(const Args& a) { return a.dtype == 0 && a.channels > 64 ? 64 : 128; }
int wide_bwd(const Args& a) { return a.channels > 64 ? 64 : 128; }

}  // namespace

AttentionCut cut_fwd(const trx_node_attention_args& a) {
    const int64_t G = a.heads / a.kv_heads;
    return cut(std::min(a.max_queries, a.num_queries) * G, std::min(a.max_nodes, a.num_nodes),
               a.num_queries * G, a.num_graphs, a.kv_heads, a.num_queries * a.heads * (a.channels + 2) * 4, wide_rows(a), 64);
}
AttentionCut cut_bwd_q(const trx_node_attention_args& a) {
    const int64_t G = a.heads / a.kv_heads;
    return cut(std::min(a.max_queries, a.num_queries) * G, std::min(a.max_nodes, a.num_nodes),
               a.num_queries * G, a.num_graphs, a.kv_heads, a.num_queries * a.heads * (a.channels + 4) * 4, wide_bwd(a), 256);
}
AttentionCut cut_bwd_kv(const trx_node_attention_args& a) {
    const int64_t G = a.heads / a.kv_heads;
    return cut(std::min(a.max_nodes, a.num_nodes), std::min(a.max_queries, a.num_queries) * G,
               a.num_nodes, a.num_graphs, a.kv_heads, a.num_nodes * a.kv_heads * a.channels * 8, wide_bwd(a), 256);
}

// each row's <go, out>, inverse of its weights' sum and slope gradient, the slope chunks' sums; the splits of one pass
// after the other follow
size_t attention_row_floats(const trx_node_attention_args& a) {
    return ((size_t)a.num_queries * a.heads * 3 + (size_t)kSlopeChunks * a.heads + 3) / 4 * 4;
}

size_t node_attention_workspace(const trx_node_attention_args& a, bool backward) {
    if (!backward) {
        const int splits = cut_fwd(a).splits;
        return splits > 1 ? (size_t)splits * a.num_queries * a.heads * (a.channels + 2) * sizeof(float) : 0;
    }
    const int sq = cut_bwd_q(a).splits, skv = cut_bwd_kv(a).splits;
    const size_t q = sq > 1 ? (size_t)sq * a.num_queries * a.heads * (a.channels + 4) : 0;
    const size_t kv = skv > 1 ? (size_t)skv * a.num_nodes * a.kv_heads * a.channels * 2 : 0;
    return (attention_row_floats(a) + std::max(q, kv)) * sizeof(float);
}

hipError_t launch_node_attention_fwd(const trx_node_attention_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) { return launch_attention_fwd<std::remove_pointer_t<decltype(t)>>(a, stream); });
}

hipError_t launch_node_attention_bwd(const trx_node_attention_args& a, hipStream_t stream) {
    return by_dtype(a.dtype, [&](auto* t) { return launch_attention_bwd<std::remove_pointer_t<decltype(t)>>(a, stream); });
}

}  // namespace trx
