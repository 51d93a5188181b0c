// node_attention_bf16.hip -- node_attention's kernels for __bf16.
#include "node_attention_bwd.h"
#include "node_attention_fwd.h"

namespace trx {
template hipError_t launch_attention_fwd<__bf16>(const trx_node_attention_args&, hipStream_t);
template hipError_t launch_attention_bwd<__bf16>(const trx_node_attention_args&, hipStream_t);
}  // namespace trx
