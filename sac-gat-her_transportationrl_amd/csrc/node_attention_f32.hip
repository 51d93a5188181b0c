// node_attention_f32.hip -- node_attention's kernels for float.
#include "node_attention_bwd.h"
#include "node_attention_fwd.h"

namespace trx {
template hipError_t launch_attention_fwd<float>(const trx_node_attention_args&, hipStream_t);
template hipError_t launch_attention_bwd<float>(const trx_node_attention_args&, hipStream_t);
}  // namespace trx
