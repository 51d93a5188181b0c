// node_attention_f16.hip -- node_attention's kernels for _Float16.
#include "node_attention_bwd.h"
#include "node_attention_fwd.h"

namespace trx {
template hipError_t launch_attention_fwd<_Float16>(const trx_node_attention_args&, hipStream_t);
template hipError_t launch_attention_bwd<_Float16>(const trx_node_attention_args&, hipStream_t);
}  // namespace trx
