from .attention import node_attention  # noqa: F401
from .dropout import dropout_add  # noqa: F401
from .gat_encoder import GATConv, GATEncoder, global_max_pool, global_mean_pool  # noqa: F401
