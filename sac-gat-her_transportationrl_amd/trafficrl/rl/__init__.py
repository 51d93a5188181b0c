from .policy import ActionLogProbs, action_log_probs  # noqa: F401
from .sac import Actor, Critic, DiscreteSAC, SACOutput, scatter_sum, segment_softmax  # noqa: F401
