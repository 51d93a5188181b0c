"""Discrete SAC with GAT encoders (src/rl/sac.py:23-291).

Same classes, constructor arguments, forward signatures, update() batch tuple,
returned metrics and checkpoint dict keys as the reference, so
src/train.py-style callers and old checkpoints keep working.  Changes are in
how the work maps to MI355X:

* the edge MLP's first layer on cat([h_src, h_dst, e, ctx]) (sac.py:42-43,
  1030 -> hidden) is evaluated as h @ W_src^T gathered at src + h @ W_dst^T at
  dst + e @ W_e^T + (ctx @ W_ctx^T)[graph]: algebraically identical, but the
  big GEMM runs per NODE (B*N rows) instead of per EDGE (B*E rows) -- 6x fewer
  FLOPs on Sioux Falls, all in MFMA GEMMs;
* PyG softmax / torch_scatter.scatter_sum over edge_batch become segment ops
  (index_add / dense [B,E] reshapes when every graph has the same links);
* update() runs the three independent backward passes (critic, actor, alpha:
  none depends on another's optimizer step, sac.py:204-243) before any step,
  so multi-GPU data parallelism needs ONE bucketed all-reduce of all
  gradients per update (`grad_sync`, RCCL over xGMI) instead of three.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Callable, Dict, Optional, Tuple

import numpy as np
import torch
from torch import nn
import torch.nn.functional as F

from ..models import fused
from ..models.gat_encoder import GATEncoder, is_regular_batch
from ..models.skinny import regular_gather, skinny_linear, splitk_linear
from ..models.tensor_cache import TensorKeyed, owner
from .policy import ActionLogProbs, action_log_probs


@dataclass
class SACOutput:
    action: int
    log_prob: torch.Tensor
    probs: torch.Tensor


def scatter_sum(src: torch.Tensor, index: torch.Tensor, num: int, regular: bool = False) -> torch.Tensor:
    """torch_scatter.scatter_sum; `regular` (index = arange(num) repeated
    equally, contiguous) reduces a [num, k] view: no atomics, deterministic."""
    if regular:
        return src.view(num, -1, *src.shape[1:]).sum(1)
    out = torch.zeros(num, *src.shape[1:], device=src.device, dtype=src.dtype)
    return out.index_add_(0, index, src)


class _SmallLN(torch.autograd.Function):
    """input_layer_norm on the GPU: one thread per row each way
    (csrc/small_ln.hip) instead of ~8 launches forward and ~12 backward."""

    @staticmethod
    def forward(ctx, x, w, b, eps: float):
        from .. import _lib
        L = _lib.load()
        x = x.float().contiguous()
        N, d = x.shape
        wc, bc = w.detach().float().contiguous(), b.detach().float().contiguous()
        y = torch.empty_like(x)
        stats = torch.empty(N, 2, device=x.device, dtype=torch.float32)
        _lib.check(L.trx_small_ln_forward(N, d, _lib.ptr(x), _lib.ptr(wc), _lib.ptr(bc), float(eps), _lib.ptr(y),
                                          _lib.ptr(stats), _lib.stream_ptr(x.device)), "trx_small_ln_forward")
        ctx.save_for_backward(x, wc, stats)
        return y

    @staticmethod
    def backward(ctx, gy):
        from .. import _lib
        L = _lib.load()
        x, w, stats = ctx.saved_tensors
        N, d = x.shape
        gy = gy.float().contiguous()
        gx = torch.empty_like(x)
        gwb = torch.empty(2, d, device=x.device, dtype=torch.float32)
        ws = torch.empty(max(1, int(L.trx_small_ln_workspace_floats(N, d))), device=x.device, dtype=torch.float32)
        _lib.check(L.trx_small_ln_backward(N, d, _lib.ptr(gy), _lib.ptr(x), _lib.ptr(w), _lib.ptr(stats),
                                           _lib.ptr(gx), _lib.ptr(gwb), _lib.ptr(ws), _lib.stream_ptr(x.device)),
                   "trx_small_ln_backward")
        return gx, gwb[0], gwb[1], None


def input_layer_norm(ln: nn.LayerNorm, x: torch.Tensor) -> torch.Tensor:
    """nn.LayerNorm over the 4-/6-wide raw node/edge features (sac.py:27-28, 36-37).
    torch's generic row kernel spends one workgroup per row there (~0.9 ms per
    acting call at 4096 graphs); on the GPU one thread per row (_SmallLN),
    elsewhere the same math as a handful of vectorised ops.  Wide rows keep
    the library kernel."""
    if x.size(-1) >= 32:
        return ln(x)
    if x.is_cuda and x.dim() == 2 and x.size(-1) <= 8 and ln.weight is not None:
        return _SmallLN.apply(x, ln.weight, ln.bias, ln.eps)
    xf = x.float()
    mu = xf.mean(-1, keepdim=True)
    d = xf - mu
    var = (d * d).mean(-1, keepdim=True)
    return d * torch.rsqrt(var + ln.eps) * ln.weight + ln.bias


def segment_softmax(logits: torch.Tensor, index: torch.Tensor, num: int, per_segment: Optional[int] = None):
    """torch_geometric.utils.softmax: exp(x - max_seg) / (sum_seg + 1e-16)."""
    if per_segment is not None and logits.numel() == num * per_segment:
        x = logits.view(num, per_segment)
        ex = torch.exp(x - x.amax(dim=1, keepdim=True))
        return (ex / (ex.sum(dim=1, keepdim=True) + 1e-16)).view(-1)
    mx = torch.full((num,), float("-inf"), device=logits.device, dtype=logits.dtype)
    mx = mx.scatter_reduce(0, index, logits, reduce="amax", include_self=True)
    ex = torch.exp(logits - mx[index])
    return ex / (scatter_sum(ex, index, num)[index] + 1e-16)


_edge_layout_cache = TensorKeyed()


def is_regular_edges(edge_index: torch.Tensor, batch: torch.Tensor, num_graphs: int) -> bool:
    """True when the edges of graph b are the b-th of num_graphs equal
    contiguous blocks (PyG Batch of same-size graphs).  Checked once per
    (edge_index, batch) pair and cached, so steady-state calls never sync."""
    E = edge_index.shape[1]
    if num_graphs <= 0 or E % num_graphs:
        return False
    key = (edge_index.data_ptr(), edge_index._version, batch.data_ptr(), batch._version, E, num_graphs)
    r = _edge_layout_cache.get(key)
    if r is None:
        eb = batch[edge_index[0]].long()
        r = bool(torch.equal(eb, torch.arange(num_graphs, device=eb.device).repeat_interleave(E // num_graphs)))
        _edge_layout_cache.put(key, (owner(edge_index), owner(batch)), r)
    return r


_regular_cache = TensorKeyed()


def regular_layout(edge_index: torch.Tensor, batch: torch.Tensor, num_graphs: int):
    """(B, src_local, dst_local) when every graph of the batch has the same
    edge list (local node ids) in its own contiguous block, else None.
    Checked once per (edge_index, batch) pair and cached."""
    if not is_regular_edges(edge_index, batch, num_graphs) or not is_regular_batch(batch, num_graphs):
        return None
    key = (edge_index.data_ptr(), edge_index._version, batch.data_ptr(), batch._version, num_graphs)
    r = _regular_cache.get(key)
    if r is None:
        B, E, N = num_graphs, edge_index.shape[1], batch.numel()
        m, n = E // B, N // B
        if N % B:
            r = False
        else:
            loc = edge_index.long() - (torch.arange(B, device=edge_index.device) * n).repeat_interleave(m)
            loc = loc.view(2, B, m)
            r = (B, loc[0, 0].contiguous(), loc[1, 0].contiguous()) if bool((loc == loc[:, :1]).all()) else False
        _regular_cache.put(key, (owner(edge_index), owner(batch)), r)
    return r if r is not False else None


@torch.no_grad()
def clip_grad_norm_listwise_(params, max_norm: float):
    """torch.nn.utils.clip_grad_norm_ with the reference's list semantics made
    deterministic.  The reference clips list(critic1.parameters()) +
    list(critic2.parameters()) (sac.py:224-227); with a shared critic encoder
    that list holds the encoder's gradients twice.  Sequentially (torch's
    per-tensor loop) each duplicate is counted twice in the norm and scaled
    twice; torch's fused CUDA path instead scales the same tensor from two
    workgroups at once (a read-modify-write race: g*c or g*c^2).  This helper
    always applies the sequential semantics."""
    uniq, count = [], {}
    for p in params:
        if p.grad is not None:
            if id(p) not in count:
                uniq.append(p)
                count[id(p)] = 0
            count[id(p)] += 1
    if not uniq:
        return torch.zeros(())
    # one multi-tensor norm launch instead of a kernel per tensor
    norms = torch.stack(torch._foreach_norm([p.grad for p in uniq], 2.0))
    if all(count[id(p)] == 1 for p in uniq):
        total = torch.linalg.vector_norm(norms, 2.0)
    else:
        mult = torch.tensor([float(count[id(p)]) for p in uniq], device=norms.device)
        total = torch.sqrt((norms * norms * mult).sum())
    coef = torch.clamp(max_norm / (total + 1e-6), max=1.0)
    for n in sorted(set(count.values())):
        group = [p.grad for p in uniq if count[id(p)] == n]
        torch._foreach_mul_(group, coef if n == 1 else coef ** n)
    return total


FUSED_INFERENCE = True   # module switch (tests compare both paths)
FUSED_EDGE_TRAIN = True  # training-path edge scorer kernels (tests compare both paths)
FUSED_UPDATE = True      # whole-update fused path (rl/fused_update.py) for regular bf16 batches
FLAT_ADAM = True         # optimizer step over the fused update's flat gradient buffer (rl/flat_adam.py)


def _fused_topology(encoder, node_x, edge_index, batch, B, head=None):
    """Topology for the fused inference kernels, or None -> general path.
    Taken only without autograd, under bf16 autocast, on the GPU."""
    if (not FUSED_INFERENCE or torch.is_grad_enabled() or not node_x.is_cuda or not fused.autocast_bf16()
            or not fused.encoder_supported(encoder) or (head is not None and not fused.head_supported(head))):
        return None
    return fused.topology(edge_index, batch, B)


class _EdgeHead(nn.Module):
    """Owner of edge_mlp (state_dict keys edge_mlp.0.*, edge_mlp.2.*)."""

    def __init__(self, embed: int, edge_in: int, hidden: int):
        super().__init__()
        self.embed, self.edge_in = embed, edge_in
        self.edge_mlp = nn.Sequential(nn.Linear(embed * 4 + edge_in, hidden), nn.ReLU(), nn.Linear(hidden, 1))

    def _fused(self, node_x, edge_index, edge_attr, batch, B, mask=None, u=None):
        """Fused inference (models/fused.py) from the raw features: prologue
        (input LayerNorms + edge logits), one kernel per GAT layer, edge head
        (+ masked softmax, + one draw per graph when u is given).  None when
        the general path must run."""
        topo = _fused_topology(self.encoder, node_x, edge_index, batch, B, self)
        if topo is None or not fused.prologue_supported(self):
            return None
        x0, ea, a_all = fused.prologue(self, node_x, edge_attr, topo)
        if fused.tail_supported(self, topo):   # last layer + edge head as one MFMA kernel
            x_prev = fused.encoder_infer(self.encoder, x0, ea, topo, a_edge=a_all, upto=len(self.encoder.layers) - 1)
            return fused.tail_infer(self, x_prev, ea, a_all, topo, mask=mask, u=u)
        emb, ctx = fused.encoder_infer(self.encoder, x0, ea, topo, a_edge=a_all)
        return fused.edge_head_infer(self, emb, ctx, ea, topo, mask=mask, u=u)

    def edge_scores(self, node_emb, global_ctx, edge_attr, src, dst, edge_batch, regular=None):
        """regular = (B, src_local, dst_local) for fixed-topology batches: the
        gathers then scatter back with incidence products (models/skinny.py)."""
        W1, b1 = self.edge_mlp[0].weight, self.edge_mlp[0].bias
        d, k = self.embed, self.edge_in
        # torch.split: the backward is one cat, not a zero-fill + add per slice
        w_src, w_dst, w_e, w_ctx = torch.split(W1, [d, d, k, W1.shape[1] - 2 * d - k], dim=1)
        w_nodes = torch.cat([w_src, w_dst], 0)                        # [2H, embed]
        p = splitk_linear(node_emb, w_nodes)                          # per-node projections
        hdim = W1.shape[0]
        c = global_ctx @ w_ctx.t() + b1                               # [B, H] per-graph context
        W2, b2 = self.edge_mlp[2].weight, self.edge_mlp[2].bias
        if (FUSED_EDGE_TRAIN and regular is not None and p.is_cuda and fused.autocast_bf16() and hdim % 4 == 0
                and hdim <= 256
                and k <= 8 and node_emb.shape[0] % regular[0] == 0 and node_emb.shape[0] // regular[0] <= 64):
            # one kernel each way for the gathers, link term, context, ReLU and 256->1 product
            B = regular[0]
            return fused.edge_scores_train(p, c, edge_attr, w_e, W2, b2, src, dst, B, node_emb.shape[0] // B)
        # fp32 from the per-node GEMM's output on (the fused kernels' rounding
        # points): the link's hidden units and the 256 -> 1 product.  Under bf16
        # autocast the logits keep fp32 resolution (a graph's logits differ by
        # ~1e-2 while bf16 resolves ~1e-3 at their magnitude)
        up = lambda t: t.float() if t.dtype in (torch.bfloat16, torch.float16) else t  # noqa: E731
        pf, c = up(p), up(c)
        with torch.autocast("cuda", enabled=False):
            ew = skinny_linear(up(edge_attr), w_e)
            if regular is not None:
                B, src_l, dst_l = regular
                z = regular_gather(pf[:, :hdim], src_l, B) + regular_gather(pf[:, hdim:], dst_l, B)
                z = z + ew
                z = z + c.unsqueeze(1).expand(B, src_l.numel(), hdim).reshape(-1, hdim)
            else:
                z = pf[src, :hdim] + pf[dst, hdim:]
                z = z + ew
                z = z + c[edge_batch]
            return skinny_linear(torch.relu(z), W2, b2).squeeze(-1)


class Actor(_EdgeHead):
    def __init__(self, node_in: int, edge_in: int, hidden: int, embed: int, num_layers: int = 3):
        super().__init__(embed, edge_in, hidden)
        self.node_norm = nn.LayerNorm(node_in)
        self.edge_norm = nn.LayerNorm(edge_in)
        self.encoder = GATEncoder(node_in, hidden, embed, edge_dim=edge_in, num_layers=num_layers)

    def forward(self, node_x, edge_index, edge_attr, action_mask, batch, return_attention: bool = False,
                num_graphs: Optional[int] = None):
        B = num_graphs if num_graphs is not None else int(batch.max()) + 1
        if not return_attention:
            out = self._fused(node_x, edge_index, edge_attr, batch, B, mask=action_mask)
            if out is not None:
                logits, probs = out
                return logits, probs, None
        node_x = input_layer_norm(self.node_norm, node_x)
        edge_attr = input_layer_norm(self.edge_norm, edge_attr)
        node_emb, global_ctx, attn = self.encoder(node_x, edge_index, edge_attr, batch,
                                                  return_attention=return_attention, num_graphs=B)
        src, dst = edge_index
        edge_batch = batch[src]
        logits = self.edge_scores(node_emb, global_ctx, edge_attr, src, dst, edge_batch,
                                  regular_layout(edge_index, batch, B)).float()
        logits = logits.masked_fill(action_mask <= 0, -1e9)
        per = logits.numel() // B if is_regular_edges(edge_index, batch, B) else None
        probs = segment_softmax(logits, edge_batch, B, per)
        return logits, probs, attn


class Critic(_EdgeHead):
    def __init__(self, node_in: int, edge_in: int, hidden: int, embed: int, num_layers: int = 3,
                 encoder: GATEncoder | None = None):
        super().__init__(embed, edge_in, hidden)
        self.node_norm = nn.LayerNorm(node_in)
        self.edge_norm = nn.LayerNorm(edge_in)
        self.encoder = encoder if encoder is not None else GATEncoder(node_in, hidden, embed, edge_dim=edge_in,
                                                                      num_layers=num_layers)

    def forward(self, node_x, edge_index, edge_attr, batch, num_graphs: Optional[int] = None):
        B = num_graphs if num_graphs is not None else int(batch.max()) + 1
        out = self._fused(node_x, edge_index, edge_attr, batch, B)
        if out is not None:
            return out
        node_x = input_layer_norm(self.node_norm, node_x)
        edge_attr = input_layer_norm(self.edge_norm, edge_attr)
        node_emb, global_ctx, _ = self.encoder(node_x, edge_index, edge_attr, batch, num_graphs=B)
        src, dst = edge_index
        return self.edge_scores(node_emb, global_ctx, edge_attr, src, dst, batch[src],
                                regular_layout(edge_index, batch, B)).float()


class DiscreteSAC:
    def __init__(self, node_in: int, edge_in: int, hidden: int, embed: int, num_layers: int = 3, lr: float = 3e-4,
                 actor_lr: float | None = None, critic_lr: float | None = None, alpha_lr: float | None = None,
                 grad_clip: float | None = None, gamma: float = 0.99, target_tau: float = 0.005,
                 target_entropy: float = None, target_entropy_ratio: float = 0.1, alpha_init: float = 0.1,
                 share_critic_encoder: bool = True, device=None, amp_dtype: Optional[torch.dtype] = None,
                 capturable: bool = False, fp32_actor: bool = True):
        self.actor = Actor(node_in, edge_in, hidden, embed, num_layers=num_layers)
        self.share_critic_encoder = share_critic_encoder
        if share_critic_encoder:
            self.critic_encoder = GATEncoder(node_in, hidden, embed, edge_dim=edge_in, num_layers=num_layers)
            self.target_encoder = GATEncoder(node_in, hidden, embed, edge_dim=edge_in, num_layers=num_layers)
            self.critic1 = Critic(node_in, edge_in, hidden, embed, num_layers, encoder=self.critic_encoder)
            self.critic2 = Critic(node_in, edge_in, hidden, embed, num_layers, encoder=self.critic_encoder)
            self.target1 = Critic(node_in, edge_in, hidden, embed, num_layers, encoder=self.target_encoder)
            self.target2 = Critic(node_in, edge_in, hidden, embed, num_layers, encoder=self.target_encoder)
            self.target_encoder.load_state_dict(self.critic_encoder.state_dict())
        else:
            self.critic1 = Critic(node_in, edge_in, hidden, embed, num_layers)
            self.critic2 = Critic(node_in, edge_in, hidden, embed, num_layers)
            self.target1 = Critic(node_in, edge_in, hidden, embed, num_layers)
            self.target2 = Critic(node_in, edge_in, hidden, embed, num_layers)
            self.target1.load_state_dict(self.critic1.state_dict())
            self.target2.load_state_dict(self.critic2.state_dict())
        if device is not None:
            for m in (self.actor, self.critic1, self.critic2, self.target1, self.target2):
                m.to(device)
        actor_lr = lr if actor_lr is None else actor_lr
        critic_lr = lr if critic_lr is None else critic_lr
        alpha_lr = lr if alpha_lr is None else alpha_lr
        # capturable: Adam keeps its step count on the device so update() can be
        # replayed from a HIP graph (train.py); same arithmetic otherwise
        self.capturable = capturable
        adam = dict(capturable=True, fused=True) if capturable else {}
        self.actor_opt = torch.optim.Adam(self.actor.parameters(), lr=actor_lr, **adam)
        if share_critic_encoder:
            critic_params = (list(self.critic_encoder.parameters()) + list(self.critic1.edge_mlp.parameters())
                             + list(self.critic2.edge_mlp.parameters()))
        else:
            critic_params = list(self.critic1.parameters()) + list(self.critic2.parameters())
        self.critic_params = critic_params
        self.critic_opt = torch.optim.Adam(critic_params, lr=critic_lr, **adam)
        dev = device if device is not None else "cpu"
        self.log_alpha = torch.tensor(float(np.log(max(alpha_init, 1e-8))), requires_grad=True, device=dev)
        if self.log_alpha.is_cuda:   # before any update can be captured (fused_update._mm32)
            from . import fused_update
            fused_update.probe_mm32(self.log_alpha.device)
        self.alpha_opt = torch.optim.Adam([self.log_alpha], lr=alpha_lr, **adam)
        self.gamma = gamma
        self.target_tau = target_tau
        self.target_entropy = target_entropy
        self.target_entropy_ratio = target_entropy_ratio
        self.grad_clip = grad_clip
        self.amp_dtype = amp_dtype
        # fused update under bf16 autocast: the actor's passes in float32
        # (rl/fused_update.py exact_nets; the critics keep bf16 GEMMs)
        self.fp32_actor = fp32_actor
        # data-parallel hook: called once per update with every gradient tensor
        self.grad_sync: Optional[Callable[[list], None]] = None
        # independent forwards (and their backwards) on side streams (_concurrent),
        # at most max_streams at once (3: the fastest measured, tools/agent_profile.py).
        # The result is the same bit for bit as with max_streams = 1
        # (tests/test_concurrent_update.py; the round-4 replay-to-replay differences
        # were a gfx950 packed-FP32 hazard under CU sharing, compiled out: DESIGN §5)
        self.concurrent = True
        self.max_streams = 3
        self._side = None
        self._warm = False
        self.last_update_path = None   # "fused" (rl/fused_update.py) or "autograd"
        self.grad_flat = None          # fused path: the one buffer every gradient is a view of

    @property
    def alpha(self):
        return self.log_alpha.exp()

    def _amp(self):
        if self.amp_dtype is None:
            return torch.autocast("cuda", enabled=False)
        # the autocast context opens and closes inside every (captured) forward
        # pass, so its weight-cast cache never outlives one graph replay
        return torch.autocast("cuda", dtype=self.amp_dtype)

    # ------------------------------------------------------------ acting
    def select_action(self, node_x, edge_index, edge_attr, action_mask, deterministic: bool = False) -> SACOutput:
        batch = torch.zeros(node_x.size(0), dtype=torch.long, device=node_x.device)
        with torch.no_grad(), self._amp():
            _, probs, _ = self.actor(node_x, edge_index, edge_attr, action_mask, batch, num_graphs=1)
        if deterministic:
            action = torch.argmax(probs).item()
        else:
            action = torch.multinomial(probs, 1).item()
        log_prob = torch.log(probs[action] + 1e-8)
        return SACOutput(action=action, log_prob=log_prob, probs=probs)

    def select_actions(self, node_x, edge_index, edge_attr, action_mask, batch, num_graphs: int,
                       deterministic: bool = False, generator=None, u: torch.Tensor = None) -> torch.Tensor:
        """Batched acting for B graphs with identical link counts (VecRepairEnv):
        one actor forward, one multinomial draw per graph, no host sync.
        `u`: the B uniforms of the fused draw, if already drawn (a captured
        acting graph reads them from a static buffer)."""
        with torch.no_grad(), self._amp():
            if not deterministic:  # fused path: the draw happens inside the edge-head kernel
                if u is None:
                    u = torch.rand(num_graphs, device=node_x.device, generator=generator)
                out = self.actor._fused(node_x, edge_index, edge_attr, batch, num_graphs, mask=action_mask, u=u)
                if out is not None:
                    self.last_act_path = "fused"
                    return out[2]
            self.last_act_path = "general"
            _, probs, _ = self.actor(node_x, edge_index, edge_attr, action_mask, batch, num_graphs=num_graphs)
        p = probs.view(num_graphs, -1)
        if deterministic:
            return p.argmax(dim=1)
        return torch.multinomial(p, 1, generator=generator).squeeze(1)

    def evaluate_actions(self, node_x, edge_index, edge_attr, action_mask, batch, num_graphs: int, actions,
                         top_k: int = 0) -> ActionLogProbs:
        """Log probabilities of given actions (one per graph, link ids), the
        policy's entropy and its top_k best alternatives, for B graphs with
        identical link counts; differentiable in the actor's parameters where
        gradients are enabled (imitation losses, probability ratios)."""
        with self._amp():
            logits, _, _ = self.actor(node_x, edge_index, edge_attr, action_mask, batch, num_graphs=num_graphs)
        return action_log_probs(logits.view(num_graphs, -1), actions, mask=action_mask.view(num_graphs, -1),
                                top_k=top_k)

    # ------------------------------------------------------------ update
    def update(self, batch, weights=None, alpha_max: float = None, sync_metrics: bool = True):
        """sac.py:157-263.  sync_metrics=True returns python floats and a
        td_errors list like the reference; False keeps them as device tensors
        (no host synchronisation, for the vectorised trainer)."""
        out = self.compute_gradients(batch, weights)
        if self.grad_sync is not None:
            self.grad_sync(self.gradients())
        self.apply_gradients(alpha_max)
        if sync_metrics:
            out = {k: (v.cpu().numpy().tolist() if k == "td_errors" else float(v)) for k, v in out.items()}
        return out

    def gradients(self):
        return [p.grad for p in self._all_params() if p.grad is not None]

    def compute_gradients(self, batch, weights=None, on_td=None):
        """Losses and the three backward passes of sac.py:157-243.  None of
        critic, actor and alpha backward depends on another's optimizer step,
        so all gradients exist before any step: one synchronisation point for
        data parallelism.  No host synchronisation (HIP-graph capturable).
        on_td(td_errors): work that needs only the TD errors (the trainer's
        priority write-back, src/train.py:1017-1019), run beside the backward
        passes on the fused path, after them otherwise."""
        if isinstance(batch, list) and len(batch) == 1:
            batch = batch[0]
        (node_x, edge_index, edge_attr, action_mask, batch_vec, action, reward, next_node_x, next_edge_attr,
         next_action_mask, next_batch_vec, done) = batch
        B = reward.shape[0]
        if FUSED_UPDATE and reward.is_cuda and next_batch_vec is batch_vec:
            from . import fused_update
            topo = fused.topology(edge_index, batch_vec, B)
            if fused_update.supported(self, topo):
                self.last_update_path = "fused"
                return fused_update.compute_gradients_fused(self, batch, weights, topo, on_td=on_td)
        self.last_update_path = "autograd"
        self.grad_flat = None
        if weights is None:
            weights_tensor = torch.ones_like(reward)
        else:
            weights_tensor = torch.as_tensor(weights, device=reward.device, dtype=reward.dtype)
            if weights_tensor.dim() == 0:
                weights_tensor = weights_tensor.unsqueeze(0).expand_as(reward)
        edge_batch = batch_vec[edge_index[0]]
        reg = is_regular_edges(edge_index, batch_vec, B)
        # The no-grad passes get an autocast region of their own: autocast caches
        # a weight's bf16 cast for the rest of its region, and a cast made under
        # no_grad carries no autograd history -- reused by the actor's training
        # forward below it would silently cut the gradient of every weight cast
        # in both passes (the actor's GAT lin weights).
        # The three networks of each phase are independent until the losses:
        # on the GPU they run on three side streams (after a first sequential
        # call has built every topology cache), so their hundreds of small
        # kernels overlap instead of queueing behind each other; each has an
        # autocast region of its own (no cached cast is shared across streams).
        def no_grad_pass(net, *args):
            def run():
                with self._amp(), torch.no_grad():
                    return net(*args)
            return run

        next_out, qt1, qt2 = self._concurrent([
            no_grad_pass(self.actor, next_node_x, edge_index, next_edge_attr, next_action_mask, next_batch_vec,
                         False, B),
            no_grad_pass(self.target1, next_node_x, edge_index, next_edge_attr, next_batch_vec, B),
            no_grad_pass(self.target2, next_node_x, edge_index, next_edge_attr, next_batch_vec, B)])
        with torch.no_grad():
            next_probs = next_out[1]
            q_next = torch.min(qt1, qt2)
            v_next = scatter_sum(next_probs * (q_next - self.alpha * torch.log(next_probs + 1e-8)), edge_batch, B,
                                 reg)
            target = reward + (1.0 - done) * self.gamma * v_next

        def train_pass(net, *args):
            def run():
                with self._amp():
                    return net(*args)
            return run

        # The training forwards (autograd recording) run in order on the current
        # stream: with the recorded graphs on side streams, repeated updates in one
        # process came out different from the sequential ones now and then (an
        # unsynchronised reuse somewhere between the side-stream forwards and the
        # backward; tools/fused_vs_autograd_probe.py).  The fused update, whose
        # kernels take their stream explicitly, keeps its side streams.
        q1_all, q2_all, act_out = [fn() for fn in (
            train_pass(self.critic1, node_x, edge_index, edge_attr, batch_vec, B),
            train_pass(self.critic2, node_x, edge_index, edge_attr, batch_vec, B),
            train_pass(self.actor, node_x, edge_index, edge_attr, action_mask, batch_vec, False, B))]
        logits, probs = act_out[0], act_out[1]
        q1 = q1_all[action]
        q2 = q2_all[action]
        td_error = (target - q1).detach().abs()
        loss1 = F.mse_loss(q1, target, reduction="none")
        loss2 = F.mse_loss(q2, target, reduction="none")
        critic_loss = (weights_tensor * (loss1 + loss2)).mean()
        q_all = torch.min(q1_all, q2_all).detach()
        # alpha detached: the reference zeroes log_alpha.grad (alpha_opt.zero_grad,
        # sac.py:236) after actor_loss.backward, so this term never reaches it
        actor_terms = probs * (self.alpha.detach() * torch.log(probs + 1e-8) - q_all)
        actor_loss = scatter_sum(actor_terms, edge_batch, B, reg).mean()
        if self.target_entropy is None:
            valid = scatter_sum((action_mask > 0).float(), edge_batch, B, reg)
            target_entropy = (self.target_entropy_ratio * torch.log(valid + 1e-8)).mean()
        else:
            target_entropy = self.target_entropy
        log_probs = torch.log(probs + 1e-8).detach()
        alpha_term = scatter_sum(probs.detach() * (log_probs + target_entropy), edge_batch, B, reg)
        alpha_loss = -(self.log_alpha * alpha_term).mean()
        entropy = scatter_sum(-(probs.detach() * log_probs), edge_batch, B, reg).mean()
        q_taken = torch.min(q1, q2).detach()
        logp_mean = scatter_sum(probs.detach() * log_probs, edge_batch, B, reg).mean().detach()

        # set_to_none (torch's default, as the reference's zero_grad()): backward
        # hands each parameter its gradient tensor instead of accumulating into
        # zeros -- one fill + one add launch fewer per parameter and update; the
        # tensors autograd allocates inside the captured update keep their
        # addresses on every replay
        self.critic_opt.zero_grad(set_to_none=True)
        self.actor_opt.zero_grad(set_to_none=True)
        self.alpha_opt.zero_grad(set_to_none=True)
        critic_loss.backward()
        actor_loss.backward()
        alpha_loss.backward()
        if on_td is not None:
            on_td(td_error)
        self._warm = True
        return {
            "critic_loss": critic_loss.detach(),
            "actor_loss": actor_loss.detach(),
            "alpha": self.alpha.detach(),
            "alpha_loss": alpha_loss.detach(),
            "policy_entropy": entropy,
            "q_taken": q_taken.mean(),
            "q_mean": q_all.mean(),
            "logp_mean": logp_mean,
            "td_errors": td_error,
        }

    def _concurrent(self, fns, streams=None):
        """Run the callables on side streams forked from (and joined back into)
        the current stream -- fns[i] on side stream streams[i] (default i) --;
        sequentially on the CPU, with concurrent=False, or before the first
        compute_gradients has completed."""
        dev = self.log_alpha.device
        if dev.type != "cuda" or not self.concurrent or not self._warm:
            return [fn() for fn in fns]
        main = torch.cuda.current_stream(dev)
        streams = list(range(len(fns))) if streams is None else list(streams)
        # logical stream k runs on side stream k % max_streams: at most max_streams
        # branches at once (the calls of one side stream run in order)
        width = max(1, int(self.max_streams))
        if self._side is None or len(self._side) < width:
            self._side = [torch.cuda.Stream(dev) for _ in range(width)]
        used = [self._side[k % width] for k in streams]
        outs = []
        forked = set()
        for st, fn in zip(used, fns):
            if id(st) not in forked:
                st.wait_stream(main)
                forked.add(id(st))
            with torch.cuda.stream(st):
                outs.append(fn())
        for st in {id(s): s for s in used}.values():
            main.wait_stream(st)
        def record(o):   # consumed (and freed) on the main stream from here on
            if isinstance(o, torch.Tensor):
                o.record_stream(main)
            elif isinstance(o, (tuple, list)):
                for t in o:
                    record(t)
        record(outs)
        return outs

    def _flat_opt(self):
        """The flat-buffer optimizer step (rl/flat_adam.py), or None where it
        does not apply (CPU, shared critic encoder, non-default Adam options)."""
        fa = getattr(self, "_flat_adam", None)
        if fa is None:
            if not (FLAT_ADAM and self.log_alpha.is_cuda and not self.share_critic_encoder):
                return None
            for opt in (self.critic_opt, self.actor_opt, self.alpha_opt):
                d = opt.defaults
                if d.get("weight_decay", 0) != 0 or d.get("amsgrad") or d.get("maximize") or len(opt.param_groups) != 1:
                    return None
            from .flat_adam import FlatAdam
            fa = self._flat_adam = FlatAdam(self)
        return fa

    def apply_gradients(self, alpha_max: float = None):
        """Clipping, the three optimizer steps, the log_alpha clamps and the
        Polyak target update (sac.py:224-263), in the reference's order.  After
        a fused update: one trx_sac_adam call over the flat gradient buffer."""
        fa = self._flat_opt()
        if fa is not None and getattr(self, "last_update_path", None) == "fused" and fa.usable():
            fa.step([o.param_groups[0]["lr"] for o in (self.critic_opt, self.actor_opt, self.alpha_opt)],
                    self.grad_clip, self.target_tau, alpha_max)
            fused.weights_changed()
            return
        if fa is not None and fa.owner == "flat":
            fa.export_torch()
        clip = self.grad_clip is not None and self.grad_clip > 0
        if clip:
            clip_grad_norm_listwise_(list(self.critic1.parameters()) + list(self.critic2.parameters()), self.grad_clip)
        self.critic_opt.step()
        if clip:
            clip_grad_norm_listwise_(list(self.actor.parameters()), self.grad_clip)
        self.actor_opt.step()
        if clip:
            clip_grad_norm_listwise_([self.log_alpha], self.grad_clip)
        self.alpha_opt.step()
        fused.weights_changed()   # prepared inference weights are stale now
        with torch.no_grad():
            if alpha_max is not None:
                self.log_alpha.clamp_(max=float(np.log(alpha_max)))
            self.log_alpha.clamp_(min=float(np.log(0.01)))
        if self.share_critic_encoder:
            self._soft_update(self.critic_encoder, self.target_encoder)
            self._soft_update(self.critic1.edge_mlp, self.target1.edge_mlp)
            self._soft_update(self.critic2.edge_mlp, self.target2.edge_mlp)
        else:
            self._soft_update(self.critic1, self.target1)
            self._soft_update(self.critic2, self.target2)

    def _all_params(self):
        seen, out = set(), []
        for p in list(self.critic_params) + list(self.actor.parameters()) + [self.log_alpha]:
            if id(p) not in seen:
                seen.add(id(p))
                out.append(p)
        return out

    def save(self, path: str):
        torch.save({"actor": self.actor.state_dict(), "critic1": self.critic1.state_dict(),
                    "critic2": self.critic2.state_dict(), "target1": self.target1.state_dict(),
                    "target2": self.target2.state_dict(), "log_alpha": self.log_alpha.detach().cpu()}, path)

    def load(self, path: str, map_location: str = "cpu"):
        fa = getattr(self, "_flat_adam", None)
        if fa is not None:   # hand the moments back before log_alpha / alpha_opt are replaced
            if fa.owner == "flat":
                fa.export_torch()
            self._flat_adam = None
        state = torch.load(path, map_location=map_location, weights_only=True)
        self.actor.load_state_dict(state["actor"])
        self.critic1.load_state_dict(state["critic1"])
        self.critic2.load_state_dict(state["critic2"])
        self.target1.load_state_dict(state["target1"])
        self.target2.load_state_dict(state["target2"])
        self.log_alpha = state["log_alpha"].to(map_location).requires_grad_()
        lr = self.alpha_opt.param_groups[0]["lr"]
        adam = dict(capturable=True, fused=True) if self.capturable else {}
        self.alpha_opt = torch.optim.Adam([self.log_alpha], lr=lr, **adam)

    @torch.no_grad()
    def _soft_update(self, src, tgt):
        """tp <- tp*(1-tau) + p*tau (sac.py:288-291), as two multi-tensor ops."""
        ps = [p.data for p in src.parameters()]
        tps = [tp.data for tp in tgt.parameters()]
        scaled = torch._foreach_mul(ps, self.target_tau)
        torch._foreach_mul_(tps, 1.0 - self.target_tau)
        torch._foreach_add_(tps, scaled)
