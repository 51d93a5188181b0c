"""node_attention, dropout_add and action_log_probs together, as a node-attention
policy uses them, against the same policy in float64; and the agent's call of
action_log_probs."""
import math

import pytest
import torch

from test_dropout_add import keep_mask
from test_sac_e2e import flat, make_agent, observations

pytestmark = pytest.mark.gpu


def policy(x, w, p, src, dst, row_ptr, dist, mask, action, rng, attend, drop, score):
    """Two blocks of attention with residual dropout, then a score for each link."""
    for i in range(2):
        qkv = (x @ w["qkv"][i]).view(-1, 3, 4, 16)
        o = attend(qkv[:, 0], qkv[:, 1], qkv[:, 2], w["slope"][i])
        x = drop(o.reshape(-1, 64) @ w["out"][i], x, i)
    z = torch.tanh(x[src] @ w["src"] + x[dst] @ w["dst"])
    return score((z * w["head"]).sum(1))


def test_policy_forward_and_gradients():
    from trafficrl.models import dropout_add, node_attention
    from trafficrl.rl import action_log_probs
    g = torch.Generator("cuda").manual_seed(0)
    sizes = [24, 30, 7, 24]
    ends = [0, 24, 54, 61, 85]
    p = torch.tensor(ends, device="cuda")
    links = [50, 76, 9, 76]
    c = torch.Generator().manual_seed(1)
    src = torch.cat([torch.randint(a, a + n, (m,), generator=c) for a, n, m in zip(ends, sizes, links)]).cuda()
    dst = torch.cat([torch.randint(a, a + n, (m,), generator=c) for a, n, m in zip(ends, sizes, links)]).cuda()
    row_ends = [0, 50, 126, 135, 211]
    row_ptr = torch.tensor(row_ends, device="cuda")
    mask = (torch.rand(211, device="cuda", generator=g) < 0.4).float()
    action = torch.tensor([int(torch.nonzero(mask[a:b])[0]) for a, b in zip(row_ends[:-1], row_ends[1:])], device="cuda")
    dist = torch.rand(4, 30, 30, device="cuda", generator=g) * 4
    rng = torch.tensor([42, 7], device="cuda")
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g) / math.sqrt(s[-2] if len(s) > 1 else 1)  # noqa: E731
    w = {"qkv": rnd(2, 64, 192), "out": rnd(2, 64, 64), "slope": rnd(2, 4).abs(), "src": rnd(64, 32), "dst": rnd(64, 32),
         "head": rnd(32)}
    x0 = torch.randn(85, 64, device="cuda", generator=g)
    coef = torch.randn(4, device="cuda", generator=g)
    names = sorted(w)

    leaves = {n: t.clone().requires_grad_() for n, t in w.items()}
    out = policy(x0, leaves, p, src, dst, row_ptr, dist, mask, action, rng,
                 lambda q, k, v, s: node_attention(q, k, v, p, dist=dist, slope=s, cap=8.0, max_nodes=30, max_queries=30),
                 lambda y, x, i: dropout_add(y, rng, 0.2, residual=x, site=i),
                 lambda z: action_log_probs(z, action, mask=mask, row_ptr=row_ptr, max_row=76, top_k=3))
    loss = (coef * out.log_prob).sum() + 0.1 * out.entropy.sum()
    grads = torch.autograd.grad(loss, [leaves[n] for n in names])

    def attend(q, k, v, s):
        parts = []
        for b, (a, e) in enumerate(zip(ends[:-1], ends[1:])):
            d = dist[b, :e - a, :e - a].double()
            z = torch.einsum("ihc,jhc->hij", q[a:e], k[a:e]) / 4.0
            z = 8.0 * torch.tanh(z / 8.0) - s.view(-1, 1, 1) * d
            parts.append(torch.einsum("hij,jhc->ihc", torch.softmax(z, -1), v[a:e]))
        return torch.cat(parts)

    def drop(y, x, i):
        keep, scale = keep_mask(y.numel(), 42, 7, i, 0.2)
        return x + torch.where(keep.view(y.shape), y * scale, 0.0)

    def score(z):
        lps, hs = [], []
        for r, (a, e) in enumerate(zip(row_ends[:-1], row_ends[1:])):
            may = mask[a:e] > 0
            lp = torch.log_softmax(z[a:e][may], 0)
            lps.append(lp[int(may[:int(action[r])].sum())])
            hs.append(-(lp.exp() * lp).sum())
        return torch.stack(lps), torch.stack(hs)

    ref = {n: t.double().requires_grad_() for n, t in w.items()}
    lp, h = policy(x0.double(), ref, p, src, dst, row_ptr, dist, mask, action, rng, attend, drop, score)
    want = torch.autograd.grad((coef.double() * lp).sum() + 0.1 * h.sum(), [ref[n] for n in names])
    # float32 through two blocks of 64-term products, 30-term softmaxes and a 64 + 64 + 32-term head: each output
    # is off by at most some 400 roundings of values of order one (rows of x grow to about 4); a gradient adds as
    # many again on the way back, relative to its tensor's largest entry
    tol = 4 * 400 * 2.0 ** -24
    assert float((out.log_prob.double() - lp).abs().max()) <= tol * (1 + float(lp.abs().max()))
    assert float((out.entropy.double() - h).abs().max()) <= tol * (1 + float(h.abs().max()))
    for n, a, b in zip(names, grads, want):
        assert float((a.double() - b).abs().max()) <= 2 * tol * (1 + float(b.abs().max())), n


@pytest.mark.parametrize("grad", [False, True])
def test_agent_evaluates_actions(grad):
    """DiscreteSAC.evaluate_actions agrees with the actor's own probabilities."""
    B = 6
    env, obs, _ = observations(B)
    agent = make_agent()
    nx_, ei, ex_, mask, bv = flat(env, obs, B)
    actions = torch.stack([torch.nonzero(m)[1, 0] for m in mask.view(B, -1)])
    with torch.set_grad_enabled(grad):
        r = agent.evaluate_actions(nx_, ei, ex_, mask, bv, B, actions, top_k=5)
        with agent._amp():
            logits, probs, _ = agent.actor(nx_, ei, ex_, mask, bv, num_graphs=B)
    z = torch.where(mask.view(B, -1) > 0, logits.detach().view(B, -1).double(), -math.inf)
    lp = torch.log_softmax(z, 1)
    # the two forward passes are the same kernels: float32 roundings of the log-softmax alone
    assert float((r.log_prob.double() - lp.gather(1, actions.unsqueeze(1)).squeeze(1)).abs().max()) <= 200 * 2.0 ** -24
    best = torch.sort(lp, stable=True, dim=1, descending=True)
    assert torch.equal(r.top_action, best[1][:, :5])
    assert bool((mask.view(B, -1).gather(1, r.top_action) > 0).all())
    if grad:
        params = [q for q in agent.actor.parameters()]
        got = torch.autograd.grad(r.log_prob.sum() - r.entropy.sum(), params, allow_unused=True)
        assert any(t is not None and bool(t.abs().max() > 0) for t in got)
        assert all(t is None or bool(torch.isfinite(t).all()) for t in got)


def test_second_derivatives_are_refused():
    """create_graph works, but what comes back is no constant: differentiating it
    raises, also where the incoming gradient does not require one."""
    from trafficrl.models import dropout_add, node_attention
    from trafficrl.rl import action_log_probs
    rng, p = torch.tensor([1, 2], device="cuda"), torch.tensor([0, 10], device="cuda")
    x = torch.randn(10, 2, 32, device="cuda", requires_grad=True)
    logits = torch.randn(4, 9, device="cuda", requires_grad=True)
    for y, leaf in ((node_attention(x, x, x, p), x), (dropout_add(x, rng, 0.5, residual=x), x),
                    (action_log_probs(logits, torch.zeros(4, dtype=torch.int64, device="cuda")).log_prob, logits)):
        g, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
        want, = torch.autograd.grad(y.sum(), leaf, retain_graph=True)
        assert torch.equal(g, want)
        with pytest.raises(RuntimeError, match="once, not twice"):
            ((g * g).sum() + leaf.sum()).backward()


def test_broadcast_inputs_and_one_leaf_in_several_places():
    """Inputs of stride zero, and a leaf that is query, key, value and residual:
    the gradients add up to those of separate copies."""
    from trafficrl.models import dropout_add, node_attention
    from trafficrl.rl import action_log_probs
    g = torch.Generator("cuda").manual_seed(21)
    ptr = torch.tensor([0, 20, 50], device="cuda")
    one = torch.randn(50, 1, 32, device="cuda", generator=g).requires_grad_()
    s1 = torch.rand(1, device="cuda", generator=g).requires_grad_()
    d1 = torch.rand(1, 30, device="cuda", generator=g).expand(30, 30)     # every row alike
    go = torch.randn(50, 4, 32, device="cuda", generator=g)

    def attend(q, k, v, s, d):
        return node_attention(q, k, v, ptr, dist=d, slope=s)
    wide = one.expand(50, 4, 32)
    got = torch.autograd.grad(attend(wide, wide, wide, s1.expand(4), d1), [one, s1], go)
    parts = [one.detach().expand(50, 4, 32).clone().requires_grad_() for _ in range(3)]
    s4 = s1.detach().expand(4).clone().requires_grad_()
    apart = torch.autograd.grad(attend(*parts, s4, d1.contiguous()), [*parts, s4], go)
    # the same bits three times over, added in another order: 12 terms and 4 terms of float32
    want = sum(t.double() for t in apart[:3]).sum(1, keepdim=True)
    size = sum(t.double().abs() for t in apart[:3]).sum(1, keepdim=True)
    assert ((got[0].double() - want).abs() <= 12 * 2.0 ** -24 * size).all()
    assert abs(float(got[1].double() - apart[3].double().sum())) <= 4 * 2.0 ** -24 * float(apart[3].double().abs().sum())

    row = torch.randn(1, 76, device="cuda", generator=g).requires_grad_()
    mask = (torch.rand(1, 76, device="cuda", generator=g) > 0.3).expand(9, 76)
    action = torch.randint(0, 76, (9, 3), device="cuda", generator=g)[:, 1]
    a = action_log_probs(row.expand(9, 76), action, mask=mask, top_k=3)
    many = row.detach().expand(9, 76).clone().requires_grad_()
    b = action_log_probs(many, action.contiguous(), mask=mask.contiguous(), top_k=3)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    w = torch.randn(9, device="cuda", generator=g)
    ga, = torch.autograd.grad(a.entropy, row, w)
    gb, = torch.autograd.grad(b.entropy, many, w)
    assert ((ga.double() - gb.double().sum(0)).abs() <= 9 * 2.0 ** -24 * gb.double().abs().sum(0)).all()

    rng = torch.tensor([3, 4], device="cuda")
    x = torch.randn(40, 33, device="cuda", generator=g).requires_grad_()
    gx, = torch.autograd.grad(dropout_add(x, rng, 0.25, residual=x), x, torch.ones(40, 33, device="cuda"))
    kept = dropout_add(torch.ones(40, 33, device="cuda"), rng, 0.25)
    assert torch.equal(gx, kept + 1)


def test_two_streams_at_once():
    """The same operators on two streams share nothing: the bits of one after the other."""
    from trafficrl.models import node_attention
    from trafficrl.rl import action_log_probs
    g = torch.Generator("cuda").manual_seed(22)
    ptr = torch.tensor([0, 700], device="cuda")
    sets = [[torch.randn(700, 2, 64, device="cuda", generator=g).bfloat16().requires_grad_() for _ in range(3)]
            for _ in range(2)]
    go = torch.randn(700, 2, 64, device="cuda", generator=g).bfloat16()
    rows = [torch.randn(3, 50001, device="cuda", generator=g) for _ in range(2)]
    action = torch.tensor([0, 7, 50000], device="cuda")

    def run(i):
        out = node_attention(*sets[i], ptr)
        return [out.detach(), *torch.autograd.grad(out, sets[i], go), *action_log_probs(rows[i], action, top_k=8)]
    want = [run(0), run(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(4):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, run(i)))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(x, y) for x, y in zip(r, want[i]))
