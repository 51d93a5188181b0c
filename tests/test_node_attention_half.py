"""node_attention in float16 where its range is short: gradients are linear in the
incoming one, so a power of two on it (exact in the type here) must come out
again, whatever that does to the score gradients in between."""
import math

import pytest
import torch

from attention_reference import reference
from test_node_attention import F16, ints, make

pytestmark = pytest.mark.gpu
STEP, LEAST = 2.0 ** -11, 2.0 ** -25     # half a step: relative, and below the normal numbers

SHAPES = [([1500], None), ([24, 70, 3], None), ([4001], [2]), ([2000, 416], [1, 1]), ([40], [1200])]


def assert_scaled(name, got, value, bound, by):
    """`bound` holds the value's own half step; at the new size that may lie below the normal numbers."""
    got, value = got.detach().double(), value * by
    over = (got - value).abs() - (bound * by + LEAST)
    assert bool(torch.isfinite(got).all()), f"{name} x {by}: not finite"
    assert float(over.max()) <= 0.0, (f"{name} x {by}: {int((over > 0).sum())} of {over.numel()} outside, worst by "
                                      f"{float(over.max()):.3g}")


@pytest.mark.parametrize("sizes,queries", SHAPES, ids=str)
@pytest.mark.parametrize("kind,cap", [("none", 0.0), ("shared", 0.0), ("shared", 20.0)], ids=str)
def test_small_and_large_gradients(sizes, queries, kind, cap):
    from trafficrl.models import node_attention
    q, k, v, qp, kp, dist, slope, go = make(sizes, 4, 2, 64, F16, kind, queries, seed=2)
    go = (go.float() * 16).round().clamp(-48, 48).half() / 16      # six bits: any of the powers below is exact
    want = reference(q, k, v, qp, kp, dist, slope, None, cap, go)
    leaves = [t.requires_grad_() for t in (q, k, v)] + ([slope.requires_grad_()] if slope is not None else [])
    out = node_attention(q, k, v, ints(qp), k_ptr=ints(kp) if queries else None, dist=dist, slope=slope, cap=cap)
    for by in (1.0, 2.0 ** -10, 2.0 ** -13, 2.0 ** -17, 2.0 ** 10):
        scaled = (go.float() * by).half()
        assert torch.equal(scaled.double(), go.double() * by)
        got = torch.autograd.grad(out, leaves, scaled, retain_graph=True)
        for name, t in zip("qkv", got):
            # the type's numbers end: what a result of that size cannot be held in is not asked for
            value, bound = want[name]
            if float(value.abs().max()) * by < 60000.0:
                assert_scaled(name, t, value, bound, by)
        if slope is not None:
            over = (got[3].double() - want["slope"][0] * by).abs() - want["slope"][1] * by
            assert float(over.max()) <= 0.0


@pytest.mark.parametrize("n", [1000, 4001])
def test_small_gradients_as_a_whole(n):
    """Incoming gradients of 1e-3 and 1e-4, on keys of size 32 so that the results are normal numbers: the error of all
    of grad_q and grad_k together is that of gradients of size one, within the factor that two runs of independent
    roundings differ by (sqrt(n) of them and more: a tenth)."""
    from trafficrl.models import node_attention
    g = torch.Generator("cuda").manual_seed(n)
    p = ints([0, n])
    rnd = lambda: torch.randn(n, 1, 64, device="cuda", generator=g)  # noqa: E731
    q, k, v, go = (rnd() * 8).half(), (rnd() * 8).half(), rnd().half(), (rnd() * 16).round().half() / 16
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = node_attention(q, k, v, p, scale=1.0 / 512)
    want = reference(q, k, v, [0, n], [0, n], None, None, 1.0 / 512, 0.0, go)

    def off(by):
        got = torch.autograd.grad(out, leaves, (go.float() * by).half(), retain_graph=True)
        # what the result's own rounding costs at this size is the type's, not the kernels'
        r = []
        for name, t in zip("qkv", got):
            value = want[name][0] * by
            own = (value.half().double() - value).pow(2).sum()
            r.append(float((((t.double() - value).pow(2).sum() - own).clamp_min(0) / value.pow(2).sum()).sqrt()))
        return r

    base = off(1.0)
    for by in (2.0 ** -10, 2.0 ** -13):
        for name, a, b in zip("qkv", off(by), base):
            assert a <= 1.1 * b + STEP / 4, (name, by, a, b)


def test_score_gradients_beyond_the_type():
    """p (gp - D) above 65504, results well inside."""
    from trafficrl.models import node_attention
    q, k, v, qp, kp, _, _, go = make([24, 200], 2, 2, 64, F16, seed=3)
    q, k, v, go = (q.float() / 16).half(), (k.float() / 256).half(), (v.float() * 32).half(), (go.float() * 4096).half()
    gp = go[:24, 0].double() @ v[:24, 0].double().T      # scores near zero: every weight is about 1 / 24
    assert float((gp - gp.mean(1, keepdim=True)).abs().max()) / 24 > 1.5 * 65504
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = node_attention(*leaves, ints(qp))
    want = reference(q, k, v, qp, kp, None, None, None, 0.0, go)
    assert all(float(want[name][0].abs().max()) < 60000 for name in "qkv")
    for name, t in zip("qkv", torch.autograd.grad(out, leaves, go)):
        assert_scaled(name, t, *want[name], 1.0)


@pytest.mark.parametrize("n", [70000, 200])
@pytest.mark.parametrize("bits", [16, 20, 26])
def test_many_small_weights(n, bits):
    """One key far above all others: what they weigh together counts, though each is small."""
    from trafficrl.models import node_attention
    q = torch.zeros(1, 1, 32, device="cuda", dtype=F16)
    k = torch.zeros(n + 1, 1, 32, device="cuda", dtype=F16)
    v = torch.ones(n + 1, 1, 32, device="cuda", dtype=F16)
    v[0] = 0
    dist = torch.full((1, n + 1), bits * math.log(2.0), device="cuda")
    dist[0, 0] = 0.0
    out = node_attention(q, k, v, ints([0, 1]), k_ptr=ints([0, n + 1]), dist=dist, slope=torch.ones(1, device="cuda"))
    small = torch.exp(-dist[0, 1].double())
    want = n * small / (1 + n * small)
    # weights are held from 2^7 down in float16: off by its half step, and by 2^-25 2^-7 at least; the sum is float32
    near = want * (2 * STEP + (n + 40) * 2.0 ** -24 / 16) + n * 2.0 ** -32 + LEAST
    assert float((out.double() - want).abs().max()) <= float(near), (float(out[0, 0, 0]), float(want))
