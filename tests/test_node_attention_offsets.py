"""node_attention where a row's scores are large and alike: weights depend on the
scores' differences alone, so a common offset, exact in float32, must leave every
result within the bounds of the row without it (attention_reference.py, whose
bounds grow with the scores: here those of the small ones)."""
import math

import pytest
import torch

from attention_reference import HALF, assert_within, reference
from test_node_attention import BF16, F16, F32, ints

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# (query rows, nodes) of each network: one wave, four waves, split keys, split query rows
SHAPES = [([24, 7], [24, 7]), ([200, 33], [200, 33]), ([1, 1], [416, 2000]), ([1500], [1500])]


def grid(q_sizes, sizes, H, Hk, C, dt, seed):
    """Inputs whose scores are multiples of 1/8 below 2^7: small whole numbers, scale 1/8, slopes and distances of few bits."""
    g = torch.Generator("cuda").manual_seed(seed)
    whole = lambda *s: torch.randint(-2, 3, s, device="cuda", generator=g).to(dt)  # noqa: E731
    q, k, v = whole(sum(q_sizes), H, C), whole(sum(sizes), Hk, C), whole(sum(sizes), Hk, C)
    v = v + torch.randn(v.shape, device="cuda", generator=g).to(dt)
    go = torch.randn(q.shape, device="cuda", generator=g).to(dt)
    dist = torch.randint(0, 25, (max(q_sizes), max(sizes)), device="cuda", generator=g).float() / 4
    dist[torch.rand(dist.shape, device="cuda", generator=g) < 0.1] = math.inf
    slope = torch.tensor([0.5, 1.0, 0.5, 0.25], device="cuda")[:H].contiguous()
    ends = lambda s: [0, *torch.tensor(s).cumsum(0).tolist()]  # noqa: E731
    return q, k, v, go, dist, slope, ends(q_sizes), ends(sizes)


def run(q, k, v, go, dist, slope, qp, kp, **kw):
    from trafficrl.models import node_attention
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    if slope is not None:
        leaves.append(slope.clone().requires_grad_())
    out = node_attention(*leaves[:3], ints(qp), k_ptr=ints(kp), dist=dist, slope=None if slope is None else leaves[3], **kw)
    return dict(zip(["out", "q", "k", "v", "slope"], [out, *torch.autograd.grad(out, leaves, go)]))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_common_distance(shape, dt):
    """A constant added to every distance; the gradient of the slopes, which it multiplies, against its own reference."""
    q, k, v, go, dist, slope, qp, kp = grid(*shape, 4, 2, 16, dt, 1)
    want = reference(q, k, v, qp, kp, dist, slope, 0.125, 0.0, go)
    # up to 2^20 / 4 + 2^7 in steps of 1/16: 22 bits
    for shift in (0.0, 2.0 ** 11, 2.0 ** 15, 2.0 ** 18, 2.0 ** 20):
        got = run(q, k, v, go, dist + shift, slope, qp, kp, scale=0.125)
        for name in ("out", "q", "k", "v"):
            assert_within(f"{name} + {shift}", got[name], *want[name])
        own = reference(q, k, v, qp, kp, dist + shift, slope, 0.125, 0.0, go)
        assert_within(f"slope + {shift}", got["slope"], *own["slope"])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("cap", [0.0, 20.0])
def test_unreachable(shape, dt, cap):
    """Every node at one large finite distance, and alike otherwise: each weighs the same.  Up to the type's largest."""
    q, k, v, go, dist, _, qp, kp = grid(*shape, 4, 2, 16, dt, 2)
    k = k[:1].expand_as(k).contiguous()
    slope = torch.full((4,), 0.5, device="cuda")
    hidden = dist == math.inf
    want = reference(q, k, v, qp, kp, torch.where(hidden, math.inf, 0.0), slope, 0.125, cap, go)
    for far in (0.0, 1e5, 1e7, 1e9, 1e12, 1e30, torch.finfo(F32).max):
        got = run(q, k, v, go, torch.where(hidden, math.inf, far), slope, qp, kp, scale=0.125, cap=cap)
        for name in ("out", "q", "k", "v"):
            assert_within(f"{name} at {far}", got[name], *want[name])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_common_score(shape, dt):
    """A constant vector added to every key: the scores of a row move together."""
    q, k, v, go, _, _, qp, kp = grid(*shape, 4, 2, 64, dt, 3)
    want = reference(q, k, v, qp, kp, None, None, 0.125, 0.0, go)
    base = torch.zeros_like(k)
    for size in (0.0, 128.0, 1024.0, 8192.0):
        base[..., ::3] = size          # 22 channels x 2 x 8192 / 8: up to 2^16 in steps of 1/8
        step = {F32: 0, BF16: 8, F16: 11}[dt]
        if step and size * 2.0 ** -step > 0.5:
            continue                   # keys near it would not be whole in the type
        got = run(q, k + base, v, go, None, None, qp, kp, scale=0.125)
        for name in ("out", "v"):
            assert_within(f"{name} + {size}", got[name], *want[name])


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_weights_sum_to_one(shape, dt, cap):
    """At distances where float32 keeps nothing of the scores beside them any weights may come out, but a row's still
    sum to one: grad_v's sum over a network's nodes is that of the incoming gradients of the rows that see any."""
    q_sizes, sizes = shape
    q, k, v, go, dist, slope, qp, kp = grid(q_sizes, sizes, 4, 2, 16, dt, 4)
    g = torch.Generator("cuda").manual_seed(5)
    q = torch.randn(q.shape, device="cuda", generator=g).to(dt)
    k = torch.randn(k.shape, device="cuda", generator=g).to(dt)
    for far in (3e3, 1e5, 3e7, 1e9, 1e11):
        d = torch.where(dist == math.inf, math.inf, far * (1 + dist / 1e6))
        got = run(q, k, v, go, d, slope, qp, kp, cap=cap)
        assert all(bool(torch.isfinite(t).all()) for t in got.values())
        for b in range(len(sizes)):
            nq, nk = q_sizes[b], sizes[b]
            sees = torch.isfinite(d[:nq, :nk]).any(1).view(nq, 1, 1, 1)
            rows = (go[qp[b]:qp[b + 1]].double().view(nq, 2, 2, 16) * sees)
            have = got["v"][kp[b]:kp[b + 1]].double().sum(0)
            # each p is off by its sum's roundings ((nk + 64) u) and its own step, each of the sums by n u and the step
            near = (2 * HALF[dt] + (nk + 2 * nq + 64) * U + 2.0 ** -14 * (dt != F32)) * rows.abs().sum((0, 2))
            near = near + (HALF[dt] + U) * got["v"][kp[b]:kp[b + 1]].double().abs().sum(0) + nk * 2.0 ** -25
            assert bool(((have - rows.sum((0, 2))).abs() <= near).all()), (far, b)


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("n", [24, 40, 200])
def test_capped_scores_do_not_depend_on_their_tile(dt, n):
    """Scores of 1e-9 beside a bias that lies halfway between two float32 numbers 64 apart: their sum's rounding hangs
    on the last bit of the capped score.  One large score among them sends some tiles another way; both backward
    passes must still see the same scores, or a row's weights do not sum to one."""
    m = 7000001                                    # 1 mod 4: the tie goes to the number below
    q, k = (torch.zeros(n, 1, 16, device="cuda", dtype=dt) for _ in range(2))
    q[..., 0], k[..., 0] = 2.0 ** -14, 2.0 ** -14
    q[..., 1] = 1.0
    k[min(20, n - 1), 0, 1] = 8.0
    g = torch.Generator("cuda").manual_seed(n)
    v, go = (torch.randn(n, 1, 16, device="cuda", generator=g).to(dt) for _ in range(2))
    dist = torch.full((n, n), 128.0 * m, device="cuda")
    got = run(q, k, v, go, dist, torch.full((1,), 0.75, device="cuda"), [0, n], [0, n], scale=0.25, cap=3.0)
    have, rows = got["v"].double().sum(0), go.double()
    near = (2 * HALF[dt] + (3 * n + 64) * U + 2.0 ** -14 * (dt != F32)) * rows.abs().sum(0)
    near = near + (HALF[dt] + U) * got["v"].double().abs().sum(0) + n * 2.0 ** -25
    assert bool(((have - rows.sum(0)).abs() <= near).all())
    assert all(bool(torch.isfinite(t).all()) for t in got.values())
