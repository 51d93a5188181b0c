"""trafficrl.models.node_attention (csrc/node_attention.hip) against its
definition in float64, elementwise within derived bounds (attention_reference.py)."""
import itertools
import math

import pytest
import torch

from attention_reference import assert_within, reference

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(sizes, H, Hk, C, dt, kind="none", queries=None, seed=0, spread=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    k_ptr = [0] + list(itertools.accumulate(sizes))
    q_sizes = sizes if queries is None else queries
    q_ptr = [0] + list(itertools.accumulate(q_sizes))
    rnd = lambda *s: (torch.randn(*s, device="cuda", generator=g) * spread).to(dt)  # noqa: E731
    q, k, v = rnd(q_ptr[-1], H, C), rnd(k_ptr[-1], Hk, C), rnd(k_ptr[-1], Hk, C)
    dist = slope = None
    if kind != "none":
        mq, mk = max(q_sizes, default=0), max(sizes, default=0)
        shape = (len(sizes), mq, mk) if kind == "each" else (mq, mk)
        dist = torch.rand(*shape, device="cuda", generator=g) * 6
        gone = torch.rand(*shape, device="cuda", generator=g) < 0.15
        dist = dist.masked_fill(gone, math.inf)
        if mq > 2:
            dist[..., 1, :] = math.inf      # a row that sees nothing
        slope = 2.0 ** -torch.arange(1, H + 1, device="cuda", dtype=F32)
    go = rnd(q_ptr[-1], H, C)
    return q, k, v, q_ptr, k_ptr, dist, slope, go


def ints(p):
    return torch.tensor(p, dtype=torch.int64, device="cuda")


def check(sizes, H, Hk, C, dt, kind="none", queries=None, cap=0.0, seed=0, backward=True, **kw):
    from trafficrl.models import node_attention
    q, k, v, q_ptr, k_ptr, dist, slope, go = make(sizes, H, Hk, C, dt, kind, queries, seed)
    leaves = [t for t in (q, k, v, slope) if t is not None]
    if backward:
        for t in leaves:
            t.requires_grad_()
    out = node_attention(q, k, v, ints(q_ptr), k_ptr=ints(k_ptr) if queries is not None else None, dist=dist,
                         slope=slope, cap=cap, **kw)
    assert out.dtype == dt and out.shape == q.shape
    want = reference(q, k, v, q_ptr, k_ptr, dist, slope, None, cap, go if backward else None)
    assert_within("out", out, *want["out"])
    if backward:
        grads = torch.autograd.grad(out, leaves, go)
        for name, t in zip(["q", "k", "v", "slope"], grads):
            assert_within(name, t, *want[name])


# sizes around the 16-, 32-, 64- and 128-row tiles, empty and single-node networks among them
SIZES = [[1], [24] * 5, [0, 1, 2, 0, 15, 16, 17], [31, 32, 33], [63, 64, 65], [127, 128, 129, 5], [200, 3, 77], [0, 0]]


@pytest.mark.parametrize("sizes", SIZES, ids=str)
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_sizes(sizes, dt):
    check(sizes, 4, 4, 64, dt, "shared")
    check(sizes, 2, 2, 32, dt, "none", seed=1)


@pytest.mark.parametrize("C", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 128])
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_channels(C, dt):
    check([24, 70, 1], 2, 2, C, dt, "each")


@pytest.mark.parametrize("H,Hk", [(1, 1), (3, 3), (4, 2), (6, 2), (8, 1), (16, 2), (5, 1)])
@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_shared_heads(H, Hk, dt):
    """Key/value heads shared by several query heads: their gradients are sums
    over the group, and the slopes of a group differ."""
    check([24, 90, 3], H, Hk, 64, dt, "each")
    check([24, 90, 3], H, Hk, 32, dt, "shared", queries=[1, 5, 2])


@pytest.mark.parametrize("cap", [0.5, 10.0, 50.0, 1e4])
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_cap(cap, dt):
    check([24, 100], 4, 2, 64, dt, "each", cap=cap)
    check([24, 100], 4, 2, 64, dt, "none", cap=cap)


@pytest.mark.parametrize("queries,sizes", [([1], [416]), ([1] * 4, [5000, 1, 0, 64]), ([2, 0, 7], [300, 20, 0]),
                                           ([1], [70001]), ([130], [9]), ([300, 1], [1, 700])], ids=str)
@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_queries_apart(queries, sizes, dt):
    """Query rows of their own: one to a network (serving), a few, more than nodes."""
    check(sizes, 4, 2, 64, dt, "each", queries=queries)
    check(sizes, 4, 4, 128, dt, "none", queries=queries, backward=False)


@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_large_network(dt):
    check([1500], 2, 1, 64, dt, "shared", cap=20.0)


def test_hints_only_shape_the_launch():
    """max_queries / max_nodes far too small or too large leave no row out."""
    for m in (0, 1, 7, 10 ** 6):
        check([24, 200, 90], 2, 2, 32, BF16, "shared", max_queries=m, max_nodes=m)


def test_distance_matrix_smaller_than_network():
    """Pairs outside the matrix are not seen."""
    from trafficrl.models import node_attention
    q, k, v, p, _, _, _, go = make([50, 20], 2, 2, 32, F32)
    dist = torch.rand(30, 17, device="cuda") * 3
    slope = torch.tensor([0.3, -0.2], device="cuda")
    out = node_attention(q, k, v, ints(p), dist=dist, slope=slope)
    assert_within("out", out, *reference(q, k, v, p, p, dist, slope)["out"])
    assert bool((out[30:50] == 0).all())


def test_odd_distances():
    """NaN and -inf distances hide a pair like +inf; without a slope dist only masks."""
    from trafficrl.models import node_attention
    q, k, v, p, _, dist, _, _ = make([40, 33], 2, 2, 32, F32, "shared")
    dist[3, 4], dist[3, 5], dist[7, :] = math.nan, -math.inf, -math.inf
    out = node_attention(q, k, v, ints(p), dist=dist)
    assert_within("out", out, *reference(q, k, v, p, p, dist, None)["out"])
    assert bool((out[7] == 0).all())


@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_strides(dt):
    """Views of one projection [rows, 3, heads, channels], heads before rows, an
    unaligned view, one query for all heads: the same bits as contiguous copies."""
    from trafficrl.models import node_attention
    g = torch.Generator("cuda").manual_seed(3)
    p = ints([0, 24, 60])
    x = torch.randn(60, 3, 4, 64, device="cuda", generator=g).to(dt)
    y = torch.randn(4, 60, 64, device="cuda", generator=g).to(dt).transpose(0, 1)
    z = torch.randn(60, 4, 67, device="cuda", generator=g).to(dt)[..., 3:]
    e = torch.randn(60, 1, 64, device="cuda", generator=g).to(dt).expand(60, 4, 64)
    big = torch.rand(60, 80, device="cuda", generator=g)
    for q, k, v, dist in [(x[:, 0], x[:, 1], x[:, 2], None), (y, x[:, 1], y, big[:, ::2]), (z, z, x[:, 0], big),
                          (e, x[:, 0], e, big.t())]:
        a = node_attention(q, k, v, p, dist=dist)
        b = node_attention(q.contiguous(), k.contiguous(), v.contiguous(), p,
                           dist=None if dist is None else dist.contiguous())
        assert torch.equal(a, b)


@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_other_networks_do_not_leak(dt):
    """Rows of no network and of other networks hold NaN and inf: a network's
    results and gradients stay the same bits; rows of no network get zeros."""
    from trafficrl.models import node_attention
    for sizes, lo, hi in [([30, 24, 41], 5, 7), ([200, 33, 64], 0, 90)]:
        q, k, v, p, _, dist, slope, go = make(sizes, 4, 2, 64, dt, "shared")
        p = [lo + x for x in p]
        pad = lambda t, x: torch.cat([t.new_full((lo, *t.shape[1:]), x), t, t.new_full((hi, *t.shape[1:]), x)])  # noqa: E731
        results = []
        for bad in (0.0, math.nan, math.inf):
            qq, kk, vv, gg = (pad(t, bad) for t in (q, k, v, go))
            if bad != 0.0:      # the middle network too
                for t in (qq, kk, vv, gg):
                    t[p[1]:p[2]] = bad
            leaves = [t.requires_grad_() for t in (qq, kk, vv)]
            out = node_attention(qq, kk, vv, ints(p), dist=dist, slope=slope)
            r = [out.detach()] + list(torch.autograd.grad(out, leaves, gg))
            for t in r:
                assert bool((t[:lo] == 0).all()) and bool((t[p[-1]:] == 0).all())
            results.append([torch.cat([t[p[0]:p[1]], t[p[2]:p[3]]]) for t in r])
        for other in results[1:]:
            for a, b in zip(results[0], other):
                assert torch.equal(a, b)


def test_extreme_scores():
    """Scores in the thousands: one key takes a row, nothing overflows."""
    check([70], 2, 2, 64, F32)
    from trafficrl.models import node_attention
    q, k, v, p, _, _, _, _ = make([70, 9], 2, 2, 64, F32, spread=30.0)
    out = node_attention(q, k, v, ints(p))
    assert_within("out", out, *reference(q, k, v, p, p)["out"])
    # a slope that sends every score of far pairs below any float: weights of zero
    dist = torch.full((70, 70), 3e38, device="cuda").fill_diagonal_(0.0)
    out = node_attention(q, k, v, ints(p), dist=dist, slope=torch.full((2,), 3e38, device="cuda"))
    # the one key left has some weight p, and out = fl(fl(p v) fl(1 / p)): three roundings, under 4 u |v|
    assert_within("out", out, v.double(), 4 * 2.0 ** -24 * v.double().abs())


@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_scale_and_slope_signs(dt):
    """A scale of zero, negative and tiny ones; slopes of zero, negative and mixed ones."""
    from trafficrl.models import node_attention
    for sizes in ([30, 24], [150, 70]):
        q, k, v, p, _, dist, _, go = make(sizes, 4, 2, 32, dt, "shared")
        for scale in (0.0, -0.2, 1e-25, 0.3):
            for slope in ([0.0] * 4, [-0.5] * 4, [0.5, -0.25, 0.0, 1.0], [1.0] * 4):
                s = torch.tensor(slope, device="cuda").requires_grad_()
                leaves = [t.detach().requires_grad_() for t in (q, k, v)] + [s]
                out = node_attention(*leaves[:3], ints(p), dist=dist, slope=s, scale=scale)
                want = reference(q, k, v, p, p, dist, s.detach(), scale, 0.0, go)
                assert_within("out", out, *want["out"])
                for name, t in zip(["q", "k", "v", "slope"], torch.autograd.grad(out, leaves, go)):
                    assert_within(name, t, *want[name])


def test_large_cap_is_no_cap():
    """cap = 1e6: a capped score differs from the plain one by z^3 / 3e12, below float32's resolution of z here, so the
    half types' fast tanh must not show."""
    from trafficrl.models import node_attention
    for dt in (F32, BF16, F16):
        q, k, v, p, _, dist, slope, _ = make([40, 200], 4, 2, 64, dt, "shared")
        out = node_attention(q, k, v, ints(p), dist=dist, slope=slope, cap=1e6)
        assert_within("out", out, *reference(q, k, v, p, p, dist, slope)["out"])


def test_pointers_outside_the_tensors():
    """ptr values past the rows, or negative, are clamped; an empty distance matrix shows no pair."""
    from trafficrl.models import node_attention
    q, k, v, _, _, _, _, _ = make([40, 30], 2, 2, 32, F32)
    a = node_attention(q, k, v, ints([-5, 40, 10 ** 12]))
    assert torch.equal(a, node_attention(q, k, v, ints([0, 40, 70])))
    a = node_attention(q, k, v, ints([10 ** 12, 10 ** 12 + 1]))
    assert bool((a == 0).all())
    for shape in ((0, 0), (40, 0), (0, 40)):
        assert bool((node_attention(q, k, v, ints([0, 40, 70]), dist=torch.zeros(shape, device="cuda")) == 0).all())


def test_no_rows():
    from trafficrl.models import node_attention
    for sizes in ([], [0], [0, 0, 0]):
        q, k, v, p, _, _, _, go = make(sizes, 2, 2, 32, F32)
        out = node_attention(q.requires_grad_(), k.requires_grad_(), v, ints(p))
        gq, gk = torch.autograd.grad(out, [q, k], go)
        assert out.shape == gq.shape == gk.shape == (0, 2, 32)
    # queries without nodes, nodes without queries
    q, k, v, qp, kp, _, _, go = make([0, 0], 2, 2, 32, F32, queries=[3, 1])
    assert bool((node_attention(q, k, v, ints(qp), k_ptr=ints(kp)) == 0).all())
    q, k, v, qp, kp, _, _, go = make([3, 4], 2, 2, 32, F32, queries=[0, 0])
    out = node_attention(q, k.requires_grad_(), v.requires_grad_(), ints(qp), k_ptr=ints(kp))
    assert all(bool((t == 0).all()) for t in torch.autograd.grad(out, [k, v], go))


def test_gradient_against_differences():
    """<gradient, direction> against a central difference of the float64 definition."""
    from trafficrl.models import node_attention
    q, k, v, p, _, dist, slope, go = make([20, 7], 4, 2, 16, F32, "shared", seed=5)
    leaves = [t.requires_grad_() for t in (q, k, v, slope)]
    out = node_attention(q, k, v, ints(p), dist=dist, slope=slope, cap=3.0)
    grads = torch.autograd.grad(out, leaves, go)
    bounds = reference(q, k, v, p, p, dist, slope, None, 3.0, go)
    g = torch.Generator("cuda").manual_seed(9)
    eps = 1e-5
    for i, name in enumerate(["q", "k", "v", "slope"]):
        step = torch.randn(leaves[i].shape, device="cuda", generator=g, dtype=torch.float64)
        values = []
        for sign in (1, -1):
            moved = [t.detach().double() for t in leaves]
            moved[i] = moved[i] + sign * eps * step
            o = _definition(*moved, p, dist.double(), 3.0)
            values.append(float((o * go.double()).sum()))
        numeric = (values[0] - values[1]) / (2 * eps)
        got = float((grads[i].double() * step).sum())
        # the kernel's bound along the direction, and the difference's own error: eps^2 times a third
        # derivative of order one, and 1e-15 / eps of cancellation, both on sums of a few hundred terms
        assert abs(got - numeric) <= float((bounds[name][1] * step.abs()).sum()) + 1e-6 * (1 + abs(numeric)), name


def _definition(q, k, v, slope, p, dist, cap):
    out = torch.zeros_like(q)
    for a, b in zip(p[:-1], p[1:]):
        n = b - a
        kk, vv = (t[a:b].repeat_interleave(q.shape[1] // k.shape[1], 1) for t in (k, v))
        z = torch.stack([q[a:b, h] @ kk[:, h].T for h in range(q.shape[1])]) / math.sqrt(q.shape[2])
        z = cap * torch.tanh(z / cap)
        d = dist[:n, :n]
        w = torch.where(torch.isfinite(d), z - slope.view(-1, 1, 1) * torch.where(torch.isfinite(d), d, 0.0), -math.inf)
        w = torch.where(torch.isfinite(d).any(-1, keepdim=True), torch.softmax(w, -1), 0.0)
        out[a:b] = torch.stack([w[h] @ vv[:, h] for h in range(q.shape[1])], 1)
    return out


def test_repeatable():
    """Two runs, and a run beside work on another stream, give the same bits."""
    from trafficrl.models import node_attention
    q, k, v, p, _, dist, slope, go = make([300, 24, 511, 64], 4, 2, 64, BF16, "each")
    leaves = [t.requires_grad_() for t in (q, k, v, slope)]
    ptr = ints(p)

    def both():
        out = node_attention(q, k, v, ptr, dist=dist, slope=slope, cap=5.0)
        return [out.detach()] + list(torch.autograd.grad(out, leaves, go))

    first = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
    again = both()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, again):
        assert torch.equal(a, b) and torch.equal(a, c)


def test_captured():
    """Forward and backward in a captured graph, replayed on new inputs between
    eager calls: every replay equals the eager result."""
    from trafficrl.models import node_attention
    sizes = [24] * 6 + [150]
    q, k, v, p, _, dist, slope, go = make(sizes, 4, 2, 64, BF16, "each")
    ptr = ints(p)

    def both(q, k, v, slope):
        leaves = [t.detach().requires_grad_() for t in (q, k, v, slope)]
        out = node_attention(*leaves[:3], ptr, dist=dist, slope=leaves[3])
        return [out.detach()] + list(torch.autograd.grad(out, leaves, go))

    both(q, k, v, slope)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both(q, k, v, slope)
    for seed in (11, 12, 13):
        nq, nk, nv = make(sizes, 4, 2, 64, BF16, "each", seed=seed)[:3]
        q.copy_(nq), k.copy_(nk), v.copy_(nv)
        want = both(q, k, v, slope)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, want):
            assert torch.equal(a, b)
        both(nk.repeat_interleave(2, 1), nk, nv, slope)
        torch.cuda.synchronize()


def test_long_offsets():
    """Rows past 2^31 elements of a strided cache are found."""
    from trafficrl.models import node_attention
    rows, C = 40, 64
    base = torch.empty(2 ** 31 + 2 ** 20, device="cuda", dtype=BF16)     # 4 GiB
    stride = (2 ** 31) // (rows - 1) // 8 * 8
    view = base.as_strided((rows, 1, C), (stride, C, 1), 2 ** 19)
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(rows, 1, C, device="cuda", generator=g).to(BF16)
    view.copy_(x)
    p = ints([0, 17, rows])
    assert torch.equal(node_attention(x, view, view, p), node_attention(x, x, x, p))


@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_many_small_networks_and_a_large_one(dt):
    """More networks than a launch has tiles for: the large one's further tiles
    are looped over, whether the hints say so or not."""
    from trafficrl.models import node_attention
    many, n, H, C = 40000, 700, 4, 16
    g = torch.Generator("cuda").manual_seed(11)
    rnd = lambda: torch.randn(many + n, H, C, device="cuda", generator=g).to(dt)  # noqa: E731
    q, k, v, go = rnd(), rnd(), rnd(), rnd()
    dist = torch.rand(n, n, device="cuda", generator=g) * 6
    ptr = torch.arange(many + 2, device="cuda")
    ptr[-1] = many + n
    # A single node sees itself: out = v, grad_v = go, up to p = 2^(w - statistics), which is 1 only if w is the same in
    # both.  attention_reference's bounds with n = 1 and M the largest scale sum |q||k| (scores and statistics are
    # below M): dw <= (C + 1) u M + 12 u M, p off by 2 dw + 9 u, the result by 9 u more, and by the type's roundings
    # of p (2 h) and of the result (h).
    M = float((q.double() * k.double()).abs().sum(-1).max()) / math.sqrt(C)
    h = {F32: 0.0, BF16: 2.0 ** -8}[dt]
    near = 2 * (C + 13) * 2.0 ** -24 * max(M, 1.0) + 18 * 2.0 ** -24 + 3 * h
    want = reference(q[many:], k[many:], v[many:], [0, n], [0, n], dist, None, None, 0.0, go[many:])
    for hints in ({}, {"max_queries": n, "max_nodes": n}):
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        out = node_attention(*leaves, ptr, dist=dist, **hints)
        grads = torch.autograd.grad(out, leaves, go)
        for got, own in ((out, v), (grads[2], go)):
            assert ((got[:many].double() - own[:many].double()).abs() <= near * own[:many].double().abs()).all()
        assert_within("out", out[many:], *want["out"])
        for name, t in zip("qkv", grads):
            assert_within(name, t[many:], *want[name])
