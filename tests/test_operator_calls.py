"""Calls of node_attention, dropout_add and action_log_probs that their
documentation allows and ordinary programs make rarely: other default types,
views whose strides say nothing, sizes at the limits, forward-mode tangents."""
import math

import pytest
import torch


class _Recorder:
    """Stands in for the library on a CPU: every entry succeeds and does nothing."""

    def __getattr__(self, name):
        return lambda *a: 0


@pytest.fixture
def no_library(monkeypatch):
    from trafficrl import _lib
    monkeypatch.setattr(_lib, "load", lambda: _Recorder())
    monkeypatch.setattr(_lib, "raw_stream", lambda device: 0)
    monkeypatch.setattr(_lib, "same_device", lambda what, first, *others: None)
    monkeypatch.setattr(_lib, "on_device", lambda device, f, *a: f(*a))


@pytest.fixture(params=[torch.float64, torch.float32, torch.float16, torch.bfloat16], ids=str)
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


def test_buffers_have_the_kernels_types(no_library, default_dtype):
    """Whatever torch's default type is: a two-byte one would leave the kernels half the memory that they write."""
    from trafficrl.models import dropout_add, node_attention
    from trafficrl.rl import action_log_probs
    logits = torch.zeros(3, 9, dtype=torch.float32, requires_grad=True)
    r = action_log_probs(logits, torch.zeros(3, dtype=torch.int64), top_k=2)
    assert r.log_prob.dtype == r.entropy.dtype == r.top_log_prob.dtype == torch.float32
    assert r.top_action.dtype == torch.int64
    saved = r.log_prob.grad_fn.saved_tensors
    stats = [t for t in saved if t is not None and t.shape == (3, 4)]
    assert len(stats) == 1 and stats[0].dtype == torch.float32
    q = torch.zeros(6, 2, 32, dtype=torch.bfloat16, requires_grad=True)
    out = node_attention(q, q, q, torch.tensor([0, 6]))
    assert out.dtype == torch.bfloat16
    lse = [t for t in out.grad_fn.saved_tensors if t is not None and t.shape == (6, 2)]
    assert len(lse) == 1 and lse[0].dtype == torch.float32
    assert dropout_add(q, torch.zeros(2, dtype=torch.int64), 0.5).dtype == torch.bfloat16


@pytest.mark.gpu
def test_default_type_does_not_matter():
    from trafficrl.rl import action_log_probs
    x = torch.randn(5, 76, device="cuda")
    a = torch.arange(5, device="cuda")

    def both():
        leaf = x.clone().requires_grad_()
        r = action_log_probs(leaf, a, top_k=3)
        return [*r, *torch.autograd.grad(r.log_prob.sum() + r.entropy.sum(), leaf)]
    want = both()
    torch.set_default_dtype(torch.float64)
    try:
        got = both()
    finally:
        torch.set_default_dtype(torch.float32)
    assert all(torch.equal(s, t) and s.dtype == t.dtype for s, t in zip(want, got))


def _odd_strides(rows, heads, channels, dt, **kw):
    """Tensors with a dimension of one whose stride is no multiple of 16 bytes and never used."""
    base = torch.randn(4096, **kw).to(dt)
    if rows == 1:      # one row of a wider one
        yield base.as_strided((1, heads, channels), (heads * channels + 3, channels, 1), 0)
    if heads == 1:     # one head out of a layout with heads innermost but one
        yield base.as_strided((rows, 1, channels), (channels, 5, 1), 0)
        yield base.as_strided((rows, 1, channels), (channels + 8, 7, 1), 8)
    yield base.as_strided((rows, heads, channels), (heads * channels, channels, 1), 1)   # not aligned


@pytest.mark.parametrize("rows,heads", [(1, 4), (1, 1), (6, 1)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16], ids=str)
def test_dimensions_of_one_have_any_stride(rows, heads, dt):
    """contiguous() leaves such a stride as it is; the kernels' boundary takes multiples of 16 bytes."""
    from trafficrl.models.attention import _strided
    unit = 16 // torch.zeros(0, dtype=dt).element_size()
    for t in _odd_strides(rows, heads, 32, dt):
        s = _strided(t)
        assert s.stride(2) == 1 and s.stride(0) % unit == 0 and s.stride(1) % unit == 0 and s.data_ptr() % 16 == 0
        assert torch.equal(s, t)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,heads", [(1, 4), (1, 1), (6, 1)])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16], ids=str)
def test_attention_of_dimensions_of_one(rows, heads, dt):
    from trafficrl.models import node_attention
    p = torch.tensor([0, rows], device="cuda")
    for t in _odd_strides(rows, heads, 32, dt, device="cuda"):
        c = torch.empty(t.shape, device="cuda", dtype=dt).copy_(t)
        leaf, plain = t.detach().requires_grad_(), c.requires_grad_()
        a, b = node_attention(leaf, t, leaf, p), node_attention(plain, c.detach(), plain, p)
        go = torch.randn(t.shape, device="cuda").to(dt)
        assert torch.equal(a, b)
        assert torch.equal(torch.autograd.grad(a, leaf, go)[0], torch.autograd.grad(b, plain, go)[0])


@pytest.mark.parametrize("nodes,code", [((1 << 31) - (1 << 16) + 1, -3), ((1 << 31) - 1, -3), (1 << 31, -3)])
def test_nodes_below_the_kernels_counters(nodes, code):
    """Keys (a stride of zero makes that many out of one) that a 32-bit counter would step over the end of."""
    from test_operators_cpu import _attention_args
    from trafficrl import _lib
    L = _lib.load()
    a = _attention_args()
    a.num_nodes = a.max_nodes = nodes
    a.workspace_bytes = 0     # never launched: without the limit the workspace's check refuses the call
    a.workspace = None
    assert L.trx_node_attention_forward(a, None) == code and L.trx_node_attention_backward(a, None) == code
    assert b"nodes" in L.trx_last_error()
    assert L.trx_node_attention_workspace_bytes(a, 0) == -1
    a.num_nodes = a.max_nodes = (1 << 31) - (1 << 16)
    assert L.trx_node_attention_workspace_bytes(a, 1) > 0


def test_tangents_are_refused():
    """Forward-mode inputs that need no gradient would come back as constants."""
    from torch.autograd import forward_ad
    from trafficrl.models import dropout_add, node_attention
    from trafficrl.rl import action_log_probs
    p, rng = torch.tensor([0, 6]), torch.tensor([1, 2])
    x, logits = torch.randn(6, 2, 32), torch.randn(4, 9)
    act = torch.zeros(4, dtype=torch.int64)
    with forward_ad.dual_level():
        dx, dl = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(logits, torch.ones_like(logits))
        for call in (lambda: node_attention(dx, x, x, p), lambda: node_attention(x, dx, x, p),
                     lambda: node_attention(x, x, dx, p),
                     lambda: node_attention(x, x, x, p, dist=torch.zeros(6, 6),
                                            slope=forward_ad.make_dual(torch.ones(2), torch.ones(2))),
                     lambda: dropout_add(dx, rng, 0.5), lambda: dropout_add(x, rng, 0.5, residual=dx),
                     lambda: action_log_probs(dl, act)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        # without one the call goes on, here to where there is no device
        with pytest.raises(ValueError, match="HIP device"):
            node_attention(x, x, x, p)


def test_distances_bound_the_launch(no_library, monkeypatch):
    """Without hints a launch is shaped by dist, which holds the largest of several networks; a single one by its rows."""
    from trafficrl import _lib
    from trafficrl.models import node_attention
    seen = []

    class Keep(_Recorder):
        def trx_node_attention_forward(self, a, stream):
            seen.append((a.max_queries, a.max_nodes))
            return 0
    monkeypatch.setattr(_lib, "load", lambda: Keep())
    x, many, one = torch.zeros(48, 2, 32), torch.tensor([0, 24, 48]), torch.tensor([0, 48])
    q, qp = torch.zeros(2, 2, 32), torch.tensor([0, 1, 2])
    for kw, want in [
            (dict(dist=torch.zeros(24, 24)), (24, 24)), (dict(dist=torch.zeros(2, 30, 26)), (30, 26)),
            (dict(dist=torch.zeros(90, 90)), (48, 48)), (dict(), (48, 48)),
            (dict(dist=torch.zeros(24, 24), max_queries=7, max_nodes=9), (7, 9)),
            (dict(ptr=one, dist=torch.zeros(5, 5)), (48, 48)),
            (dict(q=q, ptr=qp, k_ptr=many, dist=torch.zeros(1, 24)), (1, 24))]:
        a = dict(q=x, ptr=many) | kw
        node_attention(a.pop("q"), x, x, a.pop("ptr"), **a)
        assert seen[-1] == want, kw


@pytest.mark.gpu
def test_launch_shaped_by_distances():
    """The same bits as with the hints given; a matrix smaller than the networks leaves no row out."""
    from trafficrl.models import node_attention
    from test_node_attention import assert_within, ints, make, reference
    q, k, v, p, _, dist, slope, _ = make([24] * 40 + [7, 90], 4, 2, 32, torch.bfloat16, "shared", seed=6)
    a = node_attention(q, k, v, ints(p), dist=dist, slope=slope)
    assert torch.equal(a, node_attention(q, k, v, ints(p), dist=dist, slope=slope, max_queries=90, max_nodes=90))
    small = dist[:10, :5].contiguous()
    out = node_attention(q, k, v, ints(p), dist=small, slope=slope)
    assert_within("out", out, *reference(q, k, v, p, p, small, slope)["out"])
