"""trafficrl.models.dropout_add (csrc/dropout_add.hip) against Philox4x32-10
restated in Python whole numbers."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def philox(counter, key):
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def keep_mask(n, seed, step, site, p):
    border = int(np.floor(p * 65536 + 0.5))
    seed &= 2 ** 64 - 1
    bits = []
    for g in range((n + 7) // 8):
        for w in philox((g & 0xFFFFFFFF, g >> 32, step & 0xFFFFFFFF, site), (seed & 0xFFFFFFFF, seed >> 32)):
            bits += [w & 0xFFFF, w >> 16]
    return torch.tensor(bits[:n], device="cuda") >= border, 65536.0 / (65536 - border)


def test_published_answer():
    """The generator's known answers (Salmon et al., the paper's test vectors)."""
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    f = 0xFFFFFFFF
    assert philox((f, f, f, f), (f, f)) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]


@pytest.mark.parametrize("n", [1, 7, 8, 9, 64, 1000, 4097, 70001])
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("residual", [False, True])
def test_values_and_gradients(n, dt, residual):
    from trafficrl.models import dropout_add
    g = torch.Generator("cuda").manual_seed(n)
    x = torch.randn(n, device="cuda", generator=g).to(dt).requires_grad_()
    r = torch.randn(n, device="cuda", generator=g).to(dt).requires_grad_() if residual else None
    go = torch.randn(n, device="cuda", generator=g).to(dt)
    for seed, step, site, p in [(12345, 0, 0, 0.1), (-7, 2 ** 33 + 5, 3, 0.5), (2 ** 62 + 99, 17, 2 ** 32 - 1, 0.9)]:
        rng = torch.tensor([seed, step], device="cuda")
        y = dropout_add(x, rng, p, residual=r, site=site)
        keep, scale = keep_mask(n, seed, step, site, p)
        want = torch.where(keep, x.detach().double() * scale, 0.0)
        total = want if r is None else want + r.detach().double()
        # the product's rounding in float32, the sum's, and the one to the type
        bound = 2.0 ** -24 * (2 * want.abs() + total.abs()) + HALF[dt] * total.abs() + 2.0 ** -25
        assert bool(((y.double() - total).abs() <= bound).all())
        rng += 1      # the state moves on before the backward pass
        grads = torch.autograd.grad(y, [x] if r is None else [x, r], go)
        want = torch.where(keep, go.double() * scale, 0.0)
        assert bool(((grads[0].double() - want).abs() <= (2.0 ** -23 + HALF[dt]) * want.abs() + 2.0 ** -25).all())
        if r is not None:
            assert torch.equal(grads[1], go)


def test_edges():
    from trafficrl.models import dropout_add
    rng = torch.tensor([1, 2], device="cuda")
    x = torch.randn(300, 7, device="cuda")
    assert torch.equal(dropout_add(x, rng, 0.0), x)
    assert dropout_add(x[:0], rng, 0.5).shape == (0, 7)
    bad = torch.full((4096,), float("nan"), device="cuda")
    y = dropout_add(bad, rng, 0.5)
    keep, _ = keep_mask(4096, 1, 2, 0, 0.5)
    assert torch.equal(y.isnan(), keep) and bool((y[~keep] == 0).all())      # a dropped element adds nothing
    # strided and unaligned inputs, a broadcast residual and its gradient
    wide = torch.randn(64, 33, device="cuda")
    v, r = wide[:, 1:9], torch.randn(8, device="cuda", requires_grad=True)
    y = dropout_add(v, rng, 0.3, residual=r.expand(64, 8))
    assert torch.equal(y, dropout_add(v.contiguous(), rng, 0.3, residual=r.detach().expand(64, 8).contiguous()))
    assert torch.equal(torch.autograd.grad(y.sum(), r)[0], torch.full((8,), 64.0, device="cuda"))


def test_share_sites_and_steps():
    """The kept share is 1 - p within six deviations of a binomial; masks of other
    sites, steps and seeds agree with it no more often than chance has it."""
    from trafficrl.models import dropout_add
    n, p = 1 << 20, 0.25
    x = torch.ones(n, device="cuda")
    masks = [dropout_add(x, torch.tensor(rng, device="cuda"), p, site=s) > 0
             for rng, s in (([5, 0], 0), ([5, 1], 0), ([5, 0], 1), ([6, 0], 0), ([5 + 2 ** 32, 0], 0))]
    for m in masks:
        assert abs(float(m.double().mean()) - 0.75) < 6 * (p * (1 - p) / n) ** 0.5
    agree = p * p + (1 - p) ** 2
    for m in masks[1:]:
        assert abs(float((m == masks[0]).double().mean()) - agree) < 6 * (agree * (1 - agree) / n) ** 0.5


def test_captured_graph_draws_anew():
    """rng raised inside the graph: every replay draws the mask of its own step."""
    from trafficrl.models import dropout_add
    rng = torch.tensor([77, 0], device="cuda")
    one = torch.tensor([0, 1], device="cuda")
    x = torch.randn(999, device="cuda")

    def step():
        leaf = x.detach().requires_grad_()
        y = dropout_add(leaf, rng, 0.4, residual=x, site=9)
        rng.add_(one)
        return y.detach(), torch.autograd.grad(y, leaf, x)[0]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        before = rng.clone()
        graph.replay()
        torch.cuda.synchronize()
        after = rng.clone()
        assert int(after[1]) == int(before[1]) + 1
        rng.copy_(before)
        want = step()
        assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]) and torch.equal(rng, after)


def test_beyond_32_bits():
    """Elements behind 2^32 are reached, with counters of their own."""
    from trafficrl.models import dropout_add
    n = 2 ** 32 + 24
    x = torch.ones(n, device="cuda", dtype=F16)
    y = dropout_add(x, torch.tensor([3, 4], device="cuda"), 0.5)
    first = (n - 64) // 8
    bits = []
    for g in range(first, first + 8):
        for w in philox((g & 0xFFFFFFFF, g >> 32, 4, 0), (3, 0)):
            bits += [w & 0xFFFF, w >> 16]
    assert torch.equal(y[-64:] > 0, torch.tensor(bits, device="cuda") >= 32768)
    assert torch.equal(y[:1000] > 0, keep_mask(1000, 3, 4, 0, 0.5)[0])
