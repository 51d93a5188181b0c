"""Gradients of trafficrl.rl.action_log_probs entry by entry, within bounds that
shrink with the probability they are about, on rows whose logits share a large
offset or fill.

Bounds, with u = 2^-24, d = x - m (m the row's largest logit), L = log sum e^d and
lp = d - L.  Every term e^d is off by (2 |d| + 4) u, a sum of n of them by another
(n / 64 + 20) u (a lane adds n / 64 at most, then a tree); so with Q = sum p (2 |d|
+ 4) + n / 64 + 20
  L by Q u + 3 u |L|,  lp by that + 2 u |d| + u |lp|,  p relative by lp's error + (3 |lp| + 4) u,
  the entropy H = L - t / s by 2 (Q + 6) u (|L| + sum p |d| + 1),
  -p (A + g (lp + H)) + E by p times the errors of its parts + 12 roundings of them;
A: the incoming log probability gradients' sum, E: what the link itself got of them.
The hardware's exponential gives 0 below the smallest normal number, 2^-126: p is off by that much
besides, the product by 2^-126 (|A| + |g| |lp + H|), which may pass 2^-126 itself.
Last the half step of the result's type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -126, BF16: 2.0 ** -126, F16: 2.0 ** -25}
U = 2.0 ** -24


def gradient(x, action, g1, g2, top=(), gt=()):
    """One row in float64: (gradient, softmax part, bound without the type's step)."""
    may = x > -math.inf
    d = torch.where(may, x - x[may].max(), 0.0)
    L = torch.log(torch.where(may, torch.exp(d), 0.0).sum())
    lp = torch.where(may, d - L, 0.0)
    p = torch.where(may, torch.exp(lp), 0.0)
    H = -(p * lp).sum()
    given = torch.zeros_like(x)
    given[action] += g1
    absolute = abs(g1)
    for j, t in zip(top, gt):
        given[j] += t
        absolute += abs(t)
    A = g1 + sum(gt)
    soft = -p * (A + g2 * (lp + H))
    Q = (p * (2 * d.abs() + 4)).sum() + x.numel() / 64 + 20
    e_lp = U * (Q + 3 * L.abs() + 2 * d.abs() + lp.abs())
    e_H = 2 * (Q + 6) * U * (L.abs() + (p * d.abs()).sum() + 1)
    parts = absolute + abs(g2) * (lp.abs() + H.abs())
    bound = p * (parts * (e_lp + (3 * lp.abs() + 16) * U) + abs(g2) * (e_lp + e_H)) + 2 * U * (given.abs() + absolute * p)
    bound = bound + 2.0 ** -126 * parts
    return soft + given, soft, bound


def run(logits, action, g1, g2, top_k=0, gt=None, **kw):
    from trafficrl.rl import action_log_probs
    leaf = logits.detach().requires_grad_()
    r = action_log_probs(leaf, action, top_k=top_k, **kw)
    outs, gs = [r.log_prob, r.entropy], [g1, g2]
    if top_k:
        outs.append(r.top_log_prob), gs.append(gt)
    return r, torch.autograd.grad(outs, leaf, gs)[0]


def assert_row(got, x, action, g1, g2, dt, top=(), gt=(), what=""):
    want, soft, bound = gradient(x, action, g1, g2, top, gt)
    bound = bound + HALF[dt] * want.abs() + TINY[dt]
    over = (got.double() - want).abs() > bound
    assert not bool(over.any()), (f"{what}: {int(over.sum())} of {x.numel()}, link {int(over.nonzero()[0])}: "
                                  f"{float(got[over][0])} for {float(want[over][0])}")
    # the bound can fail: where the softmax part of a link that got nothing else is a number of the type at all, the
    # bound is far below it, so a gradient without that part is outside
    plain = x > -math.inf      # links that may not be chosen have no softmax part
    plain[action] = False
    for j in top:
        plain[j] = False
    soft = soft.abs().masked_fill(~plain, 0.0)
    most = soft.argmax()
    if float(soft[most]) > 64 * TINY[dt]:
        assert float(bound[most]) < 0.05 * float(soft[most]), what


def incoming(rows, seed, top=0):
    c = torch.Generator().manual_seed(seed)
    # of size one and of no zero, so that nothing cancels by chance
    rnd = lambda *s: (torch.rand(*s, generator=c) + 0.5).cuda()  # noqa: E731
    return rnd(rows), rnd(rows) * 0.25, rnd(rows, max(1, top))


@pytest.mark.parametrize("n", [76, 914, 1025, 8193, 20011])
@pytest.mark.parametrize("dt,step,shifts", [(F32, 0.125, [0.0, 2.0 ** 14, -2.0 ** 14, 2.0 ** 20, -2.0 ** 20]),
                                            (BF16, 1.0, [0.0, 192.0, -192.0]), (F16, 1.0, [0.0, 1800.0, -1800.0])], ids=str)
def test_shift_leaves_the_gradient(n, dt, step, shifts):
    """Logits on a grid that the shifted values lie on too: every result's bits
    but log_prob's sums stay, and each entry is within its bound."""
    g = torch.Generator("cuda").manual_seed(n)
    base = torch.randint(-24, 25, (n,), device="cuda", generator=g).double() * step
    rows = torch.stack([base + s for s in shifts])
    logits = rows.to(dt)
    assert torch.equal(logits.double(), rows)
    action = torch.full((len(shifts),), n // 3, device="cuda")
    g1, g2, gt = (t[:1].expand(len(shifts), *t.shape[1:]).contiguous() for t in incoming(1, n, 4))
    for top in (0, 4):
        r, got = run(logits, action, g1, g2, top, gt)
        assert all(torch.equal(t[0], t[i]) for t in (r.log_prob, r.entropy, got) for i in range(len(shifts)))
        links = r.top_action[0].tolist() if top else []
        assert_row(got[0], rows[0], n // 3, float(g1[0]), float(g2[0]), dt, links, gt[0].tolist() if top else [], f"{n}")


FILLS = {F32: [-1e9, -1e30, torch.finfo(F32).min, 1e9], BF16: [-1e9, torch.finfo(BF16).min, 1e30],
         F16: [-30000.0, torch.finfo(F16).min, 60000.0]}


@pytest.mark.parametrize("n", [1, 2, 76, 914, 5000, 20011])
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_rows_of_one_value(n, dt):
    """Rows in which every link that may be chosen holds the same large value (a
    fill): each has its 1 / count, in log_prob, entropy and the gradient."""
    fills = torch.tensor(FILLS[dt], device="cuda").to(dt)
    rows = fills.unsqueeze(1).expand(-1, n).contiguous()
    mask = torch.ones_like(rows, dtype=torch.bool)
    mask[:, 1::3] = False
    count = int(mask[0].sum())
    action = torch.zeros(len(fills), dtype=torch.int64, device="cuda")
    g1, g2, _ = incoming(len(fills), n)
    r, got = run(rows, action, g1, g2, mask=mask)
    # log: two units in the last place of it and the sum's count of roundings
    near = (n / 64 + 24 + 3 * math.log(count)) * U
    assert float((r.log_prob.double() + math.log(count)).abs().max()) <= near
    assert float((r.entropy.double() - math.log(count)).abs().max()) <= near
    for i in range(len(fills)):
        x = torch.where(mask[i], rows[i].double(), -math.inf)
        assert_row(got[i], x, 0, float(g1[i]), float(g2[i]), dt, what=f"{n} x {float(fills[i])}")
    assert bool((got[~mask] == 0).all())


@pytest.mark.parametrize("n", [76, 914, 3000, 50001])
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("top", [0, 8])
def test_each_entry(n, dt, top):
    """Ordinary rows, some with few links at ordinary values above a fill."""
    g = torch.Generator("cuda").manual_seed(n + top)
    rows = (torch.randn(3, n, device="cuda", generator=g) * 3).to(dt)
    fill = FILLS[dt][0]
    rows[1, torch.rand(n, device="cuda", generator=g) < 0.7] = fill
    rows[2] = (rows[2].double() * 10).to(dt)
    action = rows.double().topk(20, 1)[1][:, 19]
    g1, g2, gt = incoming(3, n, top)
    r, got = run(rows, action, g1, g2, top, gt)
    for i in range(3):
        links = r.top_action[i].tolist() if top else []
        assert_row(got[i], rows[i].double(), int(action[i]), float(g1[i]), float(g2[i]), dt, links,
                   gt[i].tolist() if top else [], f"row {i}")


@pytest.mark.parametrize("hint", [None, 0, 20011])
def test_packed_entries(hint):
    """Packed rows of different lengths and offsets, each way a launch is shaped."""
    g = torch.Generator("cuda").manual_seed(7)
    sizes, shifts = [76, 20011, 1, 914, 0, 300], [-2.0 ** 20, 2.0 ** 14, 5.0, -2.0 ** 18, 0.0, 0.0]
    rows = [torch.randint(-24, 25, (s,), device="cuda", generator=g).double() / 8 + b for s, b in zip(sizes, shifts)]
    ends = torch.tensor([0, *sizes]).cumsum(0)
    action = torch.tensor([s // 2 for s in sizes], device="cuda")
    g1, g2, _ = incoming(len(sizes), 9)
    _, got = run(torch.cat(rows).float(), action, g1, g2, row_ptr=ends.cuda(), max_row=hint)
    for i, x in enumerate(rows):
        if sizes[i]:
            assert_row(got[ends[i]:ends[i + 1]], x, int(action[i]), float(g1[i]), float(g2[i]), F32, what=f"row {i}")
