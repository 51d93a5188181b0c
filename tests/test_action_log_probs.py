"""trafficrl.rl.action_log_probs (csrc/action_log_probs.hip) against its
definition in float64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
U = 2.0 ** -24


def reference_row(x, action, top, g=None):
    """One row in float64: log_prob, entropy, top values and links, gradient."""
    n = x.numel()
    may = x > -math.inf
    if not bool(may.any()):
        return -math.inf, 0.0, [-math.inf] * top, [-1] * top, torch.zeros_like(x)
    lp = torch.where(may, x - torch.logsumexp(x, 0), -math.inf)
    p = torch.where(may, torch.exp(lp), 0.0)
    plp = torch.where(p > 0, p * lp, 0.0)
    entropy = float(-plp.sum())
    chosen = float(lp[action]) if 0 <= action < n else -math.inf
    values = x.tolist()
    order = sorted(range(n), key=lambda j: (-values[j], j))
    order = [j for j in order[:top] if bool(may[j])]
    links = order + [-1] * (top - len(order))
    values = [float(lp[j]) for j in order] + [-math.inf] * (top - len(order))
    grad = torch.zeros_like(x)
    if g is not None:
        g1, g2, gt = g
        if chosen > -math.inf:
            grad -= g1 * p
            grad[action] += g1
        grad -= g2 * torch.where(p > 0, p * (lp + entropy), 0.0)
        for t, j in enumerate(order):
            grad -= gt[t] * p
            grad[j] += gt[t]
    return chosen, entropy, values, links, grad


def near(got, want, bound, what):
    got, want = float(got.detach()) if torch.is_tensor(got) else got, float(want)
    if not math.isfinite(want):
        assert got == want, f"{what}: {got} for {want}"
    else:
        assert abs(got - want) <= bound, f"{what}: {got} for {want}, bound {bound:.3g}"


def check(rows, dt, top, mask, action, grads, row_ptr=None, stride=None, mask_type=F32, **kw):
    """rows: list of float64 rows (values of dt); mask: list of bool rows or None."""
    from trafficrl.rl import action_log_probs
    lengths = [r.numel() for r in rows]
    if row_ptr is None:
        logits = torch.stack(rows).to(dt)
        m = None if mask is None else torch.stack(mask).to(mask_type)
        if stride:
            wide = torch.full((len(rows), stride), 7.0, device="cuda", dtype=dt)
            wide[:, :lengths[0]] = logits
            logits = wide[:, :lengths[0]]
    else:
        logits = torch.full((row_ptr["total"],), math.nan, device="cuda", dtype=dt)
        m = None if mask is None else torch.ones(row_ptr["total"], device="cuda").to(mask_type)
        for r, at in zip(range(len(rows)), row_ptr["at"]):
            logits[at:at + lengths[r]] = rows[r].to(dt)
            if m is not None:
                m[at:at + lengths[r]] = mask[r].to(mask_type)
        kw["row_ptr"] = torch.tensor(row_ptr["at"], device="cuda")
    logits = logits.detach().requires_grad_()
    r = action_log_probs(logits, torch.tensor(action, device="cuda"), mask=m, top_k=top, **kw)
    outs, gs = [r.log_prob, r.entropy], [torch.tensor(grads[0], device="cuda"), torch.tensor(grads[1], device="cuda")]
    if top:
        outs, gs = outs + [r.top_log_prob], gs + [torch.tensor(grads[2], device="cuda").view(len(rows), top)]
    got, = torch.autograd.grad(outs, logits, gs)
    assert got.dtype == dt and r.log_prob.dtype == r.entropy.dtype == F32
    touched = torch.zeros(got.shape, dtype=torch.bool, device="cuda")
    for i, row in enumerate(rows):
        x = row if mask is None else torch.where(mask[i], row, -math.inf)
        g = (grads[0][i], grads[1][i], grads[2][i] if top else [])
        chosen, entropy, values, links, grad = reference_row(x, action[i], top, g)
        # x - m is exact to u |x - m|; sums of n terms lose at most n u; log and exp a few u
        fin = torch.where(x > -math.inf, x, 0.0)
        size = float(fin.abs().max()) if row.numel() else 0.0
        span = 2 * size + math.log(max(2, row.numel()))
        err = U * (row.numel() + 12 + 6 * span)
        near(r.log_prob[i], chosen, err * 2 + U * span, f"row {i} log_prob")
        near(r.entropy[i], entropy, err * (2 + 2 * span), f"row {i} entropy")
        if top:
            assert r.top_action[i].tolist() == links, f"row {i}"
            for a, b in zip(r.top_log_prob[i].tolist(), values):
                near(a, b, err * 2 + U * span, f"row {i} top")
        if row_ptr is None:
            mine = got[i]
            touched[i] = True
        else:
            at = row_ptr["at"][i]
            mine = got[at:at + row.numel()]
            touched[at:at + row.numel()] = True
        total = abs(g[0]) + sum(abs(t) for t in g[2]) + abs(g[1]) * (2 * span + 2)
        bound = 6 * err * total + HALF[dt] * grad.abs() + 2.0 ** -25
        assert bool(((mine.double() - grad).abs() <= bound).all()), f"row {i} gradient"
        if row.numel():
            assert bool((mine[~(x > -math.inf)] == 0).all())
    assert bool((got[~touched] == 0).all())


def case(count, n, dt, seed, masked=0.4, top=4):
    g = torch.Generator("cuda").manual_seed(seed)
    sizes = [n] * count if isinstance(n, int) else n
    rows = [(torch.randn(s, device="cuda", generator=g) * 3).to(dt).double() for s in sizes]
    mask = [torch.rand(s, device="cuda", generator=g) >= masked for s in sizes] if masked else None
    c = torch.Generator().manual_seed(seed)
    action = [int(torch.randint(-1, max(1, s) + 1, (1,), generator=c)) if s < 50 else
              int(torch.randint(0, s, (1,), generator=c)) for s in sizes]
    grads = [torch.randn(len(sizes), generator=c).tolist(), torch.randn(len(sizes), generator=c).tolist(),
             torch.randn(len(sizes), max(1, top), generator=c).tolist()]
    return rows, mask, action, grads


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 76, 255, 914, 1024, 1025, 4095])
@pytest.mark.parametrize("dt", [F32, BF16, F16], ids=str)
def test_lengths(n, dt):
    for top, masked in ((0, 0.0), (4, 0.4), (16, 0.95)):
        rows, mask, action, grads = case(5, n, dt, n + top, masked, top)
        check(rows, dt, top, mask, action, grads)


@pytest.mark.parametrize("n", [16384, 16385, 50001, 131072])
@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_long_rows(n, dt):
    """Rows longer than one workgroup holds; in bfloat16 the best values tie."""
    rows, mask, action, grads = case(2, n, dt, n, 0.3, 8)
    check(rows, dt, 8, mask, action, grads)
    rows, _, action, grads = case(1, n, dt, n + 1, 0.0, 16)
    check(rows, dt, 16, None, action, grads)


@pytest.mark.parametrize("dt", [F32, BF16], ids=str)
def test_packed(dt):
    """Rows of different lengths, empty ones among them, elements of no row before
    and behind them (NaN there stays unread)."""
    sizes = [76, 0, 1, 914, 20011, 5, 0, 300]
    rows, mask, action, grads = case(0, sizes, dt, 3, 0.4, 8)
    at = [11]
    for s in sizes:
        at.append(at[-1] + s)
    layout = {"at": at, "total": at[-1] + 40}
    for hint in (None, 0, 76, 20011):
        check(rows, dt, 8, mask, action, grads, row_ptr=layout, max_row=hint)
    check(rows, dt, 8, mask, action, grads, row_ptr=layout, mask_type=torch.bool)


def test_mask_types_and_strides():
    rows, mask, action, grads = case(7, 76, F32, 1)
    for t in (F32, torch.bool, torch.uint8, torch.int64, BF16, torch.float64):
        check(rows, F32, 4, mask, action, grads, mask_type=t)
    check(rows, F32, 4, mask, action, grads, stride=91)
    check([r.to(BF16).double() for r in rows], BF16, 4, mask, action, grads, stride=77)


def test_rows_of_no_choice():
    """Everything masked; logits of -inf; one link left; ties; the type's lowest value."""
    n = 40
    low = torch.finfo(F32).min
    rows = [torch.linspace(-2, 2, n, device="cuda", dtype=torch.float64) for _ in range(6)]
    mask = [torch.ones(n, dtype=torch.bool, device="cuda") for _ in range(6)]
    mask[0][:] = False
    rows[1][:] = -math.inf
    mask[2][:] = False
    mask[2][17] = True
    rows[3][:] = 1.5
    rows[4][:] = low
    rows[5][:39] = low
    check(rows, F32, 6, mask, [3, 4, 17, 39, 2, 5],
          [[1.0] * 6, [0.5] * 6, [[1.0, -1.0, 2.0, 0.5, 0.25, 3.0]] * 6])


@pytest.mark.parametrize("n", [200, 3000, 40000])
def test_equal_and_sorted_rows(n):
    """Constant, rising and falling rows: ties go to the lower link, and the best
    links may all lie in one lane's share."""
    flat = torch.full((n,), 0.25, device="cuda", dtype=torch.float64)
    rise = (torch.arange(n, device="cuda") / 4096).to(F32).double()
    block = torch.zeros(n, device="cuda", dtype=torch.float64)
    block[::64] = 1.0 + torch.arange((n + 63) // 64, device="cuda").double() / 2048
    block8 = torch.zeros(n, device="cuda", dtype=torch.float64)
    block8[80:88] = 2.0
    zeros = torch.zeros(n, device="cuda", dtype=torch.float64)
    zeros[1::2] = -0.0
    rows = [flat, rise, rise.flip(0), block, block8, zeros]
    check(rows, F32, 16, None, [0, 1, 2, 3, 4, 5], [[1.0] * 6, [1.0] * 6, [[0.5] * 16] * 6])


def test_nan_and_inf():
    from trafficrl.rl import action_log_probs
    for n in (30, 5000, 40000):
        x = torch.randn(4, n, device="cuda")
        x[1, 7], x[2, 8] = math.nan, math.inf
        mask = torch.ones(4, n, device="cuda")
        x[3, 9:12] = torch.tensor([math.nan, math.inf, -math.inf], device="cuda")
        mask[3, 9:12] = 0.0
        mask[0, 5] = math.nan        # not > 0
        r = action_log_probs(x, torch.zeros(4, dtype=torch.int64, device="cuda"), mask=mask, top_k=3)
        bad = torch.tensor([False, True, True, False], device="cuda")
        assert torch.equal(r.log_prob.isnan(), bad) and torch.equal(r.entropy.isnan(), bad)
        assert int(r.top_action[1, 0]) == 7 and int(r.top_action[2, 0]) == 8


def test_gradient_against_differences():
    """<gradient, direction> against a central difference of the float64 definition."""
    from trafficrl.rl import action_log_probs
    rows, _, _, _ = case(3, 50, F32, 4, 0.0)
    x = torch.stack(rows).float().requires_grad_()
    action = torch.tensor([4, 0, 49], device="cuda")
    r = action_log_probs(x, action, top_k=3)
    g, = torch.autograd.grad([r.log_prob.sum() + 2 * r.entropy.sum() - r.top_log_prob.sum()], x)

    def value(y):
        lp = torch.log_softmax(y, 1)
        best = torch.gather(lp, 1, r.top_action)
        return float(lp.gather(1, action.unsqueeze(1)).sum() - 2 * (lp.exp() * lp).sum() - best.sum())

    step = torch.randn(3, 50, device="cuda", dtype=torch.float64)
    y, eps = x.detach().double(), 1e-5
    numeric = (value(y + eps * step) - value(y - eps * step)) / (2 * eps)
    # float32 terms of size up to 60 u each along 150 components; the difference's own error 1e-15 / eps
    assert abs(float((g.double() * step).sum()) - numeric) <= 60 * 150 * U * 8 + 1e-8 * 60


def test_captured_and_streams():
    from trafficrl.rl import action_log_probs
    x = torch.randn(3, 40001, device="cuda")
    action = torch.tensor([1, 2, 3], device="cuda")

    def both():
        leaf = x.detach().requires_grad_()
        r = action_log_probs(leaf, action, top_k=8)
        return [t.detach() for t in r] + list(torch.autograd.grad([r.log_prob, r.entropy], leaf,
                                                                  [torch.ones(3, device="cuda")] * 2))

    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    for seed in range(3):
        x.copy_(torch.randn(3, 40001, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)))
        want = both()
        graph.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        torch.cuda.synchronize()
        for a, b, c in zip(held, want, other):
            assert torch.equal(a, b) and torch.equal(b, c)


def test_no_rows():
    from trafficrl.rl import action_log_probs
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    r = action_log_probs(torch.zeros(0, 76, device="cuda"), none, top_k=2)
    assert r.log_prob.shape == (0,) and r.top_action.shape == (0, 2)
    r = action_log_probs(torch.zeros(3, 0, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), top_k=2)
    assert bool((r.log_prob == -math.inf).all()) and bool((r.top_action == -1).all()) and bool((r.entropy == 0).all())
    x = torch.zeros(9, device="cuda", requires_grad=True)
    r = action_log_probs(x, none, row_ptr=torch.tensor([4], device="cuda"))
    assert bool((torch.autograd.grad(r.log_prob.sum() + r.entropy.sum(), x)[0] == 0).all())


def test_beyond_32_bits():
    """Packed elements behind 2^31 are found."""
    from trafficrl.rl import action_log_probs
    n = 2 ** 31 + 5000
    x = torch.zeros(n, device="cuda", dtype=BF16)
    x[-300:] = torch.randn(300, device="cuda").to(BF16)
    ptr = torch.tensor([n - 300, n - 100, n], device="cuda")
    a = torch.tensor([5, 6], device="cuda")
    r = action_log_probs(x, a, row_ptr=ptr, max_row=200, top_k=4)
    s = action_log_probs(x[-300:].clone(), a, row_ptr=torch.tensor([0, 200, 300], device="cuda"), max_row=200, top_k=4)
    assert all(torch.equal(u, v) for u, v in zip(r, s))


def test_many_short_rows_and_a_long_one():
    """More rows than a launch has workgroups for: the long row's further chunks
    are looped over; without the hint the same bits as alone, links in order."""
    from trafficrl.rl import action_log_probs
    many, n = 40000, 50001
    g = torch.Generator("cuda").manual_seed(5)
    x = torch.randn(3 * many + n, device="cuda", generator=g)
    ptr = torch.cat([torch.arange(many + 1, device="cuda") * 3, torch.tensor([3 * many + n], device="cuda")])
    act = torch.zeros(many + 1, dtype=torch.int64, device="cuda")
    act[-1] = n - 1
    y = x.clone().requires_grad_()
    r = action_log_probs(y, act, row_ptr=ptr)
    grad, = torch.autograd.grad(r.log_prob.sum(), y)
    # float64, and the bounds: exp, sums of n terms in any order and the division, each 2^-24 relative to values <= 1
    for part, rows, links in ((slice(0, 3 * many), many, 3), (slice(3 * many, None), 1, n)):
        p = torch.softmax(x[part].double().view(rows, links), 1)
        onehot = torch.nn.functional.one_hot(act[:many] if rows > 1 else act[-1:], links)
        assert ((grad[part].view(rows, links) - (onehot - p)).abs() <= (links + 64) * U).all()
