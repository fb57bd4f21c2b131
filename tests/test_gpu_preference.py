"""The preference loss over label pairs against its formulas in 64 bits (oracle/label_oracle.py) and against differences: rows without pairs,
masked pairs that hold anything, labels that occur often, many pairs in few rows, labels in fp16 and in MX4."""
import math

import pytest
import torch

from oracle import label_oracle as O
from renee_amd import MX4Labels, XFCLayer, pair_margins, preference, preference_loss

pytestmark = pytest.mark.gpu


def _pairs(B, L, most, seed, few=None):
    """rowptr, chosen, rejected: up to `most` pairs a row (of two numbers the second is a middle row's), some rows without; labels among the
    first `few` repeat."""
    g = torch.Generator().manual_seed(seed)
    most, long = most if isinstance(most, tuple) else (most, None)
    n = torch.randint(0, most + 1, (B,), generator=g)
    n[0::5] = 0
    if B == 1:
        n[0] = most
    if long is not None:
        n[B // 2] = long
    rowptr = torch.cat([torch.zeros(1, dtype=torch.long), n.cumsum(0)]).int()
    P = int(rowptr[-1])
    c = torch.randint(0, few or L, (P,), generator=g).int()
    r = torch.randint(0, L, (P,), generator=g).int()
    return rowptr, c, r, torch.randn(P, generator=g) * 0.1, torch.rand(P, generator=g) + 0.5


def _problem(B, L, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, d, generator=g).to(dtype) / math.sqrt(d), torch.randn(L, d, generator=g).half()


def _check(got, want, scale, steps, what):
    """A sum in fp32 that a term goes through `steps` roundings of: 2^-24 of the magnitudes summed, `scale`, for each."""
    tol = scale * 2.0 ** -24 * steps + torch.finfo(torch.float32).tiny
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (what, float((err / tol).max()))


@pytest.mark.parametrize("mx", [False, True])
@pytest.mark.parametrize("B,L,d,most,dtype", [(1, 2, 8, 1, torch.float32), (1, 50, 64, 700, torch.float32), (5, 100, 200, 3, torch.float16), (33, 1000, 768, 9, torch.float32),
                                              (64, 300, 136, 70, torch.bfloat16), (3, 5000, 1024, 400, torch.float16), (1100, 200, 96, 4, torch.float32),
                                              (7, 90, 2048, 20, torch.float32), (4, 70, 4096, 9, torch.float16), (1, 300, 768, 9000, torch.float32),
                                              (700, 300, 200, (4, 3000), torch.float16)])
def test_loss_margins_and_gradient(dev, B, L, d, most, dtype, mx):
    x, w = _problem(B, L, d, dtype, B + d)
    rowptr, c, r, ref, wt = _pairs(B, L, most, L + d)
    labels = MX4Labels.from_weight(w.to(dev)) if mx else w.to(dev)
    wide = O.rounded(w, 4) if mx else w.double()
    beta, eps, scale = 0.7, 0.1, 3.0
    loss, margin, slope, grad, row = O.preference(x, wide, rowptr, c, r, ref, wt, beta, eps)
    got_l, got_m, got_g = preference(x.to(dev), labels, rowptr.to(dev), c.to(dev), r.to(dev), ref.to(dev), wt.to(dev), beta, eps, scale)
    # a margin's products: |x| . |w_c - w_r|
    mass = ((x.double().abs()[row.clamp(min=0)] * (wide[c.long()] - wide[r.long()]).abs()).sum(1) if len(c) else torch.zeros(0, dtype=torch.float64)) + ref.abs()
    dot = 8 * -(-d // 512) + 8  # products of a lane, then six halvings, the difference and the reference
    _check(got_m, margin, mass, dot, "margin")
    # the slope's derivative by the margin is at most a beta^2 / 4
    each = wt.double() * (beta + beta ** 2 * mass)
    total = torch.zeros_like(x, dtype=torch.float64)
    count = 1
    if len(c):
        total.index_add_(0, row.clamp(min=0), each[:, None] * (wide[c.long()] - wide[r.long()]).abs())
        count = int((rowptr[1:] - rowptr[:-1]).max())
    # exp and the quotient of the slope are within some four units, then every pair of the row and the splits are added
    _check(got_g, scale * grad, scale * total, dot + 8 + count, "grad_input")
    assert abs(float(got_l) - float(loss)) <= 2.0 ** -24 * ((dot + 8) * float((wt * beta * mass).sum()) + 8 * float(loss) + 1e-30)
    # the same loss as a differentiable scalar, in the embeddings' own type
    leaf = x.to(dev).requires_grad_(True)
    out = preference_loss(leaf, labels, rowptr.to(dev), c.to(dev), r.to(dev), ref.to(dev), wt.to(dev), beta, eps, scale)
    (out * 2.0).backward()
    assert float(out.detach()) == float(got_l)
    assert torch.equal(leaf.grad, got_g.to(dtype) * 2)
    # forward only, and what it leaves for a reference
    none = preference(x.to(dev), labels, rowptr.to(dev), c.to(dev), r.to(dev), need_grad=False)
    assert none[2] is None and torch.equal(pair_margins(x.to(dev), labels, rowptr.to(dev), c.to(dev), r.to(dev)), none[1])


def test_gradient_against_differences(dev):
    x, w = _problem(6, 40, 64, torch.float32, 3)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(6, 40, 5, 4))
    wd = w.to(dev)
    _, _, grad = preference(x.to(dev), wd, rowptr, c, r, ref, wt, 1.3, 0.2)
    g = torch.Generator().manual_seed(9)
    for _ in range(4):
        v = torch.randn(6, 64, generator=g)
        h = 1e-2
        up, down = (float(preference((x + s * h * v).to(dev), wd, rowptr, c, r, ref, wt, 1.3, 0.2)[0]) for s in (1, -1))
        along = float((grad.cpu() * v).sum())
        # A central difference is off by at most h^2 / 6 of the third derivative: a pair's margin moves by u along v, its loss's third
        # derivative is beta^3 sigmoid'', and |sigmoid''| <= 1 / (6 sqrt 3).  The two losses are off by some 2^-22 each, in inputs and sums.
        row = torch.repeat_interleave(torch.arange(6), (rowptr[1:] - rowptr[:-1]).cpu().long())
        u = (v[row] * (w[c.cpu().long()].float() - w[r.cpu().long()].float())).sum(1)
        bound = h * h / 6 * 1.3 ** 3 / (6 * math.sqrt(3)) * float((wt.cpu() * u.abs() ** 3).sum()) + (up + down) * 2.0 ** -22 / (2 * h)
        assert abs((up - down) / (2 * h) - along) <= bound


def test_masked_pairs_are_not_there(dev):
    """Labels outside the matrix, weights of zero: whatever reference, labels and weights hold there."""
    x, w = _problem(4, 30, 72, torch.float32, 5)
    w[0], w[29] = float("nan"), float("inf")
    rowptr = torch.tensor([0, 4, 4, 9, 9], dtype=torch.int32)
    c = torch.tensor([1, -1, 5, 30, 2, 0, 3, 29, 7], dtype=torch.int32)
    r = torch.tensor([2, 3, -7, 4, 2 ** 31 - 1, 4, 6, 8, 9], dtype=torch.int32)
    ref = torch.tensor([0.1, float("nan"), float("inf"), 0, 0, float("nan"), 0.2, 0, -0.3])
    wt = torch.tensor([1.0, 1, 1, 1, 1, 0, 2, 0, 1])
    kept = torch.tensor([0, 6, 8])
    loss, margin, slope, grad, row = O.preference(x, w, rowptr, c, r, ref, wt, 0.5, 0.0)
    assert row.ge(0).nonzero().flatten().tolist() == kept.tolist()
    got = preference(x.to(dev), w.to(dev), rowptr.to(dev), c.to(dev), r.to(dev), ref.to(dev), wt.to(dev), 0.5)
    assert abs(float(got[0]) - float(loss)) < 1e-6 * float(loss)
    assert torch.allclose(got[1].cpu().double(), margin, rtol=0, atol=1e-5) and torch.equal(got[1].cpu() == 0, margin == 0)
    assert torch.allclose(got[2].cpu().double(), grad, rtol=0, atol=1e-5) and bool((got[2][1] == 0).all()) and bool((got[2][3] == 0).all())
    g0 = torch.zeros(4, 32, dtype=torch.float16, device=dev)
    g0[:, 30:] = 5
    preference(x.to(dev), w.to(dev), rowptr.to(dev), c.to(dev), r.to(dev), ref.to(dev), wt.to(dev), 0.5, g=g0)
    want = O.add_to_g(torch.zeros(4, 30), row, c.long(), r.long(), slope)
    assert torch.equal(g0[:, :30].cpu() != 0, want != 0) and bool((g0[:, 30:] == 5).all())


@pytest.mark.parametrize("B,L,most,few", [(1, 20, 1, None), (9, 500, 30, 2), (40, 64, 200, 1), (2, 3000, 1500, 3), (300, 1000, 8, None),
                                            (3, 70, 513, None), (1, 2000, 1024, None)])
def test_pairs_added_to_g(dev, B, L, most, few):
    x, w = _problem(B, L, 64, torch.float16, B + L)
    rowptr, c, r, ref, wt = _pairs(B, L, most, B, few)
    g0 = torch.rand(B, L + 16, generator=torch.Generator().manual_seed(2)).half()
    _, _, slope, _, row = O.preference(x, w, rowptr, c, r, ref, wt, 2.0, 0.05)
    want = O.add_to_g(g0, row, c.long(), r.long(), slope)
    g = g0.to(dev)
    _, _, grad = preference(x.to(dev), w.to(dev), rowptr.to(dev), c.to(dev), r.to(dev), ref.to(dev), wt.to(dev), 2.0, 0.05, g=g)
    assert grad is None
    # half a step of fp16 for every 512 pairs of the row, and fp32 sums of the slopes
    amount = torch.zeros_like(want)
    if len(c):
        amount = O.add_to_g(torch.zeros_like(want), row, c.long(), torch.zeros_like(r).long(), 0 * slope)
        for k in (c, r):
            amount.index_put_((row.clamp(min=0), k.long()), slope.abs(), accumulate=True)
    rounds = -(-most // 512)
    tol = rounds * 2.0 ** -11 * (want.abs() + (amount if rounds > 1 else 0)) + 2.0 ** -18 * amount + 2.0 ** -25
    tol = torch.where(amount > 0, tol, 0.0)
    err = (g.cpu().double() - want).abs()
    assert bool((err <= tol).all()), float((err / tol.clamp(min=1e-30)).max())
    again = g0.to(dev)
    preference(x.to(dev), w.to(dev), rowptr.to(dev), c.to(dev), r.to(dev), ref.to(dev), wt.to(dev), 2.0, 0.05, g=again)
    assert torch.equal(again, g)


def test_row_pointers_that_do_not_ascend_or_leave_the_list(dev):
    """Pairs of no row have no margin; row pointers beyond the list end with it; those that do not ascend do no harm."""
    x, w = _problem(4, 30, 64, torch.float32, 7)
    c = torch.arange(10, dtype=torch.int32)
    r = c + 10
    for rowptr in ([3, 5, 5, 6, 8], [0, 0, 4, 6, 99], [-3, 1, 2, 2, 2]):
        rp = torch.tensor(rowptr, dtype=torch.int32)
        _, margin, _, grad, row = O.preference(x, w, rp, c, r, beta=0.5)
        got = preference(x.to(dev), w.to(dev), rp.to(dev), c.to(dev), r.to(dev), beta=0.5)
        assert torch.allclose(got[2].cpu().double(), grad, rtol=0, atol=1e-5)
        assert torch.equal(got[1].cpu() != 0, row >= 0)
    preference(x.to(dev), w.to(dev), torch.tensor([2, 5, 3, 8, 99], dtype=torch.int32, device=dev), c.to(dev), r.to(dev), beta=0.5)
    torch.cuda.synchronize()


def test_large_margins_do_not_overflow(dev):
    x = torch.ones(2, 64, device=dev)
    w = torch.zeros(4, 64, dtype=torch.float16, device=dev)
    w[1], w[2] = 1000.0, -1000.0
    rowptr = torch.tensor([0, 1, 2], dtype=torch.int32, device=dev)
    c, r = torch.tensor([1, 2], dtype=torch.int32, device=dev), torch.tensor([2, 1], dtype=torch.int32, device=dev)
    loss, margin, grad = preference(x, w, rowptr, c, r, beta=1.0)
    assert margin.tolist() == [128000.0, -128000.0] and float(loss) == 128000.0
    assert bool((grad[0] == 0).all()) and bool((grad[1] == 2000.0).all())
    assert float(preference(x, w, rowptr, c, r, beta=1.0, label_smoothing=0.25)[0]) == 128000.0


def test_a_step_of_the_classifier_with_pairs(dev):
    """fwd_grad, preference_grad, backward_pass: dX, W and the momentum are those of G with the pairs' slopes in it."""
    B, L, d = 48, 700, 128
    x, w = _problem(B, L, d, torch.float16, 13)
    w = w * 0.05
    rowptr, c, r, ref, _ = _pairs(B, L, 6, 14)
    px, py = torch.arange(B), torch.randint(0, L, (B,), generator=torch.Generator().manual_seed(3))
    layer = XFCLayer(L, d, B, dev, weight=w, lr=0.1)
    with pytest.raises(RuntimeError, match="fwd_grad"):
        layer.preference_grad(x.to(dev), rowptr, c, r)
    layer.fwd_grad(x.to(dev), px, py)
    layer.preference_grad(x.to(dev), rowptr, c, r, ref, beta=2.0)
    grad = layer.backward_pass(x.to(dev)).cpu().double()
    G = torch.sigmoid(x.double() @ w.double().t())
    G[px, py] -= 1
    _, _, slope, _, row = O.preference(x, w, rowptr, c, r, ref, None, 2.0)
    G = O.add_to_g(G, row, c.long(), r.long(), slope)
    dX, M = G @ w.double(), G.t() @ x.double()
    W = w.double() - 0.1 * M
    for got, want in ((grad, dX), (layer.momentum_buffer, M), (layer.xfc_weight, W)):
        assert float((got.cpu().double() - want).norm() / want.norm()) < 1e-3


@pytest.mark.parametrize("B,d,most", [(40, 128, 7), (2, 64, 200)])
def test_captured(dev, B, d, most):
    """Replays follow new embeddings, with eager calls between them."""
    x, w = _problem(B, 300, d, torch.float32, 21)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(B, 300, most, 1))
    labels = MX4Labels.from_weight(w.to(dev))
    static = x.to(dev)
    preference(static, labels, rowptr, c, r, ref, wt, 0.9, 0.1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = preference(static, labels, rowptr, c, r, ref, wt, 0.9, 0.1)
    for k in range(3):
        static.copy_(x.to(dev) * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, preference(static, labels, rowptr, c, r, ref, wt, 0.9, 0.1)))


def test_captured_with_its_backward_pass(dev):
    x, w = _problem(20, 300, 128, torch.float32, 27)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(20, 300, 7, 1))
    labels = MX4Labels.from_weight(w.to(dev))
    leaf = x.to(dev).requires_grad_(True)

    def step():
        preference_loss(leaf, labels, rowptr, c, r, ref, wt, 0.9, 0.1).backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    leaf.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        with torch.no_grad():
            leaf.copy_(x.to(dev) * (k + 1))
        leaf.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = preference(leaf.detach(), labels, rowptr, c, r, ref, wt, 0.9, 0.1)[2]
        assert torch.equal(leaf.grad, want)


def test_a_second_derivative_is_refused(dev):
    x, w = _problem(3, 30, 64, torch.float32, 29)
    rowptr, c, r, _, _ = (t.to(dev) for t in _pairs(3, 30, 4, 2))
    leaf = x.to(dev).requires_grad_(True)
    (grad,) = torch.autograd.grad(preference_loss(leaf, w.to(dev), rowptr, c, r), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_embeddings_that_are_expanded_strided_or_on_the_cpu(dev):
    x, w = _problem(6, 50, 64, torch.float32, 33)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(6, 50, 6, 4))
    one = x[:1].to(dev).requires_grad_(True)
    preference_loss(one.expand(6, 64), w.to(dev), rowptr, c, r, ref, wt, 0.5).backward()
    want = preference(x[:1].expand(6, 64).to(dev), w.to(dev), rowptr, c, r, ref, wt, 0.5)[2]
    assert torch.allclose(one.grad, want.sum(0, keepdim=True), rtol=1e-6, atol=1e-6)
    wide = torch.zeros(6, 130, device=dev)
    wide[:, 3:67] = x.to(dev)
    full = preference(x.to(dev), w.to(dev), rowptr, c, r, ref, wt, 0.5)
    assert all(torch.equal(a, b) for a, b in zip(preference(wide[:, 3:67], w.to(dev), rowptr, c, r, ref, wt, 0.5), full))
    leaf = x.clone().requires_grad_(True)
    preference_loss(leaf, w.to(dev), rowptr.cpu(), c.cpu(), r.cpu(), ref.cpu(), wt.cpu(), 0.5).backward()
    assert leaf.grad.device.type == "cpu" and torch.equal(leaf.grad, full[2].cpu())


def test_both_gradients_in_one_call(dev):
    from renee_amd._lib import check, lib

    x, w = _problem(12, 100, 64, torch.float32, 37)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(12, 100, 9, 6))
    xd, wd = x.to(dev), w.to(dev)
    want = preference(xd, wd, rowptr, c, r, ref, wt, 0.5)
    g0 = torch.rand(12, 104, device=dev).half()
    gw = g0.clone()
    preference(xd, wd, rowptr, c, r, ref, wt, 0.5, g=gw)
    P, g = len(c), g0.clone()
    loss, margin, dx = torch.empty((), device=dev), torch.empty(P, device=dev), torch.full((12, 72), 7.0, device=dev)
    need = lib().xfc_preference_workspace_bytes(12, P, 64)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    check(lib().xfc_preference(xd.data_ptr(), 2, 64, wd.data_ptr(), 64, None, 100, 64, rowptr.data_ptr(), c.data_ptr(), r.data_ptr(), ref.data_ptr(), wt.data_ptr(),
                               12, P, 0.5, 0.0, 1.0, loss.data_ptr(), margin.data_ptr(), dx.data_ptr(), 2, 72, g.data_ptr(), 104, ws.data_ptr(), need,
                               torch.cuda.current_stream().cuda_stream), "xfc_preference")
    assert torch.equal(loss, want[0]) and torch.equal(margin, want[1]) and torch.equal(dx[:, :64], want[2]) and torch.equal(g, gw)
    assert bool((dx[:, 64:] == 7).all())


def test_on_another_stream(dev):
    x, w = _problem(40, 300, 128, torch.float32, 23)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(40, 300, 7, 2))
    labels, xd = MX4Labels.from_weight(w.to(dev)), x.to(dev)
    want = preference(xd, labels, rowptr, c, r, ref, wt)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = preference(xd, labels, rowptr, c, r, ref, wt)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_no_rows_and_no_pairs(dev):
    w = torch.ones(5, 64, dtype=torch.float16, device=dev)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    loss, margin, grad = preference(torch.empty(0, 64, device=dev), w, torch.zeros(1, dtype=torch.int32, device=dev), none, none)
    assert float(loss) == 0 and margin.numel() == 0 and grad.shape == (0, 64)
    loss, margin, grad = preference(torch.ones(3, 64, device=dev), w, torch.zeros(4, dtype=torch.int32, device=dev), none, none)
    assert float(loss) == 0 and bool((grad == 0).all())


def test_scoring_and_tuning_together(dev):
    """Quantise a layer's labels, keep their margins as the reference, tune the embeddings on pairs, score again: the first steps' losses
    fall below that of no change, log 2 a pair, along the gradient."""
    x, w = _problem(16, 400, 96, torch.float32, 31)
    layer = XFCLayer(400, 96, 16, dev, weight=w * 0.1)
    labels = layer.quantize_labels()
    rowptr, c, r, _, _ = (t.to(dev) for t in _pairs(16, 400, 5, 3))
    leaf = x.to(dev).requires_grad_(True)
    ref = pair_margins(leaf, labels, rowptr, c, r)
    loss = preference_loss(leaf, labels, rowptr, c, r, ref, beta=1.0)
    used = len(c)
    assert abs(float(loss.detach()) - used * math.log(2)) < 1e-5 * used
    loss.backward()
    assert leaf.grad.shape == x.shape and bool(torch.isfinite(leaf.grad).all())
    values, best = labels.topk(leaf, 5)
    z = labels.xfc_forward(leaf).float()
    assert torch.allclose(values, z.gather(1, best), rtol=2.0 ** -11, atol=1e-6)


@pytest.mark.parametrize("empty", ["behind", "before", "between", "no rows"])
def test_rows_without_pairs_are_not_gone_through(dev, empty):
    """65,536 rows of which almost none has pairs, and pairs that no row has (a slice of a list's rows): waves go on at the next row that has
    any, wherever it is.  (Row by row 8.9 ms; 0.13 for all pairs in the first row.)"""
    B, P = 65536, 1024
    x, w = _problem(B, 100, 64, torch.float16, 47)
    g = torch.Generator().manual_seed(1)
    c, r = (torch.randint(0, 100, (P,), generator=g).int() for _ in range(2))
    xd, wd, cd, rd = x.to(dev), w.to(dev), c.to(dev), r.to(dev)

    def timed(rowptr):
        rp, best = rowptr.to(dev), math.inf
        out = preference(xd, wd, rp, cd, rd)
        for _ in range(5):
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            preference(xd, wd, rp, cd, rd)
            end.record()
            torch.cuda.synchronize()
            best = min(best, start.elapsed_time(end))
        return best, out

    def pointers(*ends):
        """Of rows that end at these pairs from the given rows on; the first is where row 0 begins."""
        rp = torch.zeros(B + 1, dtype=torch.int32)
        for row, pair in ends:
            rp[row:] = pair
        return rp

    usual, _ = timed(pointers((0, 0), (1, P)))
    for rp in {"behind": [pointers((0, 0), (1, 503)), pointers((0, 0), (1, 4))],
               "before": [pointers((0, 0), (B, P)), pointers((0, 2), (B, P)), pointers((0, 501), (B // 2, 503))],
               "between": [pointers((0, 0), (1, 2), (B, P)), pointers((0, 1), (3, 2), (70, 3), (40000, 5), (B - 1, 1001), (B, 1022))],
               "no rows": [pointers((0, P - 4), (1, P)), pointers((0, 500), (1, 503)), pointers((0, P)), pointers((0, 7))]}[empty]:
        time, got = timed(rp)
        rows, has, beta = (rp[1:] > rp[:-1]).nonzero().flatten(), torch.zeros(P, dtype=torch.bool), 0.1
        assert torch.equal((got[2] != 0).any(1).nonzero().flatten().cpu(), rows)
        for b in rows.tolist():
            s = slice(int(rp[b]), int(rp[b + 1]))
            has[s] = True
            _, margin, _, grad, _ = O.preference(x[b:b + 1], w, torch.tensor([0, s.stop - s.start]), c[s], r[s], beta=beta)
            # as in test_loss_margins_and_gradient: a lane's eight products, six halvings and the two differences; then the slope and the row's pairs
            diff = (w.double()[c[s].long()] - w.double()[r[s].long()]).abs()
            mass = diff @ x[b].double().abs()
            _check(got[1][s], margin, mass, 16, "margin")
            _check(got[2][b], grad[0], (beta + beta ** 2 * mass) @ diff, 16 + 8 + s.stop - s.start, "grad_input")
        assert not got[1].cpu()[~has].any()
        assert time < 4 * usual
