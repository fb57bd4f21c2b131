"""What preference_loss hands to autograd: the gradient in the embeddings' type, rounded once behind the factor that comes down the graph, so that a
loss scale keeps what a narrower type would lose before it; equal to the bit to the fp32 gradient (tests/test_gpu_preference.py holds that
against 64 bits) times the factor, rounded by torch."""
import pytest
import torch

from renee_amd import preference, preference_loss
from tests.test_gpu_preference import _pairs, _problem

pytestmark = pytest.mark.gpu


def _both(dev, x, w, lists, factor, **how):
    leaf = x.to(dev).requires_grad_(True)
    lists = [t.to(dev) for t in lists]
    (preference_loss(leaf, w.to(dev), *lists, **how) * factor).backward()
    return leaf.grad, preference(x.to(dev), w.to(dev), *lists, **how)[2]


@pytest.mark.parametrize("factor", [65536.0, 1.0, 2.0 ** -20])
@pytest.mark.parametrize("size", [1e-6, 1.0, 6e4])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_factor_is_applied_before_the_rounding(dev, dtype, size, factor):
    x, w = _problem(9, 50, 64, dtype, 41)
    w = (w.float() * 0.25 * size).clamp(-65504, 65504).half()
    got, exact = _both(dev, x, w, _pairs(9, 50, 6, 42)[:3], factor, beta=0.25)
    assert exact.dtype == torch.float32 and bool(torch.isfinite(exact).all()) and float(exact.abs().max()) > 0
    if size == 1e-6:
        assert float(exact.abs().max()) < 2.0 ** -20  # in fp16 a few steps, most of them none
    assert got.dtype == dtype and torch.equal(got, (exact * factor).to(dtype))


def test_a_gradient_under_a_factor_is_off_by_half_a_step(dev):
    """2 g of 140,000 numbers, some below fp16's normal ones, where rounding g and then doubling is off by up to a whole step."""
    x, w = _problem(700, 300, 200, torch.float16, 900)
    lists = _pairs(700, 300, (4, 3000), 500)
    got, exact = _both(dev, x, w, lists, 2.0, beta=0.7, label_smoothing=0.1, scale=3.0)
    want = exact.double() * 2
    step = torch.exp2(torch.floor(torch.log2(want.abs().clamp(min=2.0 ** -14))) - 10)
    assert bool(((got.double() - want).abs() <= step / 2).all())
    assert bool(((exact.half().double() * 2 - want).abs() > step / 2).any())  # (what rounding first would give)


def test_the_gradient_is_a_saved_tensor(dev):
    """Hooks on saved tensors see it, and a backward pass frees it."""
    x, w = _problem(5, 40, 64, torch.float16, 43)
    rowptr, c, r = (t.to(dev) for t in _pairs(5, 40, 4, 44)[:3])
    leaf, seen = x.to(dev).requires_grad_(True), []

    def pack(t):
        seen.append((t.shape, t.dtype))
        return t.cpu()

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t.to(dev)):
        loss = preference_loss(leaf, w.to(dev), rowptr, c, r)
    assert seen == [((5, 64), torch.float32)]
    loss.backward()
    assert torch.equal(leaf.grad, preference(x.to(dev), w.to(dev), rowptr, c, r)[2].half())
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    again = preference_loss(leaf, w.to(dev), rowptr, c, r)
    leaf.grad = None
    again.backward(retain_graph=True)
    again.backward()
    assert torch.equal(leaf.grad, 2 * preference(x.to(dev), w.to(dev), rowptr, c, r)[2].half())


def test_a_label_matrix_that_requires_grad_gets_none(dev):
    x, w = _problem(5, 40, 64, torch.float32, 45)
    rowptr, c, r = (t.to(dev) for t in _pairs(5, 40, 4, 46)[:3])
    leaf, labels = x.to(dev).requires_grad_(True), w.to(dev).requires_grad_(True)
    preference_loss(leaf, labels, rowptr, c, r).backward()
    assert labels.grad is None and torch.equal(leaf.grad, preference(x.to(dev), w.to(dev), rowptr, c, r)[2])
    assert not preference_loss(x.to(dev), labels, rowptr, c, r).requires_grad


@pytest.mark.parametrize("most", [4, (3, 700)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_gradient_asked_for_in_a_narrow_type_is_rounded_once(dev, dtype, most):
    """preference(grad_dtype=): rows of one chunk of pairs and of several."""
    x, w = _problem(40, 60, 72, torch.float32, 51)
    lists = [t.to(dev) for t in _pairs(40, 60, most, 52)]
    exact = preference(x.to(dev), w.to(dev), *lists, 0.5, 0.1, 1.5)[2]
    got = preference(x.to(dev), w.to(dev), *lists, 0.5, 0.1, 1.5, grad_dtype=dtype)[2]
    assert got.dtype == dtype and torch.equal(got, exact.to(dtype))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_captured_with_a_loss_scale(dev, dtype):
    """A captured forward and backward pass of narrow embeddings, replayed with new embeddings and scales beside eager calls."""
    x, w = _problem(20, 300, 128, torch.float32, 53)
    rowptr, c, r, ref, wt = (t.to(dev) for t in _pairs(20, 300, 7, 54))
    x, w, scale = x.to(dev), w.to(dev), torch.tensor(65536.0, device=dev)
    leaf = x.to(dtype).requires_grad_(True)

    def step():
        (preference_loss(leaf, w, rowptr, c, r, ref, wt, 1e-3) * scale).backward()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    leaf.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(4):
        with torch.no_grad():
            leaf.copy_(x * (k + 1))
        scale.fill_(2.0 ** (16 - 4 * k))
        leaf.grad.zero_()
        graph.replay()
        torch.cuda.synchronize()
        exact = preference(leaf.detach(), w, rowptr, c, r, ref, wt, 1e-3)[2]
        assert bool(exact.any()) and torch.equal(leaf.grad, (exact * scale).to(dtype))
