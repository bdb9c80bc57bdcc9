"""Masked classes together with label smoothing, whose loss has the mean of all scores in it."""
import pytest

torch = pytest.importorskip("torch")

from test_head_loss_gpu import TYPES, _make, _reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "mean"])
@pytest.mark.parametrize("n,k,v", [(150, 64, 700), (300, 300, 90), (200, 64, 90), (70, 256, 33), (140, 128, 128)])
def test_lowest_values_with_smoothing(cuda, n, k, v, reduction, dtype):
    """Several classes at the type's lowest value: their sum leaves fp32 for bfloat16, their mean does not, and the loss is the finite number that
    the formula gives: 2^-20 relative (a sum of up to v / 128 + 32 terms of one size, 1 / v and a product; 0.1 is 2^-26 off
    in 32 bits) beside the errors of the scores that are not masked, which the bound without smoothing has. Gradients do not depend on that mean:
    they have the bounds of classes masked by -inf."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, g = _make(n + k + v, n, k, v, dtype, True, cuda)
    masked = torch.zeros(v, dtype=torch.bool, device=cuda)
    masked[:3] = True
    masked[v // 2:v // 2 + 9] = True
    b[masked] = torch.finfo(TYPES[dtype]).min
    labels = torch.where(labels >= 0, 3 + labels % (v // 2 - 3), labels).int()          # none of the masked ones
    g = g if reduction == "none" else torch.full((), 8.0, device=cuda)
    gone = b.masked_fill(masked, float("-inf"))
    want = _reference(x, w, b, labels, 0.1, reduction, g, dtype)[0][0]
    off = _reference(x, w, gone, labels, 0.0, reduction, g, dtype)[1][0]
    wants, tols = (r[1:] for r in _reference(x, w, gone, labels, 0.1, reduction, g, dtype))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = P.linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2], label_smoothing=0.1, reduction=reduction)
    assert bool(torch.isfinite(loss).all()) and bool(((loss.double() - want).abs() <= want.abs() * 2.0 ** -20 + off).all())
    for got, exact, tol in zip(torch.autograd.grad(loss, leaves, g if reduction == "none" else torch.full_like(loss, 8.0)), wants, tols):
        assert bool(((got.double() - exact).abs() <= tol).all())


@pytest.mark.parametrize("n,k,v", [(150, 64, 700), (200, 64, 90)])
def test_minus_infinity_with_smoothing(cuda, n, k, v):
    """The formula's loss is +inf for rows that count; gradients are finite."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(n, n, k, v, "fp16", True, cuda)
    b[5:8] = float("-inf")
    labels = torch.where(labels >= 0, 8 + labels % (v - 8), labels).int()
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    loss = P.linear_cross_entropy(leaves[0], leaves[1], labels, leaves[2], label_smoothing=0.1, reduction="none")
    assert torch.equal(torch.isinf(loss), labels >= 0) and bool((loss >= 0).all())
    assert all(bool(torch.isfinite(t).all()) for t in torch.autograd.grad(loss, leaves, torch.ones_like(loss)))
