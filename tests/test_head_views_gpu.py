"""Views whose bytes are not their values: the negation of a conjugate's imaginary part is still to come when the view is made."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def test_negated_views(cuda):
    from rocal_b200 import kernels as K
    from rocal_b200.plugin import pytorch as P
    g = torch.Generator(device=cuda).manual_seed(2)
    x, w, b = (torch.randn(s, generator=g, device=cuda).half() for s in ((20, 16), (9, 16), (9,)))
    labels = torch.arange(20, device=cuda) % 9
    nx, nw, nb = (torch._neg_view(t) for t in (x, w, b))
    assert nx.is_neg() and nx.is_contiguous()
    assert torch.equal(P.linear(nx, nw, nb), P.linear(-x, -w, -b)) and torch.equal(P.linear(nx, w, b), P.linear(-x, w, b))
    assert torch.equal(P.linear_cross_entropy(nx, w, labels, nb), P.linear_cross_entropy(-x, w, labels, -b))
    dx = [torch.autograd.grad(P.linear_cross_entropy(leaf, w, labels), leaf, dl)[0]
          for leaf in (x.clone().requires_grad_(True),) for dl in (torch._neg_view(torch.ones((), device=cuda)), -torch.ones((), device=cuda))]
    assert torch.equal(dx[0], dx[1])
    with pytest.raises(ValueError, match="out has shape"):
        K.linear(x, w, out=torch._neg_view(torch.zeros((20, 9), device=cuda).half()))


def test_clipping_of_negated_views(cuda):
    """As a real program has them: the imaginary part of a conjugate, and one that happens to be contiguous."""
    from rocal_b200.plugin import pytorch as P
    z = torch.tensor([[1 + 2j], [3 - 4j]], device=cuda, dtype=torch.complex64)
    part = z.conj().imag                                      # -2, 4
    assert part.is_neg()
    out = torch.zeros((2, 1), device=cuda)
    norm = P.clip_grad_norm([part], 1e9, out=[out])
    assert abs(float(norm) - 20 ** 0.5) <= 1e-6 and out[:, 0].tolist() == [-2.0, 4.0]
    P.clip_grad_norm([part], 20 ** 0.5 / 2)                   # in place: halved
    assert part[:, 0].tolist() == pytest.approx([-1.0, 2.0], rel=1e-6) and z.real[:, 0].tolist() == [1.0, 3.0]
    values = torch.ones(300, device=cuda)
    target = torch.zeros(300, device=cuda)
    P.clip_grad_norm([torch._neg_view(values)], 1e9, out=[target])
    assert bool((target == -1).all())
    P.clip_grad_norm([values], 1e9, out=[torch._neg_view(target)])
    assert bool((target == -1).all()) and bool((torch._neg_view(target) == 1).all())
    P.clip_grad_norm([torch._neg_view(values)], 0.0)
    assert not values.any()
