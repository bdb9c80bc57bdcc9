"""Forms of differentiation, on the GPU: what goes through, and what is refused instead of giving a wrong result."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad as fw  # noqa: E402

pytestmark = pytest.mark.gpu


def test_forward_over_reverse_is_refused(cuda):
    """A tangent on the gradient that comes back into the backward pass is not dropped either; without one the pass works."""
    from rocal_b200.plugin import pytorch as P
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn((6, 16), generator=g, device=cuda).half().requires_grad_(True)
    w = torch.randn((5, 16), generator=g, device=cuda).half()
    labels = torch.arange(6, device=cuda) % 5
    for y in (P.linear(x, w), P.linear_cross_entropy(x, w, labels)):
        with fw.dual_level():
            dy = fw.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="has no forward-mode derivative"):
                torch.autograd.grad(y, x, dy, retain_graph=True)
        assert torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x.shape


@pytest.mark.parametrize("grad", [False, True])
def test_tangents_are_refused(cuda, grad):
    """On the device itself: no plain result for a dual input, whether or not it requires a gradient."""
    from rocal_b200.plugin import pytorch as P
    x, w = torch.ones((6, 16), device=cuda).half().requires_grad_(grad), torch.ones((5, 16), device=cuda).half()
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            P.linear(dual, w)
        with pytest.raises(NotImplementedError):
            P.linear_cross_entropy(dual, w, torch.arange(6, device=cuda) % 5)
