"""What the head operators say to forms of differentiation that they do not have. The checks come before the device's, so that
none of this needs a GPU."""
import pytest

torch = pytest.importorskip("torch")
from torch.autograd import forward_ad as fw  # noqa: E402


def _half(*shape):
    return torch.ones(shape, dtype=torch.float16)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "residual"])
def test_tangents_are_refused(which, grad):
    """A dual tensor that does not require a gradient came out as a plain tensor, its tangent lost; one that does was refused
    by autograd."""
    from rocal_b200.plugin import pytorch as P
    args = dict(x=_half(4, 8), weight=_half(3, 8), bias=_half(3), residual=_half(4, 3))
    args[which].requires_grad_(grad)
    with fw.dual_level():
        args[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError, match="linear has no forward-mode derivative"):
            P.linear(**args)
        if which != "residual":
            del args["residual"]
            with pytest.raises(NotImplementedError, match="linear_cross_entropy has no forward-mode derivative"):
                P.linear_cross_entropy(labels=torch.zeros(4, dtype=torch.int32), **args)


def test_tangents_of_gradients_are_refused():
    from rocal_b200.plugin import pytorch as P
    g = _half(4, 8)
    with fw.dual_level():
        dual = fw.make_dual(g, torch.ones_like(g))
        with pytest.raises(NotImplementedError, match="grad_clip has no forward-mode derivative"):
            P.clip_grad_norm([g.clone(), dual], 1.0)
        with pytest.raises(NotImplementedError, match="grad_clip has no forward-mode derivative"):
            P.clip_grad_norm([g.clone()], 1.0, out=[dual])
    # behind the level a tensor is an ordinary one again: what is refused then is the device
    with pytest.raises(ValueError, match="run on a GPU"):
        P.clip_grad_norm([dual], 1.0)
