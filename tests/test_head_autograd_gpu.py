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


@pytest.mark.parametrize("behind", ["cast", "view", "both"])
def test_stale_leaves_behind_other_operations_are_refused(cuda, behind):
    """A capture whose leaf goes through a cast or a transposition first (32-bit weights of a 16-bit head), while an eager graph of that leaf
    lives on the default stream: refused like the leaf itself, since autograd would end the process. Without it the capture works."""
    from rocal_b200.plugin import pytorch as P
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn((12, 32), generator=g, device=cuda).half()
    leaf = torch.randn((32, 9) if behind != "cast" else (9, 32), generator=g, device=cuda)
    leaf = (leaf if behind != "view" else leaf.half()).requires_grad_(True)
    labels = torch.arange(12, device=cuda) % 9

    def weight():
        return {"cast": lambda: leaf.half(), "view": lambda: leaf.t(), "both": lambda: leaf.t().half() * 1.0}[behind]()

    def step():
        loss = P.linear_cross_entropy(x, weight(), labels)
        return loss.detach(), torch.autograd.grad(loss, leaf)[0]
    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    alive = P.linear(x, weight())
    for call in (lambda: P.linear(x, weight()), lambda: P.linear_cross_entropy(x, weight(), labels)):
        with pytest.raises(RuntimeError, match="still alive"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
    torch.cuda.synchronize()
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_eager_inputs_of_a_capture_stay_allowed(cuda):
    """What comes out of an eager graph may go into a captured forward pass, as before."""
    from rocal_b200.plugin import pytorch as P
    w = torch.ones((8, 16), device=cuda).half().requires_grad_(True)
    h = P.linear(torch.ones((4, 16), device=cuda).half(), w)
    graph = torch.cuda.CUDAGraph()
    c = torch.ones((5, 8), device=cuda).half()
    P.linear(h, c)
    with torch.cuda.graph(graph):
        y = P.linear(h, c)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((y == 128).all())
