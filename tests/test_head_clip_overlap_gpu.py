"""Clipping refuses outputs that meet themselves, one another or other gradients, before anything is written - tensors with gaps
too, whose columns may interleave with others without meeting them."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def _columns(cuda, *slices):
    base = torch.arange(1, 61, device=cuda, dtype=torch.float32).view(10, 6)
    return base, [base[:, s] for s in slices]


def test_overlapping_outputs_with_gaps(cuda):
    import rocal_b200
    from rocal_b200.plugin import pytorch as P
    grads = [torch.ones((10, 3), device=cuda), torch.full((10, 3), 2.0, device=cuda)]
    for slices in ((slice(0, 3), slice(2, 5)), (slice(0, 6, 2), slice(0, 3))):
        base, out = _columns(cuda, *slices)
        kept = base.clone()
        with pytest.raises(rocal_b200.Rb200Error, match="overlaps"):
            P.clip_grad_norm(grads, 1.0, out=out)
        assert torch.equal(base, kept) and bool((grads[0] == 1).all())
    base, (a, b) = _columns(cuda, slice(0, 3), slice(3, 6))                      # side by side
    norm = P.clip_grad_norm(grads, 1e9, out=[a, b])
    assert abs(float(norm) - 150.0 ** 0.5) <= 1e-5 and torch.equal(base[:, :3], grads[0]) and torch.equal(base[:, 3:], grads[1])


def test_overlapping_gradients_with_gaps_in_place(cuda):
    import rocal_b200
    from rocal_b200.plugin import pytorch as P
    base, (a, b) = _columns(cuda, slice(0, 3), slice(2, 5))
    kept = base.clone()
    for tensors in ([a, b], [a, a], [a, base.view(-1)[7:9]], [base.view(-1)[7:9], a]):
        with pytest.raises(rocal_b200.Rb200Error, match="overlaps"):
            P.clip_grad_norm(tensors, 1.0)
        assert torch.equal(base, kept)
    base, (a, b) = _columns(cuda, slice(0, 3), slice(3, 6))
    P.clip_grad_norm([a, b], 0.0)
    assert not base.any()


def test_outputs_over_other_gradients_with_gaps(cuda):
    import rocal_b200
    from rocal_b200.plugin import pytorch as P
    base, (a, b) = _columns(cuda, slice(0, 3), slice(3, 6))
    kept, other = base.clone(), torch.zeros((10, 3), device=cuda)
    for grads, out in (([a, b], [b, other]), ([torch.ones(3, device=cuda), a], [base.view(-1)[1:4], other]), ([a, torch.ones(2, device=cuda)], [other, base[4, 1:3]])):
        with pytest.raises(rocal_b200.Rb200Error, match="overlaps"):
            P.clip_grad_norm(grads, 1.0, out=out)
        assert torch.equal(base, kept) and not other.any()
    P.clip_grad_norm([a, torch.ones(2, device=cuda)], 1e9, out=[other, base[4, 3:5]])          # between the columns
    assert torch.equal(other, kept[:, :3]) and bool((base[4, 3:5] == 1).all())


def test_an_output_of_repeated_elements(cuda):
    """An expanded gradient, clipped in place: copying back failed behind the launch, with the other gradients already clipped."""
    import rocal_b200
    from rocal_b200.plugin import pytorch as P
    first, repeated = torch.full((100,), 3.0, device=cuda), torch.ones(1, device=cuda).expand(5)
    with pytest.raises(rocal_b200.Rb200Error, match="overlaps"):
        P.clip_grad_norm([first, repeated], 1.0)
    assert bool((first == 3).all())
    out = [torch.empty_like(first), torch.empty(5, device=cuda)]
    assert abs(float(P.clip_grad_norm([first, repeated], 1e9, out=out)) - 905.0 ** 0.5) <= 1e-5 and bool((out[1] == 1).all())
