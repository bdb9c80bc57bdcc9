"""linear_cross_entropy for few classes and features (one sweep over x each way) and for many rows, against the formulas in 64
bits with the tolerances derived in test_head_loss_gpu."""
import pytest

torch = pytest.importorskip("torch")

import test_head_loss_gpu as loss_tests   # noqa: E402
from test_head_loss_gpu import _close, _make, _reference   # noqa: E402

pytestmark = pytest.mark.gpu

# rows around tiles of 128 and the 148 of one round, features around chunks of 64 and pairs of them, classes around strips of 32,
# and around the limits 128, 256 (and 96 above 128 features), beyond which the general way is taken
SHAPES = [(1, 1, 2), (1, 64, 33), (2, 8, 128), (5, 65, 32), (127, 63, 31), (128, 128, 64), (129, 129, 65), (255, 192, 96), (256, 256, 96),
          (257, 256, 97), (300, 128, 128), (301, 136, 128), (400, 257, 20), (777, 130, 95), (1000, 127, 127), (128 * 148, 72, 10),
          (128 * 148 + 1, 256, 81), (128 * 148 * 2 - 3, 120, 90), (60001, 200, 81), (40000, 64, 128), (100000, 16, 3)]


def _check(x, w, b, labels, smooth, reduction, g, dtype, ignore=-100):
    """The other file's check, except that fp16 has no number beyond 65504: what is 65520 or more rounds to infinity (half a step of
    32 above 65504), so a sum whose exact value is at most its tolerance below that may be infinite with the exact value's sign."""
    def close(got, want, tol, what):
        if dtype == "fp16" and what != "loss" and what != "loss without gradient":
            full = torch.isinf(got) & (want.abs() + tol >= 65520) & (torch.sign(got.double()) == torch.sign(want))
            got = torch.where(full, want, got.double())
        _close(got, want, tol, what)
    with pytest.MonkeyPatch.context() as m:
        m.setattr(loss_tests, "_close", close)
        return loss_tests._check(x, w, b, labels, smooth, reduction, g, dtype, ignore)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,v", SHAPES)
@pytest.mark.parametrize("smooth,reduction,bias", [(0.0, "mean", True), (0.1, "sum", False), (0.1, "none", True), (0.0, "none", False)])
def test_sizes(cuda, n, k, v, smooth, reduction, bias, dtype):
    x, w, b, labels, g = _make(n + 5 * k + 11 * v, n, k, v, dtype, bias, cuda)
    _check(x, w, b, labels, smooth, reduction, g if reduction == "none" else torch.full((), 256.0, device=cuda), dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_that_do_not_count(cuda, dtype):
    """Ignored rows hold inf and NaN; whole tiles are ignored; a label that is a class is the ignored one."""
    x, w, b, labels, _ = _make(3, 1000, 200, 81, dtype, True, cuda, ignored=0.3)
    labels[128:512] = -100
    x[labels == -100] = float("nan")
    x[(labels == -100).nonzero()[0, 0], 5] = float("inf")
    _check(x, w, b, labels, 0.0, "mean", torch.full((), 256.0, device=cuda), dtype)
    labels[labels == -100] = 7
    _check(x, w, b, labels, 0.1, "sum", torch.full((), 16.0, device=cuda), dtype, ignore=7)


def test_no_row_counts(cuda):
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(4, 300, 64, 20, "fp16", True, cuda)
    labels.fill_(-100)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    loss = P.linear_cross_entropy(x, w, labels, b)
    assert float(loss.detach()) == 0
    assert all(float(g.abs().max()) == 0 for g in torch.autograd.grad(loss, leaves))


def test_a_label_that_is_no_class(cuda):
    """Its row is NaN: the sum, the row's dx and all of dweight; other rows keep their loss and dx."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(6, 400, 64, 20, "bf16", True, cuda, ignored=0.0)
    want = P.linear_cross_entropy(x, w, labels, b, reduction="none")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    clean = torch.autograd.grad(P.linear_cross_entropy(x, w, labels, b, reduction="sum"), leaves)
    labels[17] = 20
    got = P.linear_cross_entropy(x, w, labels, b, reduction="none").detach()
    keep = torch.arange(400, device=cuda) != 17
    assert torch.equal(got[keep], want[keep]) and bool(torch.isnan(got[17]))
    dx, dw, db = torch.autograd.grad(P.linear_cross_entropy(x, w, labels, b, reduction="sum"), leaves)
    assert torch.equal(dx[keep], clean[0][keep]) and bool(torch.isnan(dx[17]).all()) and bool(torch.isnan(dw).all()) and bool(torch.isnan(db).all())


def test_masked_classes_and_large_scores(cuda):
    """Biases of -inf take classes out; scores of some thousands; nothing but -inf beside the label."""
    x, w, b, labels, _ = _make(8, 513, 96, 70, "bf16", True, cuda, spread=300.0)
    b[3:40] = float("-inf")
    labels[(labels >= 3) & (labels < 40)] = 50
    _check(x, w, b, labels, 0.0, "sum", torch.full((), 1.0, device=cuda), "bf16")


@pytest.mark.parametrize("need", [(True, False, False), (False, True, False), (False, False, True), (True, False, True), (False, True, True)])
def test_gradients_one_by_one(cuda, need):
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(12, 20000, 192, 81, "fp16", True, cuda)
    g = torch.full((), 64.0, device=cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    full = torch.autograd.grad(P.linear_cross_entropy(x, w, labels, b), leaves, g)
    some = [t for t, n in zip(leaves, need) if n]
    for got, want in zip(torch.autograd.grad(P.linear_cross_entropy(x, w, labels, b), some, g), [f for f, n in zip(full, need) if n]):
        assert torch.equal(got, want)


def test_captured_replays_and_bits(cuda):
    """Two captured steps that share the graph pool, replayed with other inputs: the eager call's bits."""
    from rocal_b200 import kernels as K
    x, w, b, labels, g = _make(14, 50000, 256, 81, "bf16", True, cuda)
    one = torch.ones((), device=cuda)

    def step():
        loss, stats, info = K.linear_cross_entropy(x, w, labels, b)
        return (loss,) + tuple(K.linear_cross_entropy_backward(one, x, w, labels, stats, info, b, need=(True, True, True)))
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first = step()
        second = step()
    for seed in range(3):
        x.copy_(torch.randn(x.shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)))
        graph.replay()
        for a, c, d in zip(first, second, step()):
            assert torch.equal(a, d) and torch.equal(c, d)


@pytest.mark.parametrize("pitch,lead", [(208, 8), (201, 0), (208, 3)])
def test_pitches_and_offsets(cuda, pitch, lead):
    x0, w, b, labels, g = _make(16, 700, 200, 40, "fp16", True, cuda)
    wide = torch.full((700 * pitch + 16,), float("nan"), device=cuda, dtype=torch.float16)
    x = wide[lead:].as_strided((700, 200), (pitch, 1))
    x.copy_(x0)
    _check(x.detach(), w, b, labels, 0.0, "none", g, "fp16")


@pytest.mark.parametrize("n,k,v", [(279424, 16, 5), (5000, 520, 200), (2049, 64, 10), (2048, 64, 10)])
def test_a_gradient_for_every_row_of_many(cuda, n, k, v):
    """The largest of the rows' gradients is found by many blocks; it lies in the last row here, and some are inf where nothing counts."""
    x, w, b, labels, g = _make(n, n, k, v, "fp16", True, cuda)
    labels[-1] = 1
    g[-1] = 37.0
    g[labels == -100] = float("inf")
    keep = torch.where(labels == -100, torch.zeros_like(g), g)
    wants, tols = _reference(x, w, b, labels, 0.0, "none", keep, "fp16")
    from rocal_b200.plugin import pytorch as P
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(P.linear_cross_entropy(x, w, labels, b, reduction="none"), leaves, g)
    for a, want, tol, what in zip(got, wants[1:], tols[1:], ("dx", "dweight", "dbias")):
        _close(a, want, tol, what)


def test_statistics_in_pieces_of_the_classes(cuda):
    """A million rows: the partial statistics of 1500 classes are made in two launches. The reference in pieces of the rows."""
    from rocal_b200.plugin import pytorch as P
    n, k, v = 1000000, 16, 1500
    x, w, b, labels, g = _make(21, n, k, v, "fp16", True, cuda)
    got = P.linear_cross_entropy(x, w, labels, b, label_smoothing=0.1, reduction="none")
    for i in range(0, n, 100000):
        s = slice(i, i + 100000)
        wants, tols = _reference(x[s], w, b, labels[s], 0.1, "none", g[s], "fp16")
        _close(got[s], wants[0], tols[0], "loss")


@pytest.mark.parametrize("n,k,v", [(130, 64, 40), (128, 64, 40), (333, 200, 81), (333, 300, 200)])
def test_a_weight_of_inf_that_masks_a_class(cuda, n, k, v):
    """Where an infinite weight makes a class' scores -inf in every row, the other gradients are those of the class masked by its
    bias, to the bit; the rows that fill up the last tile (zeros times that weight) must not show."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(n + v, n, k, v, "bf16", True, cuda, ignored=0.0)
    x[:, 3] = -x[:, 3].abs() - 0.5
    labels[labels == 5] = 6

    def grads(weight, bias):
        leaves = [weight.clone().requires_grad_(True), bias.clone().requires_grad_(True)]
        loss = P.linear_cross_entropy(x, leaves[0], labels, leaves[1], reduction="sum")
        return [loss.detach()] + list(torch.autograd.grad(loss, leaves))
    w[5] = 0
    b_masked = b.clone()
    b_masked[5] = float("-inf")
    want = grads(w, b_masked)
    w_inf = w.clone()
    w_inf[5, 3] = float("inf")
    for got, expect in zip(grads(w_inf, b), want):
        assert bool(torch.isfinite(expect).all()) and torch.equal(got, expect)


@pytest.mark.parametrize("n,k,v", [(300, 4096, 700), (1000, 2056, 300), (64, 3301, 1000)])
def test_long_sums(cuda, n, k, v):
    """More than 2048 features: the scores' sums are spread over two accumulators, which the epilogue adds."""
    x, w, b, labels, g = _make(n + k, n, k, v, "fp16", True, cuda)
    _check(x, w, b, labels, 0.1, "none", g, "fp16")
