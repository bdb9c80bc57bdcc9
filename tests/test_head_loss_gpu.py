"""rb200k_linear_ce and its backward pass (plugin.pytorch.linear_cross_entropy) against the formulas in 64 bits.

Tolerances from the arithmetic alone, element by element. u = eps / 2 of the element type bounds one rounding to it.
A score z is a 32-bit sum of k products: off by at most tz = k * 2^-23 * sum |x||w| (+ the bias' rounding). The sum of
exponentials is off by 2^-21 + (64 + classes / 64) * 2^-24 relative (exponentials, at most 64 + classes / 64 additions one
after another) and by the scores' errors. Hence for the loss: the scores' errors (an average of them in lse, the label's own) +
that, and one rounding of each term; for a probability: p * (tz + the row's largest tz + that + |z - lse| * 2^-22). The gradient
of the scores is rounded to the element type, then multiplied and summed in 32 bits, and rounded once more."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0}


def _make(seed, n, k, v, dtype, bias, device, spread=2.0, ignored=0.2):
    g = torch.Generator(device=device).manual_seed(seed)

    def normal(shape, scale):
        return (torch.randn(shape, generator=g, device=device) * scale).to(TYPES[dtype])
    x, w, b = normal((n, k), 1.0), normal((v, k), spread * k ** -0.5), normal((v,), 0.3) if bias else None
    labels = torch.randint(0, v, (n,), generator=g, device=device, dtype=torch.int32)
    labels[torch.rand((n,), generator=g, device=device) < ignored] = -100
    return x, w, b, labels, torch.rand((n,), generator=g, device=device) + 0.5


def _reference(x, w, b, labels, smooth, reduction, g, dtype, ignore=-100):
    """loss, gradients and their tolerances; ignored rows of x are taken as zeros, which is what "takes no part" means."""
    u = torch.finfo(TYPES[dtype]).eps / 2
    keep = labels.long() != ignore
    x, w, b = x.detach(), w.detach(), None if b is None else b.detach()
    x, w = torch.where(keep[:, None], x.double(), torch.zeros((), dtype=torch.float64, device=x.device)), w.double()
    v, k = w.shape
    z = x @ w.t()
    tz = k * 2.0 ** -23 * (x.abs() @ w.abs().t())
    if b is not None:
        z = z + b.double()
        tz = tz + torch.where(torch.isfinite(z), 2.0 ** -23 * z.abs(), torch.zeros_like(z))
    top = z.max(1, keepdim=True).values
    e = torch.exp(z - top)
    s = e.sum(1, keepdim=True)
    rel = 2.0 ** -21 + (64 + v / 64) * 2.0 ** -24
    at = labels.long().clamp(0, v - 1)[:, None]
    zy, ty = z.gather(1, at)[:, 0], tz.gather(1, at)[:, 0]
    p = e / s
    big = tz.max(1, keepdim=True).values
    one = torch.log(s)[:, 0] + (top[:, 0] - zy)
    t_one = (p * tz).sum(1) + ty + rel + 2.0 ** -22 * (torch.log(s)[:, 0].abs() + (top[:, 0] - zy).abs())
    t_one = t_one + 2.0 ** -22 * torch.where(top[:, 0].abs() < 1e30, top[:, 0].abs(), torch.zeros_like(zy))
    loss, tol = (1 - smooth) * one, t_one
    if smooth:
        loss = loss + smooth * (torch.log(s)[:, 0] + (top[:, 0] - z.mean(1)))
        tol = tol + smooth * (tz.mean(1) + (64 + v / 64) * 2.0 ** -24 * z.abs().mean(1))
    loss, tol = torch.where(keep, loss, torch.zeros_like(loss)), torch.where(keep, tol, torch.zeros_like(tol)) + 2.0 ** -23 * loss.abs()
    count = max(1, int(keep.sum())) if reduction == "mean" else 1
    if reduction != "none":
        loss, tol = loss.sum() / count, tol.sum() / count + 2.0 ** -23 * loss.abs().sum() / count
    c = (g.double() if reduction == "none" else g.double().expand(len(labels)) / count) * keep
    dz = p - smooth / v
    dz = dz.scatter_add(1, at, torch.full_like(at, -(1 - smooth), dtype=torch.float64)) * c[:, None]
    # |z - lse| <= 60 wherever p is not vanishing
    e_p = p * (tz + big + rel + 60 * 2.0 ** -22)
    e_dz = c.abs()[:, None] * (e_p + 2.0 ** -23) + u * dz.abs() + c.abs().max() * 2.0 ** -39
    e_dz = e_dz * keep[:, None]
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    tx = u * dx.abs() + e_dz @ w.abs() + 1.01 * v * 2.0 ** -23 * (dz.abs() @ w.abs()) + TINY[dtype]
    tw = u * dw.abs() + e_dz.t() @ x.abs() + 1.01 * len(labels) * 2.0 ** -23 * (dz.abs().t() @ x.abs()) + TINY[dtype]
    tb = u * db.abs() + e_dz.sum(0) + len(labels) * 2.0 ** -24 * dz.abs().sum(0) + TINY[dtype]
    return (loss, dx, dw, db), (tol, tx, tw, tb)


def _close(got, want, tol, what):
    assert got.shape == want.shape, what
    assert not torch.isnan(got).any(), what
    got = got.double()
    same = got == want                          # infinities among them
    off = torch.where(same, torch.full_like(want, -1.0), (got - want).abs() - tol)
    assert off.numel() == 0 or float(off.max()) <= 0, "%s: %g beyond the bound at %d places" % (what, float(off.max()), int((off > 0).sum()))


def _check(x, w, b, labels, smooth, reduction, g, dtype, ignore=-100):
    from rocal_b200._lib import lib
    from rocal_b200.plugin import pytorch as P
    wants, tols = _reference(x, w, b, labels, smooth, reduction, g, dtype, ignore)
    with torch.no_grad():
        _close(P.linear_cross_entropy(x, w, labels, b, ignore, smooth, reduction), wants[0], tols[0], "loss without gradient")
    leaves = [t.requires_grad_(True) for t in (x, w, b) if t is not None]
    loss = P.linear_cross_entropy(x, w, labels, b, ignore, smooth, reduction)
    _close(loss.detach(), wants[0], tols[0], "loss")
    grads = torch.autograd.grad(loss, leaves, g.expand(loss.shape) if reduction == "none" else g)
    for got, want, tol, what in zip(grads, wants[1:], tols[1:], ("dx", "dweight", "dbias")):
        _close(got, want, tol, what)
    torch.cuda.synchronize()
    assert lib.rb200k_device_status() == 0
    return loss.detach(), grads


SHAPES = [(1, 16, 2), (1, 1, 1), (3, 17, 5), (2, 100, 1), (64, 2048, 1000), (65, 72, 81), (127, 200, 257), (130, 1001, 515), (1000, 256, 81),
          (300, 64, 5003), (1025, 520, 999), (5000, 32, 10)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,v", SHAPES)
@pytest.mark.parametrize("smooth,reduction,bias", [(0.0, "mean", True), (0.1, "sum", False), (0.1, "none", True)])
def test_loss_and_gradients(cuda, n, k, v, smooth, reduction, bias, dtype):
    x, w, b, labels, g = _make(n + 3 * k + 7 * v, n, k, v, dtype, bias, cuda)
    _check(x, w, b, labels, smooth, reduction, g if reduction == "none" else torch.full((), 256.0, device=cuda), dtype)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,v,smooth,reduction", [(1100, 24, 128000, 0.0, "mean"), (140000, 24, 1000, 0.1, "sum"), (140000, 16, 961, 0.0, "none")])
def test_scores_that_are_made_in_pieces(cuda, n, k, v, smooth, reduction, dtype):
    """More than 256 MB of scores: pieces of the classes, pieces of the rows; the statistics of the second in pieces, too."""
    x, w, b, labels, g = _make(n + k, n, k, v, dtype, True, cuda)
    _check(x, w, b, labels, smooth, reduction, g if reduction == "none" else torch.full((), 64.0, device=cuda), dtype)
