"""rb200k_linear and its backward pass (plugin.pytorch.linear) against the formulas in 64 bits.

Tolerances, element by element, from the arithmetic alone. u = eps / 2 of the element type bounds one rounding to it. A sum
of k products in 32 bits is off by at most k * 2^-23 * sum |a||b| (2^-23: the tensor cores may cut instead of round). An
activation has slope <= 1.13 and is evaluated to 4e-6 relative. The backward pass of an activation reads z rounded to the
element type (slope changes by at most 0.8 per unit of z) and rounds dz to it."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {"fp16": 2.0 ** -25, "bf16": 0.0}         # half a step of fp16's subnormals


def _act(z, name):
    f = torch.nn.functional
    return {"none": lambda v: v, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}[name](z)


def _slope(z, name):
    z = z.clone().requires_grad_(True)
    return torch.autograd.grad(_act(z, name).sum(), z)[0]


def _make(seed, n, k, m, dtype, bias, period, device):
    g = torch.Generator(device=device).manual_seed(seed)
    t = TYPES[dtype]

    def normal(shape, scale):
        return (torch.randn(shape, generator=g, device=device) * scale).to(t)
    return (normal((n, k), 1.0), normal((m, k), k ** -0.5), normal((m,), 0.3) if bias else None,
            normal((period, m), 0.5) if period else None, normal((n, m), 1.0))


def _sum_bound(a, b):
    """Bound of a 32-bit sum of products over a's columns."""
    return a.shape[1] * 2.0 ** -23 * (a.abs() @ b.abs().t())


def _forward(x, w, b, r, act, dtype):
    """(y, z) in 64 bits and their tolerances."""
    u = torch.finfo(TYPES[dtype]).eps / 2
    x, w = x.double(), w.double()
    z = x @ w.t()
    tz = _sum_bound(x, w)
    if b is not None:
        z = z + b.double()
        tz = tz + 2.0 ** -23 * z.abs()
    a = _act(z, act)
    y = a if r is None else a + r.double().repeat(x.shape[0] // r.shape[0], 1)
    return y, z, u * y.abs() + 1.13 * tz + 5e-6 * a.abs() + 2.0 ** -22 * y.abs() + TINY[dtype], tz


def _backward(x, w, dy, z, tz, act, period, dtype):
    u = torch.finfo(TYPES[dtype]).eps / 2
    x, w, dy = x.double(), w.double(), dy.double()
    dz = dy * _slope(z, act)
    if act == "none":
        e = torch.zeros_like(dz)
    elif act == "relu":
        e = dy.abs() * (z.abs() <= tz + TINY[dtype])
    else:
        e = u * dz.abs() + dy.abs() * (0.8 * (u * z.abs() + tz) + 8e-6) + TINY[dtype]
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    tx = u * dx.abs() + e @ w.abs() + 1.01 * _sum_bound(dz, w.t()) + TINY[dtype]
    tw = u * dw.abs() + e.t() @ x.abs() + 1.01 * _sum_bound(dz.t(), x.t()) + TINY[dtype]
    tb = u * db.abs() + e.sum(0) + dz.shape[0] * 2.0 ** -24 * dz.abs().sum(0) + TINY[dtype]
    dr = tr = None
    if period:
        parts = dy.view(-1, period, dy.shape[1])
        dr = parts.sum(0)
        tr = u * dr.abs() + parts.shape[0] * 2.0 ** -24 * parts.abs().sum(0) + TINY[dtype]
    return (dx, dw, db, dr), (tx, tw, tb, tr)


def _close(got, want, tol, what):
    assert got.shape == want.shape, what
    off = (got.double() - want).abs() - tol
    assert not torch.isnan(got).any(), what
    assert float(off.max()) <= 0, "%s: off by %g more than the bound at %d places" % (what, float(off.max()), int((off > 0).sum()))


SHAPES = [(1, 16, 16), (1, 2048, 1000), (3, 17, 5), (2, 1, 1), (64, 72, 33), (127, 64, 130), (129, 200, 257), (200, 1001, 515),
          (513, 256, 640), (1000, 1000, 1000), (4100, 320, 96), (700, 8, 2100), (20, 8192, 24), (2500, 1032, 2056)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,m", SHAPES)
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_forward_and_gradients(cuda, n, k, m, act, dtype):
    from rocal_b200.plugin import pytorch as P
    period = {"none": n, "relu": 0, "gelu": 1, "silu": next(p for p in (7, 5, 4, 3, 2, 1) if n % p == 0)}[act]
    x, w, b, r, dy = _make(n * 7 + k * 3 + m, n, k, m, dtype, act != "silu", period, cuda)
    y64, z64, ty, tz = _forward(x, w, b, r, act, dtype)
    with torch.no_grad():
        _close(P.linear(x, w, b, r, act), y64, ty, "y without gradient")
    leaves = [t for t in (x, w, b, r) if t is not None]
    for t in leaves:
        t.requires_grad_(True)
    y = P.linear(x, w, b, r, act)
    _close(y.detach(), y64, ty, "y")
    got = dict(zip([id(t) for t in leaves], torch.autograd.grad(y, leaves, dy)))
    wants, tols = _backward(x.detach(), w.detach(), dy, z64, tz, act, period, dtype)
    for t, want, tol, what in zip((x, w, b, r), wants, tols, ("dx", "dweight", "dbias", "dresidual")):
        if t is not None:
            _close(got[id(t)], want, tol, what)
    torch.cuda.synchronize()
    from rocal_b200._lib import lib
    assert lib.rb200k_device_status() == 0
