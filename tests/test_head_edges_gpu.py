"""The head operators where they can go wrong: masked classes and rows, infinities and NaN, odd strides and alignments,
outputs inside larger buffers, other streams, captured graphs, threads, waits that run out."""
import math
import os
import subprocess
import sys
import threading

import pytest

torch = pytest.importorskip("torch")

from test_head_clip_gpu import _close as _clip_close, _grads, _reference as _clip_reference
from test_head_linear_gpu import TYPES, _backward, _close as _linear_close, _forward, _make as _linear_make
from test_head_loss_gpu import _check, _close, _make, _reference

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
WAIT_CYCLES = 2_000_000      # about a millisecond of SM clock


def _status():
    from rocal_b200._lib import lib
    return lib.rb200k_device_status()


# ---- linear ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_linear_takes_views(cuda, dtype):
    """Row pitches, columns cut out of wider rows at odd places, transposed and overlapping operands."""
    from rocal_b200.plugin import pytorch as P
    g = torch.Generator(device=cuda).manual_seed(3)
    t = TYPES[dtype]
    wide = torch.randn((300, 400), generator=g, device=cuda).to(t)
    weights = torch.randn((400, 300), generator=g, device=cuda).to(t) * 0.05
    bias = torch.randn((900,), generator=g, device=cuda).to(t)
    for x, w, b in ((wide[:, 8:136], weights[:200, 16:144], bias[:200]),                # pitch 400, on 16-byte boundaries
                    (wide[:, 3:130], weights[1:100:2, 5:132], bias[1:199:2][:50]),      # odd places, every other row
                    (wide.t()[:128], weights.t()[:77, :300], bias[7:84]),               # transposed: copied
                    (wide[:1].expand(50, 400)[:, :64], weights[:33, :64], bias[:33]),   # one row, repeated without a copy
                    (wide[5:6, 1:66], weights[0:1, 1:66], bias[899:])):                 # single rows at odd addresses
        y64, _, tol, _ = _forward(x, w, b, None, "relu", dtype)
        _linear_close(P.linear(x, w, b, activation="relu"), y64, tol, "%s %s" % (tuple(x.shape), x.stride()))


def test_linear_shapes_and_residual_tails(cuda):
    """Leading dimensions are rows; the residual is a tail of the result's shape."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, _ = _linear_make(5, 24, 40, 16, "fp16", True, 0, cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    flat = P.linear(x, w, b)
    assert torch.equal(P.linear(x.view(2, 3, 4, 40), w, b), flat.view(2, 3, 4, 16))
    assert torch.equal(P.linear(x[0], w, b), flat[0])                 # one vector
    for shape in ((16,), (4, 16), (3, 4, 16), (2, 3, 4, 16)):
        r = torch.randn(shape, generator=g, device=cuda).half()
        y64, _, tol, _ = _forward(x, w, b, r.reshape(-1, 16), "none", "fp16")
        _linear_close(P.linear(x.view(2, 3, 4, 40), w, b, r).view(24, 16), y64, tol, str(shape))
    for shape in ((5, 16), (4, 15), (3, 16), (2, 2, 3, 4, 16)):
        with pytest.raises(ValueError, match="not a tail"):
            P.linear(x.view(2, 3, 4, 40), w, b, torch.zeros(shape, device=cuda, dtype=torch.float16))
    with pytest.raises(ValueError, match="do not divide"):
        P.linear(x, w, b, torch.zeros((5, 16), device=cuda, dtype=torch.float16))
    for bad in (w.float(), w.bfloat16(), w.cpu()):
        with pytest.raises(ValueError, match="weight is"):
            P.linear(x, bad, b)
    with pytest.raises(ValueError, match="bias has shape"):
        P.linear(x, w, b[:-1])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_linear_without_rows(cuda, dtype):
    from rocal_b200.plugin import pytorch as P
    t = TYPES[dtype]
    x, w, b = torch.empty((0, 24), device=cuda, dtype=t), torch.randn((9, 24), device=cuda).to(t), torch.randn((9,), device=cuda).to(t)
    r = torch.randn((3, 9), device=cuda).to(t)
    leaves = [v.requires_grad_(True) for v in (x, w, b, r)]
    y = P.linear(x, w, b, r, "gelu")
    assert y.shape == (0, 9)
    dx, dw, db, dr = torch.autograd.grad(y, leaves, torch.empty((0, 9), device=cuda, dtype=t), allow_unused=True)
    assert dx.shape == (0, 24) and not dw.any() and not db.any() and (dr is None or not dr.any())


def test_linear_writes_nothing_but_its_rows(cuda):
    """An output that is a window of a larger buffer: what lies around it stays."""
    from rocal_b200 import kernels as K
    for n, m, ld, at in ((130, 65, 80, 3), (64, 96, 128, 16), (1, 33, 40, 5), (257, 40, 41, 0)):
        x, w, b, _, _ = _linear_make(n + m, n, 72, m, "fp16", True, 0, cuda)
        whole = torch.full((n + 2, ld), 7.0, device=cuda, dtype=torch.float16)
        K.linear(x, w, b, out=whole[1:n + 1, at:at + m] if at + m <= ld else whole[1:n + 1, :m])
        y64, _, tol, _ = _forward(x, w, b, None, "none", "fp16")
        got = whole[1:n + 1, at:at + m]
        _linear_close(got, y64, tol, "window")
        rest = torch.ones_like(whole, dtype=torch.bool)
        rest[1:n + 1, at:at + m] = False
        assert bool((whole[rest] == 7.0).all())


@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
def test_linear_special_values_stay_in_their_rows(cuda, act):
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, _ = _linear_make(9, 140, 64, 70, "bf16", True, 0, cuda)
    clean = P.linear(x, w, b, None, act)
    x = x.clone()
    x[3, 5], x[100, 0], x[139, 63] = float("nan"), float("inf"), float("-inf")
    got = P.linear(x, w, b, None, act)
    touched = [3, 100, 139]
    rest = [i for i in range(140) if i not in touched]
    assert torch.equal(got[rest], clean[rest]) and bool(torch.isnan(got[3]).all())
    z = x[100].double() @ w.double().t()
    if act in ("none", "relu", "gelu"):
        want = z if act == "none" else z.clamp(min=0)          # the limits of relu and gelu
        assert torch.equal(got[100].double(), want)


def test_linear_gelu_over_its_range(cuda):
    """The activation alone (weight = identity), both tails, against 64 bits. One rounding to bf16 is half of eps = 2^-7, 2^-8
    relative. The tail is a ratio good to 2.3e-6 times the exponential of -z^2 / 2, whose argument (in powers of two at
    most 26 for |z| <= 6) has two roundings of 2^-24: 26 * 2 * 2^-24 * ln 2 = 2.2e-6; 8e-6 in all with the products'
    roundings. Beyond 6, where the value is below 6e-9, the ratio is that at 6, 2% off at most."""
    from rocal_b200.plugin import pytorch as P
    z = torch.linspace(-12, 12, 4096, device=cuda).bfloat16().view(64, 64)
    eye = torch.eye(64, device=cuda, dtype=torch.bfloat16)
    got = P.linear(z, eye, activation="gelu").double()
    want = z.double() * 0.5 * torch.erfc(-z.double() * math.sqrt(0.5))
    tol = want.abs() * (2.0 ** -8 + 8e-6) + torch.where(z < -6, want.abs() * 0.02, torch.zeros_like(want))
    assert bool(((got - want).abs() <= tol).all())


def test_linear_bounded_wait(cuda):
    """Copies from the third block of the contracted axis on are left out: every role gives up, the status word reads 1, the
    next launch is right."""
    from rocal_b200 import kernels as K
    for n in (40, 300):                                       # one CTA a tile, CTA pairs
        x, w, b, _, _ = _linear_make(n, n, 512, 200, "fp16", True, 0, cuda)
        y64, _, tol, _ = _forward(x, w, b, None, "none", "fp16")
        status = torch.zeros(1, dtype=torch.int32, device=cuda)
        K.linear(x, w, b, status=status, probe=(WAIT_CYCLES, 2))
        torch.cuda.synchronize()
        assert int(status.item()) == 1 and _status() == 0
        status.zero_()
        _linear_close(K.linear(x, w, b, status=status), y64, tol, "after")
        assert int(status.item()) == 0
        K.linear(x, w, b, probe=(WAIT_CYCLES, 0))
        torch.cuda.synchronize()
        assert _status() == 1 and _status() == 0
        _linear_close(K.linear(x, w, b, probe=(WAIT_CYCLES * 1000, -1)), y64, tol, "a probe that skips nothing")


def test_gradients_pass_through_other_operations(cuda):
    """Gradients that are expanded scalars, non-contiguous, or not wanted at all."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, r, _ = _linear_make(11, 96, 48, 40, "bf16", True, 12, cuda)
    for t in (x, w, b, r):
        t.requires_grad_(True)
    y64, z64, _, tz = _forward(x.detach(), w.detach(), b.detach(), r.detach(), "silu", "bf16")
    ones = torch.ones((96, 40), device=cuda, dtype=torch.bfloat16)
    wants, tols = _backward(x.detach(), w.detach(), ones, z64, tz, "silu", 12, "bf16")
    got = torch.autograd.grad(P.linear(x, w, b, r, "silu").sum(), (x, w, b, r))        # an expanded scalar
    for g, want, tol, name in zip(got, wants, tols, "xwbr"):
        _linear_close(g, want, tol, name)
    turned = torch.ones((40, 96), device=cuda, dtype=torch.bfloat16).t()                 # columns contiguous
    got = torch.autograd.grad(P.linear(x, w, b, r, "silu"), (x, w, b, r), turned)
    for g, want, tol, name in zip(got, wants, tols, "xwbr"):
        _linear_close(g, want, tol, name)
    for wanted in ((x,), (w,), (b,), (r,), (x, r), (w, b)):
        for t in (x, w, b, r):
            t.requires_grad_(any(t is v for v in wanted))
        got = torch.autograd.grad(P.linear(x, w, b, r, "silu"), wanted, ones)
        for g, v in zip(got, wanted):
            i = [j for j, t in enumerate((x, w, b, r)) if t is v][0]
            _linear_close(g, wants[i], tols[i], "xwbr"[i] + " alone")
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad(P.linear(x, w, b, r, "silu").sum(), (x,), create_graph=True)


# ---- the loss ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("mask", ["-inf", "lowest"])
def test_masked_classes(cuda, dtype, mask):
    """Classes whose bias is -inf or the type's lowest value have probability 0 and no gradient; whole strips and tiles of them,
    and the first ones among them."""
    n, k, v = 150, 64, 700
    x, w, b, labels, g = _make(8, n, k, v, dtype, True, cuda)
    low = float("-inf") if mask == "-inf" else torch.finfo(TYPES[dtype]).min
    b[0:64] = low
    b[300:620] = low
    b[699] = low
    labels = torch.where(labels >= 0, 64 + labels % 236, labels).int()       # none of the masked ones
    _, grads = _check(x, w, b, labels, 0.0, "none", g, dtype)
    assert not grads[2][0:64].any() and not grads[1][300:620].any()


def test_all_classes_masked_but_one_and_all(cuda):
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, _ = _make(4, 40, 32, 90, "bf16", True, cuda)
    labels = torch.full((40,), 17, dtype=torch.int32, device=cuda)
    only = torch.full_like(b, float("-inf"))
    only[17] = 0.5
    loss = P.linear_cross_entropy(x, w, labels, only, reduction="none")
    assert not loss.any()                                                     # probability 1
    lowest = torch.full_like(b, torch.finfo(torch.bfloat16).min)              # all alike: uniform
    loss = P.linear_cross_entropy(x, w, labels, lowest, reduction="none")
    assert bool(((loss.double() - math.log(90)).abs() <= 1e-5).all())
    nothing = torch.full_like(b, float("-inf"))
    assert bool(torch.isnan(P.linear_cross_entropy(x, w, labels, nothing, reduction="none")).all())
    masked = P.linear_cross_entropy(x, w, torch.full_like(labels, 3), only, reduction="none")
    assert bool((masked == float("inf")).all())                               # the label itself is masked


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("n", [5, 300])
def test_ignored_rows_may_hold_anything(cuda, n, reduction, dtype):
    """inf and NaN in the features of rows that do not count reach neither the loss nor any gradient."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, g = _make(n, n, 80, 210, dtype, True, cuda, ignored=0.4)
    labels[0], labels[-1] = -100, 3
    bad = (labels == -100).nonzero()[:, 0]
    dirty = x.clone()
    dirty[bad[::2], 7] = float("nan")
    dirty[bad[1::2], 0] = float("inf")
    g = g if reduction == "none" else torch.full((), 8.0, device=cuda)
    loss, grads = _check(dirty, w, b, labels, 0.1, reduction, g, dtype)
    clean_loss, clean = _check(x, w, b, labels, 0.1, reduction, g, dtype)
    assert torch.equal(loss, clean_loss)
    for a, c in zip(grads, clean):
        assert torch.equal(a, c)
    assert not grads[0][bad].any()
    # scalar gradients of rows that do not count may hold anything, too
    if reduction == "none":
        wild = torch.where(labels == -100, torch.full_like(g, float("nan")), g)
        for t in (x, w, b):
            t.requires_grad_(True)
        again = torch.autograd.grad(P.linear_cross_entropy(x, w, labels, b, -100, 0.1, "none"), (x, w, b), wild)
        for a, c in zip(again, clean):
            assert torch.equal(a, c)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_no_row_counts(cuda, reduction):
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(2, 70, 40, 130, "fp16", True, cuda)
    labels.fill_(-7)
    for n in (70, 0):
        leaves = [t.detach().clone().requires_grad_(True) for t in (x[:n], w, b)]
        loss = P.linear_cross_entropy(leaves[0], leaves[1], labels[:n], leaves[2], -7, 0.1, reduction)
        assert loss.shape == ((n,) if reduction == "none" else ()) and not loss.any()
        grads = torch.autograd.grad(loss, leaves, torch.ones_like(loss))
        assert all(not g.any() for g in grads)


def test_labels(cuda):
    """64-bit labels, labels that are no class, an ignored label that is a class, the last class, several dimensions."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, labels, _ = _make(6, 90, 48, 97, "fp16", True, cuda, ignored=0.0)
    with torch.no_grad():
        want = P.linear_cross_entropy(x, w, labels, b, reduction="none")
        assert torch.equal(P.linear_cross_entropy(x, w, labels.long(), b, reduction="none"), want)
        assert torch.equal(P.linear_cross_entropy(x.view(3, 30, 48), w, labels.view(3, 30), b, reduction="none"), want.view(3, 30))
        assert torch.equal(P.linear_cross_entropy(x[4], w, labels[4], b, reduction="none"), want[4])
    odd = labels.long().clone()
    odd[3], odd[40], odd[89] = 97, -1, 1 << 40
    leaf = x.clone().requires_grad_(True)
    loss = P.linear_cross_entropy(leaf, w, odd, b, reduction="none")
    bad = torch.isnan(loss)
    assert bad.nonzero()[:, 0].tolist() == [3, 40, 89] and torch.equal(loss[~bad], want[~bad])
    dx = torch.autograd.grad(loss, leaf, torch.ones_like(loss))[0]
    assert bool(torch.isnan(dx[bad]).all()) and not bool(torch.isnan(dx[~bad]).any())
    assert torch.isnan(P.linear_cross_entropy(x, w, odd, b))
    labels[5], labels[6] = 96, 11
    _check(x, w, b, labels, 0.0, "sum", torch.ones((), device=cuda), "fp16", ignore=11)
    for wrong in (labels[:-1], labels.short(), labels.float(), labels.cpu()):
        with pytest.raises(ValueError):
            P.linear_cross_entropy(x, w, wrong, b)


def test_scores_far_from_zero(cuda):
    """Scores in the hundreds: the running maximum is needed; rows that are certain have loss 0 and no gradient."""
    x, w, b, labels, g = _make(12, 200, 64, 333, "bf16", True, cuda, spread=60.0)
    _check(x, w, b, labels, 0.0, "none", g, "bf16")


def test_loss_against_differences(cuda):
    """The gradient of single features and weights against central differences of the operator's own loss. Steps are exact in
    fp16 (inputs are multiples of 2^-6). The difference is off by the third derivative (a softmax moment, at most |w|^3 times
    the row's factor: step^2 / 6 of it) and by the rounding of two losses (2^-20 of their size, from the loss test's bounds)."""
    from rocal_b200.plugin import pytorch as P
    n, k, v, step = 6, 16, 50, 2.0 ** -5
    g = torch.Generator(device=cuda).manual_seed(2)
    x = (torch.randn((n, k), generator=g, device=cuda) * 64).round().clamp(-128, 128) / 64
    w = (torch.randn((v, k), generator=g, device=cuda) * 32).round().clamp(-96, 96) / 64
    x, w = x.half(), w.half()
    labels = torch.randint(0, v, (n,), generator=g, device=cuda)
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
    grads = torch.autograd.grad(P.linear_cross_entropy(leaves[0], leaves[1], labels, label_smoothing=0.1, reduction="sum"), leaves)
    for which, (r, c) in ((0, (0, 0)), (0, (3, 7)), (0, (5, 15)), (1, (int(labels[0]), 2)), (1, (int(labels[4]), 9)), (1, (49, 15))):
        sides = []
        for sign in (1, -1):
            ts = [x.clone(), w.clone()]
            ts[which][r, c] += sign * step
            sides.append(P.linear_cross_entropy(ts[0], ts[1], labels, label_smoothing=0.1, reduction="none").double().sum())
        diff = float(sides[0] - sides[1]) / (2 * step)
        third = (2.0 if which == 0 else float(x.abs().max())) ** 3 * (1 if which == 0 else n) * 2
        tol = third * step ** 2 / 6 + float(sides[0].abs()) * 2.0 ** -20 / step + 2.0 ** -10 * abs(diff)
        assert abs(float(grads[which][r, c]) - diff) <= tol, (which, r, c)


def test_linear_against_differences(cuda):
    """Gradients of sum(y * c) against central differences along single entries, in fp16 with 32 columns of weight 2^-k: the
    sums stay exact enough for the difference of two rounded outputs (each off by 2^-12 of its size)."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, dy = _linear_make(31, 10, 12, 14, "fp16", True, 0, cuda)
    x, w, step = (x * 64).round() / 64, (w * 64).round() / 64, 2.0 ** -3
    leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
    grads = torch.autograd.grad(P.linear(*leaves, activation="silu"), leaves, dy)
    for which, at in ((0, (2, 3)), (1, (5, 11)), (2, (7,))):
        sides, size = [], 0.0
        for sign in (1, -1):
            ts = [x.clone(), w.clone(), b.clone()]
            ts[which][at] += sign * step
            y = P.linear(*ts, activation="silu").double() * dy.double()
            sides.append(float(y.sum()))
            size = max(size, float(y.abs().sum()))
        moved = float((ts[which][at] - [x, w, b][which][at]).abs())
        diff = (sides[0] - sides[1]) / (2 * moved)
        scale = 3.0 ** 3 if which < 2 else 1.0                    # |x|, |w| stay below 3
        tol = 0.6 * scale * moved ** 2 / 6 * float(dy.abs().sum()) + size * 2.0 ** -11 / moved + 2.0 ** -9 * abs(diff)
        assert abs(float(grads[which][at]) - diff) <= tol, (which, at)


# ---- clipping ------------------------------------------------------------------------------------------


def test_clip_values(cuda):
    from rocal_b200.plugin import pytorch as P
    big = [torch.full((1000,), 1e30, device=cuda), torch.full((70000,), 1e-30, device=cuda)]         # squares beyond fp32
    norm = P.clip_grad_norm(big, 1.0)
    assert abs(float(norm) / (1e30 * math.sqrt(1000)) - 1) <= 2.0 ** -23 and abs(float(big[0][0]) * math.sqrt(1000) - 1) <= 1e-6
    small = [torch.full((400,), 1e-30, device=cuda)]
    assert abs(float(P.clip_grad_norm(small, 1.0)) / 2e-29 - 1) <= 2.0 ** -23 and bool((small[0] == 1e-30).all())
    huge = [torch.full((300,), 3e38, device=cuda, dtype=torch.bfloat16)]
    assert float(P.clip_grad_norm(huge, float("inf"))) == float("inf")                                # beyond fp32 itself
    for n in (100, 400000):                                                                           # one launch, two launches
        inf = [torch.ones((n,), device=cuda), torch.ones((5,), device=cuda)]
        inf[0][n // 2] = float("-inf")
        assert float(P.clip_grad_norm(inf, 1.0)) == float("inf") and torch.isnan(inf[0][n // 2]) and not inf[1].any()
        nan = [torch.ones((n,), device=cuda), torch.ones((5,), device=cuda)]
        nan[1][4] = float("nan")
        assert torch.isnan(P.clip_grad_norm(nan, 1.0)) and bool(torch.isnan(nan[0]).all())
        ones = [torch.ones((n,), device=cuda, dtype=torch.float16)]
        assert float(P.clip_grad_norm(ones, 0.0)) == float(torch.tensor(math.sqrt(n))) and not ones[0].any()
        zeros = [torch.zeros((n,), device=cuda, dtype=torch.bfloat16)]
        assert float(P.clip_grad_norm(zeros, 1.0)) == 0.0 and not zeros[0].any()


def test_clip_layouts(cuda):
    """Empty and 0-d tensors, other memory orders, views with gaps, odd starts - in place and into other arrays."""
    from rocal_b200.plugin import pytorch as P
    g = torch.Generator(device=cuda).manual_seed(9)

    def made(shape):
        return torch.randn(shape, generator=g, device=cuda).bfloat16()
    whole = made((40, 60))
    base = made((5000,))
    grads = [torch.empty((0,), device=cuda, dtype=torch.bfloat16), made(()), made((6, 8, 5, 5)).contiguous(memory_format=torch.channels_last),
             made((30, 20)).t(), whole[3:33, 7:50], base[1:4001], made((1, 1, 7))]
    rest = torch.ones((40, 60), dtype=torch.bool, device=cuda)
    rest[3:33, 7:50] = False
    kept, edge = whole[rest].clone(), base[[0, 4001, 4999]].clone()
    norm, wants = _clip_reference([t.clone() for t in grads], 0.5, 1.0)
    outs = [torch.empty_like(t, dtype=torch.float32) for t in grads]
    outs[3] = torch.empty((20, 30), device=cuda)                   # another order than its gradient
    outs[4] = torch.zeros((30, 50), device=cuda)[:, 3:46]          # gaps
    before = [t.clone() for t in grads]
    assert abs(float(P.clip_grad_norm(grads, 0.5, out=outs)) - norm) <= 2.0 ** -23 * norm
    for o, w, t, k in zip(outs, wants, grads, before):
        _clip_close(o, w)
        assert torch.equal(t, k)
    assert abs(float(P.clip_grad_norm(grads, 0.5)) - norm) <= 2.0 ** -23 * norm
    for t, w in zip(grads, wants):
        _clip_close(t, w)
    assert torch.equal(whole[rest], kept) and torch.equal(base[[0, 4001, 4999]], edge)


def test_clip_refusals_and_parameters(cuda):
    import rocal_b200
    from rocal_b200.plugin import pytorch as P
    t = torch.ones((64,), device=cuda)
    with pytest.raises(rocal_b200.Rb200Error, match="overlaps"):
        P.clip_grad_norm([t, t], 1.0)
    with pytest.raises(rocal_b200.Rb200Error, match="overlaps"):
        P.clip_grad_norm([t[:40], t[30:]], 1.0)
    out = torch.empty_like(t)
    assert abs(float(P.clip_grad_norm([t, t], 100.0, out=[out, torch.empty_like(t)])) - math.sqrt(128)) <= 1e-5   # listed twice, counts twice
    for bad in (t.double(), t.int(), t.cpu()):
        with pytest.raises(ValueError):
            P.clip_grad_norm([t, bad], 1.0)
    with pytest.raises(ValueError):
        P.clip_grad_norm([t], 1.0, out=[out[:10]])
    with pytest.raises(ValueError):
        P.clip_grad_norm([t.half()], 1.0, out=[out.bfloat16()])
    with pytest.raises(ValueError):
        P.clip_grad_norm([t], -1.0)
    assert bool((t == 1).all())
    params = [torch.nn.Parameter(torch.zeros((10,), device=cuda)) for _ in range(3)]
    params[0].grad, params[2].grad = torch.full((10,), 3.0, device=cuda), torch.full((10,), 4.0, device=cuda)
    norm = P.clip_grad_norm_(params, 1.0)
    assert abs(float(norm) - math.sqrt(250)) <= 1e-5 and abs(float(params[2].grad[0]) - 4 / math.sqrt(250)) <= 1e-6 and params[1].grad is None
    assert float(P.clip_grad_norm_([torch.nn.Parameter(torch.zeros((1,), device=cuda))], 1.0)) == 0.0


# ---- sizes beyond 32 bits, what autograd is told -----------------------------------------------------


def test_offsets_beyond_32_bits(cuda):
    """Rows of 40000 elements apart: the last rows lie beyond 2^31 elements; gradients of more than 2^31 elements."""
    from rocal_b200 import kernels as K
    from rocal_b200.plugin import pytorch as P
    n, ld, k, m = 60000, 40000, 64, 40
    whole = torch.zeros((n, ld), dtype=torch.float16, device=cuda)           # 4.8 GB
    g = torch.Generator(device=cuda).manual_seed(4)
    x = whole[:, 16:16 + k]
    x.copy_(torch.randn((n, k), generator=g, device=cuda))
    w, b = torch.randn((m, k), generator=g, device=cuda).half() / 8, torch.randn((m,), generator=g, device=cuda).half()
    out = whole[:, 2000:2000 + m]
    K.linear(x, w, b, activation="relu", out=out)
    y64, _, tol, _ = _forward(x, w, b, None, "relu", "fp16")
    _linear_close(out, y64, tol, "y")
    odd = whole[:, 3001:3001 + k]                                             # not on 16-byte boundaries: packed
    odd.copy_(x)
    assert torch.equal(K.linear(odd, w, b, activation="relu"), out)
    dy = out
    _, dw, db, _ = K.linear_backward(dy, x, w, need=(False, True, True, False))
    _, dw2, db2, _ = K.linear_backward(dy.contiguous(), x.contiguous(), w, need=(False, True, True, False))
    assert torch.equal(dw, dw2) and torch.equal(db, db2)
    labels = torch.randint(0, m, (n,), generator=g, device=cuda)
    assert torch.equal(P.linear_cross_entropy(x, w, labels, b), P.linear_cross_entropy(x.contiguous(), w, labels, b))
    del whole, x, out, odd, dy
    big = torch.full(((1 << 31) + 77,), 2.0 ** -10, dtype=torch.bfloat16, device=cuda)
    small = torch.ones((3,), device=cuda)
    norm = P.clip_grad_norm([big, small], 1.0)
    want = math.sqrt(((1 << 31) + 77) * 2.0 ** -20 + 3)
    assert abs(float(norm) / want - 1) <= 2.0 ** -23
    c = torch.tensor(2.0 ** -10 / want, device=cuda).bfloat16()
    assert bool((big[:1000] == c).all()) and bool((big[-1000:] == c).all()) and bool((big[(1 << 30) - 500:(1 << 30) + 500] == c).all())


def test_in_place_writes_are_known_to_autograd(cuda):
    from rocal_b200 import kernels as K
    from rocal_b200.plugin import pytorch as P
    a = torch.ones((8,), device=cuda, requires_grad=True)
    saved = torch.full((8,), 2.0, device=cuda)
    y = (a * saved).sum()                       # saves `saved`
    P.clip_grad_norm([saved], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    out = torch.zeros((4, 8), device=cuda, dtype=torch.float16)
    before = out._version
    K.linear(torch.ones((4, 16), device=cuda, dtype=torch.float16), torch.ones((8, 16), device=cuda, dtype=torch.float16), out=out)
    assert out._version > before


@pytest.mark.parametrize("period", [1, 2, 60, 1024, 1500, 3000])
def test_residual_gradients_of_any_period(cuda, period):
    """Few and many rows to a residual row, with and without the bias' sums."""
    from rocal_b200 import kernels as K
    n, k, m = 3000 // period * period, 24, 300
    x, w, _, _, dy = _linear_make(period, n, k, m, "bf16", False, 0, cuda)
    z = torch.zeros((n, m), dtype=torch.float64, device=cuda)
    wants, tols = _backward(x, w, dy, z, z, "none", period, "bf16")
    for need in ((False, False, False, True), (False, False, True, True), (True, True, True, True)):
        got = K.linear_backward(dy, x, w, residual_rows=period, need=need)
        for g, want, tol, name in zip(got, wants, tols, ("dx", "dweight", "dbias", "dresidual")):
            if g is not None:
                _linear_close(g, want, tol, name)


# ---- streams, graphs, threads --------------------------------------------------------------------------


def _step(x, w, b, wc, labels, r):
    """A head's forward and backward pass and the clipping of its gradients, through the kernel layer."""
    from rocal_b200 import kernels as K
    h, z = K.linear(x, w, b, r, "gelu", want_preact=True)
    loss, stats, info = K.linear_cross_entropy(h, wc, labels, label_smoothing=0.1)
    dh, dwc, _ = K.linear_cross_entropy_backward(torch.ones_like(loss), h, wc, labels, stats, info, label_smoothing=0.1, need=(True, True, False))
    dx, dw, db, dr = K.linear_backward(dh, x, w, z, "gelu", r.shape[0])
    norm = K.grad_clip([dwc, dw, db, dr], 0.01)
    return [h, loss, dx, dwc, dw, db, dr, norm]


def _step_inputs(seed, cuda, n=384, k=96, m=128, v=300):
    x, w, b, r, _ = _linear_make(seed, n, k, m, "bf16", True, 12, cuda)
    _, wc, _, labels, _ = _make(seed + 1, n, m, v, "bf16", False, cuda)
    return x, w, b, wc, labels, r


def test_results_do_not_depend_on_the_run(cuda):
    """The same inputs give the same bits: no sum depends on timing."""
    args = _step_inputs(50, cuda)
    first = _step(*args)
    for _ in range(5):
        for a, c in zip(first, _step(*args)):
            assert torch.equal(a, c)


def test_captured_steps_replay(cuda):
    """Two captured steps, replayed in turn and on new inputs; each has workspaces of its own."""
    one, two = _step_inputs(60, cuda), _step_inputs(70, cuda, n=204, v=1000)
    fresh = _step_inputs(80, cuda)
    want_one, want_two, want_fresh = _step(*one), _step(*two), _step(*fresh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _step(*one)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for args in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(*args))
        graphs.append(g)
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
    torch.cuda.synchronize()
    for want, got in ((want_one, outs[0]), (want_two, outs[1])):
        for a, c in zip(want, got):
            assert torch.equal(a, c)
    for a, c in zip(one, fresh):
        a.copy_(c)
    graphs[0].replay()
    torch.cuda.synchronize()
    for a, c in zip(want_fresh, outs[0]):
        assert torch.equal(a, c)
    assert _status() == 0


def test_captured_backward_pass(cuda):
    """autograd's backward pass in a capture - refused while an eager graph of the same leaf lives on the default stream,
    which CUDA would answer by ending the process."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, wc, labels, r = _step_inputs(90, cuda)
    w.requires_grad_(True)
    wc.requires_grad_(True)

    def step():
        loss = P.linear_cross_entropy(P.linear(x, w, b, r, "gelu"), wc, labels)
        return (loss,) + torch.autograd.grad(loss, (w, wc))
    want = [t.detach().clone() for t in step()]
    alive = P.linear(x, w, b, r, "gelu")                       # holds w's gradient node
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="still alive"):
        with torch.cuda.graph(g):
            step()
    torch.cuda.synchronize()
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for _ in range(2):
        g.replay()
    torch.cuda.synchronize()
    for a, c in zip(want, got):
        assert torch.equal(a, c.detach())


def test_other_streams(cuda):
    """Calls on a stream of the caller's choice, tensors of the default stream; two streams at a time."""
    from rocal_b200 import kernels as K
    args = [_step_inputs(100 + i, cuda) for i in range(2)]
    wants = [_step(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    gots = []
    for _ in range(3):
        gots = []
        for a, s in zip(args, streams):
            with torch.cuda.stream(s):
                gots.append(_step(*a))
    torch.cuda.synchronize()
    for want, got in zip(wants, gots):
        for a, c in zip(want, got):
            assert torch.equal(a, c)
    y = K.linear(args[0][0], args[0][1], stream=streams[0])
    streams[0].synchronize()
    assert torch.equal(y, K.linear(args[0][0], args[0][1]))
    assert _status() == 0


def test_concurrent_threads(cuda):
    args = [_step_inputs(110 + i, cuda) for i in range(4)]
    wants = [_step(*a) for a in args]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = _step(*args[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, c) for a, c in zip(wants[i], got)):
                    wrong.append(i)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_threads_that_have_not_used_cuda(cuda):
    """The first CUDA work of a thread is the operator's: a backward pass in a fresh process (autograd's own thread), a new
    thread of this one."""
    code = ("import torch\n"
            "from rocal_b200.plugin import pytorch as P\n"
            "x, w = torch.ones(8, 128).half().cuda(), torch.ones(10, 128).half().cuda().requires_grad_(True)\n"
            "loss = P.linear_cross_entropy(x, w, torch.arange(8, device='cuda'))\n"
            "loss.backward()\n"
            "print('gradient', float(w.grad.float().abs().sum()) > 0)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "gradient True" in r.stdout, r.stderr[-2000:]
    from rocal_b200 import kernels as K
    x, w, b, _, _ = _linear_make(1, 20, 64, 30, "fp16", True, 0, cuda)
    want, got = K.linear(x, w, b), []
    thread = threading.Thread(target=lambda: got.append(K.linear(x, w, b)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert torch.equal(want, got[0])


def test_loss_bound_is_not_vacuous(cuda):
    """The oracle with a planted mistake (one label moved) is far outside the bounds that the operator meets."""
    x, w, b, labels, g = _make(3, 64, 32, 50, "fp16", True, cuda, ignored=0.0)
    right, tols = _reference(x, w, b, labels, 0.0, "none", g, "fp16")
    labels[7] = (labels[7] + 1) % 50
    wrong, _ = _reference(x, w, b, labels, 0.0, "none", g, "fp16")
    assert all(float(((a - c).abs() - t).max()) > 0 for a, c, t in zip(right, wrong, tols))
    with pytest.raises(AssertionError):
        _close(wrong[0].float(), right[0], tols[0], "planted")
