"""Sums that are exact: small whole numbers, whose 32-bit sums lose nothing in any order, so that results have to be equal to the
last bit. A bound for rounded sums grows with their length and would not notice a few missing elements of a long one; here every
element of the last 16 contracted ones counts in every output.

Entries are -1, 0 or 1, one in four of them not 0 (the last 16 all): a sum of k products has a spread of at most sqrt(k / 16) + 4, 36 for
16385. Results up to 256 are whole numbers of both element types; larger ones do not occur (7 spreads), which the test asserts."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _whole(g, shape, contracted, dtype, dense=16):
    """Entries -1, 0, 1 along axis `contracted`, its last `dense` places without zeros."""
    t = torch.randint(0, 8, shape, generator=g, device=g.device)
    t = (t == 0).int() - (t == 1).int()
    end = t.narrow(contracted, max(0, shape[contracted] - dense), min(dense, shape[contracted]))
    end.copy_(torch.randint(0, 2, end.shape, generator=g, device=g.device) * 2 - 1)
    return t.to(TYPES[dtype])


def _equal(got, exact, name):
    assert float(exact.abs().max()) <= 256 and bool((exact == exact.round()).all()), name
    assert torch.equal(got.double(), exact), (name, int((got.double() != exact).sum()), exact.numel())


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,m", [(1, 16384, 70), (2, 8191, 33), (3, 16383, 40), (4, 8192, 257), (5, 16385, 5), (20, 8192, 24), (20, 8191, 24), (130, 16384, 300),
                                   (300, 16385, 130), (513, 8191, 65), (1, 16385, 9), (64, 127, 64), (129, 65, 31), (260, 64, 520)])
def test_forward(cuda, n, k, m, dtype):
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(n + k + m)
    x, w = _whole(g, (n, k), 1, dtype), _whole(g, (m, k), 1, dtype)
    b = _whole(g, (1, m), 1, dtype)[0]
    exact = x.double() @ w.double().t()
    assert bool((exact != x[:, :-1].double() @ w[:, :-1].double().t()).all())      # a missing last element would show everywhere
    _equal(K.linear(x, w), exact, "y")
    y, z = K.linear(x, w, b, activation="relu", want_preact=True)
    _equal(z, exact + b.double(), "z")
    _equal(y, (exact + b.double()).clamp(min=0), "relu")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,m", [(16385, 24, 20), (8191, 130, 72), (16384, 64, 300), (8192, 257, 33), (300, 130, 16385), (20, 24, 8192), (5, 40, 8191), (2, 16, 16384), (1, 8, 16)])
def test_backward(cuda, n, k, m, dtype):
    """dx is contracted over m, dweight over n; dbias and dresidual are sums over rows."""
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(n + k + m)
    dout = _whole(g, (n, m), 0 if n > m else 1, dtype)
    x, w = _whole(g, (n, k), 0, dtype), _whole(g, (m, k), 0, dtype)
    d, x64, w64 = dout.double(), x.double(), w.double()
    for period in (p for p in (1, 5, 4) if n % p == 0):
        dx, dw, db, dr = K.linear_backward(dout, x, w, residual_rows=period)
        for got, exact, name in ((dx, d @ w64, "dx"), (dw, d.t() @ x64, "dweight")):
            _equal(got, exact, name)
        for got, exact, name in ((db, d.sum(0), "dbias"), (dr, d.view(-1, period, m).sum(0), "dresidual")):
            if float(exact.abs().max()) <= 256:       # n sixteenths at most: a spread of 64
                _equal(got, exact, name)
            assert torch.equal(got, exact.to(got.dtype)), name


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,v", [(20, 16385, 300), (300, 8192, 130), (5, 8191, 1000), (130, 4097, 20), (700, 256, 90), (129, 255, 96), (1000, 128, 128), (64, 1, 7)])
def test_scores_of_the_loss(cuda, n, k, v, dtype):
    """The statistics that the forward pass keeps: each row's largest score and its label's are whole numbers. Both ways, the general one
    with one accumulator and with two, and the one for few classes."""
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(n + k + v)
    x, w = _whole(g, (n, k), 1, dtype), _whole(g, (v, k), 1, dtype)
    labels = torch.randint(0, v, (n,), generator=g, device=cuda)
    z = x.double() @ w.double().t()
    _, stats, _ = K.linear_cross_entropy(x, w, labels)
    assert torch.equal(stats[0].double(), z.max(1).values) and torch.equal(stats[2].double(), z.gather(1, labels[:, None])[:, 0])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n,k,v", [(16385, 264, 256), (8191, 300, 256), (600001, 257, 256), (16384, 128, 128), (8193, 256, 64), (3000, 512, 16)])
def test_gradient_of_the_weights(cuda, n, k, v, dtype):
    """Weights of zero: every class has probability 1 / v, a power of two, and the gradient of a score is 1 / v or 1 / v - 1, exact in both element
    types. Sums over n rows (600001: in several pieces) are whole multiples of 1 / v, 2^23 of them at most; one rounding ends them."""
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(n + k + v)
    x, w = _whole(g, (n, k), 0, dtype), torch.zeros((v, k), dtype=TYPES[dtype], device=cuda)
    labels = torch.randint(0, v, (n,), generator=g, device=cuda)
    loss, stats, info = K.linear_cross_entropy(x, w, labels, reduction="sum")
    dx, dw, db = K.linear_cross_entropy_backward(torch.ones_like(loss), x, w, labels, stats, info, reduction="sum")
    x64 = x.double()
    mine = torch.zeros((v, k), dtype=torch.float64, device=cuda).index_add_(0, labels, x64)
    exact = x64.sum(0) / v - mine
    assert float(exact.abs().max()) * v < 2.0 ** 23
    assert torch.equal(dw, exact.to(dw.dtype)) and not dx.any()
    counts = torch.bincount(labels, minlength=v).double()
    assert torch.equal(db, (n / v - counts).to(db.dtype))


@pytest.mark.parametrize("dtype,n,k,v", [("fp16", 300, 264, 2048), ("fp16", 5000, 300, 2048), ("fp16", 40, 8, 1024), ("bf16", 300, 264, 256), ("bf16", 5, 512, 256),
                                         ("fp16", 260, 128, 128), ("bf16", 260, 100, 128), ("bf16", 129, 256, 64)])
def test_gradient_of_the_features(cuda, dtype, n, k, v):
    """Features of zero: again all classes have probability 1 / v. Labels point at classes whose weights are zero, so that a row's gradient is the
    sum of the other classes' weights over v: every class counts, and the result is exact."""
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(n + k + v)
    x, w = torch.zeros((n, k), dtype=TYPES[dtype], device=cuda), _whole(g, (v, k), 0, dtype)
    w[:3] = 0
    labels = torch.randint(0, 3, (n,), generator=g, device=cuda)
    loss, stats, info = K.linear_cross_entropy(x, w, labels, reduction="sum")
    dx, dw, _ = K.linear_cross_entropy_backward(torch.ones_like(loss), x, w, labels, stats, info, reduction="sum")
    total = w.double().sum(0)
    assert float(total.abs().max()) <= 256
    assert torch.equal(dx.double(), (total / v).expand(n, k)) and not dw.any()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_drift_of_long_sums(cuda, dtype):
    """The tensor cores cut what they add, always to the same side, so that the loss drifts with the length of an accumulator's sum: with scores
    of spread 2, -0.65e-6 to -0.77e-6 of it for 2048 products and -1.35e-6 to -1.5e-6 for 4096 (8192 rows, 16384 classes). 4096 features are
    spread over two accumulators and must not drift further than 2048 do: 1.0e-6 lies between, and the mean over 2048 rows, each
    off by some 0.4e-6 besides, is known to 1e-8."""
    from rocal_b200 import kernels as K
    drift = {}
    for k in (2048, 4096):
        g = torch.Generator(device=cuda).manual_seed(k)
        n, v = 2048, 16384
        x = torch.randn((n, k), generator=g, device=cuda).to(TYPES[dtype])
        w = (torch.randn((v, k), generator=g, device=cuda) * 2 / k ** 0.5).to(TYPES[dtype])
        labels = torch.randint(0, v, (n,), generator=g, device=cuda)
        z = x.double() @ w.double().t()
        exact = torch.logsumexp(z, 1) - z.gather(1, labels[:, None])[:, 0]
        loss = K.linear_cross_entropy(x, w, labels, reduction="none")[0].double()
        drift[k] = float((loss - exact).sum() / exact.sum())
    assert abs(drift[2048]) <= 1.0e-6 and abs(drift[4096]) <= 1.0e-6, drift


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_sums_over_very_many_rows(cuda, dtype):
    """Products of one sign, the worst that cutting can meet: a long sum in one accumulator drifts by 2.9e-9 of itself for every product (measured
    up to 65536 of them), 524288 rows by 3e-3. Split as they are, they must not drift by more than 2.44e-4, half of an fp16 result's half
    step. (The tiles alone nearly fill the GPU, so that nothing else splits the sum.)"""
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(4)
    n, m, k = 524288, 2048, 2048
    x = torch.rand((n, k), generator=g, device=cuda, dtype=torch.float32).to(TYPES[dtype])
    dout = (torch.rand((n, m), generator=g, device=cuda, dtype=torch.float32) / 16).to(TYPES[dtype])
    dw = K.linear_backward(dout, x, torch.zeros((m, k), dtype=TYPES[dtype], device=cuda), need=(False, True, False, False))[1].double()
    exact = torch.zeros((m, k), dtype=torch.float64, device=cuda)
    for a, b in zip(dout.split(65536), x.split(65536)):
        exact += a.double().t() @ b.double()
    off = (dw - exact) / exact
    half = torch.finfo(TYPES[dtype]).eps / 2
    assert float(off.abs().max()) <= half + 2.44e-4, float(off.abs().max())
    # the mean, but for the roundings' own: the sums are 8192 with a spread of 10, bfloat16's step is 32 below and 64 above it, so that its
    # roundings all go to 8192 and do not cancel
    rounded = (exact.to(TYPES[dtype]).double() - exact) / exact
    assert abs(float((off - rounded).mean())) <= 2.44e-4, float((off - rounded).mean())


def test_few_classes_over_very_many_rows(cuda):
    """The same for the way of few classes, where a block adds up all of its rows: weights of zero and one label for all rows make the other
    class' gradient half the sum of the features, all of one sign. 2^25 rows are 226720 for each of 148 blocks, which drift by 6.6e-4 and
    more. Features of 64 sizes within a binade, so that the mean of the 64 roundings is within 2^-11 / 3 ** 0.5 / 8 = 3.5e-5 (one spread)."""
    from rocal_b200 import kernels as K
    g = torch.Generator(device=cuda).manual_seed(6)
    n, k = 1 << 25, 64
    x = torch.empty((n, k), dtype=torch.float16, device=cuda)
    exact = torch.zeros(k, dtype=torch.float64, device=cuda)
    for part in x.split(1 << 21):
        part.copy_(torch.rand(part.shape, generator=g, device=cuda) * (1 + torch.arange(k, device=cuda) / k))
        exact += part.double().sum(0) / 2
    w, labels = torch.zeros((2, k), dtype=torch.float16, device=cuda), torch.zeros(n, dtype=torch.int32, device=cuda)
    loss, stats, info = K.linear_cross_entropy(x, w, labels, reduction="sum")
    dw = K.linear_cross_entropy_backward(torch.full_like(loss, 2.0 ** -12), x, w, labels, stats, info, reduction="sum", need=(False, True, False))[1].double()
    exact *= 2.0 ** -12
    assert torch.equal(dw[0], -dw[1])
    off = (dw[1] - exact) / exact
    assert float(off.abs().max()) <= 2.0 ** -11 + 2.44e-4 and abs(float(off.mean())) <= 2.44e-4, (float(off.abs().max()), float(off.mean()))
