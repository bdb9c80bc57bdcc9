"""rb200k_linear for a few rows (the form of single queries): against the formulas in 64 bits, with the tolerances derived in
test_head_linear_gpu (sums in 32 bits, one rounding), around the sizes where its vectors, slices and rules change."""
import pytest

torch = pytest.importorskip("torch")

from test_head_linear_gpu import TYPES, _close, _forward, _make   # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("k,m", [(1, 1), (7, 3), (8, 2), (255, 17), (256, 16), (257, 1001), (264, 1), (1024, 300), (1032, 301), (2048, 1000),
                                 (2049, 999), (6000, 77), (16384, 5), (16385, 5), (4096, 4100), (4104, 4096)])
def test_sizes(cuda, n, k, m, dtype):
    from rocal_b200.plugin import pytorch as P
    x, w, b, r, _ = _make(n + 3 * k + m, n, k, m, dtype, k % 2 == 0, (0, n, 1)[(n + k) % 3], cuda)
    for act in ("none", "relu", "gelu", "silu"):
        y64, _, ty, _ = _forward(x, w, b, r, act, dtype)
        _close(P.linear(x, w, b, r, act), y64, ty, act)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("n", [1, 2, 4])
@pytest.mark.parametrize("lead,pitch", [(0, 520), (8, 520), (1, 520), (0, 515), (3, 517)])
def test_pitches_and_offsets(cuda, n, lead, pitch, dtype):
    """x, weight and out inside wider arrays; what lies between the rows is NaN and stays."""
    from rocal_b200 import kernels as K
    k, m = 509, 70
    x0, w0, b, _, _ = _make(n + lead + pitch, n, k, m, dtype, True, 0, cuda)

    def inside(t):
        wide = torch.full((t.shape[0] * pitch + 16,), float("nan"), device=cuda, dtype=t.dtype)
        v = wide[lead:].as_strided((t.shape[0], t.shape[1]), (pitch, 1))
        v.copy_(t)
        return v, wide
    (x, _), (w, _) = inside(x0), inside(w0)
    out, wide = inside(torch.zeros(n, m, device=cuda, dtype=TYPES[dtype]))
    y64, z64, ty, tz = _forward(x0, w0, b, None, "gelu", dtype)
    u = torch.finfo(TYPES[dtype]).eps / 2
    _, z = K.linear(x, w, b, activation="gelu", want_preact=True, out=out)
    _close(out, y64, ty, "out")
    _close(z, z64, u * z64.abs() + (1 + u) * tz + 2.0 ** -24, "z")
    assert int(torch.isnan(wide).sum()) == wide.numel() - n * m


def test_values_that_are_not_finite_stay_in_their_rows_and_columns(cuda):
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, _ = _make(5, 3, 300, 40, "bf16", True, 0, cuda)
    want = P.linear(x, w, b)
    x2, w2 = x.clone(), w.clone()
    x2[1, 299] = float("inf")
    w2[7, 0] = float("nan")
    got = P.linear(x2, w2, b)
    keep = torch.ones(3, 40, dtype=torch.bool, device=cuda)
    keep[1] = keep[:, 7] = False
    assert torch.equal(got[keep], want[keep])
    assert bool(torch.isnan(got[:, 7]).all()) and not bool(torch.isfinite(got[1]).any())


@pytest.mark.parametrize("n", [1, 4])
def test_gradients_captured_replays_and_bits(cuda, n):
    """The forward pass of few rows keeps what the backward pass reads; replays follow their inputs; the same call gives the same bits."""
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, dy = _make(n, n, 520, 264, "fp16", True, 0, cuda)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(P.linear(x, w, b, activation="gelu"), leaves, dy)
    x64, w64, b64 = (t.detach().double().requires_grad_(True) for t in leaves)
    want = torch.autograd.grad(torch.nn.functional.gelu(x64 @ w64.t() + b64), (x64, w64, b64), dy.double())
    for g, t in zip(got, want):    # dz rounded, z rounded for its slope, the result rounded: under 4 roundings of the largest products' sum
        assert float((g.double() - t).abs().max()) <= 4 * 2.0 ** -11 * float(t.abs().max()) + 4 * 2.0 ** -11 * float(dy.abs().max())
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        P.linear(x, w, b)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            y = P.linear(x, w, b)
        for seed in range(3):
            x.copy_(torch.randn(n, 520, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)))
            graph.replay()
            assert torch.equal(y, P.linear(x, w, b))


def test_an_empty_call_and_one_output(cuda):
    from rocal_b200.plugin import pytorch as P
    x, w, b, _, _ = _make(9, 1, 33, 1, "fp16", True, 0, cuda)
    assert P.linear(x[:0], w, b).shape == (0, 1)
    y64, _, ty, _ = _forward(x, w, b, None, "none", "fp16")
    _close(P.linear(x, w, b), y64, ty, "one output")
