"""The activations and their slopes over the whole range that an element type holds, against 64 bits.

One rounding to the result's type is at most half of eps relative (bf16 2^-8, fp16 2^-11), or half of its smallest subnormal (bf16
2^-134, fp16 2^-25). The value itself, in 32 bits: the argument of the exponential, up to 126 in powers of two, has three
roundings of 2^-24 of its size (two operations and the constant), 126 * 3 * 2^-24 * ln 2 = 1.6e-5; the exponential and the reciprocal 2^-22
each (squared where its root is taken: 2^-21), the tail's ratio 1.1e-6, half a dozen operations 2^-24 each: 2e-5 in all. Exponentials below
2^-126 are flushed: gelu, at most 14 * 2^-126 * R(13) = 2^-127 off there, its slope 14 * 0.4 * 2^-126 = 2^-123."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
HALF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}
LEAST = {"fp16": 2.0 ** -25, "bf16": 2.0 ** -134}


def _values(device, dtype, n):
    """n multiples of 64 numbers: densely -14 .. 14, logarithmically out to +-120."""
    inner = torch.linspace(-14, 14, n // 2, device=device)
    outer = torch.logspace(-6, 2.079, n // 4, device=device)
    return torch.cat((inner, outer, -outer)).to(TYPES[dtype]).view(-1, 64)


def _exact(z, act):
    """(value, slope) in 64 bits, without cancellation in the tails."""
    if act == "silu":
        g, rest = torch.sigmoid(z), torch.sigmoid(-z)
        return z * g, g * (1 + z * rest)
    tail = 0.5 * torch.special.erfcx(-z * 0.5 ** 0.5) * torch.exp(-0.5 * z * z)          # Phi(z) for z < 0
    phi = torch.where(z < 0, tail, 0.5 * torch.erfc(-z * 0.5 ** 0.5))
    return z * phi, phi + z * torch.exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("few", [False, True])
def test_values_over_the_whole_range(cuda, act, dtype, few):
    """The activation alone: the weight is the identity. On the tensor cores' way and on that of a few rows."""
    from rocal_b200 import kernels as K
    z = _values(cuda, dtype, 16384)
    eye = torch.eye(64, device=cuda).to(TYPES[dtype])
    got = torch.cat([K.linear(p, eye, activation=act) for p in z.split(4 if few else z.shape[0])]).double()
    want, _ = _exact(z.double(), act)
    tol = want.abs() * (HALF[dtype] + 2e-5) + LEAST[dtype] + (2.0 ** -127 if act == "gelu" else 0.0)
    off = (got - want).abs() - tol
    assert float(off.max()) <= 0, (float(z.flatten()[off.argmax()]), float(got.flatten()[off.argmax()]), float(want.flatten()[off.argmax()]))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_slopes_over_the_whole_range(cuda, act, dtype):
    """dx behind an identity and a gradient of ones is the slope: rounded as the operand of the product, which adds zeros to it. The
    slopes cancel near their zeros (gelu -0.75, silu -1.28): the terms' sizes count there."""
    from rocal_b200 import kernels as K
    z = _values(cuda, dtype, 16384)
    eye = torch.eye(64, device=cuda).to(TYPES[dtype])
    dx, _, _, _ = K.linear_backward(torch.ones_like(z), z, eye, z, act, need=(True, False, False, False))
    d = z.double()
    _, want = _exact(d, act)
    if act == "silu":
        size = torch.sigmoid(d) * (1 + (d * torch.sigmoid(-d)).abs())
    else:
        value, _ = _exact(d, act)
        size = (value / torch.where(d == 0, torch.ones_like(d), d)).abs() + (d * torch.exp(-0.5 * d * d)).abs() / (2 * torch.pi) ** 0.5 + (d == 0)
    tol = want.abs() * HALF[dtype] + size * 2e-5 + LEAST[dtype] + (2.0 ** -123 if act == "gelu" else 0.0)
    off = (dx.double() - want).abs() - tol
    assert float(off.max()) <= 0, (float(z.flatten()[off.argmax()]), float(dx.flatten()[off.argmax()]), float(want.flatten()[off.argmax()]))
