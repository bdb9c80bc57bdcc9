"""rb200k_grad_clip (plugin.pytorch.clip_grad_norm) against the formula in 64 bits.

Squares are added in 64 bits, so the norm is off by its one rounding to fp32 (2^-24; 2^-23 is asked). The factor is made of
that norm by an addition, a division and a product, and multiplies the gradient: six roundings of 2^-24 in all, then one to
the output's type (u = eps / 2; half a step of its subnormals below them)."""
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _grads(seed, counts, dtypes, device, scale=1e-2):
    g = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn((c,), generator=g, device=device) * scale).to(TYPES[dtypes[i % len(dtypes)]]) for i, c in enumerate(counts)]


def _reference(grads, max_norm, inv_scale):
    norm = inv_scale * math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))
    c = min(1.0, max_norm / (norm + 1e-6))
    return norm, [g.double() * (inv_scale * c) for g in grads]


def _close(got, want):
    tol = want.abs() * (6 * 2.0 ** -24 + torch.finfo(got.dtype).eps / 2) + TINY[got.dtype]
    off = (got.double() - want).abs() - tol
    assert got.numel() == 0 or float(off.max()) <= 0, "%g beyond the bound" % float(off.max())


COUNTS = [[1], [7], [2048], [2049, 1, 0, 5], [100000], [3, 70000, 1, 32768, 65537, 12, 4095], [17] * 16, [33, 5000] * 100, [300 + i for i in range(1000)],
          [1 + (i * 37) % 9000 for i in range(2100)], [3000001, 5, 1 << 20]]


@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "%d_tensors_%d" % (len(c), sum(c)))
@pytest.mark.parametrize("dtypes", [("fp32",), ("fp16",), ("bf16",), ("fp32", "bf16", "fp16")], ids="-".join)
@pytest.mark.parametrize("clips", [True, False])
def test_norm_and_clipping(cuda, counts, dtypes, clips):
    from rocal_b200.plugin import pytorch as P
    grads = _grads(sum(counts) + len(counts), counts, dtypes, cuda)
    inv = 1.0 / 128 if "fp16" in dtypes else 1.0
    max_norm = 1e-2 * inv * math.sqrt(sum(counts)) * (0.3 if clips else 4.0)
    norm, wants = _reference(grads, max_norm, inv)
    # into other arrays, of the gradients' types and 32-bit, packed behind one another (any alignment)
    for out_type in (None, torch.float32):
        if out_type is None and len(dtypes) > 1:
            out = [torch.empty_like(g) for g in grads]
        else:
            flat = torch.full((sum(counts) + 1,), 7.0, dtype=out_type or grads[0].dtype, device=cuda)
            out = list(flat[1:].split(counts))
        keep = [g.clone() for g in grads]
        got = P.clip_grad_norm(grads, max_norm, out=out, inv_scale=inv)
        assert abs(float(got) - norm) <= 2.0 ** -23 * norm
        assert all(torch.equal(a, b) for a, b in zip(grads, keep))
        for o, w in zip(out, wants):
            _close(o, w)
    # in place
    got = P.clip_grad_norm(grads, max_norm, inv_scale=inv)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for g, w in zip(grads, wants):
        _close(g, w)
