"""Which tensors share memory, as the clipping decides it before it writes: strided views of one buffer, on the CPU, against
the sets of their bytes."""
import random

import pytest

torch = pytest.importorskip("torch")


def _bytes(t):
    size, at = t.element_size(), t.storage_offset() * t.element_size()
    found = [at]
    for n, stride in zip(t.shape, t.stride()):
        found = [a + i * stride * size for a in found for i in range(n)]
    return [a + k for a in found for k in range(size)]


def _view(rng, base):
    dims = rng.randint(0, 3)
    shape = [rng.choice([0, 1, 2, 3, 4, 5]) if rng.random() < 0.9 else 1 for _ in range(dims)]
    stride = [rng.choice([0, 1, 2, 3, 5, 7, 10, 20]) for _ in range(dims)]
    offset = rng.randint(0, 40)
    while offset + sum((n - 1) * s for n, s in zip(shape, stride) if n) >= base.numel():
        offset = 0
        stride = [s // 2 for s in stride]
    return torch.as_strided(base, shape, stride, offset)


@pytest.mark.parametrize("seed", range(4))
def test_shared_memory_of_any_views(seed):
    from rocal_b200._torch import head
    rng, yes = random.Random(seed), 0
    buffer = torch.zeros(400, dtype=torch.uint8)
    bases = [buffer.view(torch.float16), buffer[4:].view(torch.float32), torch.zeros(100, dtype=torch.float16)]
    for _ in range(1500):
        a, b = (_view(rng, rng.choice(bases)) for _ in range(2))
        x, y = _bytes(a), _bytes(b)
        same = a.untyped_storage().data_ptr() == b.untyped_storage().data_ptr()
        want = same and bool(set(x) & set(y))
        assert head.share_memory(a, b) == head.share_memory(b, a) == want, (a.shape, a.stride(), a.storage_offset(), b.shape, b.stride(), b.storage_offset())
        # a repeated byte is found, and only layouts that are not nested may be refused beside those
        repeated, said = len(set(x)) < len(x), head.overlaps_itself(a)
        assert said or not repeated
        yes += want
    assert 50 < yes < 1450      # the sample holds both kinds


def test_views_that_do_not_overlap_are_told_apart():
    """What programs have: columns of one matrix, every other row, halves of a channels-last tensor."""
    from rocal_b200._torch import head
    base = torch.zeros(3000, 700)
    for a, b, want in ((base[:, :350], base[:, 350:], False), (base[:, :351], base[:, 350:], True), (base[::2], base[1::2], False),
                       (base[::2], base[::3], True), (base.t()[:350], base.t()[350:], False), (base[:, 1::2], base[:, ::2], False)):
        assert head.share_memory(a, b) == want
        assert not head.overlaps_itself(a) and not head.overlaps_itself(b)
    images = torch.zeros(4, 8, 5, 5).contiguous(memory_format=torch.channels_last)
    assert not head.share_memory(images[:, :4], images[:, 4:]) and head.share_memory(images[:, :5], images[:, 4:])
    assert head.overlaps_itself(torch.zeros(1).expand(5)) and not head.overlaps_itself(images[:, 2:7])
