"""The head operators behind the framework's own sources and encoders, as a training program strings them together: the batches
of a folder of JPEGs through a patch projection, a hidden layer and a loss, backward and clipped; the anchors of the box
matcher and encoder into the loss.

The chain is compared with the same chain in 64 bits from the same batch. Every tensor between two operators is rounded to
fp16, half of 2^-10 relative at each element: u = 2^-11 of its norm at most. On the way to a gradient there are no more
than twelve such roundings, and none of the operators (projections with weights of norm about one, gelu, softmax) enlarges a
relative difference by more than two: 24 u = 1.2% of a gradient's norm."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

import synthetic as S
from test_pipeline_gpu import MEAN, STD, _jpeg_batch

pytestmark = pytest.mark.gpu


def _patches(images, size):
    """[n, 3, h, w] -> [n, patches, 3 * size * size]"""
    n, c, h, w = images.shape
    return images.view(n, c, h // size, size, w // size, size).permute(0, 2, 4, 1, 3, 5).reshape(n, -1, c * size * size)


def _model(device, classes, width=96, size=16, side=64):
    g = torch.Generator(device=device).manual_seed(5)

    def made(shape, scale):
        return (torch.randn(shape, generator=g, device=device) * scale).half().requires_grad_(True)
    k, patches = 3 * size * size, (side // size) ** 2
    return {"proj": made((width, k), k ** -0.5), "proj_b": made((width,), 0.1), "pos": made((patches, width), 0.3),
            "hidden": made((2 * width, width), width ** -0.5), "hidden_b": made((2 * width,), 0.1),
            "head": made((classes, 2 * width), (2 * width) ** -0.5), "head_b": made((classes,), 0.1)}


def _loss(m, images, labels):
    from rocal_b200.plugin import pytorch as P
    x = P.linear(_patches(images, 16), m["proj"], m["proj_b"], m["pos"])
    h = P.linear(x, m["hidden"], m["hidden_b"], activation="gelu")
    return P.linear_cross_entropy(h.float().mean(1).half(), m["head"], labels, m["head_b"], label_smoothing=0.1)


def _loss64(m, images, labels):
    f = torch.nn.functional
    x = _patches(images.double(), 16) @ m["proj"].t() + m["proj_b"] + m["pos"]
    h = f.gelu(x @ m["hidden"].t() + m["hidden_b"]).mean(1)
    return f.cross_entropy(h @ m["head"].t() + m["head_b"], labels.long(), label_smoothing=0.1)


def _off(a, b):
    return float((a.double() - b).norm() / b.norm())


def test_training_steps_on_a_folder_of_images(cuda, tmp_path):
    from rocal_b200 import fn, types
    from rocal_b200.pipeline import Pipeline
    from rocal_b200.plugin import pytorch as P
    _, streams = _jpeg_batch(S.rng_for(61), 7, (70, 120))
    for i, sb in enumerate(streams):
        d = tmp_path / ("n%02d" % (i % 3))
        d.mkdir(exist_ok=True)
        (d / ("im%d.jpg" % i)).write_bytes(sb)
    pipe = Pipeline(batch_size=4, device_id=0, seed=3)
    with pipe:
        jpegs, _ = fn.readers.file(file_root=str(tmp_path))
        dec = fn.decoders.image(jpegs, file_root=str(tmp_path), max_decoded_width=128, max_decoded_height=128, pad_last_batch=True)
        out = fn.crop_mirror_normalize(fn.resize(dec, resize_width=72, resize_height=72), crop=[64, 64], mean=MEAN, std=STD,
                                       mirror=fn.random.coin_flip(0.5), output_layout=types.NCHW, output_dtype=types.FLOAT16)
        pipe.set_outputs(out)
    pipe.build()
    m = _model(cuda, 3)
    steps = 0
    for (images,), labels in P.ROCALClassificationIterator(pipe):
        assert images.dtype == torch.float16 and images.shape == (4, 3, 64, 64)
        labels = labels.to(torch.int32)
        padded = pipe.get_last_batch_padded_size() if steps else 0
        if padded:                                     # the samples that fill up the last batch take no part
            labels[4 - padded:] = -100
        for t in m.values():
            t.grad = None
        loss = _loss(m, images, labels)
        (loss * 128).backward()                        # a loss scale
        wide = {k: t.detach().double().requires_grad_(True) for k, t in m.items()}
        loss64 = _loss64(wide, images, labels)
        grads64 = dict(zip(wide, torch.autograd.grad(loss64, list(wide.values()))))
        assert abs(float(loss.detach()) - float(loss64.detach())) <= 24 * 2.0 ** -11 * float(loss64.detach())
        for k, t in m.items():
            assert _off(t.grad / 128, grads64[k]) <= 24 * 2.0 ** -11, k
        masters = [torch.empty_like(t, dtype=torch.float32) for t in m.values()]
        norm = P.clip_grad_norm([t.grad for t in m.values()], 0.5, out=masters, inv_scale=1 / 128)
        norm64 = float(torch.sqrt(sum((g ** 2).sum() for g in grads64.values())))
        assert abs(float(norm) - norm64) <= 24 * 2.0 ** -11 * norm64
        for g, k in zip(masters, m):
            assert _off(g, grads64[k] * min(1.0, 0.5 / norm64)) <= 48 * 2.0 ** -11, k
        with torch.no_grad():
            for t, g in zip(m.values(), masters):
                t -= 0.1 * g
        steps += 1
    assert steps == 2
    pipe.rocal_release()


def test_anchor_classes_from_the_matcher_and_the_encoder(cuda):
    """box_iou_match: background below the low threshold, ignored between the thresholds; box_encode: a class for every anchor.
    Both int32 arrays go into the loss as they are."""
    from rocal_b200 import kernels as K
    from rocal_b200.plugin import pytorch as P
    rng = S.rng_for(62)
    n, k, classes = 3, 64, 81
    anchors = S.ssd300_anchors()
    boxes, labels, offs = S.random_boxes(rng, n)
    b, l, o = (torch.from_numpy(np.ascontiguousarray(t)).to(cuda) for t in (boxes, labels, offs))
    a = torch.from_numpy(anchors).to(cuda)
    _, encoded = K.box_encode(b, l, o, a, 0.5, (0, 0, 0, 0), (0.1, 0.1, 0.2, 0.2), True, 1.0, 50)
    matches = K.box_iou_match(b, o, a, 0.5, 0.4, False, 50)
    start = o[:-1, None].long()
    picked = torch.where(matches >= 0, l[(start + matches.clamp(min=0)).clamp(max=len(l) - 1)], torch.where(matches == -1, 0, -2)).int()
    assert bool((picked == -2).any()) and encoded.shape == (n, len(anchors)) and encoded.dtype == torch.int32
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn((n, len(anchors), k), generator=g, device=cuda).bfloat16().requires_grad_(True)
    w = (torch.randn((classes, k), generator=g, device=cuda) * k ** -0.5).bfloat16().requires_grad_(True)
    for target, ignore in ((encoded, -100), (picked, -2)):
        loss = P.linear_cross_entropy(x, w, target, ignore_index=ignore, reduction="sum")
        dx, dw = torch.autograd.grad(loss, (x, w))
        x64, w64 = x.detach().double().requires_grad_(True), w.detach().double().requires_grad_(True)
        want = torch.nn.functional.cross_entropy((x64 @ w64.t()).view(-1, classes), target.view(-1).long(), ignore_index=ignore, reduction="sum")
        wx, ww = torch.autograd.grad(want, (x64, w64))
        assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
        assert _off(dx, wx) <= 2 * 2.0 ** -8 and _off(dw, ww) <= 2 * 2.0 ** -8      # two roundings to bf16
        if ignore == -2:
            assert not dx[picked == -2].any()
