"""The head operators' refusals, none of which needs a GPU: the kernel C ABI checks its arguments before any CUDA call, the
torch binding before any library call."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

INVALID, LIMIT = -1, -3


def _lib():
    from rocal_b200 import _lib
    return _lib


def _buffer(nbytes, offset=0):
    """Host memory that stands for a device pointer: nothing reads it, the calls below are refused."""
    raw = np.zeros(nbytes + 512, dtype=np.uint8)
    at = raw.ctypes.data
    return raw, (at + 255) // 256 * 256 + offset


def _linear_params(**changes):
    L = _lib()
    keep, at = _buffer(1 << 16)
    p = L.LinearParams()
    p.dtype, p.activation, p.rows, p.in_features, p.out_features = 1, 0, 4, 16, 8
    p.x, p.ldx, p.weight, p.ldw, p.out, p.ldo = at, 16, at, 16, at, 8
    for k, v in changes.items():
        setattr(p, k, v)
    return p, (keep, at)


@pytest.mark.parametrize("changes,code,text", [
    (dict(dtype=0), INVALID, b"dtype 0"), (dict(dtype=2), INVALID, b"dtype 2"), (dict(activation=4), INVALID, b"activation 4"),
    (dict(activation=-1), INVALID, b"activation -1"), (dict(rows=-1), INVALID, b"rows -1"), (dict(in_features=0), INVALID, b"in_features 0"),
    (dict(out_features=0), INVALID, b"out_features 0"), (dict(rows=(1 << 30) + 1), LIMIT, b"2^30"), (dict(x=None), INVALID, b"x is null"),
    (dict(weight=None), INVALID, b"weight is null"), (dict(out=None), INVALID, b"out is null"), (dict(ldx=15), INVALID, b"leading dimension 15 of x"),
    (dict(ldw=8), INVALID, b"leading dimension 8 of weight"), (dict(ldo=7), INVALID, b"leading dimension 7 of out"),
    (dict(ldx=1 << 40), INVALID, b"leading dimension"), (dict(x=4097), INVALID, b"x is not aligned"), (dict(bias=4097), INVALID, b"bias is not aligned"),
    (dict(residual=4096, ldr=8, residual_rows=3), INVALID, b"residual_rows 3"), (dict(residual=4096, ldr=8, residual_rows=0), INVALID, b"residual_rows 0"),
    (dict(residual=4096, ldr=7, residual_rows=4), INVALID, b"leading dimension 7 of residual"),
    (dict(preact=4096, ldp=7), INVALID, b"leading dimension 7 of preact")])
def test_linear_refuses(changes, code, text):
    lib = _lib().lib
    p, _ = _linear_params(**changes)
    assert lib.rb200k_linear(ctypes.byref(p), None) == code
    assert text in lib.rb200k_last_error(), lib.rb200k_last_error()


def test_null_parameter_blocks_and_empty_batches():
    lib = _lib().lib
    for name in ("linear", "linear_backward", "linear_ce", "linear_ce_backward"):
        assert getattr(lib, "rb200k_" + name)(None, None) == INVALID
        assert getattr(lib, "rb200k_" + name + "_workspace_bytes")(None) == 0
    p, _ = _linear_params(rows=0, x=None)
    assert lib.rb200k_linear(ctypes.byref(p), None) == 0                # no rows: nothing to do
    assert lib.rb200k_linear_workspace_bytes(ctypes.byref(p)) == 0


def _backward_params(**changes):
    L = _lib()
    keep, at = _buffer(1 << 16)
    p = L.LinearBackwardParams()
    p.dtype, p.rows, p.in_features, p.out_features = 16, 6, 16, 8
    p.dout, p.lddo, p.x, p.ldx, p.weight, p.ldw = at, 8, at, 16, at, 16
    p.dx, p.lddx, p.dweight, p.lddw, p.dbias = at, 16, at, 16, at
    for k, v in changes.items():
        setattr(p, k, v)
    return p, (keep, at)


@pytest.mark.parametrize("changes,text", [
    (dict(dout=None), b"dout is null"), (dict(lddo=7), b"leading dimension 7 of dout"), (dict(x=None), b"x is null"),
    (dict(weight=None), b"weight is null"), (dict(activation=2), b"preact is null"), (dict(dresidual=4096, residual_rows=4, lddr=8), b"residual_rows 4"),
    (dict(dresidual=4096, residual_rows=3, lddr=4), b"leading dimension 4 of dresidual"), (dict(lddx=15), b"leading dimension 15 of dx"),
    (dict(lddw=15), b"leading dimension 15 of dweight"), (dict(dbias=4097), b"dbias is not aligned")])
def test_linear_backward_refuses(changes, text):
    lib = _lib().lib
    p, _ = _backward_params(**changes)
    assert lib.rb200k_linear_backward(ctypes.byref(p), None) == INVALID
    assert text in lib.rb200k_last_error(), lib.rb200k_last_error()


def _ce_params(**changes):
    L = _lib()
    keep, at = _buffer(1 << 16)
    p = L.LinearCeParams()
    p.dtype, p.reduction, p.rows, p.features, p.classes = 1, 1, 4, 16, 8
    p.x, p.ldx, p.weight, p.ldw, p.labels, p.label_bytes = at, 16, at, 16, at, 4
    p.loss, p.stats, p.info, p.dloss, p.dx, p.lddx = at, at, at, at, at, 16
    for k, v in changes.items():
        setattr(p, k, v)
    return p, (keep, at)


@pytest.mark.parametrize("changes,code,text,both", [
    (dict(dtype=0), INVALID, b"dtype 0", True), (dict(reduction=3), INVALID, b"reduction 3", True), (dict(label_bytes=2), INVALID, b"labels of 2 bytes", True),
    (dict(label_smoothing=-0.1), INVALID, b"label_smoothing", True), (dict(label_smoothing=1.5), INVALID, b"label_smoothing", True),
    (dict(label_smoothing=float("nan")), INVALID, b"label_smoothing", True), (dict(features=0), INVALID, b"features 0", True),
    (dict(classes=0), INVALID, b"classes 0", True), (dict(classes=(1 << 30) + 1), LIMIT, b"2^30", True), (dict(x=None), INVALID, b"x is null", True),
    (dict(weight=None), INVALID, b"weight is null", True), (dict(labels=None), INVALID, b"labels", True), (dict(stats=None), INVALID, b"stats", True),
    (dict(info=None), INVALID, b"info", True), (dict(labels=4098), INVALID, b"aligned", True), (dict(labels=4100, label_bytes=8), INVALID, b"aligned", True),
    (dict(stats=4098), INVALID, b"aligned", True), (dict(loss=None), INVALID, b"loss is null", False), (dict(ldw=15), INVALID, b"leading dimension 15", True)])
def test_linear_cross_entropy_refuses(changes, code, text, both):
    lib = _lib().lib
    for name in ("linear_ce", "linear_ce_backward") if both else ("linear_ce",):
        p, _ = _ce_params(**changes)
        assert getattr(lib, "rb200k_" + name)(ctypes.byref(p), None) == code, name
        assert text in lib.rb200k_last_error(), lib.rb200k_last_error()


def test_linear_cross_entropy_backward_refuses():
    lib = _lib().lib
    for changes, text in ((dict(dloss=None), b"dloss"), (dict(lddx=15), b"leading dimension 15 of dx"), (dict(dweight=4096, lddw=15), b"dweight"),
                          (dict(dbias=4097), b"dbias")):
        p, _ = _ce_params(**changes)
        assert lib.rb200k_linear_ce_backward(ctypes.byref(p), None) == INVALID
        assert text in lib.rb200k_last_error(), lib.rb200k_last_error()
    p, _ = _ce_params(dx=None)                     # no gradient asked for: nothing to do
    assert lib.rb200k_linear_ce_backward(ctypes.byref(p), None) == 0


def _clip(entries, max_norm=1.0, inv_scale=1.0, norm=4096, ws=4096, ws_bytes=1 << 20):
    from rocal_b200 import tables as T
    lib = _lib().lib
    t = np.array(entries, dtype=T.GRAD_TENSOR) if entries else np.zeros(0, dtype=T.GRAD_TENSOR)
    return lib.rb200k_grad_clip(t.ctypes.data, len(t), max_norm, inv_scale, norm, ws, ws_bytes, None), lib.rb200k_last_error()


FP32, FP16, BF16 = 0, 1, 16


@pytest.mark.parametrize("entries,text", [
    ([(4096, 4096, 8, FP32, FP32), (4096, 4096, 8, FP32, FP32)], b"overlaps"),              # the same gradient twice, in place
    ([(4096, 4096, 8, FP32, FP32), (4100, 4100, 8, FP32, FP32)], b"overlaps"),              # overlapping views, in place
    ([(4096, 8192, 8, FP32, FP32), (5000, 8220, 8, FP32, FP32)], b"overlaps"),              # overlapping outputs
    ([(4096, 8192, 8, FP32, FP32), (8200, 9000, 8, FP32, FP32)], b"overlaps"),              # an output over another's gradients
    ([(4096, 4100, 8, FP32, FP32)], b"overlaps"),                                           # an output over its own gradients, shifted
    ([(4096, 4096, 8, FP16, FP32)], b"another type"),
    ([(4096, 8192, 8, FP16, BF16)], b"types"), ([(4096, 8192, 8, FP32, FP16)], b"types"), ([(4096, 8192, 8, 2, 2)], b"types"),
    ([(4097, 8192, 8, FP16, FP16)], b"aligned"), ([(4098, 8192, 8, FP32, FP32)], b"aligned"), ([(4096, 8194, 8, FP16, FP32)], b"aligned"),
    ([(0, 8192, 8, FP32, FP32)], b"null"), ([(4096, 0, 8, FP32, FP32)], b"null"), ([(4096, 8192, -1, FP32, FP32)], b"-1 elements")])
def test_clip_refuses_tensors(entries, text):
    rc, said = _clip(entries)
    assert rc == INVALID and text in said, said


def test_clip_refuses_arguments():
    one = [(4096, 4096, 8, FP32, FP32)]
    for kw, text in ((dict(max_norm=-1.0), b"max_norm"), (dict(max_norm=float("nan")), b"max_norm"), (dict(inv_scale=0.0), b"inv_scale"),
                     (dict(inv_scale=float("inf")), b"inv_scale"), (dict(norm=None), b"norm"), (dict(norm=4098), b"norm"), (dict(ws=None), b"workspace"),
                     (dict(ws_bytes=16), b"workspace"), (dict(ws=4104), b"workspace")):
        rc, said = _clip(one, **kw)
        assert rc == INVALID and text in said, (kw, said)
    # gradients that share memory are fine where the outputs do not (a tied weight's gradient, listed twice, counts twice); the
    # call gets as far as the device query, which fails here or passes on a GPU box with a workspace that is refused
    assert _lib().lib.rb200k_grad_clip_workspace_bytes(0) == 0
    assert _lib().lib.rb200k_grad_clip_workspace_bytes(961) == 2 * _lib().lib.rb200k_grad_clip_workspace_bytes(960)


def test_binding_refuses_what_is_not_on_a_gpu():
    from rocal_b200.plugin import pytorch as P
    x, w = torch.zeros(2, 8, dtype=torch.float16), torch.zeros(3, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="run on a GPU"):
        P.linear(x, w)
    with pytest.raises(ValueError, match="run on a GPU"):
        P.linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="run on a GPU"):
        P.clip_grad_norm([x], 1.0)
    with pytest.raises(ValueError, match="no gradients"):
        P.clip_grad_norm([], 1.0)
    with pytest.raises(ValueError, match="activation 'tanh'"):
        P.linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match="reduction 'max'"):
        P.linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int32), reduction="max")
    with pytest.raises(ValueError, match="does not go with"):
        P.linear(x, torch.zeros(3, 7, dtype=torch.float16))
    with pytest.raises(ValueError, match="do not go together"):
        P.linear_cross_entropy(x, w, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="not a tail"):
        P.linear(x.view(1, 2, 8), w, residual=torch.zeros(5, 3, dtype=torch.float16))
    with pytest.raises(ValueError, match="1 outputs for 2"):
        P.clip_grad_norm([x, w], 1.0, out=[x])


def test_parameter_blocks_have_the_headers_sizes(tmp_path):
    """The ctypes mirrors and the C structs agree (compiled with the system compiler)."""
    import os
    import subprocess
    L, root = _lib(), os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "rb200_kernels.h"\nint main(void) { printf("%zu %zu %zu %zu", sizeof(rb200_linear_params), '
                   "sizeof(rb200_linear_backward_params), sizeof(rb200_linear_ce_params), sizeof(rb200_grad_tensor)); return 0; }\n")
    exe = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", exe], check=True)
    got = [int(v) for v in subprocess.run([exe], capture_output=True, text=True, check=True).stdout.split()]
    from rocal_b200 import tables as T
    assert got == [ctypes.sizeof(L.LinearParams), ctypes.sizeof(L.LinearBackwardParams), ctypes.sizeof(L.LinearCeParams), T.GRAD_TENSOR.itemsize]
