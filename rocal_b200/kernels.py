"""Thin Python front of the kernel-level C-ABI (include/rb200_kernels.h).

torch is used only to own device memory and streams; every computation is a call into
librocal_b200.so. Inputs: a uint8 CUDA tensor holding the packed source images (the arena) and
a numpy structured array with one row per sample (dtypes in rocal_b200.tables).
"""
import ctypes

import numpy as np
import torch

from . import tables as T
from ._lib import (BoxEncoderParams, BoxMatcherParams, LinearBackwardParams, LinearCeParams,
                   LinearParams, NormalizeParams, PointwiseParams,
                   ResampleParams, WarpParams, check, lib)

_TORCH_DTYPE = {T.FP32: torch.float32, T.FP16: torch.float16, T.UINT8: torch.uint8}


def _stream_ptr(stream):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def to_device_table(samples, device):
    """Uploads a structured numpy table as raw bytes."""
    raw = torch.from_numpy(np.ascontiguousarray(samples).view(np.uint8).reshape(-1))
    return raw.to(device, non_blocking=False)


def _alloc_out(n, out_w, out_h, dtype, layout, device, out):
    shape = (n, 3, out_h, out_w) if layout == T.NCHW else (n, out_h, out_w, 3)
    if out is None:
        out = torch.empty(shape, dtype=_TORCH_DTYPE[dtype], device=device)
    else:
        assert tuple(out.shape) == shape and out.dtype == _TORCH_DTYPE[dtype] and out.is_contiguous()
    return out


def _sizes(p, arena, out, arena_bytes, out_bytes):
    """The sizes a launch states to the library: the tensors' own unless the caller overrides them."""
    p.arena_bytes = int(arena.numel() * arena.element_size() if arena_bytes is None else arena_bytes)
    p.out_bytes = int(out.numel() * out.element_size() if out_bytes is None else out_bytes)


def resample(arena, samples, out_w, out_h, out_dtype=T.FP32, out_layout=T.NCHW, mul=None, add=None,
             fill_padding=True, out=None, d_samples=None, stream=None, staged=True, interpolation=0, path=0,
             status=None, probe=None, overlap=False, arena_bytes=None, out_bytes=None, strip_rows=0):
    """rb200k_resample. strip_rows: rows per CTA of the row-streaming kernel (0 = the library chooses). arena_bytes / out_bytes: the sizes stated to the library (None: those of the tensors). overlap=True states that the launch is independent of the kernel enqueued just before it. `samples`: numpy RESAMPLE_SAMPLE table (host); `d_samples`: the same table
    already on the device (uploaded here when None). staged=False withholds the host table from
    the launch so that the kernel gathers straight from global memory; path=1 (RB200_RESAMPLE_PATH_TILE)
    forces the shared-memory tile kernel. status: an int32 CUDA tensor that receives 1 when a bounded wait gives up
    (None: the library-wide word); probe=(wait_cycles, skip_row) launches through rb200k_resample_probe."""
    n = len(samples)
    out = _alloc_out(n, out_w, out_h, out_dtype, out_layout, arena.device, out)
    if d_samples is None:
        d_samples = to_device_table(samples, arena.device)
    p = ResampleParams()
    p.out = out.data_ptr()
    p.out_w, p.out_h, p.out_dtype, p.out_layout = out_w, out_h, out_dtype, out_layout
    p.normalize = 1 if mul is not None else 0
    p.fill_padding = 1 if fill_padding else 0
    p.interpolation = int(interpolation)
    p.path = int(path)
    p.strip_rows = int(strip_rows)
    for c in range(3):
        p.mul[c] = float(mul[c]) if mul is not None else 1.0
        p.add[c] = float(add[c]) if add is not None else 0.0
    p.status = status.data_ptr() if status is not None else None
    p.overlap = 1 if overlap else 0
    _sizes(p, arena, out, arena_bytes, out_bytes)
    h_ptr = samples.ctypes.data_as(ctypes.c_void_p) if staged else None
    if probe is not None:
        check(lib.rb200k_resample_probe(arena.data_ptr(), d_samples.data_ptr(), h_ptr, n, ctypes.byref(p),
                                        _stream_ptr(stream), int(probe[0]), int(probe[1])), "rb200k_resample_probe")
    else:
        check(lib.rb200k_resample(arena.data_ptr(), d_samples.data_ptr(), h_ptr, n, ctypes.byref(p),
                                  _stream_ptr(stream)), "rb200k_resample")
    return out


def pointwise(arena, samples, out_w, out_h, color_op=T.COLOR_NONE, out_dtype=T.UINT8, out_layout=T.NHWC,
              mul=None, add=None, reverse_channels=False, fill_padding=True, out=None, d_samples=None,
              stream=None, arith=0, status=None, probe=None, overlap=False, arena_bytes=None, out_bytes=None):
    """rb200k_pointwise. arena_bytes / out_bytes as for resample. arith: 0 exact, 1 fast colour arithmetic; status / probe as for resample."""
    n = len(samples)
    out = _alloc_out(n, out_w, out_h, out_dtype, out_layout, arena.device, out)
    if d_samples is None:
        d_samples = to_device_table(samples, arena.device)
    p = PointwiseParams()
    p.out = out.data_ptr()
    p.out_w, p.out_h, p.out_dtype, p.out_layout = out_w, out_h, out_dtype, out_layout
    p.color_op = color_op
    p.normalize = 1 if mul is not None else 0
    p.fill_padding = 1 if fill_padding else 0
    p.reverse_channels = 1 if reverse_channels else 0
    for c in range(3):
        p.mul[c] = float(mul[c]) if mul is not None else 1.0
        p.add[c] = float(add[c]) if add is not None else 0.0
    p.arith = int(arith)
    p.overlap = 1 if overlap else 0
    p.status = status.data_ptr() if status is not None else None
    _sizes(p, arena, out, arena_bytes, out_bytes)
    if probe is not None:
        check(lib.rb200k_pointwise_probe(arena.data_ptr(), d_samples.data_ptr(), samples.ctypes.data_as(ctypes.c_void_p), n,
                                         ctypes.byref(p), _stream_ptr(stream), int(probe[0]), int(probe[1])),
              "rb200k_pointwise_probe")
    else:
        check(lib.rb200k_pointwise(arena.data_ptr(), d_samples.data_ptr(), samples.ctypes.data_as(ctypes.c_void_p), n,
                                   ctypes.byref(p), _stream_ptr(stream)), "rb200k_pointwise")
    return out


def warp_affine(arena, samples, out_w, out_h, fill_padding=True, out=None, d_samples=None, stream=None, overlap=False,
                status=None, arena_bytes=None, out_bytes=None):
    """rb200k_warp_affine: uint8 NHWC output. status / arena_bytes / out_bytes as for resample."""
    n = len(samples)
    out = _alloc_out(n, out_w, out_h, T.UINT8, T.NHWC, arena.device, out)
    if d_samples is None:
        d_samples = to_device_table(samples, arena.device)
    p = WarpParams()
    p.out = out.data_ptr()
    p.out_w, p.out_h = out_w, out_h
    p.fill_padding = 1 if fill_padding else 0
    p.overlap = 1 if overlap else 0
    p.status = status.data_ptr() if status is not None else None
    _sizes(p, arena, out, arena_bytes, out_bytes)
    check(lib.rb200k_warp_affine(arena.data_ptr(), d_samples.data_ptr(), n, ctypes.byref(p), _stream_ptr(stream)),
          "rb200k_warp_affine")
    return out


def box_encode(boxes, labels, box_offsets, anchors, criteria, means, stds, offset, scale, max_boxes,
               out_boxes=None, out_labels=None, stream=None):
    """rb200k_box_encode. boxes [total,4] f32, labels [total] i32, box_offsets [n+1] i32, anchors
    [A,4] f32 — all CUDA tensors."""
    n = box_offsets.numel() - 1
    a = anchors.shape[0]
    if out_boxes is None:
        out_boxes = torch.empty((n, a, 4), dtype=torch.float32, device=boxes.device)
    if out_labels is None:
        out_labels = torch.empty((n, a), dtype=torch.int32, device=boxes.device)
    p = BoxEncoderParams()
    p.anchors = anchors.data_ptr()
    p.num_anchors = a
    p.criteria = float(criteria)
    for k in range(4):
        p.means[k] = float(means[k])
        p.inv_stds[k] = float(np.float32(1.0 / float(np.float32(stds[k]))))
    p.offset = 1 if offset else 0
    p.scale = float(scale)
    check(lib.rb200k_box_encode(boxes.data_ptr(), labels.data_ptr(), box_offsets.data_ptr(), n, int(max_boxes),
                                ctypes.byref(p), out_boxes.data_ptr(), out_labels.data_ptr(), _stream_ptr(stream)),
          "rb200k_box_encode")
    return out_boxes, out_labels


def box_iou_match(boxes, box_offsets, anchors, high_threshold, low_threshold, allow_low_quality_matches, max_boxes,
                  out=None, stream=None):
    """rb200k_box_iou_match. boxes [total,4] f32, box_offsets [n+1] i32, anchors [A,4] f32 - CUDA tensors.
    Returns int32 [n, A]: matched box index per anchor, -1 / -2 below the low / high threshold."""
    n = box_offsets.numel() - 1
    a = anchors.shape[0]
    if out is None:
        out = torch.empty((n, a), dtype=torch.int32, device=boxes.device)
    p = BoxMatcherParams()
    p.anchors = anchors.data_ptr()
    p.num_anchors = a
    p.high_threshold, p.low_threshold = float(high_threshold), float(low_threshold)
    p.allow_low_quality_matches = 1 if allow_low_quality_matches else 0
    check(lib.rb200k_box_iou_match(boxes.data_ptr(), box_offsets.data_ptr(), n, int(max_boxes), ctypes.byref(p),
                                   out.data_ptr(), _stream_ptr(stream)), "rb200k_box_iou_match")
    return out


def box_transform(boxes, labels, box_offsets, windows, rule, stream=None):
    """rb200k_box_transform. boxes [total,4] f32, labels [total] i32, box_offsets [n+1] i32 - CUDA tensors; windows: numpy
    BOX_WINDOW table (uploaded here) or a CUDA uint8 tensor holding one. Returns (out_boxes, out_labels, out_offsets) with
    capacity total + n; out_offsets[n] is the number of valid entries."""
    n = box_offsets.numel() - 1
    total = boxes.shape[0]
    d_win = to_device_table(windows, boxes.device) if isinstance(windows, np.ndarray) else windows
    out_boxes = torch.empty((total + n, 4), dtype=torch.float32, device=boxes.device)
    out_labels = torch.empty((total + n,), dtype=torch.int32, device=boxes.device)
    out_offsets = torch.empty((n + 1,), dtype=torch.int32, device=boxes.device)
    check(lib.rb200k_box_transform(boxes.data_ptr(), labels.data_ptr(), box_offsets.data_ptr(), n, d_win.data_ptr(), int(rule),
                                   out_boxes.data_ptr(), out_labels.data_ptr(), out_offsets.data_ptr(), _stream_ptr(stream)),
          "rb200k_box_transform")
    return out_boxes, out_labels, out_offsets


def normalize_scratch_bytes(n, max_w, max_h, axis_mask):
    return int(lib.rb200k_normalize_scratch_bytes(int(n), int(max_w), int(max_h), int(axis_mask)))


def _normalize_params(out, out_w, out_h, out_dtype, axis_mask, mean, stddev, scale, shift, fill_padding):
    p = NormalizeParams()
    p.out = out.data_ptr()
    p.out_w, p.out_h, p.out_dtype, p.axis_mask = out_w, out_h, out_dtype, int(axis_mask)
    p.compute_mean, p.compute_stddev = int(mean is None), int(stddev is None)
    p.fill_padding = 1 if fill_padding else 0
    for c in range(3):
        p.mean[c] = float(mean[c]) if mean is not None else 0.0
        p.stddev[c] = float(stddev[c]) if stddev is not None else 1.0
    p.scale, p.shift = float(scale), float(shift)
    return p


def normalize(arena, samples, out_w, out_h, axis_mask=3, mean=None, stddev=None, scale=1.0, shift=0.0, out_dtype=T.FP32,
              fill_padding=True, out=None, d_samples=None, scratch=None, stream=None):
    """rb200k_normalize: uint8 HWC windows (POINTWISE_SAMPLE table) -> [n][out_h][out_w][3] float32 / float16.
    mean / stddev None = computed over the axes of axis_mask (bit 0 height, 1 width, 2 channel). `scratch`: a uint8
    CUDA tensor of at least normalize_scratch_bytes(...) bytes (allocated here when None and needed)."""
    n = len(samples)
    out = _alloc_out(n, out_w, out_h, out_dtype, T.NHWC, arena.device, out)
    if d_samples is None:
        d_samples = to_device_table(samples, arena.device)
    p = _normalize_params(out, out_w, out_h, out_dtype, axis_mask, mean, stddev, scale, shift, fill_padding)
    _sizes(p, arena, out, None, None)
    need = normalize_scratch_bytes(n, out_w, out_h, axis_mask) if (mean is None or stddev is None) else 0
    if scratch is None and need:
        scratch = torch.empty(need, dtype=torch.uint8, device=arena.device)
    check(lib.rb200k_normalize(arena.data_ptr(), d_samples.data_ptr(), samples.ctypes.data_as(ctypes.c_void_p), n, ctypes.byref(p),
                               scratch.data_ptr() if scratch is not None else None, scratch.numel() if scratch is not None else 0,
                               _stream_ptr(stream)), "rb200k_normalize")
    return out


def transpose(arena, samples, perm, out_dims, out=None, d_samples=None, stream=None):
    """rb200k_transpose: uint8 [n][out_dims...], every sample's permuted window at the origin of its slot."""
    n = len(samples)
    if out is None:
        out = torch.zeros((n,) + tuple(int(v) for v in out_dims), dtype=torch.uint8, device=arena.device)
    if d_samples is None:
        d_samples = to_device_table(samples, arena.device)
    pm = (ctypes.c_int32 * 3)(*[int(v) for v in perm])
    od = (ctypes.c_int32 * 3)(*[int(v) for v in out_dims])
    check(lib.rb200k_transpose(arena.data_ptr(), d_samples.data_ptr(), n, pm, out.data_ptr(), od, _stream_ptr(stream)),
          "rb200k_transpose")
    return out


# ---- head operators -----------------------------------------------------------------------------
# Tensors may live on any device; the call runs there, on `stream` or that device's current stream, and takes its
# workspace from torch's allocator on that stream.
_HEAD_DTYPE = {torch.float16: T.FP16, torch.bfloat16: T.BF16}


class _on:
    """The device and stream of a head operator's launch."""

    def __init__(self, device, stream):
        self.device, self.stream = device, stream
        self.away = device.index != torch.cuda.current_device()

    def __enter__(self):
        self.guards = []
        if self.away:
            self.guards.append(torch.cuda.device(self.device))
        if self.stream is not None:
            if self.stream.device != self.device:
                raise ValueError("the stream is on %s, the tensors are on %s" % (self.stream.device, self.device))
            self.guards.append(torch.cuda.stream(self.stream))
        for g in self.guards:
            g.__enter__()
        s = self.stream if self.stream is not None else torch.cuda.current_stream(self.device)
        return s.cuda_stream

    def __exit__(self, *exc):
        for g in reversed(self.guards):
            g.__exit__(*exc)
        return False


def _matrix(t, name, like, cols=None):
    """A 2-d tensor on the device and of the type of `like`, its rows contiguous and not overlapping (copied if need be)."""
    if t.dim() != 2:
        raise ValueError("%s has %d dimensions, a matrix is needed" % (name, t.dim()))
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError("%s is %s on %s, the input is %s on %s" % (name, t.dtype, t.device, like.dtype, like.device))
    if cols is not None and t.shape[1] != cols:
        raise ValueError("%s has %d columns, %d are needed" % (name, t.shape[1], cols))
    if (t.stride(1) != 1 and t.shape[1] > 1) or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _vector(t, name, like, n):
    if t.dim() != 1 or t.shape[0] != n:
        raise ValueError("%s has shape %s, (%d,) is needed" % (name, tuple(t.shape), n))
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError("%s is %s on %s, the input is %s on %s" % (name, t.dtype, t.device, like.dtype, like.device))
    return t.contiguous()


def _head_input(x, weight):
    """Element type of a head operator and its (x, weight) as matrices."""
    if not x.is_cuda:
        raise ValueError("x is on %s: the head operators run on a GPU" % x.device)
    if x.dtype not in _HEAD_DTYPE:
        raise ValueError("x is %s: the head operators take float16 and bfloat16" % x.dtype)
    x = _matrix(x, "x", x)
    return _HEAD_DTYPE[x.dtype], x, _matrix(weight, "weight", x, x.shape[1])


def _output(out, name, shape, like):
    if out is None:
        return torch.empty(shape, dtype=like.dtype, device=like.device)
    if tuple(out.shape) != tuple(shape) or out.dtype != like.dtype or out.device != like.device:
        raise ValueError("%s is %s %s on %s, needed: %s %s on %s" % (name, tuple(out.shape), out.dtype, out.device, tuple(shape),
                                                                    like.dtype, like.device))
    if out.dim() == 2 and ((out.stride(1) != 1 and out.shape[1] > 1) or (out.shape[0] > 1 and out.stride(0) < out.shape[1])):
        raise ValueError("%s needs contiguous rows that do not overlap" % name)
    return out


def _workspace(p, sizer, device):
    need = sizer(ctypes.byref(p))
    if not need:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    p.workspace, p.workspace_bytes = ws.data_ptr(), need
    return ws


def _activation(name):
    if name not in T.ACTIVATIONS:
        raise ValueError("activation %r: one of %s is needed" % (name, ", ".join(T.ACTIVATIONS)))
    return T.ACTIVATIONS[name]


def linear(x, weight, bias=None, residual=None, activation="none", out=None, want_preact=False, stream=None, status=None, probe=None):
    """rb200k_linear: act(x weight^T + bias) + residual for x [n, k], weight [m, k], bias [m], residual [r, m] with r a
    divisor of n (row i takes residual row i % r), all float16 or all bfloat16. Returns [n, m], with want_preact also
    the value before the activation. probe=(wait_cycles, skip_block) launches through rb200k_linear_probe."""
    dtype, x, weight = _head_input(x, weight)
    n, k = x.shape
    m = weight.shape[0]
    act = _activation(activation)
    if bias is not None:
        bias = _vector(bias, "bias", x, m)
    if residual is not None:
        residual = _matrix(residual, "residual", x, m)
        if residual.shape[0] == 0 and n or residual.shape[0] and n % residual.shape[0]:
            raise ValueError("residual has %d rows, which do not divide the %d rows of x" % (residual.shape[0], n))
    with _on(x.device, stream) as s:
        out = _output(out, "out", (n, m), x)
        pre = torch.empty((n, m), dtype=x.dtype, device=x.device) if want_preact else None
        if n:
            p = LinearParams(dtype, act, n, k, m, x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0))
            p.out, p.ldo = out.data_ptr(), out.stride(0)
            if bias is not None:
                p.bias = bias.data_ptr()
            if residual is not None:
                p.residual, p.ldr, p.residual_rows = residual.data_ptr(), residual.stride(0), residual.shape[0]
            if pre is not None:
                p.preact, p.ldp = pre.data_ptr(), m
            if status is not None:
                p.status = status.data_ptr()
            ws = _workspace(p, lib.rb200k_linear_workspace_bytes, x.device)  # noqa: F841  (alive until the launch)
            if probe is not None:
                check(lib.rb200k_linear_probe(ctypes.byref(p), s, int(probe[0]), int(probe[1])), "rb200k_linear_probe")
            else:
                check(lib.rb200k_linear(ctypes.byref(p), s), "rb200k_linear")
    return (out, pre) if want_preact else out


def linear_backward(dout, x, weight, preact=None, activation="none", residual_rows=0, need=(True, True, True, True), stream=None,
                    status=None):
    """rb200k_linear_backward: (dx, dweight, dbias, dresidual), None where `need` is false. dresidual takes residual_rows."""
    dtype, x, weight = _head_input(x, weight)
    n, k = x.shape
    m = weight.shape[0]
    act = _activation(activation)
    dout = _matrix(dout, "dout", x, m)
    if dout.shape[0] != n:
        raise ValueError("dout has %d rows, x has %d" % (dout.shape[0], n))
    if act and (need[0] or need[1] or need[2]):
        if preact is None:
            raise ValueError("the backward pass of an activation needs preact")
        preact = _matrix(preact, "preact", x, m)
        if preact.shape[0] != n:
            raise ValueError("preact has %d rows, x has %d" % (preact.shape[0], n))
    if need[3] and (residual_rows < 1 or n % residual_rows):
        raise ValueError("residual_rows %d does not divide the %d rows" % (residual_rows, n))
    shapes = ((n, k), (m, k), (m,), (residual_rows, m))
    with _on(x.device, stream) as s:
        grads = [torch.empty(shape, dtype=x.dtype, device=x.device) if want else None for shape, want in zip(shapes, need)]
        dx, dw, db, dr = grads
        p = LinearBackwardParams(dtype, act, n, k, m, dout.data_ptr(), dout.stride(0), x.data_ptr(), x.stride(0), weight.data_ptr(),
                                 weight.stride(0))
        if act and preact is not None:
            p.preact, p.ldp = preact.data_ptr(), preact.stride(0)
        if dx is not None:
            p.dx, p.lddx = dx.data_ptr(), k
        if dw is not None:
            p.dweight, p.lddw = dw.data_ptr(), k
        if db is not None:
            p.dbias = db.data_ptr()
        if dr is not None:
            p.dresidual, p.lddr, p.residual_rows = dr.data_ptr(), m, residual_rows
        if status is not None:
            p.status = status.data_ptr()
        ws = _workspace(p, lib.rb200k_linear_backward_workspace_bytes, x.device)  # noqa: F841
        check(lib.rb200k_linear_backward(ctypes.byref(p), s), "rb200k_linear_backward")
    return tuple(grads)


def _ce_params(x, weight, labels, bias, ignore_index, label_smoothing, reduction):
    """(parameter block, tensors that it points into) of a linear cross entropy."""
    dtype, x, weight = _head_input(x, weight)
    n, k = x.shape
    v = weight.shape[0]
    if reduction not in T.REDUCTIONS:
        raise ValueError("reduction %r: one of %s is needed" % (reduction, ", ".join(T.REDUCTIONS)))
    if labels.dim() != 1 or labels.shape[0] != n or labels.device != x.device or labels.dtype not in (torch.int32, torch.int64):
        raise ValueError("labels are %s %s on %s, needed: int32 or int64 of shape (%d,) on %s"
                         % (labels.dtype, tuple(labels.shape), labels.device, n, x.device))
    labels = labels.contiguous()
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("label_smoothing %r outside [0, 1]" % (label_smoothing,))
    p = LinearCeParams(dtype, T.REDUCTIONS[reduction], n, k, v, x.data_ptr(), x.stride(0), weight.data_ptr(), weight.stride(0))
    if bias is not None:
        bias = _vector(bias, "bias", x, v)
        p.bias = bias.data_ptr()
    p.labels, p.label_bytes, p.label_smoothing, p.ignore_index = labels.data_ptr(), labels.element_size(), label_smoothing, ignore_index
    return p, (x, weight, labels, bias)


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, label_smoothing=0.0, reduction="mean", stream=None, status=None):
    """rb200k_linear_ce: the cross entropy of the scores x weight^T + bias for x [n, k], weight [v, k], labels [n] (int32 or
    int64), without making the [n, v] scores. Returns (loss, stats, info): the loss is fp32, [n] or a scalar; stats and info
    go to linear_cross_entropy_backward."""
    p, held = _ce_params(x, weight, labels, bias, ignore_index, label_smoothing, reduction)
    x, n = held[0], p.rows
    with _on(x.device, stream) as s:
        loss = torch.empty((n,) if reduction == "none" else (), dtype=torch.float32, device=x.device)
        stats = torch.empty((2, n), dtype=torch.float32, device=x.device)
        info = torch.empty((4,), dtype=torch.int32, device=x.device)
        p.loss, p.stats, p.info = loss.data_ptr(), stats.data_ptr(), info.data_ptr()
        if status is not None:
            p.status = status.data_ptr()
        ws = _workspace(p, lib.rb200k_linear_ce_workspace_bytes, x.device)  # noqa: F841
        check(lib.rb200k_linear_ce(ctypes.byref(p), s), "rb200k_linear_ce")
    return loss, stats, info


def linear_cross_entropy_backward(dloss, x, weight, labels, stats, info, bias=None, ignore_index=-100, label_smoothing=0.0,
                                  reduction="mean", need=(True, True, True), stream=None, status=None):
    """rb200k_linear_ce_backward: (dx, dweight, dbias), None where `need` is false. dloss: fp32, of the loss's shape."""
    p, held = _ce_params(x, weight, labels, bias, ignore_index, label_smoothing, reduction)
    x, n, k, v = held[0], p.rows, p.features, p.classes
    if dloss.dtype != torch.float32 or dloss.device != x.device or tuple(dloss.shape) != ((n,) if reduction == "none" else ()):
        raise ValueError("dloss is %s %s on %s, it has to be like the loss" % (dloss.dtype, tuple(dloss.shape), dloss.device))
    if tuple(stats.shape) != (2, n) or stats.dtype != torch.float32 or tuple(info.shape) != (4,) or info.dtype != torch.int32 or \
            stats.device != x.device or info.device != x.device or not stats.is_contiguous() or not info.is_contiguous():
        raise ValueError("stats and info are not those of this forward pass")
    dloss = dloss.contiguous()
    with _on(x.device, stream) as s:
        grads = [torch.empty(shape, dtype=x.dtype, device=x.device) if want else None for shape, want in zip(((n, k), (v, k), (v,)), need)]
        dx, dw, db = grads
        p.dloss, p.stats, p.info = dloss.data_ptr(), stats.data_ptr(), info.data_ptr()
        if dx is not None:
            p.dx, p.lddx = dx.data_ptr(), k
        if dw is not None:
            p.dweight, p.lddw = dw.data_ptr(), k
        if db is not None:
            p.dbias = db.data_ptr()
        if status is not None:
            p.status = status.data_ptr()
        ws = _workspace(p, lib.rb200k_linear_ce_backward_workspace_bytes, x.device)  # noqa: F841
        check(lib.rb200k_linear_ce_backward(ctypes.byref(p), s), "rb200k_linear_ce_backward")
    return tuple(grads)


_GRAD_DTYPE = {torch.float32: T.FP32, torch.float16: T.FP16, torch.bfloat16: T.BF16}


def _dense(t):
    """Whether the elements fill a contiguous stretch of memory, in whatever order of the dimensions."""
    order = sorted(range(t.dim()), key=lambda d: -t.stride(d))
    return t.is_contiguous() or t.permute(order).is_contiguous()


def grad_clip(grads, max_norm, out=None, inv_scale=1.0, stream=None):
    """rb200k_grad_clip: the norm (fp32 scalar tensor) of inv_scale * all of `grads`, and each of them times inv_scale * min(1,
    max_norm / (norm + 1e-6)) - in place, or written to the tensors of `out` (the gradients' types or float32)."""
    grads = list(grads)
    targets = grads if out is None else list(out)
    if not grads:
        raise ValueError("no gradients")
    device = grads[0].device
    if not grads[0].is_cuda:
        raise ValueError("the gradients are on %s: the head operators run on a GPU" % device)
    if len(targets) != len(grads):
        raise ValueError("%d outputs for %d gradients" % (len(targets), len(grads)))
    copies = []                        # (view with gaps, the dense tensor that stands for it)
    types = _GRAD_DTYPE
    for both in ((grads,) if out is None else (grads, targets)):
        for t in both:
            if t.dtype not in types or t.device != device or t.layout != torch.strided:
                raise ValueError("a tensor is %s %s on %s; float32, float16 or bfloat16 on %s are needed" % (t.layout, t.dtype, t.device, device))
    with _on(device, stream) as s:
        if out is None:
            if not all(map(torch.Tensor.is_contiguous, grads)):
                dense = [t if _dense(t) else t.contiguous() for t in grads]
                copies = [(t, d) for t, d in zip(grads, dense) if d is not t]
                grads = targets = dense
        else:
            for g, o in zip(grads, targets):
                if g.shape != o.shape or (o.dtype != g.dtype and o.dtype != torch.float32):
                    raise ValueError("an output is %s %s for a gradient %s %s" % (tuple(o.shape), o.dtype, tuple(g.shape), g.dtype))
            if not (all(map(torch.Tensor.is_contiguous, grads)) and all(map(torch.Tensor.is_contiguous, targets))):
                pairs = []
                for g, o in zip(grads, targets):
                    if g.is_contiguous() and o.is_contiguous() or g.stride() == o.stride() and _dense(g):
                        pairs.append((g, o))
                        continue
                    d = o if o.is_contiguous() else torch.empty(o.shape, dtype=o.dtype, device=device)
                    if d is not o:
                        copies.append((o, d))
                    pairs.append((g.contiguous(), d))
                grads, targets = [g for g, _ in pairs], [o for _, o in pairs]
        n = len(grads)
        table = np.empty(n, dtype=T.GRAD_TENSOR)
        table["grad"] = list(map(torch.Tensor.data_ptr, grads))
        table["out"] = table["grad"] if targets is grads else list(map(torch.Tensor.data_ptr, targets))
        table["count"] = list(map(torch.Tensor.numel, grads))
        table["grad_dtype"] = [types[t.dtype] for t in grads]
        table["out_dtype"] = table["grad_dtype"] if targets is grads else [types[t.dtype] for t in targets]
        norm = torch.empty((), dtype=torch.float32, device=device)
        need = lib.rb200k_grad_clip_workspace_bytes(n)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        check(lib.rb200k_grad_clip(table.ctypes.data, n, max_norm, inv_scale, norm.data_ptr(), ws.data_ptr(), need, s), "rb200k_grad_clip")
        for view, dense in copies:
            view.copy_(dense)
    return norm
