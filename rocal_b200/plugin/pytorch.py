"""PyTorch iterator over a built pipeline, in the spirit of amd.rocal.plugin.pytorch.ROCALGenericIterator
(rocAL_pybind/amd/rocal/plugin/pytorch.py:32-294). The reference copies every output into a fresh
torch tensor (copy_data); here outputs are handed over zero-copy through DLPack (the route the
reference's TensorFlow plugin uses, plugin/tf.py:114) and are valid until the next batch, or copied
when copy=True."""
import torch


class ROCALGenericIterator(object):
    def __init__(self, pipeline, feeder=None, copy=False, size=-1, auto_reset=False, tensor_layout=None, reverse_channels=False,
                 multiplier=None, offset=None, tensor_dtype=None, device="cuda", device_id=0, display=False,
                 fill_last_batch=True, dynamic_shape=False, last_batch_padded=False):
        """feeder(pipeline) -> bool feeds one batch through pipeline.feed_input / feed_ragged and returns
        False when the data is exhausted. The remaining arguments are those of the reference's iterators
        (plugin/pytorch.py:46, 282-290) and are accepted for source compatibility: layout, type and normalisation
        are those of the pipeline's output operators, and the tensors live on the pipeline's GPU."""
        if str(device).startswith("cpu"):
            raise ValueError("outputs live on the pipeline's GPU (device must be 'cuda' / 'gpu')")
        self.loader = pipeline
        self.feeder = feeder
        self.copy = copy
        self.auto_reset = auto_reset

    def __iter__(self):
        return self

    def _outputs(self):
        """Zero-copy views of the batch's outputs, valid until the next batch: torch.from_dlpack hands the pipeline
        the current torch stream, and the pipeline orders the reuse of these buffers behind the work queued there
        (RocalTensor.__dlpack__). Work on other streams is the caller's to order. With copy=True the views are cloned
        and the clone has finished before the tensors are returned, as the reference's synchronous copy_data."""
        outs = [torch.from_dlpack(t) for t in self.loader.get_output_tensors()]
        if self.copy:
            outs = [o.clone() for o in outs]
            torch.cuda.current_stream(outs[0].device).synchronize()
        return outs

    def __next__(self):
        if self.feeder is not None and not self.feeder(self.loader):
            if self.loader.is_empty():
                raise StopIteration
        elif self.feeder is None and self.loader.is_empty():
            raise StopIteration
        self.loader.rocal_run()
        outs = self._outputs()
        return outs

    next = __next__


class ROCALClassificationIterator(ROCALGenericIterator):
    """Yields ([outputs...], labels) for a pipeline with a file source (plugin/pytorch.py:246-294 of the reference):
    labels are an int32 CUDA tensor of the batch's class indices, or - after fn.one_hot(num_classes=k) - an int32
    [N, k] one-hot tensor filled on the device. With LAST_BATCH_PARTIAL the padding samples of the last batch are
    cut off. Iteration stops when the source is exhausted; reset() starts the next epoch."""

    def __next__(self):
        if self.loader.is_empty():
            if self.auto_reset:
                self.reset()
            raise StopIteration
        self.loader.rocal_run()
        outs = self._outputs()
        if getattr(self.loader, "_one_hot_encoding", False):
            labels = self.loader.get_one_hot_encoded_labels(self.loader._num_classes, device=outs[0].device)
        else:
            labels = torch.from_numpy(self.loader.get_image_labels()).to(outs[0].device)
        from .. import types
        if getattr(self.loader, "_last_batch_policy", None) == types.LAST_BATCH_PARTIAL:
            valid = self.loader._batch_size - self.loader.get_last_batch_padded_size()
            if valid < self.loader._batch_size:
                return [o[:valid] for o in outs], labels[:valid]
        return outs, labels

    next = __next__

    def reset(self):
        self.loader.reset()


# ---- the head of a training or serving step, on the batches above -----------------------------------
# Float16 and bfloat16 CUDA tensors; differentiable by torch.autograd, once (create_graph is refused, and so are the tangents of
# forward-mode differentiation). Everything runs on the tensors' device, on its current stream. The calls are C++ functions, not
# registered operators: torch.compile breaks its graph at them, and dispatch modes and the functions of tensor subclasses do not see
# them.
#
# Waits inside the kernels are bounded (about a second, longer for long sums); one that runs out leaves its results unfinished. The next of these
# calls then raises Rb200Error, and check_unfinished() does so behind the last one.
_head = None


def _binding():
    global _head
    if _head is None:
        from .._torch import head
        _head = head
    return _head


def linear(x, weight, bias=None, residual=None, activation="none"):
    """act(x weight^T + bias) + residual, the matrix product with its epilogue in one kernel: a projection of image
    patches with their position table, a hidden layer or the scores of a classifier.

    x [..., k]; weight [m, k]; bias [m]; residual: the trailing dimensions of the result, repeated over the leading ones
    (a position table [196, m] for x [images, 196, k]), or for a matrix x a matrix whose row count divides that of x;
    activation "none", "relu", "gelu" (with the error function) or "silu". All float16 or all bfloat16; sums in 32 bits, one
    rounding at the end. Returns [..., m]."""
    return (_head or _binding()).linear(x, weight, bias, residual, activation)


def linear_cross_entropy(x, weight, labels, bias=None, ignore_index=-100, label_smoothing=0.0, reduction="mean"):
    """Softmax cross entropy of the scores x weight^T + bias against class indices, without keeping the scores: forward
    and backward pass make them piece by piece. For the labels of the iterators above, of Pipeline.get_image_labels() and of
    the box encoder (the anchors' classes, int32).

    x [..., k] and weight [v, k], bias [v]: all float16 or all bfloat16; labels [...]: int32 or int64. Rows whose label is
    ignore_index (samples that pad the last batch, anchors that matched nothing) have loss 0 and take no part in any
    gradient, whatever their features hold; any other label outside 0 .. v-1 makes the row's loss NaN. A class is masked by
    a bias of -inf or of the type's lowest value. reduction "mean" (over the rows that count; 0 if none does), "sum" or
    "none" (the shape of labels). The loss is float32."""
    return (_head or _binding()).linear_cross_entropy(x, weight, labels, bias, ignore_index, label_smoothing, reduction)


def clip_grad_norm(grads, max_norm, out=None, inv_scale=1.0):
    """The norm over all tensors of `grads` (times inv_scale, the inverse of a loss scale), and the clipping to it: every
    tensor is multiplied by inv_scale * min(1, max_norm / (norm + 1e-6)), in place or into the tensors of `out` (of the
    gradients' types, or float32 copies for a 32-bit optimiser; contiguous ones need only the same number of elements).
    Float32, float16 and bfloat16 CUDA tensors of any shapes, mixed, on one device. Returns the norm, a float32 scalar on
    the device; nothing is read back. A gradient with inf gives the norm inf and the factor 0, one with NaN gives NaN, as
    torch.nn.utils.clip_grad_norm_. An output that overlaps itself, another output or another tensor's gradients is refused."""
    return (_head or _binding()).grad_clip(grads if isinstance(grads, list) else list(grads), max_norm, out, inv_scale)


def clip_grad_norm_(parameters, max_norm, inv_scale=1.0):
    """clip_grad_norm of the parameters' gradients, in place; parameters without one are passed over."""
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else list(parameters)
    grads = [p.grad for p in parameters if p.grad is not None]
    if not grads:
        return torch.zeros((), device=parameters[0].device if parameters else "cuda")
    return clip_grad_norm(grads, max_norm, inv_scale=inv_scale)


def check_unfinished():
    """Waits for the current device and raises Rb200Error if a call of this section gave up on a bounded wait since the last
    of these calls: its results, and what was made from them, are unfinished."""
    torch.cuda.synchronize()
    (_head or _binding()).check_unfinished()
