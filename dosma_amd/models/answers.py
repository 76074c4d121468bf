"""What a network's answers say: log probabilities of given labels, entropy, the best alternatives, and the divergence from
a teacher's stored answers -- with the gradients of all of them.

The reference keeps the thresholded masks of ``model.predict`` (``dosma/models/oaiunet2d.py:305-316``) and nothing else of
the answer.  These functions read the category scores (logits) themselves, one softmax per row (voxel, token, ...):
``p = softmax(z / temperature)`` over the classes.  ``background=True`` puts an implicit category 0 of score 0 in front
(category = class + 1): for the models of this package, whose classes have sigmoid heads, that is the distribution of the
label under the condition that a voxel carries at most one tissue.

``logits`` is a torch tensor on the GPU (float32, float16 or bfloat16, any strides; the work is enqueued on torch's current
stream of that device and nothing waits for it) or a numpy array (float16 / float32; other floats are converted), whose
results are numpy arrays.  ``dim`` is the class axis: -1 for rows, 1 for the (B, C, H, W) answers of a torch network.  The
per-row arguments and results have the shape of ``logits`` without that axis.

A score of -inf is a category that is not offered: probability 0, never an alternative.  A row of nothing but -inf has log
probability -inf, entropy 0, no alternatives, loss 0 and gradient 0.  NaN or +inf makes the row's results NaN.

Calls on tensors can be captured into a graph, their gradients as well; as with every backward pass in torch, no eager graph of
the same leaves may be alive while one is captured (a leaf's accumulation stays on the stream that it was first used on).  Derivatives are reverse mode and first order; tensors
with a forward-mode tangent are refused."""
import sys
from collections import namedtuple

import numpy as np

from dosma_amd import _hostpool, _lib

__all__ = ["LabelScores", "DistillLoss", "label_scores", "label_scores_grad", "distill_loss", "distill_loss_grad"]

#: ``log_prob`` (None without labels), ``entropy`` in nats, ``norm`` (..., 2): the row maximum M and ln sum exp((z - M) / T),
#: which the gradient needs (M / T + norm[..., 1] is log sum exp(z / T)); None unless asked for or needed by a gradient;
#: ``top_log_prob`` / ``top_label`` (..., top) or None
LabelScores = namedtuple("LabelScores", "log_prob entropy norm top_log_prob top_label")
#: ``loss`` in nats, ``norm`` as above, ``log_tail``: log probability outside the teacher's entries (None without the tail); both
#: None unless ``norm`` is asked for or a gradient needs them
DistillLoss = namedtuple("DistillLoss", "loss norm log_tail")


def _is_torch(x):
    torch = sys.modules.get("torch")
    return torch is not None and isinstance(x, torch.Tensor)


def _check_dim(ndim, dim):
    if ndim < 1:
        raise ValueError("logits need a class axis")
    if not -ndim <= dim < ndim:
        raise ValueError(f"dim={dim} is not an axis of {ndim}-dimensional logits")
    return dim % ndim


def _rows_of(shape, strides, dim, beside=None):
    """-> (row shape, Rows), or (row shape, None) where the rows need more than two strides.

    ``beside``: the strides of another tensor of this shape.  Its rows are counted together with these (one ``inner`` for both), so
    two axes are merged only where both tensors allow it; -> (row shape, Rows, Rows of the other), None for both where that takes
    more than two groups."""
    groups, rows = [], 1  # (length, stride, the other's stride)
    for i, n in enumerate(shape):
        if i == dim:
            continue
        rows *= n
        if n == 1:
            continue
        st, other = strides[i], 0 if beside is None else beside[i]
        if groups and groups[-1][1] == st * n and groups[-1][2] == other * n:
            groups[-1] = (groups[-1][0] * n, st, other)
        else:
            groups.append((n, st, other))
    row_shape = tuple(shape[:dim]) + tuple(shape[dim + 1:])
    C = shape[dim]

    def geometry(strides, at):
        sc = strides[dim] if C > 1 else 1
        if rows == 0 or not groups:
            return _lib.Rows(rows, C, 1, 0, C, sc)
        if len(groups) == 1:
            return _lib.Rows(rows, C, groups[0][0], 0, groups[0][at], sc)
        if len(groups) == 2:
            return _lib.Rows(rows, C, groups[1][0], groups[0][at], groups[1][at], sc)
        return None

    if beside is None:
        return row_shape, geometry(strides, 1)
    return row_shape, geometry(strides, 1), geometry(beside, 2)


# ---- torch ---------------------------------------------------------------------------------------------------------------
_names = {}  # torch dtype -> "float32", ..


def _name(dtype):
    name = _names.get(dtype)
    if name is None:
        name = _names[dtype] = str(dtype)[6:]
    return name


def _no_tangent(name, t):
    # (a dual tensor does not require gradients, so the derivative asked for would come back as none, which reads as zero)
    ad = sys.modules["torch"].autograd.forward_ad
    if getattr(ad, "_current_level", 0) >= 0 and ad.unpack_dual(t).tangent is not None:  # (the level: a tenth of the time of the question)
        raise ValueError(f"{name}: forward-mode derivatives are not offered")


def _tensor_logits(x, dim):
    """-> (scores, axis, shape of the rows, Rows); a copy of the scores where their rows need more than two strides."""
    if not x.is_cuda:
        raise ValueError("logits must be a tensor on the GPU or a numpy array")
    if _name(x.dtype) not in _lib.SCORE_DTYPES:
        raise ValueError(f"logits must be float32, float16 or bfloat16, got {x.dtype}")
    _no_tangent("logits", x)
    if x.is_neg():  # (``c.conj().imag``: the memory holds the values with the other sign)
        x = x.resolve_neg()
    ndim = x.ndim
    dim = _check_dim(ndim, dim)
    if dim == ndim - 1 and x.is_contiguous():
        C = x.shape[dim]
        return x, dim, x.shape[:-1], _lib.Rows(x.numel() // C if C else 0, C)
    shape, rows = _rows_of(x.shape, x.stride(), dim)
    if rows is None:
        x = x.contiguous()
        shape, rows = _rows_of(x.shape, x.stride(), dim)
    return x, dim, shape, rows


def _tensor_arg(name, t, shape, device, dtypes, last=()):
    """A per-row argument, dense.  ``last``: its extra last axis."""
    if not _is_torch(t):
        raise ValueError(f"{name} must be a tensor like the logits")
    if t.shape != shape + last:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape + last)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the logits are on {device}")
    if _name(t.dtype) not in dtypes:
        raise ValueError(f"{name} must be one of {', '.join(sorted(dtypes))}, got {t.dtype}")
    if t.is_floating_point():
        _no_tangent(name, t)
        if t.is_neg():
            t = t.resolve_neg()
    return t if t.is_contiguous() else t.contiguous()


_F32 = ("float32",)


def _ptr(t):
    return None if t is None else t.data_ptr()


class _TorchCall:
    """Results and workspace from torch's allocator, work on torch's current stream of the logits' device."""

    __slots__ = ("torch", "device", "index", "stream", "held")

    def __init__(self, x):
        self.torch = torch = sys.modules["torch"]
        self.device = x.device
        self.index = x.get_device()
        self.stream = torch._C._cuda_getCurrentRawStream(self.index)

    # (new_empty and empty_like take half the time of torch.empty with a device, and small calls are bound by such things)
    def empty(self, x, shape):
        return x.new_empty(shape, dtype=self.torch.float32)

    def like(self, t, dtype=None):
        return self.torch.empty_like(t) if dtype is None else self.torch.empty_like(t, dtype=dtype)

    def workspace(self, nbytes):
        # kept until the call is enqueued; torch's allocator hands it out again only to work behind this on the same stream
        self.held = self.torch.empty(nbytes, dtype=self.torch.uint8, device=self.device)
        return self.held.data_ptr()

    def grad_like(self, x, dim, rows):
        """-> (scores, their Rows, gradient, its Rows); ``rows``: those of the scores alone.  The gradient has the layout of the
        scores, or dense rows where the two cannot be walked through together in that; the scores are copied where not even these
        can."""
        g = self.torch.empty_like(x)
        if x.is_contiguous():
            return x, rows, g, rows
        rows, grad_rows = self._together(x, g, dim)
        if rows is None:
            g = self.torch.empty(x.shape, dtype=x.dtype, device=x.device)
            rows, grad_rows = self._together(x, g, dim)
        if rows is None:
            x = x.contiguous()
            rows, grad_rows = self._together(x, g, dim)
        return x, rows, g, grad_rows

    @staticmethod
    def _together(x, g, dim):
        if any(st == 0 and n > 1 for n, st in zip(g.shape, g.stride())):
            return None, None
        return _rows_of(x.shape, x.stride(), dim, g.stride())[1:]


def _scores_tensor(x, labels, dim, top, norm, temperature, background, ignore_label):
    x, dim, shape, rows = _tensor_logits(x, dim)
    call = _TorchCall(x)
    l_dtype = None
    if labels is not None:
        labels = _tensor_arg("labels", labels, shape, x.device, _lib.L_KINDS)
        l_dtype = _name(labels.dtype)
    entropy = call.empty(x, shape)
    top_log_prob = call.empty(x, shape + (top,)) if top > 0 else None
    out = LabelScores(None if labels is None else call.like(entropy), entropy, call.empty(x, shape + (2,)) if norm else None,
                      top_log_prob, call.like(top_log_prob, call.torch.int32) if top > 0 else None)
    _lib.label_scores(x.data_ptr(), _name(x.dtype), rows, labels_ptr=_ptr(labels), l_dtype=l_dtype, top=top,
                      ignore_label=ignore_label, temperature=temperature, background=background, log_prob=_ptr(out.log_prob),
                      entropy=_ptr(out.entropy), norm=_ptr(out.norm), top_log_prob=_ptr(out.top_log_prob),
                      top_label=_ptr(out.top_label), device=call.index, stream=call.stream, workspace=call.workspace)
    return out


def _scores_grad_tensor(x, labels, norm, grad_log_prob, entropy, grad_entropy, dim, temperature, background, ignore_label):
    x, dim, shape, rows = _tensor_logits(x, dim)
    call = _TorchCall(x)
    dev = x.device
    l_dtype = None
    if labels is not None:
        labels = _tensor_arg("labels", labels, shape, dev, _lib.L_KINDS)
        l_dtype = _name(labels.dtype)
    norm = _tensor_arg("norm", norm, shape, dev, _F32, (2,))
    if grad_log_prob is not None:
        grad_log_prob = _tensor_arg("grad_log_prob", grad_log_prob, shape, dev, _F32)
    if grad_entropy is not None:
        grad_entropy = _tensor_arg("grad_entropy", grad_entropy, shape, dev, _F32)
        if entropy is not None:
            entropy = _tensor_arg("entropy", entropy, shape, dev, _F32)
    else:
        entropy = None
    x, rows, grad, grad_rows = call.grad_like(x, dim, rows)
    _lib.label_scores_grad(x.data_ptr(), _name(x.dtype), rows, grad.data_ptr(), grad_rows, norm.data_ptr(), labels_ptr=_ptr(labels),
                           l_dtype=l_dtype, ignore_label=ignore_label, temperature=temperature, background=background,
                           entropy=_ptr(entropy), grad_log_prob=_ptr(grad_log_prob), grad_entropy=_ptr(grad_entropy),
                           device=call.index, stream=call.stream)
    return grad


def _teacher_tensors(top_label, values, shape, device):
    last = (top_label.shape[-1] if _is_torch(top_label) and top_label.ndim else 0,)
    return (_tensor_arg("top_label", top_label, shape, device, ("int32", "int64"), last),
            _tensor_arg("values", values, shape, device, _lib.SCORE_DTYPES, last))


def _distill_tensor(x, top_label, values, dim, norm, temperature, tail, background):
    x, dim, shape, rows = _tensor_logits(x, dim)
    call = _TorchCall(x)
    lab, val = _teacher_tensors(top_label, values, shape, x.device)
    loss = call.empty(x, shape)
    out = DistillLoss(loss, call.empty(x, shape + (2,)) if norm else None, call.like(loss) if norm and tail else None)
    _lib.distill(x.data_ptr(), _name(x.dtype), rows, lab.data_ptr(), _name(lab.dtype), val.data_ptr(), _name(val.dtype),
                 lab.shape[-1], tail=tail, temperature=temperature, background=background, loss=out.loss.data_ptr(),
                 norm=_ptr(out.norm), log_tail=_ptr(out.log_tail), device=call.index, stream=call.stream, workspace=call.workspace)
    return out


def _distill_grad_tensor(x, top_label, values, norm, log_tail, grad_loss, dim, temperature, tail, background):
    x, dim, shape, rows = _tensor_logits(x, dim)
    call = _TorchCall(x)
    dev = x.device
    lab, val = _teacher_tensors(top_label, values, shape, dev)
    norm = _tensor_arg("norm", norm, shape, dev, _F32, (2,))
    grad_loss = _tensor_arg("grad_loss", grad_loss, shape, dev, _F32)
    if log_tail is not None:
        log_tail = _tensor_arg("log_tail", log_tail, shape, dev, _F32)
    x, rows, grad, grad_rows = call.grad_like(x, dim, rows)
    _lib.distill_grad(x.data_ptr(), _name(x.dtype), rows, grad.data_ptr(), grad_rows, lab.data_ptr(), _name(lab.dtype),
                      val.data_ptr(), _name(val.dtype), lab.shape[-1], norm.data_ptr(), grad_loss.data_ptr(),
                      log_tail=_ptr(log_tail), tail=tail, temperature=temperature, background=background, device=call.index,
                      stream=call.stream)
    return grad


_functions = {}  # the autograd functions, made when torch is first seen


def _autograd(name):
    if not _functions:
        import torch
        from torch.autograd.function import once_differentiable

        class ScoresFunction(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, labels, kw, top):
                r = _scores_tensor(x, labels, top=top, norm=True, **kw)
                ctx.kw = kw
                ctx.set_materialize_grads(False)
                ctx.mark_non_differentiable(*[t for t in r[2:] if t is not None])
                ctx.save_for_backward(x, labels, r.norm, r.entropy)
                return tuple(r)

            @staticmethod
            @once_differentiable
            def backward(ctx, g_log_prob, g_entropy, *_):
                x, labels, norm, entropy = ctx.saved_tensors
                if g_log_prob is None and g_entropy is None:
                    return None, None, None, None
                return (_scores_grad_tensor(x, labels, norm, g_log_prob, entropy, g_entropy, **ctx.kw), None, None, None)

        class DistillFunction(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x, top_label, values, kw):
                r = _distill_tensor(x, top_label, values, norm=True, **kw)
                ctx.kw = kw
                ctx.set_materialize_grads(False)
                ctx.mark_non_differentiable(*[t for t in r[1:] if t is not None])
                ctx.save_for_backward(x, top_label, values, r.norm, r.log_tail)
                return tuple(r)

            @staticmethod
            @once_differentiable
            def backward(ctx, g_loss, *_):
                x, top_label, values, norm, log_tail = ctx.saved_tensors
                if g_loss is None:
                    return None, None, None, None
                return (_distill_grad_tensor(x, top_label, values, norm, log_tail, g_loss, **ctx.kw), None, None, None)

        _functions.update(scores=ScoresFunction, distill=DistillFunction)
    return _functions[name]


def _wants_grad(x):
    return x.requires_grad and sys.modules["torch"].is_grad_enabled()


# ---- numpy ---------------------------------------------------------------------------------------------------------------
def _array_logits(x, dim):
    x = np.asarray(x)
    if x.dtype.kind != "f":
        raise ValueError(f"logits must be floating point, got {x.dtype}")
    dim = _check_dim(x.ndim, dim)
    x = np.ascontiguousarray(np.moveaxis(x, dim, -1), dtype=np.float16 if x.dtype == np.float16 else np.float32)
    return x, dim, x.shape[:-1], _lib.Rows(int(np.prod(x.shape[:-1], dtype=np.int64)), x.shape[-1])


def _array_arg(name, a, shape, dtypes, last=None):
    a = np.asarray(a)
    a = np.asarray(a, dtype=a.dtype.newbyteorder("="), order="C")  # (one row: no axis; ascontiguousarray would add one)
    want = tuple(shape) + (() if last is None else (last,))
    if a.shape != want:
        raise ValueError(f"{name} has shape {a.shape}, expected {want}")
    if a.dtype.name not in dtypes:
        raise ValueError(f"{name} must be one of {', '.join(sorted(dtypes))}, got {a.dtype}")
    return a


def _grad_array(x, dim):
    """Dense rows for the kernel and the caller's view of them, the class axis back in its place."""
    g = _hostpool.empty(x.shape, x.dtype)
    return g, np.moveaxis(g, -1, dim)


def _address(a):
    return None if a is None else a.ctypes.data


def _scores_array(x, labels, dim, top, norm, temperature, background, ignore_label, device):
    x, dim, shape, rows = _array_logits(x, dim)
    lab = None if labels is None else _array_arg("labels", labels, shape, _lib.L_KINDS)
    out = LabelScores(None if lab is None else _hostpool.empty(shape, np.float32), _hostpool.empty(shape, np.float32),
                      _hostpool.empty(shape + (2,), np.float32) if norm else None,
                      _hostpool.empty(shape + (top,), np.float32) if top > 0 else None,
                      _hostpool.empty(shape + (top,), np.int32) if top > 0 else None)
    ptr = [_address(a) for a in out]
    _lib.label_scores(_address(x), x.dtype.name, rows, labels_ptr=_address(lab), l_dtype=None if lab is None else lab.dtype.name,
                      top=top, ignore_label=ignore_label, temperature=temperature, background=background, log_prob=ptr[0],
                      entropy=ptr[1], norm=ptr[2], top_log_prob=ptr[3], top_label=ptr[4], host=True, device=device)
    return out


def label_scores(logits, labels=None, *, dim=-1, top=0, norm=False, temperature=1.0, background=False, ignore_label=-1,
                 device=None):
    """Log probability of the given ``labels``, entropy and the ``top`` best categories of every row -> :class:`LabelScores`.

    ``labels``: int32 / uint8 / int16 / int64 categories; rows with ``ignore_label`` have none (log_prob 0), any other value
    that is not a category gives NaN.  ``top`` (0 .. 64, at most the number of categories): alternatives in falling order,
    ties to the lower category; label -1 with log probability -inf where fewer are offered.  ``norm=True``: also what
    :func:`label_scores_grad` needs.  Tensors that require gradients: ``log_prob`` and ``entropy`` are differentiable (first
    order), the alternatives are not.  ``device``: of numpy calls."""
    top = int(top)
    if not 0 <= top <= _lib.MAX_TOP:
        raise ValueError(f"top must be 0 .. {_lib.MAX_TOP}, got {top}")
    kw = dict(dim=dim, temperature=temperature, background=background, ignore_label=ignore_label)
    if not _is_torch(logits):
        return _scores_array(logits, labels, top=top, norm=norm, device=device, **kw)
    if _wants_grad(logits):
        return LabelScores(*_autograd("scores").apply(logits, labels, kw, top))
    return _scores_tensor(logits, labels, top=top, norm=norm, **kw)


def label_scores_grad(logits, labels, norm, *, grad_log_prob=None, entropy=None, grad_entropy=None, dim=-1, temperature=1.0,
                      background=False, ignore_label=-1, device=None):
    """Gradient of ``sum(grad_log_prob * log_prob + grad_entropy * entropy)`` with respect to the logits, in their type and
    layout; ``norm`` and (for ``grad_entropy``) ``entropy`` as :func:`label_scores` returned them."""
    kw = dict(dim=dim, temperature=temperature, background=background, ignore_label=ignore_label)
    if _is_torch(logits):
        return _scores_grad_tensor(logits, labels, norm, grad_log_prob, entropy, grad_entropy, **kw)
    x, dim, shape, rows = _array_logits(logits, dim)
    lab = None if labels is None else _array_arg("labels", labels, shape, _lib.L_KINDS)
    norm = _array_arg("norm", norm, shape, _F32, 2)
    rest = [None if a is None else _array_arg(n, a, shape, _F32)
            for n, a in (("entropy", entropy), ("grad_log_prob", grad_log_prob), ("grad_entropy", grad_entropy))]
    g, view = _grad_array(x, dim)
    _lib.label_scores_grad(_address(x), x.dtype.name, rows, _address(g), rows, _address(norm), labels_ptr=_address(lab),
                           l_dtype=None if lab is None else lab.dtype.name, ignore_label=ignore_label, temperature=temperature,
                           background=background, entropy=_address(rest[0]), grad_log_prob=_address(rest[1]),
                           grad_entropy=_address(rest[2]), host=True, device=device)
    return view


def _teacher_arrays(top_label, values, shape, tail):
    top_label = np.asarray(top_label)
    K = top_label.shape[-1] if top_label.ndim else 0
    values = np.asarray(values)
    if values.dtype.name == "float64":  # (of either byte order)
        values = values.astype(np.float32)
    return _array_arg("top_label", top_label, shape, ("int32", "int64"), K), _array_arg("values", values, shape, _lib.SCORE_DTYPES, K), K


def distill_loss(logits, top_label, values, *, dim=-1, norm=False, temperature=1.0, tail=False, background=False, device=None):
    """Divergence (nats, per row) of the answers ``logits`` from a teacher's best ones -> :class:`DistillLoss`.

    ``top_label`` (..., K) int32 / int64 and ``values`` (..., K), K <= 64, are the teacher's categories and either its scores
    or log probabilities (``tail=False``: the teacher is ``softmax(values / temperature)`` over the entries) or float32 log
    probabilities at this ``temperature`` (``tail=True``: the rest of its mass is compared with the student's mass outside the
    entries) -- what ``label_scores(teacher, top=K, temperature=...)`` returns.  Entries whose label is not a category (-1) are
    empty slots; a row of empty slots has loss 0.  ``norm=True``: also what :func:`distill_loss_grad` needs.  ``loss`` is
    differentiable (first order) in the student's logits."""
    kw = dict(dim=dim, temperature=temperature, tail=bool(tail), background=background)
    if _is_torch(logits):
        if _wants_grad(logits):
            return DistillLoss(*_autograd("distill").apply(logits, top_label, values, kw))
        return _distill_tensor(logits, top_label, values, norm=norm, **kw)
    x, dim, shape, rows = _array_logits(logits, dim)
    lab, val, K = _teacher_arrays(top_label, values, shape, tail)
    out = DistillLoss(_hostpool.empty(shape, np.float32), _hostpool.empty(shape + (2,), np.float32) if norm else None,
                      _hostpool.empty(shape, np.float32) if norm and tail else None)
    _lib.distill(_address(x), x.dtype.name, rows, _address(lab), lab.dtype.name, _address(val), val.dtype.name, K, tail=tail,
                 temperature=temperature, background=background, loss=_address(out.loss), norm=_address(out.norm),
                 log_tail=_address(out.log_tail), host=True, device=device)
    return out


def distill_loss_grad(logits, top_label, values, norm, *, grad_loss, log_tail=None, dim=-1, temperature=1.0, tail=False,
                      background=False, device=None):
    """Gradient of ``sum(grad_loss * loss)`` with respect to the student's logits, in their type and layout; ``norm`` and
    (with the tail) ``log_tail`` as :func:`distill_loss` returned them."""
    kw = dict(dim=dim, temperature=temperature, tail=bool(tail), background=background)
    if _is_torch(logits):
        return _distill_grad_tensor(logits, top_label, values, norm, log_tail, grad_loss, **kw)
    x, dim, shape, rows = _array_logits(logits, dim)
    lab, val, K = _teacher_arrays(top_label, values, shape, tail)
    norm = _array_arg("norm", norm, shape, _F32, 2)
    grad_loss = _array_arg("grad_loss", grad_loss, shape, _F32)
    log_tail = None if log_tail is None else _array_arg("log_tail", log_tail, shape, _F32)
    g, view = _grad_array(x, dim)
    _lib.distill_grad(_address(x), x.dtype.name, rows, _address(g), rows, _address(lab), lab.dtype.name, _address(val),
                      val.dtype.name, K, _address(norm), _address(grad_loss), log_tail=_address(log_tail), tail=tail,
                      temperature=temperature, background=background, host=True, device=device)
    return view
