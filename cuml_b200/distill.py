"""Distillation: a teacher's best scores, and losses that train a small network on them.

A large forest can be compressed into a small network by training that on the forest's answers.
These operators take a teacher's scores over classes (a forest's probabilities, or the logits of any other
model), keep the `k` best classes of each row, and compute the loss of a student and its gradient:

    top_scores                 the k best scores of each row, their classes, the row's log-sum-exp
    distillation_loss          T^2 KL(teacher || student) from the student's logits
    cross_entropy              softmax cross entropy from the student's logits
    linear_cross_entropy       softmax cross entropy from the last linear layer, logits not kept
    linear_distillation_loss   distillation_loss from the last linear layer, logits not kept

`ForestInference.predict_top`, `.teach` and `.distillation_loss` call them with a forest as the teacher.
All tensors are CUDA tensors of one device; work is enqueued on torch's current stream of that device and
nothing waits.  The losses have first derivatives by the logits, or by the layer's input and weight (backward mode
only: second and forward-mode derivatives are errors); the teacher's values are constants.  Calls and their gradients can be captured into CUDA graphs once they have run on
the device (as everywhere in torch, while no autograd graph of the same leaves from outside the capture is
alive).  All computation happens in libb2fil.so.
"""
from __future__ import annotations

import ctypes as C
import warnings
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from .fil import _lib

MOST_TOP = 256  # largest k
_TYPES = {torch.float32: 0, torch.float64: 1, torch.bfloat16: 2, torch.float16: 3}
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_TAILS = ("renormalise", "bucket")
_NO_CLASS = -(1 << 62)


class TopScores(NamedTuple):
    """The best scores of each row (see `top_scores`); `logsumexp` may be None."""
    values: torch.Tensor
    index: torch.Tensor
    logsumexp: Optional[torch.Tensor]


class CTeacher(C.Structure):
    """`b2fil_teacher`."""
    _fields_ = [("values", C.c_void_p), ("index", C.c_void_p), ("logsumexp", C.c_void_p),
                ("values_stride", C.c_int64), ("index_stride", C.c_int64), ("ignore", C.c_int64),
                ("k", C.c_int32), ("index64", C.c_int32)]


_call = None  # the compiled call path; False: not available


def _native():
    """The compiled call path (csrc/torch_call.cpp), or False where it was not built for the installed
    torch: the same calls then go through ctypes, slower by tens of microseconds."""
    global _call
    if _call is None:
        try:
            module = _lib.torch_module()
        except (ImportError, OSError) as e:
            warnings.warn(f"distillation calls take longer than they need: {e}", RuntimeWarning, stacklevel=3)
            _call = False
            return _call
        lib = _lib.load()
        module.bind(*(C.cast(getattr(lib, "b2fil_" + name), C.c_void_p).value for name in (
            "last_error", "top_scores_workspace", "top_scores", "distill_loss_workspace", "distill_loss",
            "distill_loss_grad", "linear_loss_workspace", "linear_loss", "linear_loss_grad_workspace",
            "linear_loss_grad")))
        _call = module
    return _call


def _answer(out):
    """What the compiled path returned, an error code raised."""
    if type(out) is int:
        _lib.check(out)
    return out


def _cuda(name, x, dtypes, ndim=None):
    if not isinstance(x, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(x).__name__}")
    if not x.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device, it is on {x.device}")
    if x.dtype not in dtypes:
        raise ValueError(f"{name} must be one of {', '.join(str(d) for d in dtypes)}, got {x.dtype}")
    if ndim is not None and x.ndim != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, got shape {tuple(x.shape)}")


def _rows(x):
    """`x` with unit stride within its rows and rows that do not overlap."""
    if x.stride(1) != 1 and x.shape[1] > 1 or x.stride(0) < x.shape[1] and x.shape[0] > 1:
        x = x.contiguous()
    return x


def _step(x):
    """Elements from one row to the next (a single row's stride says nothing)."""
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _temperature(t):
    t = float(t)
    if not 1e-6 <= t <= 1e6:
        raise ValueError(f"temperature must be between 1e-6 and 1e6, got {t}")
    return t


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(n_bytes, device):
    if n_bytes < 0:
        _lib.check(int(n_bytes))
    return torch.empty(n_bytes, dtype=torch.uint8, device=device)


def top_scores(scores, k: int, *, temperature: float = 1.0, probabilities: bool = False) -> TopScores:
    """The `k` largest of each row of `scores` (..., n_classes), fp32, fp64, bf16 or fp16.

    Returns `TopScores`: `values` (..., k) of the scores' type in descending order, equal ones in the
    order of their classes, NaN above everything; their classes as `index` (..., k) int32; and
    `logsumexp` (...), log sum exp(score / temperature) over the whole row (fp32, of fp64 scores fp64).
    With `probabilities` the logarithms of the scores take the scores' place in `values` and
    `logsumexp`: what a distillation loss takes as a forest's logits.  1 <= k <= min(n_classes, 256).
    The outputs are constants to autograd."""
    temperature = _temperature(temperature)
    call = _native() if isinstance(scores, torch.Tensor) and scores.is_cuda else False
    if call and (out := _answer(call.top_scores(scores, int(k), temperature, probabilities))) is not None:
        return TopScores(*out)
    _cuda("scores", scores, _TYPES)
    if scores.ndim < 1:
        raise ValueError("scores must have at least one dimension")
    shape, n_cols, k = scores.shape[:-1], scores.shape[-1], int(k)
    if not 1 <= k <= min(n_cols, MOST_TOP):
        raise ValueError(f"k must be between 1 and min(n_classes, {MOST_TOP}) = {min(n_cols, MOST_TOP)}, got {k}")
    x = scores.detach()
    x = _rows(x if x.ndim == 2 else x.reshape(-1, n_cols))
    n, dev = x.shape[0], x.device
    values = torch.empty((n, k), dtype=x.dtype, device=dev)
    index = torch.empty((n, k), dtype=torch.int32, device=dev)
    lse = torch.empty((n,), dtype=torch.float64 if x.dtype == torch.float64 else torch.float32, device=dev)
    if n:
        lib, kind = _lib.load(), _TYPES[x.dtype]
        ws = _workspace(lib.b2fil_top_scores_workspace(kind, n, n_cols, k, dev.index), dev)
        _lib.check(lib.b2fil_top_scores(kind, x.data_ptr(), n, n_cols, x.stride(0), k, bool(probabilities),
                                        temperature, values.data_ptr(), index.data_ptr(), lse.data_ptr(),
                                        ws.data_ptr(), ws.numel(), dev.index, _stream(dev)))
    if len(shape) != 1:
        values, index, lse = values.view(*shape, k), index.view(*shape, k), lse.view(shape)
    return TopScores(values, index, lse)


class _Teacher:
    """The teacher's tensors of one call, checked, and the structure that points at them."""

    def __init__(self, n, dev, values, index, lse, ignore=_NO_CLASS):
        self.tensors = (values, index, lse)  # kept while the structure is in use
        self.c = CTeacher(values.data_ptr() if values is not None else None, index.data_ptr(),
                          lse.data_ptr() if lse is not None else None,
                          values.stride(0) if values is not None else 0, index.stride(0), ignore, index.shape[1],
                          index.dtype == torch.int64)


def _top(top, n, dev, tail):
    """(values fp32, index, logsumexp fp32 or None) of `top` for n rows, checked."""
    if tail not in _TAILS:
        raise ValueError(f"tail must be one of {_TAILS}, got {tail!r}")
    if not isinstance(top, (tuple, list)) or len(top) not in (2, 3):
        raise TypeError("the teacher must be a TopScores, or (values, index[, logsumexp])")
    values, index, lse = (*top, None) if len(top) == 2 else top
    _cuda("the teacher's values", values, _TYPES)
    _cuda("the teacher's index", index, (torch.int32, torch.int64))
    if values.ndim < 1 or values.shape != index.shape:
        raise ValueError(f"the teacher's values and index differ in shape: {tuple(values.shape)}, {tuple(index.shape)}")
    k = values.shape[-1]
    if not 1 <= k <= MOST_TOP:
        raise ValueError(f"the teacher's k must be between 1 and {MOST_TOP}, got {k}")
    values, index = values.detach().reshape(-1, k), index.reshape(-1, k)
    if values.shape[0] != n:
        raise ValueError(f"the teacher has {values.shape[0]} rows, the student {n}")
    if tail == "bucket":
        if lse is None:
            raise ValueError("tail='bucket' needs the teacher's logsumexp")
        _cuda("the teacher's logsumexp", lse, _TYPES)
        if lse.numel() != n:
            raise ValueError(f"the teacher's logsumexp has {lse.numel()} rows, the student {n}")
        lse = lse.detach().reshape(-1).float().contiguous()
    else:
        lse = None
    for t in (values, index, lse):
        if t is not None and t.device != dev:
            raise ValueError(f"the teacher is on {t.device}, the student on {dev}")
    return _rows(values.float()), _rows(index), lse


def _saved(x, like):
    """A saved tensor as the kernels read it: hooks may have given back another one."""
    if (x.shape, x.dtype, x.device) != like:
        raise RuntimeError("a hook gave back another tensor than the distillation loss had saved")
    return _rows(x.detach())


def _upstream(g):
    """(fp32 gradient by the loss, elements from one row's to the next)."""
    g = g if g.dtype == torch.float32 else g.float()
    return g, (g.stride(0) if g.ndim else 0)


def _reduction(reduction):
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be one of {tuple(_REDUCTIONS)}, got {reduction!r}")
    return _REDUCTIONS[reduction]


class _Loss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, values, index, lse, temperature, ignore, reduction):
        lib, kind, dev = _lib.load(), _TYPES[logits.dtype], logits.device
        x = _rows(logits)
        n, n_cols = x.shape
        t = _Teacher(n, dev, values, index, lse, ignore)
        k = t.c.k
        ws = _workspace(lib.b2fil_distill_loss_workspace(kind, n, n_cols, k, dev.index), dev)
        # kept for the gradient: statistics and the factor; the named classes' probabilities and places
        kept = torch.empty((4 * n + 4 + 2 * n * k,), dtype=torch.float32, device=dev)
        rows = torch.empty((n,), dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev) if reduction else rows
        stats, factor, named = _kept(kept, n)
        _lib.check(lib.b2fil_distill_loss(
            kind, x.data_ptr(), n, n_cols, x.stride(0), C.byref(t.c), temperature, reduction, rows.data_ptr(), stats, named,
            named + 4 * n * k, loss.data_ptr(), factor if reduction else None, ws.data_ptr(), ws.numel(), dev.index,
            _stream(dev)))
        ctx.save_for_backward(logits)
        ctx.like = (logits.shape, logits.dtype, logits.device)
        ctx.kept, ctx.options = kept, (temperature, reduction, k)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        (logits,) = ctx.saved_tensors
        temperature, reduction, k = ctx.options
        lib, kind, dev = _lib.load(), _TYPES[logits.dtype], logits.device
        x = _saved(logits, ctx.like)
        n, n_cols = x.shape
        grad = torch.empty((n, n_cols), dtype=x.dtype, device=dev)
        g, stride = _upstream(g)
        stats, factor, named = _kept(ctx.kept, n)
        _lib.check(lib.b2fil_distill_loss_grad(
            kind, x.data_ptr(), n, n_cols, x.stride(0), k, temperature, stats, named, named + 4 * n * k, g.data_ptr(), stride,
            factor if reduction else None, grad.data_ptr(), n_cols, dev.index, _stream(dev)))
        return grad, None, None, None, None, None, None


def _kept(kept, n):
    """Addresses of the statistics, the factor and the named classes' arrays in what a forward pass keeps."""
    at = kept.data_ptr()
    return at, at + 16 * n, at + 16 * n + 16


_STUDENT = (torch.float32, torch.bfloat16, torch.float16)


def _columns(index):
    """Classes (n,) or (n, k) as (n, k)."""
    return index.unsqueeze(1) if index.ndim == 1 else index


def _loss(x, values, index, lse, temperature, reduction, ignore=_NO_CLASS, compiled_only=False):
    call = _native() if isinstance(x, torch.Tensor) and x.is_cuda else False
    if call:
        out = _answer(call.distill_loss(x, values, index, lse, temperature, ignore, reduction))
        if out is not None:
            return out
    if compiled_only:
        return None
    return _Loss.apply(x, values, _columns(index), lse, temperature, ignore, reduction)


def distillation_loss(logits, top, *, temperature: float = 1.0, tail: str = "renormalise", reduction: str = "mean"):
    """T^2 KL(teacher || softmax(logits / T)) over the classes that the teacher names.

    logits : (..., n_classes) fp32, bf16 or fp16; rows whose logits are all -inf do not count.
    top : `TopScores`, or (values, index[, logsumexp]) with values and index of shape (..., k), k <= 256.
        Entries whose class is outside [0, n_classes) do not count, a class that is named twice has the sum of its
        probabilities; rows without an entry do not count (but with tail='bucket', see there).
    tail : what becomes of the classes that the teacher does not name.  'renormalise': nothing, the named ones'
        probabilities are scaled to a sum of 1.  'bucket': together they are one more class on both sides;
        this takes the teacher's `logsumexp` over all its classes at the same temperature, and at most 2^20 classes.
        Less than 2^-20, or 2^-22 of the log-sum-exp's size, counts as nothing: what 32 bits of that leave.  A row without an
        entry has all of the teacher's mass there: it counts, with a loss of 0, unless its `logsumexp` is -inf (to be
        given to rows of padding).
    reduction : 'mean' over the rows that count (0 where none does), 'sum', or 'none': (...), 0 for others.

    The loss is fp32, the gradient by the logits has their type."""
    if (reduction in _REDUCTIONS and tail in _TAILS and type(top) is TopScores and top.values is not None
            and (tail != "bucket" or top.logsumexp is not None)):
        loss = _loss(logits, top.values, top.index, top.logsumexp if tail == "bucket" else None, _temperature(temperature),
                     _REDUCTIONS[reduction], compiled_only=True)
        if loss is not None:
            return loss
    _cuda("logits", logits, _STUDENT)
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape (..., n_classes), got {tuple(logits.shape)}")
    shape, n_cols = logits.shape[:-1], logits.shape[-1]
    x = logits if logits.ndim == 2 else logits.reshape(-1, n_cols)
    values, index, lse = _top(top, x.shape[0], x.device, tail)
    if lse is not None and n_cols > 1 << 20:
        raise ValueError(f"tail='bucket' takes at most 2^20 classes, got {n_cols}")
    loss = _loss(x, values, index, lse, _temperature(temperature), _reduction(reduction))
    return loss.view(shape) if reduction == "none" and len(shape) != 1 else loss


def cross_entropy(logits, target, *, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of `logits` (..., n_classes), fp32, bf16 or fp16, and the classes `target` (...), int32
    or int64: `distillation_loss` of a teacher that is sure.  Rows whose target is `ignore_index` or outside
    [0, n_classes), or whose logits are all -inf, do not count; reduction and types as there."""
    if reduction in _REDUCTIONS:
        loss = _loss(logits, None, target, None, 1.0, _REDUCTIONS[reduction], int(ignore_index), compiled_only=True)
        if loss is not None:
            return loss
    _cuda("logits", logits, _STUDENT)
    if logits.ndim < 1 or logits.shape[-1] < 1:
        raise ValueError(f"logits must have shape (..., n_classes), got {tuple(logits.shape)}")
    shape = logits.shape[:-1]
    target = _target(target, shape, logits.device)
    x = logits if logits.ndim == 2 else logits.reshape(-1, logits.shape[-1])
    loss = _loss(x, None, target, None, 1.0, _reduction(reduction), int(ignore_index))
    return loss.view(shape) if reduction == "none" and len(shape) != 1 else loss


def _target(target, shape, dev):
    """Classes of rows of that leading shape as (n,), checked."""
    _cuda("target", target, (torch.int32, torch.int64))
    if target.shape != shape:
        raise ValueError(f"target must have shape {tuple(shape)}, got {tuple(target.shape)}")
    if target.device != dev:
        raise ValueError(f"target is on {target.device}, the student on {dev}")
    return target.reshape(-1)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, weight, values, index, temperature, ignore, reduction):
        lib, kind, dev = _lib.load(), _TYPES[hidden.dtype], hidden.device
        (n, width), n_cols = hidden.shape, weight.shape[0]
        t = _Teacher(n, dev, values, index, None, ignore)
        k = t.c.k
        layer = (hidden.data_ptr(), _step(hidden), weight.data_ptr(), _step(weight), n, n_cols, width)
        ws = _workspace(lib.b2fil_linear_loss_workspace(kind, *layer, k, dev.index), dev)
        # kept for the gradient: statistics and the factor; the named classes' logits, probabilities and places
        kept = torch.empty((4 * n + 4 + 3 * n * k,), dtype=torch.float32, device=dev)
        rows = torch.empty((n,), dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev) if reduction else rows
        stats, factor, named = _kept(kept, n)
        _lib.check(lib.b2fil_linear_loss(
            kind, *layer, C.byref(t.c), temperature, reduction, rows.data_ptr(), stats, named, named + 4 * n * k, named + 8 * n * k,
            loss.data_ptr(), factor if reduction else None, ws.data_ptr(), ws.numel(), dev.index, _stream(dev)))
        ctx.save_for_backward(hidden, weight)
        ctx.like = [(x.shape, x.dtype, x.device) for x in (hidden, weight)]
        ctx.kept, ctx.options = kept, (temperature, reduction, k)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        hidden, weight = map(_saved, ctx.saved_tensors, ctx.like)
        temperature, reduction, k = ctx.options
        lib, kind, dev = _lib.load(), _TYPES[hidden.dtype], hidden.device
        (n, width), n_cols = hidden.shape, weight.shape[0]
        of_hidden, of_weight = ctx.needs_input_grad[:2]
        dh = torch.empty((n, width), dtype=hidden.dtype, device=dev) if of_hidden else None
        dw = torch.empty((n_cols, width), dtype=hidden.dtype, device=dev) if of_weight else None
        layer = (hidden.data_ptr(), _step(hidden), weight.data_ptr(), _step(weight), n, n_cols, width)
        ws = _workspace(lib.b2fil_linear_loss_grad_workspace(kind, *layer, k, of_hidden, of_weight, dev.index), dev)
        g, stride = _upstream(g)
        stats, factor, named = _kept(ctx.kept, n)
        _lib.check(lib.b2fil_linear_loss_grad(
            kind, *layer, k, temperature, stats, named, named + 4 * n * k, named + 8 * n * k, g.data_ptr(), stride,
            factor if reduction else None, dh.data_ptr() if of_hidden else None, dw.data_ptr() if of_weight else None,
            ws.data_ptr(), ws.numel(), dev.index, _stream(dev)))
        return dh, dw, None, None, None, None, None


_LAYER = (torch.bfloat16, torch.float16)


def _layer(hidden, weight):
    """(hidden (n, width), weight (n_classes, width), leading shape), checked."""
    if torch.is_autocast_enabled("cuda"):
        t = torch.get_autocast_dtype("cuda")
        hidden, weight = (x.to(t) if isinstance(x, torch.Tensor) and x.is_floating_point() else x for x in (hidden, weight))
    _cuda("hidden", hidden, _LAYER)
    _cuda("weight", weight, _LAYER, 2)
    if hidden.dtype != weight.dtype or hidden.device != weight.device:
        raise ValueError(f"hidden and weight differ in type or device: {hidden.dtype} on {hidden.device}, "
                         f"{weight.dtype} on {weight.device}")
    if hidden.ndim < 1 or hidden.shape[-1] != weight.shape[1] or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"hidden must be (..., width) and weight (n_classes, width), got {tuple(hidden.shape)} and "
                         f"{tuple(weight.shape)}")
    shape, width = hidden.shape[:-1], weight.shape[1]
    if hidden.ndim != 2:
        hidden = hidden.reshape(-1, width)
    return _rows(hidden), _rows(weight), shape


def _linear(hidden, weight, values, index, temperature, ignore, reduction, compiled_only=False):
    # (compiled_only: the layer as the caller gave it, which autocast may have to cast)
    call = _native() if isinstance(hidden, torch.Tensor) and hidden.is_cuda else False
    if call:
        out = _answer(call.linear_loss(hidden, weight, values, index, temperature, ignore, reduction, not compiled_only))
        if out is not None:
            return out
    if compiled_only:
        return None
    return _Linear.apply(hidden, weight, values, _columns(index), temperature, ignore, reduction)


def linear_cross_entropy(hidden, weight, target, *, ignore_index: int = -100, reduction: str = "mean"):
    """Softmax cross entropy of the logits `hidden @ weight.T` and `target`, without keeping the logits.

    hidden : (..., width), weight : (n_classes, width), both bf16 or both fp16 (under autocast they are cast).
    target : (...) int32 or int64 classes; rows whose target is `ignore_index` or outside [0, n_classes) do
        not count (their hidden values must be finite: they take part in weight's gradient with zeros).
    reduction : 'mean' over the rows that count (0 where none does), 'sum', or 'none': (...), 0 for others.

    The loss is fp32; products are summed in fp32.  The gradients have the layer's type; the
    differences softmax - target are rounded to it before they are multiplied (small layers: to two numbers of
    it).  Waits inside the kernels are bounded; `check_status` tells whether one ran out, and until it has,
    losses and gradients are NaN."""
    if reduction in _REDUCTIONS:
        loss = _linear(hidden, weight, None, target, 1.0, int(ignore_index), _REDUCTIONS[reduction], compiled_only=True)
        if loss is not None:
            return loss
    hidden, weight, shape = _layer(hidden, weight)
    target = _target(target, shape, hidden.device)
    loss = _linear(hidden, weight, None, target, 1.0, int(ignore_index), _reduction(reduction))
    return loss.view(shape) if reduction == "none" and len(shape) != 1 else loss


def linear_distillation_loss(hidden, weight, top, *, temperature: float = 1.0, reduction: str = "mean"):
    """`distillation_loss` (with tail='renormalise') of the logits `hidden @ weight.T`, without keeping them.

    hidden : (..., width), weight : (n_classes, width), both bf16 or both fp16 (under autocast they are cast).
    top, temperature, reduction : as in `distillation_loss`; types, rounding and waits as in
    `linear_cross_entropy`."""
    if reduction in _REDUCTIONS and type(top) is TopScores and top.values is not None:
        loss = _linear(hidden, weight, top.values, top.index, _temperature(temperature), _NO_CLASS, _REDUCTIONS[reduction],
                       compiled_only=True)
        if loss is not None:
            return loss
    hidden, weight, shape = _layer(hidden, weight)
    values, index, _ = _top(top, hidden.shape[0], hidden.device, "renormalise")
    loss = _linear(hidden, weight, values, index, _temperature(temperature), _NO_CLASS, _reduction(reduction))
    return loss.view(shape) if reduction == "none" and len(shape) != 1 else loss


def check_status(device=None) -> None:
    """Wait for all work on `device` and raise `B2FilError` (code -7) if a bounded wait inside a kernel of the
    linear losses ran out since the last check.  The losses and gradients that follow such a wait are NaN until
    then, as nothing in a stream-ordered call can raise; where a linear loss is NaN, ask here first."""
    device = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    word = C.c_int32(0)
    index = torch.cuda.current_device() if device.index is None else device.index
    _lib.check(_lib.load().b2fil_distill_status(index, C.byref(word)))
