"""Learning from a victim's answers: a teacher's top logits and the loss against them, as HIP kernels (csrc/nn/distil.hip).

A black-box victim answers an image with its best classes and their scores.  ``TopLogits`` holds such answers (``top_logits``
makes them from a local model's logits), ``distillation_loss`` is T^2 KL(teacher || student) on them -- the teacher's distribution
on the classes answered, and, where the mass it leaves to all others is known, on one more bin for those -- with its gradient in
the student's logits (the answers have none).  Attacks that take a loss take ``loss='distillation'`` and then answers in the place of labels
(``DistillationLoss``), as 'crossentropy' takes labels (transferattack/attack.py:155-162): untargeted, they move the surrogate away from
what the victim answered; targeted ([labels, answers]), towards it.  Those with a loss of their own, or that read class numbers, refuse it
when constructed (``Attack.takes_answers``).

No fallback: tensors must be on a HIP device."""
import operator

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _nn

FLOATS = (torch.float32, torch.bfloat16, torch.float16)
MAX_TOP = 1024
MAX_CLASSES = 458752                                     # of a student's row
MAX_ROW = 1 << 30                                        # of a teacher's
STATS = 5


class TopLogits:
    """A teacher's answers: ``values`` [rows, top] logits (fp32), ``classes`` [rows, top] (int64 or int32; -1: no answer in this
    place), ``rest`` [rows] fp32 log sum exp(logit / temperature) over all other classes -- or None: the classes answered are all
    there is -- and the ``temperature`` both sides are compared at.  Takes a batch of labels' place: ``len``, indexing by rows,
    ``repeat``, ``to``, ``clone`` and ``detach`` work as on a label tensor."""

    def __init__(self, values, classes, rest=None, temperature=1.0):
        if not (isinstance(values, torch.Tensor) and isinstance(classes, torch.Tensor) and values.dim() == 2 and classes.shape == values.shape):
            raise ValueError("values and classes must be tensors [rows, top] of one shape")
        if values.dtype != torch.float32 or classes.dtype not in (torch.int64, torch.int32):
            raise TypeError("values must be float32 and classes int64 or int32, got %s and %s" % (values.dtype, classes.dtype))
        if rest is not None and (not isinstance(rest, torch.Tensor) or rest.shape != values.shape[:1] or rest.dtype != torch.float32):
            raise ValueError("rest must be float32 [rows]")
        if classes.device != values.device or (rest is not None and rest.device != values.device):
            raise ValueError("values, classes and rest must be on one device")
        if not 2.0 ** -126 <= float(temperature) <= 2.0 ** 126:
            raise ValueError("temperature %r" % (temperature,))
        if not 1 <= values.shape[1] <= MAX_TOP:
            raise ValueError("%d classes answered (1 .. %d)" % (values.shape[1], MAX_TOP))
        self.values, self.classes, self.rest, self.temperature = values, classes, rest, float(temperature)

    @property
    def device(self):
        return self.values.device

    def _each(self, fn):
        return TopLogits(fn(self.values), fn(self.classes), None if self.rest is None else fn(self.rest), self.temperature)

    def __len__(self):
        return self.values.shape[0]

    def __getitem__(self, rows):
        if hasattr(rows, "__index__") and not isinstance(rows, (bool, torch.Tensor)):      # one row, still as a batch
            at, n = operator.index(rows), len(self)
            if not -n <= at < n:                         # (what ends an iteration)
                raise IndexError("row %d of %d" % (at, n))
            rows = slice(at % n, at % n + 1)
        return self._each(lambda t: t[rows])

    def repeat(self, times):
        return self._each(lambda t: t.repeat((times,) + (1,) * (t.dim() - 1)))

    def to(self, device):
        return self._each(lambda t: t.to(device))

    def clone(self):
        return self._each(torch.clone)

    def detach(self):
        return self._each(torch.Tensor.detach)


def _rows_of(logits, name="logits"):
    _nn.check_tensor(logits, name, None, FLOATS)
    if logits.dim() < 1 or not 1 <= logits.shape[-1]:
        raise ValueError("%s must be [..., classes], got %s" % (name, tuple(logits.shape)))
    if logits.shape[-1] > MAX_ROW:
        raise ValueError("%d classes (at most %d)" % (logits.shape[-1], MAX_ROW))
    rows = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    if rows.stride(1) != 1 and rows.shape[1] > 1 or rows.stride(0) < rows.shape[1] and rows.shape[0] > 1:
        rows = rows.contiguous()
    return rows


def _row_stride(rows):
    return rows.stride(0) if rows.shape[0] > 1 else rows.shape[1]


def top_logits(logits, top, temperature=1.0, rest=True):
    """The ``top`` largest logits of every row in falling order -- equal ones by the lowest class, NaN above all -- and, with
    ``rest``, log sum exp(logit / temperature) over the others.  logits [..., classes] in fp32, bf16 or fp16; no gradient."""
    rows = _rows_of(logits.detach() if isinstance(logits, torch.Tensor) else logits)
    if not 1 <= top <= min(rows.shape[1], MAX_TOP):
        raise ValueError("top %r of %d classes (at most %d)" % (top, rows.shape[1], MAX_TOP))
    if not 2.0 ** -126 <= float(temperature) <= 2.0 ** 126:
        raise ValueError("temperature %r" % (temperature,))
    n = rows.shape[0]
    values = torch.empty((n, top), dtype=torch.float32, device=rows.device)
    classes = torch.empty((n, top), dtype=torch.int64, device=rows.device)
    left = torch.empty(n, dtype=torch.float32, device=rows.device) if rest else None
    if n:
        _nn._launch("ta_nn_top_logits", rows, rows.data_ptr(), _nn.DTYPES[rows.dtype], _row_stride(rows), n, rows.shape[1], top,
                    float(temperature), values.data_ptr(), classes.data_ptr(), _nn.ptr(left))
    return TopLogits(values, classes, left, temperature)


def _checked(rows, answers, weight, reduction):
    if not isinstance(answers, TopLogits):
        raise TypeError("answers must be TopLogits, got %s" % type(answers).__name__)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction %r (mean, sum or none)" % (reduction,))
    _nn.check_tensor(answers.values, "answers", rows)
    if len(answers) != rows.shape[0]:
        raise ValueError("%d rows of logits, %d of answers" % (rows.shape[0], len(answers)))
    if rows.shape[1] > MAX_CLASSES:
        raise ValueError("%d classes (at most %d)" % (rows.shape[1], MAX_CLASSES))
    if weight is not None:
        _nn.check_tensor(weight, "weight", rows, (torch.float32,))
        if weight.numel() != rows.shape[0]:
            raise ValueError("weight must have %d entries, got %s" % (rows.shape[0], tuple(weight.shape)))
        if weight.requires_grad:
            raise ValueError("the weights of the rows have no gradient")
        weight = weight.reshape(-1).contiguous()
    _nn.no_tangents(rows, answers.values, answers.rest, weight)
    return (answers.values.contiguous(), answers.classes.contiguous(), None if answers.rest is None else answers.rest.contiguous(),
            answers.temperature, weight, reduction)


def _head(rows, o):
    values, classes, rest, temperature, weight, _ = o
    return (rows.data_ptr(), _nn.DTYPES[rows.dtype], _row_stride(rows), rows.shape[0], rows.shape[1], values.data_ptr(), classes.data_ptr(),
            int(classes.dtype == torch.int64), values.shape[1], _nn.ptr(rest), _nn.ptr(weight), temperature)


def _total(row_loss, weight, n, mean, loss, scale):
    _nn._launch("ta_nn_distil_total", row_loss if row_loss is not None else weight, _nn.ptr(row_loss), _nn.ptr(weight), n, int(mean),
                _nn.ptr(loss), _nn.ptr(scale))


def _loss(rows, o, save):
    """-> loss, statistics of the rows and the mean's scale for a backward pass (or None)"""
    weight, reduction = o[4], o[5]
    n, dev = rows.shape[0], rows.device
    row_loss = torch.empty(n, dtype=torch.float32, device=dev)
    stats = torch.empty((n, STATS), dtype=torch.float32, device=dev) if save else None
    _nn._launch("ta_nn_distil", rows, *_head(rows, o), 1.0, None, row_loss.data_ptr(), _nn.ptr(stats), None, 0)
    if reduction == "none":
        return row_loss, stats, None
    loss = torch.empty((), dtype=torch.float32, device=dev)
    scale = torch.empty((), dtype=torch.float32, device=dev) if save and weight is not None and reduction == "mean" else None
    _total(row_loss, weight, n, reduction == "mean", loss, scale)
    return loss, stats, scale


class _Distillation(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, o):
        loss, stats, scale = _loss(rows, o, True)
        values, classes, rest, temperature, weight, reduction = o
        ctx.save_for_backward(rows, stats, scale, *_nn.kept(values, classes, rest, weight))      # (one changed before the backward pass is an error)
        ctx.options = temperature, reduction
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, upstream):
        rows, stats, scale, values, classes, rest, weight = ctx.saved_tensors
        temperature, reduction = ctx.options
        o = values, classes, rest, temperature, weight, reduction
        grad = torch.empty(rows.shape, dtype=rows.dtype, device=rows.device)
        upstream = upstream.contiguous()
        factor = 1.0 / rows.shape[0] if reduction == "mean" and weight is None else 1.0
        _nn._launch("ta_nn_distil_backward", rows, *_head(rows, o), factor, _nn.ptr(scale), upstream.data_ptr(), int(reduction == "none"),
                    stats.data_ptr(), grad.data_ptr(), grad.shape[1])
        return grad, None


def distillation_loss(logits, answers, weight=None, reduction="mean"):
    """T^2 KL(teacher || student) of every row at the answers' temperature T, differentiable in the student's ``logits``
    [..., classes] (fp32, bf16 or fp16; rows in the order of the answers').

    weight     fp32, one for each row, or None; a row of weight 0 is not looked at (padding may hold anything).  Weights and answers have
               no gradient, and must not change before a backward pass
    reduction  'mean': sum of weight * loss / sum of weights (0 if no row counts); 'sum'; 'none': weight * loss for each row
    The loss is fp32, the gradient has the logits' type."""
    rows = _rows_of(logits)
    o = _checked(rows, answers, weight, reduction)
    if rows.shape[0] == 0:
        return rows.float().sum(dim=1).view(logits.shape[:-1]) if reduction == "none" else rows.float().sum()
    if torch.is_grad_enabled() and rows.requires_grad:
        loss = _Distillation.apply(rows, o)
    else:
        loss = _loss(rows, o, False)[0]
    return loss.view(logits.shape[:-1]) if reduction == "none" else loss


def distillation_loss_and_grad(logits, answers, weight=None, reduction="mean"):
    """(loss, d loss / d logits) in one pass over the logits -- for a step that has no other use for the loss's graph: hand
    the gradient on with ``logits.backward(grad)``.  ``reduction`` 'mean' or 'sum'."""
    if reduction == "none":
        raise ValueError("reduction 'none' has no single loss to differentiate")
    rows = _rows_of(logits.detach() if isinstance(logits, torch.Tensor) else logits)
    _nn.no_tangents(logits)                              # (detach drops them)
    o = _checked(rows, answers, weight, reduction)
    weight = o[4]
    n, dev = rows.shape[0], rows.device
    grad = torch.empty(logits.shape, dtype=rows.dtype, device=dev)
    loss = torch.zeros((), dtype=torch.float32, device=dev) if n == 0 else torch.empty((), dtype=torch.float32, device=dev)
    if n == 0:
        return loss, grad
    scale = None
    if weight is not None and reduction == "mean":
        scale = torch.empty((), dtype=torch.float32, device=dev)
        _total(None, weight, n, True, None, scale)
    row_loss = torch.empty(n, dtype=torch.float32, device=dev)
    factor = 1.0 / n if reduction == "mean" and weight is None else 1.0
    _nn._launch("ta_nn_distil", rows, *_head(rows, o), factor, _nn.ptr(scale), row_loss.data_ptr(), None, grad.data_ptr(), rows.shape[1])
    _total(row_loss, weight, n, reduction == "mean", loss, None)
    return loss, grad


class DistillationLoss(nn.Module):
    """``distillation_loss`` in the shape of a criterion: (logits, TopLogits) -> mean loss"""

    def forward(self, logits, label):
        return distillation_loss(logits, label)
