"""Distillation from a teacher's top logits (concord_distill_loss / _grad).

What a training run stores of a teacher is its K best token ids and logits
per position.  The loss of a student's logits z against them, with hard
labels beside if wanted, over the rows that count:

    p = softmax(t / T) over the entries present
    KL = sum_k p_k (log p_k - log softmax(z / T)_k)
    loss = mean of (alpha T^2 KL + (1 - alpha) CE(z, label))

The full teacher distribution is never formed, and neither are the student's
probabilities: one pass reads the logits and, in `distill_loss_and_grad`,
writes their gradient.
"""
import torch

from . import _ops

_INTS = (torch.int64, torch.int32)
_REDUCTIONS = ("mean", "sum", "none")


def _check(logits, top_ids, top_logits, labels, temperature, alpha):
    _ops.need_cuda(("logits", logits), ("top_ids", top_ids), ("top_logits", top_logits), ("labels", labels))
    _ops.need_type("logits", logits, _ops.TYPES)
    _ops.need_type("top_ids", top_ids, _INTS)
    _ops.need_type("top_logits", top_logits, _ops.TYPES)
    if logits.dim() < 2 or logits.shape[-1] < 1:
        raise ValueError(f"logits must be [..., V], got shape {tuple(logits.shape)}")
    if top_ids.shape[:-1] != logits.shape[:-1] or top_ids.dim() != logits.dim():
        raise ValueError(f"top_ids must be [..., K] beside logits {tuple(logits.shape)}, got {tuple(top_ids.shape)}")
    if top_logits.shape != top_ids.shape:
        raise ValueError(f"top_logits must have top_ids' shape {tuple(top_ids.shape)}, got {tuple(top_logits.shape)}")
    if not 1 <= top_ids.shape[-1] <= 512:
        raise ValueError(f"1 to 512 teacher entries per row, got {top_ids.shape[-1]}")
    if not 0 < temperature < float("inf"):
        raise ValueError(f"temperature must be positive, got {temperature}")
    if not 0 <= alpha <= 1:
        raise ValueError(f"alpha must be in [0, 1], got {alpha}")
    if labels is not None:
        _ops.need_type("labels", labels, _INTS)
        if labels.shape != logits.shape[:-1]:
            raise ValueError(f"labels must have shape {tuple(logits.shape[:-1])}, got {tuple(labels.shape)}")
    elif alpha != 1:
        raise ValueError("alpha < 1 weighs hard labels: pass labels")


def distill_loss(logits, top_ids, top_logits, labels=None, temperature=1.0, alpha=1.0, ignore_index=-100,
                 reduction="mean"):
    """Distillation loss of `logits` [..., V] against a teacher's top logits.

    top_ids [..., K] (int32 or int64) and top_logits [..., K]: the teacher's K
    best entries, 1 to 512; an id outside [0, V) (pad with -1) or a logit of
    -inf is an absent entry, and an id that comes twice counts with the sum of
    its probabilities.  labels [...]: hard labels, needed where alpha < 1.
    A row whose label is `ignore_index` or outside [0, V) is left out (loss
    and gradient 0); without labels, a row without teacher entries is.  With
    labels, a row without teacher entries keeps its (1 - alpha) CE alone.

    reduction: "mean" over the rows that count (0 if none does), "sum", or
    "none" (one loss per row).  The loss is fp32; the gradient, for the logits
    alone, has their type.  Differentiable once, backward only.
    """
    temperature, alpha = float(temperature), float(alpha)
    _check(logits, top_ids, top_logits, labels, temperature, alpha)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    return _ops.native().distill_loss(logits, top_ids, top_logits, labels, temperature, alpha, ignore_index,
                                      _REDUCTIONS.index(reduction))


def distill_loss_and_grad(logits, top_ids, top_logits, labels=None, temperature=1.0, alpha=1.0, ignore_index=-100,
                          reduction="mean", grad_scale=1.0):
    """(loss, d loss / d logits * grad_scale) in one pass over the logits, for
    `logits.backward(dlogits)`: the arguments of `distill_loss`, reduction
    "mean" or "sum".  `grad_scale` (a number, such as 1 / accumulation steps
    or a loss scale) is applied in fp32 before the gradient's rounding; the
    loss is not scaled."""
    temperature, alpha = float(temperature), float(alpha)
    _check(logits, top_ids, top_logits, labels, temperature, alpha)
    if reduction not in ("mean", "sum"):
        raise ValueError(f"reduction must be 'mean' or 'sum', not {reduction!r}")
    return _ops.native().distill_loss_and_grad(logits, top_ids, top_logits, labels, temperature, alpha, ignore_index,
                                               reduction == "mean", grad_scale)
