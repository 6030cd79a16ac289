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
from torch.autograd.function import once_differentiable

from . import _abi, _ops

_INTS = (torch.int64, torch.int32)


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


def _flat(logits, top_ids, top_logits, labels):
    V, K = logits.shape[-1], top_ids.shape[-1]
    z = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if not z.is_contiguous() and (z.stride(1) != 1 or (z.shape[0] > 1 and z.stride(0) < V)):
        z = z.contiguous()
    ids = top_ids if top_ids.dim() == 2 else top_ids.reshape(-1, K)
    t = top_logits if top_logits.dim() == 2 else top_logits.reshape(-1, K)
    if labels is not None:
        labels = (labels if labels.dim() == 1 else labels.reshape(-1)).contiguous()
    return z, ids.contiguous(), t.float().contiguous(), labels


def _params(ids, labels, temperature, alpha, ignore_index, mean, scale=1.0):
    return _abi.DistillParams(temperature, alpha, scale, mean, ids.dtype == torch.int64,
                              labels is not None and labels.dtype == torch.int64, ignore_index)


def _loss(z, ids, t, labels, params, loss, row_loss, stats, dz):
    N, V = z.shape
    nbytes = 512 + 8 * N          # concord_distill_workspace_bytes(N)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=z.device)
    _ops.call("concord_distill_loss", z.get_device(), _ops.byref(params), z.data_ptr(), _ops.TYPES[z.dtype],
              z.stride(0) if N > 1 else V, ids.data_ptr(), t.data_ptr(), _ops.ptr(labels), _ops.ptr(loss),
              _ops.ptr(row_loss), _ops.ptr(stats), _ops.ptr(dz), N, V, ids.shape[1], ws.data_ptr(), nbytes)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, top_ids, top_logits, labels, temperature, alpha, ignore_index, reduction):
        z, ids, t, lab = _flat(logits, top_ids, top_logits, labels)
        params = _params(ids, lab, temperature, alpha, ignore_index, reduction == "mean")
        f32 = dict(dtype=torch.float32, device=z.device)
        per_row = reduction == "none"
        out = torch.empty(logits.shape[:-1] if per_row else (), **f32)
        stats = torch.empty(3 * z.shape[0] + 1, **f32) if ctx.needs_input_grad[0] else None
        _loss(z, ids, t, lab, params, None if per_row else out, out if per_row else None, stats, None)
        if stats is not None:
            ctx.save_for_backward(z, ids, t, lab, stats)
            ctx.params, ctx.shape, ctx.per_row = params, logits.shape, per_row
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        z, ids, t, lab, stats = ctx.saved_tensors
        N, V = z.shape
        grad = grad.contiguous()
        dz = torch.empty(ctx.shape, dtype=z.dtype, device=z.device)
        _ops.call("concord_distill_grad", z.get_device(), _ops.byref(ctx.params), z.data_ptr(), _ops.TYPES[z.dtype],
                  z.stride(0) if N > 1 else V, ids.data_ptr(), t.data_ptr(), _ops.ptr(lab), stats.data_ptr(),
                  grad.data_ptr(), ctx.per_row, dz.data_ptr(), N, V, ids.shape[1])
        return dz, None, None, None, None, None, None, None


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
    alone, has their type.  Differentiable once.
    """
    temperature, alpha = float(temperature), float(alpha)
    _check(logits, top_ids, top_logits, labels, temperature, alpha)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"reduction must be 'mean', 'sum' or 'none', not {reduction!r}")
    return _Distill.apply(logits, top_ids, top_logits, labels, temperature, alpha, ignore_index, reduction)


@torch.no_grad()
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
    z, ids, t, lab = _flat(logits, top_ids, top_logits, labels)
    params = _params(ids, lab, temperature, alpha, ignore_index, reduction == "mean", float(grad_scale))
    loss = torch.empty((), dtype=torch.float32, device=z.device)
    dz = torch.empty(z.shape, dtype=z.dtype, device=z.device)
    _loss(z, ids, t, lab, params, loss, None, None, dz)
    return loss, dz.view(logits.shape)
