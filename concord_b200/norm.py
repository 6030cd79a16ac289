"""Layer norm with its gradient (concord_layer_norm_fwd / _bwd).

The reference's trained models normalise with torch's nn.LayerNorm around
the packed layers (notebook/src/nanogpt.py:15-101); these kernels take its
place: statistics and the sums of the weight's gradient in fp32, the output
rounded once to the type that the next layer reads.
"""
import functools

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _abi, _ops


def _rows(x, D):
    """x as [N, D] with contiguous columns (a copy only where it has none)."""
    if x.dim() != 2:
        x = x.reshape(-1, D)
    if not x.is_contiguous() and (x.stride(1) != 1 or (x.shape[0] > 1 and x.stride(0) < D)):
        x = x.contiguous()
    return x


def _ld(x2, D):
    return x2.stride(0) if x2.shape[0] > 1 else D


@functools.lru_cache(maxsize=1024)
def _workspace_floats(N, D, index):
    """fp32 values of the backward's workspace on device `index`."""
    with torch.cuda.device(index):
        return _abi.load().concord_layer_norm_bwd_workspace_bytes(N, D) // 4


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, out_dtype):
        D = x.shape[-1]
        x2 = _rows(x, D)
        N = x2.shape[0]
        y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
        mean = rstd = None
        if any(ctx.needs_input_grad):
            stats = torch.empty(2 * N, dtype=torch.float32, device=x.device)      # means, then 1 / deviations
            mean = stats.data_ptr()
            rstd = mean + 4 * N
            ctx.save_for_backward(x2, weight, stats)
            ctx.shape = x.shape
        _ops.call("concord_layer_norm_fwd", x.get_device(), x2.data_ptr(), _ops.TYPES[x.dtype], _ld(x2, D),
                  _ops.ptr(weight), _ops.ptr(bias), y.data_ptr(), _ops.TYPES[out_dtype], mean, rstd, N, D, eps)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, weight, stats = ctx.saved_tensors
        N, D = x2.shape
        index = x2.get_device()
        dy2 = _rows(dy, D)
        dx = torch.empty(ctx.shape, dtype=x2.dtype, device=x2.device)
        _, need_w, need_b, _, _ = ctx.needs_input_grad
        dw = stats.new_empty(D) if need_w else None
        db = stats.new_empty(D) if need_b else None
        ws, floats = None, 0
        if need_w or need_b:
            floats = _workspace_floats(N, D, index)
            ws = stats.new_empty(max(floats, 1))
        mean = stats.data_ptr()
        _ops.call("concord_layer_norm_bwd", index, x2.data_ptr(), _ops.TYPES[x2.dtype], _ld(x2, D), dy2.data_ptr(),
                  _ops.TYPES[dy2.dtype], _ld(dy2, D), _ops.ptr(weight), mean, mean + 4 * N, dx.data_ptr(),
                  _ops.ptr(dw), _ops.ptr(db), N, D, _ops.ptr(ws), 4 * floats)
        return dx, dw, db, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, out_dtype=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.

    x: fp32, bf16 or fp16, of any shape and strides, at most 16384 wide (a
    last dimension that is not contiguous is copied).  weight and bias [D]
    (either may be None); fp32 is read as it is, other types are converted.
    The result has `out_dtype` (default: x's type); statistics, sums and the
    gradients of weight and bias are fp32.  Differentiable once.
    """
    _ops.need_cuda(("x", x), ("weight", weight), ("bias", bias))
    _ops.need_type("x", x, _ops.TYPES)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype not in _ops.TYPES:
        raise TypeError(f"out_dtype must be one of {[str(t) for t in _ops.TYPES]}, got {out_dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x needs a last dimension of at least 1, got shape {tuple(x.shape)}")
    D = x.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and tuple(t.shape) != (D,):
            raise ValueError(f"{name} must have shape ({D},), got {tuple(t.shape)}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    weight = weight if weight is None else weight.float().contiguous()
    bias = bias if bias is None else bias.float().contiguous()
    return _LayerNorm.apply(x, weight, bias, float(eps), out_dtype)


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over one dimension on `layer_norm`; `out_dtype` as there
    (bf16 hands the next packed layer its input without another cast)."""

    def __init__(self, dim, eps=1e-5, elementwise_affine=True, bias=True, out_dtype=None, device=None, dtype=None):
        super().__init__(dim, eps=eps, elementwise_affine=elementwise_affine, bias=bias, device=device, dtype=dtype)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm normalises over the last dimension only")
        self.out_dtype = out_dtype

    def forward(self, x):
        if x.shape[-1] != self.normalized_shape[0]:
            raise ValueError(f"expected a last dimension of {self.normalized_shape[0]}, got {x.shape[-1]}")
        return layer_norm(x, self.weight, self.bias, self.eps, self.out_dtype)
